/*
 * The norm at a block's exit, its gate, the scaled residual and the norm at the next block's entry in one pass
 * (ace_block_norm_forward), and its gradients (ace_block_norm_backward).
 *
 * Bound by memory: forward reads x and block and writes r and y, backward reads those four's counterparts and writes two.  A
 * row belongs to one workgroup of W wavefronts and stays in registers, eight neighbouring elements per lane and step (16- and
 * 32-byte accesses), from its first load to its last store; workgroups walk over many rows and ask for a row's data before
 * they compute the one before it.
 *
 * A row's mean and sum of squared deviations are taken per lane around the lane's own mean and joined pair by pair
 * (n, mean, M2), so that neither a large mean nor a channel far from the others costs digits, in one exchange per norm.
 *
 * Gradients of the parameters are sums over rows.  A workgroup takes a run of consecutive rows, keeps its sums in registers
 * and leaves them as one row of partial sums; a second launch adds those up in a fixed order.  With A = sum dr' n2 and
 * B = sum dr' over the rows that share a gate, the gate's gradient is A w2 + B b2 and the exit norm's are sum g A and
 * sum g B: two sums serve three gradients.  A run that spans several gates leaves a row of A and B for each: row w + g
 * for run w and gate g (from one such pair to the next at least one of the two steps on, so no two share a row).
 */
#include "layer_common.h"

namespace {

thread_local hipError_t last_error = hipSuccess;

struct Args {
    int64_t rows, rows_per_gate, run, gates;
    int width, layer, token_gate;
    float alpha, eps;
    const void *x, *f, *gate, *w2, *b2, *w1, *b1;
    void *r, *y;
    const void *dr, *dy;
    void *dx, *df, *dgate;
    const float *stats_in;
    float *stats;
    float *sum_a, *sum_b, *sum_w1, *sum_b1;
};

struct Moments { float n, mean, m2; };

__device__ inline Moments join(const Moments &a, const Moments &b) {
    const float n = a.n + b.n, d = b.mean - a.mean, share = b.n * __builtin_amdgcn_rcpf(fmaxf(n, 1.0f));
    return {n, a.mean + d * share, a.m2 + b.m2 + d * d * a.n * share};
}

/* over the lanes of W wavefronts; `slot` alternates, so that a later exchange never writes what a slow lane still reads */
template <int W> __device__ inline Moments join_all(Moments m, float (*lds)[16][3], int slot) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = join(m, Moments{__shfl_xor(m.n, d), __shfl_xor(m.mean, d), __shfl_xor(m.m2, d)});
    if (W > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[slot][wave][0] = m.n, lds[slot][wave][1] = m.mean, lds[slot][wave][2] = m.m2;
        __syncthreads();
        m = {lds[slot][0][0], lds[slot][0][1], lds[slot][0][2]};
#pragma unroll
        for (int w = 1; w < W; ++w) m = join(m, Moments{lds[slot][w][0], lds[slot][w][1], lds[slot][w][2]});
    }
    return m;
}

template <int W> __device__ inline float2 sum_all(float2 s, float (*lds)[16][3], int slot) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s.x += __shfl_xor(s.x, d), s.y += __shfl_xor(s.y, d);
    if (W > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[slot][wave][0] = s.x, lds[slot][wave][1] = s.y;
        __syncthreads();
        s.x = lds[slot][0][0], s.y = lds[slot][0][1];
#pragma unroll
        for (int w = 1; w < W; ++w) s.x += lds[slot][w][0], s.y += lds[slot][w][1];
    }
    return s;
}

template <int NV> __device__ inline Moments lane_moments(const float (*u)[8], const int *n, bool layer) {
    Moments m = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) m.n += (float)(n[k] > 8 ? 8 : n[k] < 0 ? 0 : n[k]);
    if (layer) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += u[k][i];   /* (zero past the row's end) */
        m.mean = s * __builtin_amdgcn_rcpf(fmaxf(m.n, 1.0f));
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = i < n[k] ? u[k][i] - m.mean : 0.0f;
            m.m2 += d * d;
        }
    return m;
}

template <class T> __device__ inline void spread(float *to, const Raw8<T> &r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = (float)r.v[i];
}

template <class T> __device__ inline Raw8<T> param(const void *p, int at, int n, float otherwise) {
    if (p) return load_some((const T *)p + at, n);
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = (T)otherwise;
    return r;
}

template <class T, int W, int NV> __global__ void __launch_bounds__(W * 64) norm_forward(const Args a) {
    __shared__ float lds[2][16][3];
    const int C = a.width;
    int at[NV], n[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) at[k] = (k * W * 64 + threadIdx.x) * 8, n[k] = C - at[k];
    const bool has_f = a.f, exit_norm = a.w2, entry_norm = a.w1;
    const float inv = 1.0f / C;
    int slot = 0;
    Raw8<T> xn[NV], fn[NV];
    int64_t row = blockIdx.x;
    auto ask = [&](int64_t of) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (n[k] > 0) {
                xn[k] = load_some((const T *)a.x + of * C + at[k], n[k]);
                if (has_f) fn[k] = load_some((const T *)a.f + of * C + at[k], n[k]);
            } else
#pragma unroll
                for (int i = 0; i < 8; ++i) xn[k].v[i] = fn[k].v[i] = (T)0.0f;
    };
    if (row < a.rows) ask(row);
    for (; row < a.rows; row += gridDim.x) {
        float r[NV][8], f[NV][8];
#pragma unroll
        for (int k = 0; k < NV; ++k) spread(r[k], xn[k]);
        if (has_f)
#pragma unroll
            for (int k = 0; k < NV; ++k) spread(f[k], fn[k]);
        if (row + gridDim.x < a.rows) ask(row + gridDim.x);
        float4 st = {0.0f, 1.0f, 0.0f, 1.0f};
        if (has_f) {
            if (exit_norm) {
                const Moments m = join_all<W>(lane_moments<NV>(f, n, a.layer), lds, slot ^= 1);
                st.x = m.mean, st.y = rsqrtf(m.m2 * inv + a.eps);
            }
            const T *gate = a.gate ? (const T *)a.gate + row / a.rows_per_gate * C : nullptr;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (n[k] <= 0) continue;
                const Raw8<T> w = param<T>(a.w2, at[k], n[k], 1.0f), b = param<T>(a.b2, at[k], n[k], 0.0f), g = param<T>(gate, at[k], n[k], 1.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float z = (f[k][i] - st.x) * st.y * (float)w.v[i] + (float)b.v[i];
                    r[k][i] = i < n[k] ? a.alpha * r[k][i] + (float)g.v[i] * z : 0.0f;
                }
                Raw8<T> out;
#pragma unroll
                for (int i = 0; i < 8; ++i) out.v[i] = (T)r[k][i];
                store_some((T *)a.r + row * C + at[k], out, n[k]);
            }
        }
        if (entry_norm) {
            const Moments m = join_all<W>(lane_moments<NV>(r, n, a.layer), lds, slot ^= 1);
            st.z = m.mean, st.w = rsqrtf(m.m2 * inv + a.eps);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (n[k] <= 0) continue;
                const Raw8<T> w = param<T>(a.w1, at[k], n[k], 1.0f), b = param<T>(a.b1, at[k], n[k], 0.0f);
                Raw8<T> out;
#pragma unroll
                for (int i = 0; i < 8; ++i) out.v[i] = (T)((r[k][i] - st.z) * st.w * (float)w.v[i] + (float)b.v[i]);
                store_some((T *)a.y + row * C + at[k], out, n[k]);
            }
        }
        if (threadIdx.x == 0) ((float4 *)a.stats)[row] = st;
    }
}

template <class T, int W, int NV> __global__ void __launch_bounds__(W * 64) norm_backward(const Args a) {
    __shared__ float lds[2][16][3];
    const int C = a.width;
    int at[NV], n[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) at[k] = (k * W * 64 + threadIdx.x) * 8, n[k] = C - at[k];
    const bool has_f = a.f, exit_norm = a.w2, entry_norm = a.w1;
    const float inv = 1.0f / C;
    int slot = 0;
    float sa[NV][8], sb[NV][8], sw[NV][8], sc[NV][8];
    auto clear = [&](float (*s)[8]) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[k][i] = 0.0f;
    };
    auto leave = [&](float *to, const float (*s)[8], int64_t at_row) {
        if (!to) return;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (n[k] > 0) {
                Raw8<float> out;
#pragma unroll
                for (int i = 0; i < 8; ++i) out.v[i] = s[k][i];
                store_some(to + at_row * C + at[k], out, n[k]);
            }
    };
    clear(sa), clear(sb), clear(sw), clear(sc);
    const int64_t first = blockIdx.x * a.run, end = first + a.run < a.rows ? first + a.run : a.rows;
    int64_t group = a.gates > 1 ? first / a.rows_per_gate : 0;
    Raw8<T> xn[NV], fn[NV], drn[NV], dyn[NV];
    auto ask = [&](int64_t of) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int i = 0; i < 8; ++i) xn[k].v[i] = fn[k].v[i] = drn[k].v[i] = dyn[k].v[i] = (T)0.0f;
            if (n[k] <= 0) continue;
            const int64_t o = of * C + at[k];
            if (entry_norm) {
                xn[k] = load_some((const T *)a.x + o, n[k]);
                if (a.dy) dyn[k] = load_some((const T *)a.dy + o, n[k]);
            }
            if (has_f) fn[k] = load_some((const T *)a.f + o, n[k]);
            if (a.dr) drn[k] = load_some((const T *)a.dr + o, n[k]);
        }
    };
    if (first < end) ask(first);
    for (int64_t row = first; row < end; ++row) {
        if (a.gates > 1 && !a.token_gate && row / a.rows_per_gate != group) {
            leave(a.sum_a, sa, blockIdx.x + group), leave(a.sum_b, sb, blockIdx.x + group);
            clear(sa), clear(sb);
            group = row / a.rows_per_gate;
        }
        const float4 st = ((const float4 *)a.stats_in)[row];
        const T *gate = a.gate ? (const T *)a.gate + row / a.rows_per_gate * C : nullptr;
        Raw8<T> x[NV], f[NV], dr[NV], dy[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) x[k] = xn[k], f[k] = fn[k], dr[k] = drn[k], dy[k] = dyn[k];
        if (row + 1 < end) ask(row + 1);
        float n2[NV][8], d[NV][8], g[NV][8];
        float2 s = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            spread(d[k], dr[k]);
            if (has_f) {
                const Raw8<T> w = param<T>(a.w2, at[k], n[k], 1.0f), b = param<T>(a.b2, at[k], n[k], 0.0f);
                spread(g[k], param<T>(gate, at[k], n[k], 1.0f));
#pragma unroll
                for (int i = 0; i < 8; ++i) n2[k][i] = ((float)f[k].v[i] - st.x) * st.y;   /* (0 and 1 without an exit norm) */
            }
        }
        if (entry_norm) {
            float n1[NV][8], dn[NV][8];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const Raw8<T> w2 = param<T>(a.w2, at[k], n[k], 1.0f), b2 = param<T>(a.b2, at[k], n[k], 0.0f), w = param<T>(a.w1, at[k], n[k], 1.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float r = (float)x[k].v[i];
                    if (has_f) r = a.alpha * r + g[k][i] * (n2[k][i] * (float)w2.v[i] + (float)b2.v[i]);
                    n1[k][i] = (r - st.z) * st.w;
                    const float gy = (float)dy[k].v[i];
                    dn[k][i] = gy * (float)w.v[i];
                    s.x += dn[k][i], s.y += dn[k][i] * n1[k][i];
                    sw[k][i] += gy * n1[k][i], sc[k][i] += gy;
                }
            }
            s = sum_all<W>(s, lds, slot ^= 1);
            const float c1 = a.layer ? s.x * inv : 0.0f, c2 = s.y * inv;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[k][i] += st.w * (dn[k][i] - c1 - n1[k][i] * c2);
        }
        if (a.dx)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (n[k] > 0) {
                    Raw8<T> out;
#pragma unroll
                    for (int i = 0; i < 8; ++i) out.v[i] = (T)(has_f ? a.alpha * d[k][i] : d[k][i]);
                    store_some((T *)a.dx + row * C + at[k], out, n[k]);
                }
        if (!has_f) continue;
        s = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Raw8<T> w = param<T>(a.w2, at[k], n[k], 1.0f), b = param<T>(a.b2, at[k], n[k], 0.0f);
            Raw8<T> dg;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float dz = d[k][i] * g[k][i], by = a.token_gate ? dz : d[k][i];
                sa[k][i] += by * n2[k][i], sb[k][i] += by;
                dg.v[i] = (T)(d[k][i] * (n2[k][i] * (float)w.v[i] + (float)b.v[i]));
                d[k][i] = dz * (float)w.v[i];
                if (i < n[k]) s.x += d[k][i], s.y += d[k][i] * n2[k][i];
            }
            if (a.token_gate && a.dgate && n[k] > 0) store_some((T *)a.dgate + row * C + at[k], dg, n[k]);
        }
        if (exit_norm) {
            s = sum_all<W>(s, lds, slot ^= 1);
            const float c1 = a.layer ? s.x * inv : 0.0f, c2 = s.y * inv;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[k][i] = st.y * (d[k][i] - c1 - n2[k][i] * c2);
        }
        if (a.df)
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (n[k] > 0) {
                    Raw8<T> out;
#pragma unroll
                    for (int i = 0; i < 8; ++i) out.v[i] = (T)d[k][i];
                    store_some((T *)a.df + row * C + at[k], out, n[k]);
                }
    }
    if (first < end) {
        leave(a.sum_a, sa, blockIdx.x + (a.token_gate ? 0 : group)), leave(a.sum_b, sb, blockIdx.x + (a.token_gate ? 0 : group));
        leave(a.sum_w1, sw, blockIdx.x), leave(a.sum_b1, sc, blockIdx.x);
    }
}

/* Adds up the partial sums: workgroup y = 0 the four parameters', y = 1 + g gate g's; 64 columns and 16 shares of the rows each. */
constexpr int COLS = 64, SHARES = 16;
struct Join {
    int64_t rows, rows_per_gate, run, gates, runs;
    int width, token_gate;
    const float *sum_a, *sum_b, *sum_w1, *sum_b1;
    const void *gate, *w2, *b2;
    void *dgate, *dw2, *db2, *dw1, *db1;
};

template <class T> __global__ void __launch_bounds__(COLS * SHARES) norm_join(const Join a) {
    __shared__ float lds[4][SHARES][COLS];
    const int col = threadIdx.x % COLS, share = threadIdx.x / COLS, C = a.width;
    const int64_t c = (int64_t)blockIdx.x * COLS + col;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool grouped = a.gate && !a.token_gate;
    if (c < C) {
        if (blockIdx.y == 0) {
            for (int64_t w = share; w < a.runs; w += SHARES) {
                if (a.sum_a) {
                    const int64_t last = (w + 1) * a.run < a.rows ? (w + 1) * a.run - 1 : a.rows - 1;
                    const int64_t g0 = a.gates > 1 && grouped ? w * a.run / a.rows_per_gate : 0, g1 = a.gates > 1 && grouped ? last / a.rows_per_gate : 0;
                    for (int64_t g = g0; g <= g1; ++g) {
                        const float by = grouped ? (float)((const T *)a.gate)[g * C + c] : 1.0f;
                        s[0] += by * a.sum_a[(w + g) * C + c];
                        s[1] += by * a.sum_b[(w + g) * C + c];
                    }
                }
                if (a.sum_w1) s[2] += a.sum_w1[w * C + c], s[3] += a.sum_b1[w * C + c];
            }
        } else {
            const int64_t g = blockIdx.y - 1;
            const int64_t end = (g + 1) * a.rows_per_gate < a.rows ? (g + 1) * a.rows_per_gate : a.rows;
            const int64_t w1 = (end - 1) / a.run;
            for (int64_t w = g * a.rows_per_gate / a.run + share; w <= w1; w += SHARES) s[0] += a.sum_a[(w + g) * C + c], s[1] += a.sum_b[(w + g) * C + c];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) lds[k][share][col] = s[k];
    __syncthreads();
    if (share >= 4 || c >= C) return;
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < SHARES; ++k) total += lds[share][k][col];
    if (blockIdx.y == 0) {
        void *to = share == 0 ? a.dw2 : share == 1 ? a.db2 : share == 2 ? a.dw1 : a.db1;
        if (to) ((T *)to)[c] = (T)total;
    } else if (share == 0) {
        float b = 0.0f;
#pragma unroll
        for (int k = 0; k < SHARES; ++k) b += lds[1][k][col];
        const float w2 = a.w2 ? (float)((const T *)a.w2)[c] : 1.0f, b2 = a.b2 ? (float)((const T *)a.b2)[c] : 0.0f;
        ((T *)a.dgate)[(blockIdx.y - 1) * (int64_t)C + c] = (T)(total * w2 + b * b2);
    }
}

/* Wavefronts and vectors of eight per lane of a row: the fewest lanes that hold it with few vectors each. */
#define FOR_WIDTH(CALL)                                  \
    const int vectors = (a.width + 7) / 8;               \
    if (vectors <= 64) CALL(1, 1)                        \
    else if (vectors <= 128) CALL(2, 1)                  \
    else if (vectors <= 256) CALL(4, 1)                  \
    else if (vectors <= 512) CALL(4, 2)                  \
    else if (vectors <= 768) CALL(4, 3)                  \
    else if (vectors <= 1024) CALL(8, 2)                 \
    else if (vectors <= 1536) CALL(8, 3)                 \
    else if (vectors <= 2048) CALL(16, 2)                \
    else if (vectors <= 3072) CALL(16, 3)                \
    else CALL(16, 4)

int waves_of(int width) {
    const int vectors = (width + 7) / 8;
    return vectors <= 64 ? 1 : vectors <= 128 ? 2 : vectors <= 768 ? 4 : vectors <= 1536 ? 8 : 16;
}

int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

template <class T> int forward(const Args &a, hipStream_t stream) {
    const dim3 grid((uint32_t)least(a.rows, 256 * 32 / waves_of(a.width)));
#define CALL(W, NV) norm_forward<T, W, NV><<<grid, W * 64, 0, stream>>>(a);
    FOR_WIDTH(CALL)
#undef CALL
    return layer_launched();
}

/* Runs of consecutive rows of the backward pass, one per workgroup. */
int64_t runs_of(const ace_block_norm_t *a) {
    const int64_t most = waves_of(a->width) >= 8 ? 256 : 512;
    const int64_t run = (a->rows + most - 1) / most;
    return (a->rows + run - 1) / run;
}

int64_t gates_of(const ace_block_norm_t *a) { return a->d_gate ? (a->rows + a->rows_per_gate - 1) / a->rows_per_gate : 1; }

bool token_gate(const ace_block_norm_t *a) { return a->d_gate && a->rows_per_gate == 1 && a->rows > 1; }

template <class T> int backward(const Args &a, const Join &j, hipStream_t stream) {
    const dim3 grid((uint32_t)j.runs);
#define CALL(W, NV) norm_backward<T, W, NV><<<grid, W * 64, 0, stream>>>(a);
    FOR_WIDTH(CALL)
#undef CALL
    int rc = layer_launched();
    if (rc != ACE_OK || !(j.sum_a || j.sum_w1)) return rc;
    norm_join<T><<<dim3((a.width + COLS - 1) / COLS, (uint32_t)(1 + (j.dgate ? j.gates : 0))), COLS * SHARES, 0, stream>>>(j);
    return layer_launched();
}

int check(const ace_block_norm_t *a) {
    if (!a || a->rows < 0 || a->width < 1 || a->dtype < ACE_T_F32 || a->dtype > ACE_T_F16) return ACE_EINVAL;
    if (a->width > ACE_NORM_MAX_WIDTH || a->rows > ((int64_t)1 << 40)) return ACE_ETOOBIG;
    if (a->rows == 0) return ACE_OK;   /* (tensors without elements may have no address) */
    if (!a->d_block && (a->d_gate || a->d_exit_weight)) return ACE_EINVAL;
    if ((a->d_exit_bias && !a->d_exit_weight) || (a->d_entry_bias && !a->d_entry_weight)) return ACE_EINVAL;
    if (!a->d_block && !a->d_entry_weight) return ACE_EINVAL;
    if (a->d_gate && a->rows_per_gate < 1) return ACE_EINVAL;
    if (!a->d_x) return ACE_EINVAL;
    return ACE_OK;
}

Args args_of(const ace_block_norm_t *a) {
    Args k = {};
    k.rows = a->rows, k.rows_per_gate = a->d_gate ? a->rows_per_gate : a->rows + 1, k.gates = gates_of(a);
    k.width = a->width, k.layer = a->layer, k.alpha = a->residual_scale, k.eps = a->eps;
    k.x = a->d_x, k.f = a->d_block, k.gate = a->d_gate, k.w2 = a->d_exit_weight, k.b2 = a->d_exit_bias, k.w1 = a->d_entry_weight, k.b1 = a->d_entry_bias;
    return k;
}

}  // namespace

int layer_hip_status(hipError_t e) {
    if (e == hipSuccess) return ACE_OK;
    last_error = e;
    return ACE_EHIP;
}

extern "C" int ace_layer_abi_version(void) { return ACE_LAYER_ABI_VERSION; }

extern "C" const char *ace_layer_last_hip_error(void) { return last_error == hipSuccess ? "" : hipGetErrorString(last_error); }

extern "C" const char *ace_layer_strerror(int code) {
    switch (code) {
    case ACE_OK: return "ok";
    case ACE_EINVAL: return "invalid argument";
    case ACE_ETOOBIG: return "larger than the kernels hold";
    case ACE_EHIP: return "HIP error";
    default: return "unknown error";
    }
}

extern "C" int ace_block_norm_forward(const ace_block_norm_t *a, void *d_residual, void *d_normed, float *d_stats, void *stream) {
    const int rc = check(a);
    if (rc != ACE_OK || a->rows == 0) return rc;
    if (!d_stats || (a->d_block && !d_residual) || (a->d_entry_weight && !d_normed)) return ACE_EINVAL;
    Args k = args_of(a);
    k.r = d_residual, k.y = d_normed, k.stats = d_stats;
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == ACE_T_F32 ? forward<float>(k, s) : a->dtype == ACE_T_BF16 ? forward<bf16>(k, s) : forward<f16>(k, s);
}

extern "C" size_t ace_block_norm_workspace_bytes(const ace_block_norm_t *a) {
    if (check(a) != ACE_OK || a->rows == 0) return 0;
    const int64_t runs = runs_of(a);
    const int64_t rows = (a->d_block ? 2 * (runs + (token_gate(a) ? 0 : gates_of(a) - 1)) : 0) + (a->d_entry_weight ? 2 * runs : 0);
    return (size_t)(rows * a->width) * sizeof(float);
}

extern "C" int ace_block_norm_backward(const ace_block_norm_t *a, const void *g_residual, const void *g_normed, const float *d_stats, void *d_dx,
                                       void *d_dblock, void *d_dgate, void *d_dexit_weight, void *d_dexit_bias, void *d_dentry_weight,
                                       void *d_dentry_bias, void *d_workspace, size_t workspace_bytes, void *stream) {
    const int rc = check(a);
    if (rc != ACE_OK || a->rows == 0) return rc;   /* (the caller clears the sums over no rows) */
    if ((d_dblock && !a->d_block) || (d_dgate && !a->d_gate) || ((d_dexit_weight || d_dexit_bias) && !a->d_exit_weight) ||
        ((d_dentry_weight || d_dentry_bias) && !a->d_entry_weight))
        return ACE_EINVAL;
    if (!d_stats || !d_workspace || workspace_bytes < ace_block_norm_workspace_bytes(a)) return ACE_EINVAL;
    if (gates_of(a) > 65534 && d_dgate && !token_gate(a)) return ACE_ETOOBIG;
    Args k = args_of(a);
    k.dr = g_residual, k.dy = g_normed, k.stats_in = d_stats, k.dx = d_dx, k.df = d_dblock;
    k.token_gate = token_gate(a);
    const int64_t runs = runs_of(a), slots = runs + (k.token_gate ? 0 : k.gates - 1);
    k.run = (a->rows + runs - 1) / runs;
    float *ws = (float *)d_workspace;
    if (a->d_block) k.sum_a = ws, k.sum_b = ws + slots * a->width, ws += 2 * slots * a->width;
    if (a->d_entry_weight) k.sum_w1 = ws, k.sum_b1 = ws + runs * a->width;
    k.dgate = k.token_gate ? d_dgate : nullptr;
    Join j = {};
    j.rows = k.rows, j.rows_per_gate = k.rows_per_gate, j.run = k.run, j.gates = k.gates, j.runs = runs;
    j.width = a->width, j.token_gate = k.token_gate;
    j.sum_a = k.sum_a, j.sum_b = k.sum_b, j.sum_w1 = k.sum_w1, j.sum_b1 = k.sum_b1;
    j.gate = a->d_gate, j.w2 = a->d_exit_weight, j.b2 = a->d_exit_bias;
    j.dgate = k.token_gate ? nullptr : d_dgate, j.dw2 = d_dexit_weight, j.db2 = d_dexit_bias, j.dw1 = d_dentry_weight, j.db1 = d_dentry_bias;
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == ACE_T_F32 ? backward<float>(k, j, s) : a->dtype == ACE_T_BF16 ? backward<bf16>(k, j, s) : backward<f16>(k, j, s);
}
