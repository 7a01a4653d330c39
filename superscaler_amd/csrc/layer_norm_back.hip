/*
 * Gradients of the norms around a block (ace_block_norm_backward; formulas in ace_layer.h and layer.py).
 *
 * Bound by memory: x, block and the two results' gradients are read, two gradients written.  Rows are laid out over lanes as in
 * the forward pass; a workgroup takes a run of consecutive rows and asks for a row's data in the middle of the one before it.
 *
 * Gradients of the parameters are sums over rows.  A workgroup keeps its run's sums in registers (one of them in LDS where lanes have
 * two vectors) and leaves them as one row of
 * partial sums; a second launch adds those up in a fixed order.  With A = sum dr' n2 and B = sum dr' over the rows that share
 * a gate, the gate's gradient is A w2 + B b2 and the exit norm's are sum g A and sum g B: two sums serve three
 * gradients.  A run that spans several gates leaves a row of A and B for each: row w + g for run w and gate g (from one
 * such pair to the next at least one of the two steps on, so no two share a row).
 *
 * 4 x 2,048 rows of 12,288 elements of bfloat16, both norms and a gate per sequence: 283 us and 19 for the second launch, 4.3 TB/s of six
 * rows' traffic; 16 x 509 of 1,024 of float32: 42 and 8.  A CU holds one workgroup of the wide rows, whose lanes all wait for two
 * sums over the row: that, and not the traffic, is what is left.  (The second launch with one sum to a workgroup, twice as many
 * loads in the air, took 28 us instead of 19.)
 */
#include "layer_norm.h"

namespace {

enum { W2, B2, GATE, W1, PARAMS };

__device__ inline f32x8 join8(const f32x4 *v) { return f32x8{v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w}; }

/* HAS_F, ENTRY: whether there are a block and an entry norm.  A result's gradient that is not given is a row of zeros that every
 * row reads, an exit norm that is not there one of mean 0 and deviation 1. */
__device__ uint4 zero_row[ACE_NORM_MAX_WIDTH / 4];

template <class T, int CAP, int NV, bool EVEN, bool HAS_F, bool ENTRY> __global__ void __launch_bounds__(CAP) norm_backward(const NormArgs a) {
    __shared__ NormExchange lds;
    extern __shared__ f32x4 room[];
    constexpr bool AHEAD = norm_params_in_lds<NV>(), SC_IN_LDS = NV == 2;
    const int C = a.width;
    uint32_t at[NV];
    int n[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) at[k] = (k * blockDim.x + threadIdx.x) * 8, n[k] = C - (int)at[k];
    const float inv = 1.0f / C, exit_inv = a.w2 ? inv : 0.0f, exit_layer = a.layer ? exit_inv : 0.0f, entry_layer = a.layer ? inv : 0.0f;
    const void *dr_base = a.dr ? a.dr : zero_row, *dy_base = a.dy ? a.dy : zero_row;
    const int dr_step = a.dr ? C : 0, dy_step = a.dy ? C : 0;
    int slot = 0;
    f32x4 sa[NV][2], sb[NV][2], sw[NV][2], sc[NV][2];
    auto leave = [&](float *to, const f32x4 (*s)[2], int64_t at_row) {
        if (!to) return;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            row_store<float, EVEN>(row_at<float>(to, at_row, C), C, at[k], join8(s[k]), n[k]);
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) sa[k][0] = sa[k][1] = sb[k][0] = sb[k][1] = sw[k][0] = sw[k][1] = sc[k][0] = sc[k][1] = 0.0f;
    const int64_t first = blockIdx.x * a.run, end = first + a.run < a.rows ? first + a.run : a.rows;
    packed8<T> x[NV], f[NV], dr[NV], dy[NV], f_next[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = f[k] = f_next[k] = dr[k] = dy[k] = 0;
    f32x4 st_next = {0.0f, 1.0f, 0.0f, 1.0f};
    auto ask = [&](int64_t of) {
        st_next = ((const f32x4 *)a.stats)[of];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (ENTRY) {
                x[k] = row_load<T, EVEN>(row_at<T>(a.x, of, C), C, at[k], n[k]);
                dy[k] = row_load<T, EVEN>(row_at<T>(dy_base, of, dy_step), C, at[k], n[k]);
            }
            dr[k] = row_load<T, EVEN>(row_at<T>(dr_base, of, dr_step), C, at[k], n[k]);
            if (HAS_F) f_next[k] = row_load<T, EVEN>(row_at<T>(a.f, of, C), C, at[k], n[k]);
        }
    };
    NormParams<T, NV, EVEN> params = {(T *)room, (int)blockDim.x * NV * 8, C};
    params.put(W2, a.w2, at, n, 1.0f), params.put(B2, a.b2, at, n, 0.0f), params.put(W1, a.w1, at, n, 1.0f);
    /* the sum of one result's gradients, for which 168 registers have no room: behind the parameters, a lane's own four elements each */
    f32x4 *held = (f32x4 *)((T *)room + PARAMS * params.pitch) + threadIdx.x;
    if (SC_IN_LDS)
#pragma unroll
        for (int i = 0; i < 2 * NV; ++i) held[i * blockDim.x] = 0.0f;
    int64_t group = first / a.rows_per_gate, group_end = (group + 1) * a.rows_per_gate;
    params.put(GATE, a.gate ? (const T *)a.gate + group * C : nullptr, at, n, 1.0f);
    if (AHEAD && first < end) ask(first);
    for (int64_t row = first; row < end; ++row) {
        if (row >= group_end) {
            if (!a.token_gate) {
                leave(a.sum_a, sa, blockIdx.x + group), leave(a.sum_b, sb, blockIdx.x + group);
#pragma unroll
                for (int k = 0; k < NV; ++k) sa[k][0] = sa[k][1] = sb[k][0] = sb[k][1] = 0.0f;
            }
            group = row / a.rows_per_gate, group_end = (group + 1) * a.rows_per_gate;
            params.put(GATE, (const T *)a.gate + group * C, at, n, 1.0f);
        }
        const T *gate = a.gate ? (const T *)a.gate + group * C : nullptr;
        if (!AHEAD) ask(row);
        const f32x4 st = st_next;
#pragma unroll
        for (int k = 0; k < NV; ++k) f[k] = f_next[k];
        /* Four elements at a time, each step on its own: the scheduler would rather have many in the air than leave a row's sums their
         * registers.  The exit norm's result is taken from the block again each time it is needed. */
        auto apart = [] { __builtin_amdgcn_sched_barrier(0); };
        auto now = [](f32x4 &v) { asm volatile("" : "+v"(v)); };   /* a sum is taken here, not at the row's end with all its terms kept until then */
        auto n2 = [&](int k, int h) { return (open4<T>(f[k], h) - st.x) * st.y; };   /* (0 and 1 without an exit norm) */
        auto w2 = [&](int k, int h) { return params.get4(W2, a.w2, at[k], n[k], 1.0f, h); };
        auto b2 = [&](int k, int h) { return params.get4(B2, a.b2, at[k], n[k], 0.0f, h); };
        auto w1 = [&](int k, int h) { return params.get4(W1, a.w1, at[k], n[k], 1.0f, h); };
        auto by = [&](int k, int h) { return params.get4(GATE, gate, at[k], n[k], 1.0f, h); };
        f32x4 d[NV][2];
        if (ENTRY) {
            float2 s = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    apart();
                    f32x4 r = open4<T>(x[k], h);
                    if (HAS_F) r = a.alpha * r + by(k, h) * (n2(k, h) * w2(k, h) + b2(k, h));
                    d[k][h] = (r - st.z) * st.w;
                    const f32x4 gy = open4<T>(dy[k], h), dn = gy * w1(k, h);
                    sw[k][h] += gy * d[k][h];
                    if (SC_IN_LDS) held[(2 * k + h) * blockDim.x] += gy;
                    else sc[k][h] += gy, now(sc[k][h]);
                    now(sw[k][h]), now(d[k][h]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s.x += dn[i], s.y += dn[i] * d[k][h][i];
                }
            s = sum_all(s, lds, slot ^= 1);
            const float c1 = s.x * entry_layer, c2 = s.y * inv;
#pragma unroll
            for (int k = 0; k < NV; ++k) again<T>(dy[k]), again<T>(f[k]);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    apart();
                    d[k][h] = open4<T>(dr[k], h) + st.w * (open4<T>(dy[k], h) * w1(k, h) - c1 - d[k][h] * c2);
                    now(d[k][h]);
                }
        } else
#pragma unroll
            for (int k = 0; k < NV; ++k) d[k][0] = open4<T>(dr[k], 0), d[k][1] = open4<T>(dr[k], 1);
        apart();
        if (a.dx)
#pragma unroll
            for (int k = 0; k < NV; ++k) row_store<T, EVEN>(row_at<T>(a.dx, row, C), C, at[k], pack8<T>(a.alpha * join8(d[k])), n[k]);
        /* x and the gradients are done with: their registers take the next row's while this one's second half is computed */
        if (AHEAD && row + 1 < end) ask(row + 1);
        if (!HAS_F) continue;
        float2 s = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (a.token_gate && a.dgate) {
                const f32x4 z[2] = {d[k][0] * (n2(k, 0) * w2(k, 0) + b2(k, 0)), d[k][1] * (n2(k, 1) * w2(k, 1) + b2(k, 1))};
                row_store<T, EVEN>(row_at<T>(a.dgate, row, C), C, at[k], pack8<T>(join8(z)), n[k]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                apart();
                const f32x4 z = n2(k, h), dz = d[k][h] * by(k, h), share = a.token_gate ? dz : d[k][h];
                sa[k][h] += share * z, sb[k][h] += share;
                now(sa[k][h]), now(sb[k][h]);
                d[k][h] = dz * w2(k, h);   /* (zero past the row's end: so are the parameters) */
#pragma unroll
                for (int i = 0; i < 4; ++i) s.x += d[k][h][i], s.y += d[k][h][i] * z[i];
                now(d[k][h]);
            }
        }
        s = sum_all(s, lds, slot ^= 1);
        const float c1 = s.x * exit_layer, c2 = s.y * exit_inv;
#pragma unroll
        for (int k = 0; k < NV; ++k) again<T>(f[k]);
        if (a.df)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                apart();
#pragma unroll
                for (int h = 0; h < 2; ++h) d[k][h] = st.y * (d[k][h] - c1 - n2(k, h) * c2);
                row_store<T, EVEN>(row_at<T>(a.df, row, C), C, at[k], pack8<T>(join8(d[k])), n[k]);
            }
    }
    if (first < end) {
        leave(a.sum_a, sa, blockIdx.x + (a.token_gate ? 0 : group)), leave(a.sum_b, sb, blockIdx.x + (a.token_gate ? 0 : group));
        if (SC_IN_LDS)
#pragma unroll
            for (int i = 0; i < 2 * NV; ++i) sc[i / 2][i % 2] = held[i * blockDim.x];
        leave(a.sum_w1, sw, blockIdx.x), leave(a.sum_b1, sc, blockIdx.x);
    }
}

/* Adds up the partial sums: workgroup y = 0 the entry norm's, y = 1 the exit norm's, y = 2 + g gate g's (JOINS of them to a layer z of the
 * grid); 32 columns and 32 shares of the rows each. */
constexpr int COLS = 32, SHARES = 32, JOINS = 65535;

template <class T> __global__ void __launch_bounds__(COLS * SHARES) norm_join(const NormArgs a) {
    __shared__ float lds[2][SHARES][COLS + 1];
    const int col = threadIdx.x % COLS, share = threadIdx.x / COLS, C = a.width;
    const int64_t what = (int64_t)blockIdx.z * JOINS + blockIdx.y;
    if (what >= 2 + (a.dgate && !a.token_gate ? a.gates : 0)) return;
    const int64_t c = (int64_t)blockIdx.x * COLS + col;
    float s[2] = {0.0f, 0.0f};
    const bool grouped = a.gate && !a.token_gate && a.gates > 1;
    if (c < C) {
        if (what == 0) {
#pragma unroll 4
            for (int64_t w = share; a.sum_w1 && w < a.runs; w += SHARES) s[0] += a.sum_w1[w * C + c], s[1] += a.sum_b1[w * C + c];
        } else if (what == 1 && !grouped) {
            const float by = a.gate && !a.token_gate ? (float)((const T *)a.gate)[c] : 1.0f;
#pragma unroll 4
            for (int64_t w = share; a.sum_a && w < a.runs; w += SHARES) s[0] += by * a.sum_a[w * C + c], s[1] += by * a.sum_b[w * C + c];
        } else if (what == 1) {
            for (int64_t w = share; a.sum_a && w < a.runs; w += SHARES) {
                const int64_t last = (w + 1) * a.run < a.rows ? (w + 1) * a.run - 1 : a.rows - 1;
                const int64_t g1 = last / a.rows_per_gate;
                for (int64_t g = w * a.run / a.rows_per_gate; g <= g1; ++g) {
                    const float by = (float)((const T *)a.gate)[g * C + c];
                    s[0] += by * a.sum_a[(w + g) * C + c], s[1] += by * a.sum_b[(w + g) * C + c];
                }
            }
        } else {
            const int64_t g = what - 2;
            const int64_t end = (g + 1) * a.rows_per_gate < a.rows ? (g + 1) * a.rows_per_gate : a.rows;
            const int64_t w1 = (end - 1) / a.run;
            for (int64_t w = g * a.rows_per_gate / a.run + share; w <= w1; w += SHARES) s[0] += a.sum_a[(w + g) * C + c], s[1] += a.sum_b[(w + g) * C + c];
        }
    }
    lds[0][share][col] = s[0], lds[1][share][col] = s[1];
    __syncthreads();
    if (share >= 2 || c >= C) return;
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < SHARES; ++k) total += lds[share][k][col];
    if (what < 2) {
        void *to = what == 0 ? (share == 0 ? a.dw1 : a.db1) : share == 0 ? a.dw2 : a.db2;
        if (to) ((T *)to)[c] = (T)total;
    } else if (share == 0) {
        float b = 0.0f;
#pragma unroll
        for (int k = 0; k < SHARES; ++k) b += lds[1][k][col];
        const float w2 = a.w2 ? (float)((const T *)a.w2)[c] : 1.0f, b2 = a.b2 ? (float)((const T *)a.b2)[c] : 0.0f;
        ((T *)a.dgate)[(what - 2) * C + c] = (T)(total * w2 + b * b2);
    }
}

template <class T, int CAP, int NV, bool EVEN, bool HAS_F, bool ENTRY> int launch(const NormArgs &a, const NormShape &shape, hipStream_t stream) {
    const auto kernel = norm_backward<T, CAP, NV, EVEN, HAS_F, ENTRY>;
    static std::atomic<uint64_t> done;
    const int ready = norm_params_in_lds<NV>() ? layer_allow_lds((const void *)kernel, 155 * 1024, done) : ACE_OK;
    if (ready != ACE_OK) return ready;
    kernel<<<(uint32_t)a.runs, shape.lanes, norm_params_in_lds<NV>() ? norm_pitch(shape) * (PARAMS * (int)sizeof(T) + (NV == 2 ? 4 : 0)) : 0, stream>>>(a);
    return layer_launched();
}

template <class T> int backward(const NormArgs &a, hipStream_t stream) {
    int rc = ACE_OK;
#define CALL(CAP, NV, EVEN)                                                                                       \
    {                                                                                                             \
        if (!a.f) rc = launch<T, CAP, NV, EVEN, false, true>(a, shape, stream);                             \
        else if (!a.w1) rc = launch<T, CAP, NV, EVEN, true, false>(a, shape, stream);                       \
        else rc = launch<T, CAP, NV, EVEN, true, true>(a, shape, stream);                                   \
    }
    NORM_FOR_SHAPE(CALL, false)
#undef CALL
    if (rc != ACE_OK) return rc;
    const int64_t joins = 2 + (a.dgate && !a.token_gate ? a.gates : 0);
    norm_join<T><<<dim3((a.width + COLS - 1) / COLS, joins < JOINS ? (uint32_t)joins : JOINS, (uint32_t)((joins + JOINS - 1) / JOINS)), COLS * SHARES, 0, stream>>>(a);
    return layer_launched();
}

}  // namespace

int norm_backward_launch(const NormArgs &a, int dtype, hipStream_t stream) {
    return dtype == ACE_T_F32 ? backward<float>(a, stream) : dtype == ACE_T_BF16 ? backward<bf16>(a, stream) : backward<f16>(a, stream);
}
