/*
 * Log-probabilities of taken tokens and the clipped policy loss (ace_token_logprobs, ace_policy_loss), with gradients.
 *
 * Rows of logits, thousands to a hundred thousand elements each, are read once. A lane keeps a maximum of its own and the sum of exponentials
 * around it, 32 bits each (of rows too large to be held, 32 terms at a time); lanes and wavefronts are joined in 64 bits, and one lane goes on in 64 bits from the row's
 * maximum and sum to its log-probability, loss and derivative. So nothing but the lanes' sums is rounded before a ratio is held against the border of its clipping: it
 * falls on the side that it belongs to unless it is nearer to the border than those sums are exact (2^-24 of a ratio for each term of a lane, some hundreds at most).
 *
 * Bound by memory.  A workgroup's registers hold a whole row (held_rows), so that the gradient needs no second look at the logits: 8,192 rows of
 * 51,200 in bfloat16, a fifth of them without a target, 293 us, 5.2 TB/s of what is read and written, as a large copy does; with a second look (loss_rows,
 * loss_back) 414.  Two workgroups of 512 lanes are resident on a CU with rows of up to 53,248 elements of 16 bits (half as many of 32), one with up to
 * 131,072 (98,304), past which a row is looked at twice.  800 MB of log-probabilities alone, two inputs in turn, from 8,192 to 65,536 elements a row: 136 to 161 us, 5.0 to
 * 5.9 TB/s, slowest in half precision; of 100,000 and 131,072 of 16 bits, one workgroup on a CU, 200 to 211 and 172 to 178; of 1,000, by a wavefront each, 197 to 209 (with four
 * for each it was twice that).
 */
#include <type_traits>
#include "layer_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LOG2E_REST = (float)(1.4426950408889634 - (double)1.4426950408889634f);

struct Loss {
    int64_t rows, stride, out_stride;
    int vocab, wide;                     /* wide: targets of 64 bits */
    const void *logits, *targets;
    const float *old, *advantage, *ref, *weight, *g;
    double low, high, kl_weight, even_weight;
    float *logp, *stats, *d_logp, *loss;
    double *row_loss;
    void *d_logits;
};

__device__ inline int64_t target_of(const Loss &a, int64_t row) { return a.wide ? ((const int64_t *)a.targets)[row] : ((const int32_t *)a.targets)[row]; }
__device__ inline bool there(const Loss &a, int64_t target) { return (uint64_t)target < (uint64_t)a.vocab; }

/* What a row has come to: its largest logit, and the sum of exponentials around it. */
struct Row {
    float top;
    double total;
};
/* The rows' part in 64 bits, by one lane: results of the row, and its derivative. */
struct Settled {
    double logp, log_total;
    float d;
};
template <bool POLICY> __device__ inline Settled settle(const Loss &a, int64_t row, const Row &r, float taken) {
    const double log_total = log(r.total), logp = (double)taken - (double)r.top - log_total;
    a.logp[row] = (float)logp;
    a.stats[2 * row] = r.top, a.stats[2 * row + 1] = (float)r.total;
    if (!POLICY) return {logp, log_total, 0.0f};
    const double w = a.weight ? (double)a.weight[row] : a.even_weight, A = a.advantage[row], ratio = exp(logp - (double)a.old[row]);
    if (w == 0.0) {   /* (it takes no part, whatever its numbers are) */
        a.row_loss[row] = 0.0, a.d_logp[row] = 0.0f;
        return {logp, log_total, 0.0f};
    }
    const double held = ratio < a.low ? a.low : ratio > a.high ? a.high : ratio;   /* (what is no number stays none) */
    const bool clipped = A > 0.0 ? ratio > a.high : ratio < a.low;
    double loss = -(clipped ? held : ratio) * A, d = -(clipped ? 0.0 : ratio) * A;
    if (a.ref) {
        const double away = (double)a.ref[row] - logp, e = expm1(away);
        loss += a.kl_weight * (e - away), d -= a.kl_weight * e;
    }
    a.row_loss[row] = w * loss;
    a.d_logp[row] = (float)(w * d);
    return {logp, log_total, (float)(w * d)};
}
/* a row without a target */
template <bool POLICY> __device__ inline void settle_none(const Loss &a, int64_t row) {
    a.logp[row] = 0.0f, a.stats[2 * row] = 0.0f, a.stats[2 * row + 1] = 0.0f;
    if (POLICY) a.row_loss[row] = 0.0, a.d_logp[row] = 0.0f;
}

__device__ inline float around(float top) { return top == -__builtin_inff() ? 0.0f : top; }
/* exp(x), x a difference of two logits, so that nothing is lost before.  (Without the rest of log2 e all terms of a row are off to one side, by
 * 1.3e-8 of x each, and its log-probability by some 1e-7.) */
__device__ inline float power(float x) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, LOG2E, x * LOG2E_REST)); }

/* Joins the lanes' maxima and sums; all lanes know the result.  `tops`, `sums`: one for each wavefront, not in use. */
template <int LANES, class S> __device__ inline Row join(float top, S total, float *tops, double *sums) {
    float most = top;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    double x = (double)(total * power(top - around(most)));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = most, sums[threadIdx.x >> 6] = x;
    __syncthreads();
    Row r = {-__builtin_inff(), 0.0};
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) r.top = fmaxf(r.top, tops[w]);
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) r.total += sums[w] * (double)power(tops[w] - around(r.top));
    return r;
}

/* (elements stay as they lie in memory: they are converted once more wherever they are used, which takes an operation and no register) */
template <class V> __device__ inline void keep(V &v) {
    union { V v; uint32_t u[sizeof(V) / 4]; } x;
    x.v = v;
#pragma unroll
    for (unsigned i = 0; i < sizeof(V) / 4; ++i) asm volatile("" : "+v"(x.u[i]));
    v = x.v;
}
/* 16 bytes of a row, and a row's whole ones through a buffer descriptor: a lane's place is one register for all of them. */
template <class T> constexpr int PIECE = 16 / (int)sizeof(T);
template <class T> struct Piece { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };
template <class T> using piece = typename Piece<T>::type;
template <class T, int LANES> struct RowPieces {
    __amdgpu_buffer_rsrc_t row;
    uint32_t mine;
    __device__ inline RowPieces(const T *p, int pieces) : row(__builtin_amdgcn_make_buffer_rsrc((void *)p, 0, pieces * 16, 0x00027000)), mine(threadIdx.x * 16) {}
    __device__ inline piece<T> get(int k) const { return __builtin_bit_cast(piece<T>, __builtin_amdgcn_raw_buffer_load_b128(row, mine, k * LANES * 16, 0)); }
    __device__ inline void put(int k, piece<T> v) const { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), row, mine, k * LANES * 16, 0); }
};
/* A row in whole pieces that begin at multiples of 16 bytes in memory, and the elements before and behind them, the `rest`, one for each of the first
 * lanes.  (Rows of 51,201 elements of 16 bits, which begin anywhere, take a fifth longer in pieces from their first element on.) */
template <class T> struct Layout {
    int before, pieces, rest;
    __device__ inline Layout(const T *row, int size) {
        before = (int)(-(uintptr_t)row & 15) / (int)sizeof(T);
        before = before < size ? before : size;
        pieces = (size - before) / PIECE<T>, rest = size - pieces * PIECE<T>;
    }
    __device__ inline int edge(int lane) const { return lane < before ? lane : pieces * PIECE<T> + lane; }
    /* the piece that has an element; 0 for the rest */
    __device__ inline int piece_of(int element) const { return element >= before && element < before + pieces * PIECE<T> ? (element - before) / PIECE<T> : 0; }
    /* the lane that has an element, where every `lanes` pieces go to that many lanes in turn */
    __device__ inline int owner(int element, int lanes) const {
        const int at = element - before;
        return at < 0 ? element : at / PIECE<T> < pieces ? at / PIECE<T> % lanes : element - pieces * PIECE<T>;
    }
};

/* What lanes need for a row's gradient: d (exp(x - top) / total), where the type has 16 bits as an exponential of (x - top) log2 e + more with
 * more = log2(|d| / total): an operation fewer, and what is rounded on the way, a difference of logits, more and the sum of both, is 2^-24 of at most
 * some 250, so 2^-16 of a result. (top is taken off before anything is rounded: the gradient of a row does not change with what all its logits share.) */
struct Told {
    float d, at_target, top, by, more;
};
template <class T> __device__ inline piece<T> gradients(const Told &t, piece<T> x) {
    piece<T> r;
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) r[i] = sizeof(T) == 4 ? (T)(power((float)x[i] - t.top) * t.by * -t.d) : (T)__builtin_amdgcn_exp2f(__builtin_fmaf((float)x[i] - t.top, LOG2E, t.more));
    return sizeof(T) == 4 ? r : __builtin_bit_cast(piece<T>, __builtin_bit_cast(u32x4, r) ^ (t.d > 0.0f ? 0x80008000u : 0u));
}

/* A row per workgroup whose lanes hold all of it, HELD pieces each as they lie in memory, so that its logits are read once for the loss and
 * the gradient both. */
enum { LOGPROBS, POLICY_LOSS, POLICY_GRADIENT };
template <class T, int LANES, int HELD, int WHAT> __global__ void __launch_bounds__(LANES) held_rows(const Loss a, int64_t first) {
    __shared__ float tops[LANES / 64];
    __shared__ double sums[LANES / 64];
    __shared__ Told told;
    const float inf = __builtin_inff();
    const int lane = threadIdx.x;
    const int64_t row = first + blockIdx.x, target = target_of(a, row);
    const T *z = (const T *)a.logits + row * a.stride;
    T *to = (T *)a.d_logits + row * a.out_stride;
    const Layout<T> layout(z, a.vocab);
    const int pieces = layout.pieces;
    const RowPieces<T, LANES> out(to + layout.before, pieces);
    auto clear = [&] {
#pragma unroll
        for (int k = 0; k < HELD; ++k)
            if (k * LANES + lane < pieces) out.put(k, piece<T>{});
        if (lane < layout.rest) to[layout.edge(lane)] = (T)0.0f;
    };
    if (!there(a, target)) {
        if (lane == 0) settle_none<WHAT != LOGPROBS>(a, row);
        if (WHAT == POLICY_GRADIENT) clear();
        return;
    }
    const float taken = (float)z[target];
    const RowPieces<T, LANES> from(z + layout.before, pieces);
    piece<T> v[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        if (k * LANES + lane < pieces) v[k] = from.get(k);
        else
#pragma unroll
            for (int i = 0; i < PIECE<T>; ++i) v[k][i] = (T)-inf;
    }
    piece<T> edge;
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) edge[i] = (T)-inf;
    if (lane < layout.rest) edge[0] = z[layout.edge(lane)];
    float top = (float)edge[0];
#pragma unroll
    for (int k = 0; k < HELD; ++k)
#pragma unroll
        for (int i = 0; i < PIECE<T>; ++i) top = fmaxf(top, (float)v[k][i]);
    const float base = around(top);
    float total = power((float)edge[0] - base);
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        keep(v[k]);
#pragma unroll
        for (int i = 0; i < PIECE<T>; ++i) total += power((float)v[k][i] - base);
    }
    const Row r = join<LANES>(top, total, tops, sums);
    if (lane == 0) {
        const Settled s = settle<WHAT != LOGPROBS>(a, row, r, taken);
        if (WHAT == POLICY_GRADIENT) {
            const float d = s.d * (a.g ? *a.g : 1.0f);
            told = {d, (float)(-(double)d * expm1(s.logp)), r.top, (float)(1.0 / r.total),
                    (float)((double)__builtin_amdgcn_logf(__builtin_fabsf(d)) - s.log_total * 1.4426950408889634)};
        }
    }
    if (WHAT != POLICY_GRADIENT) return;
    __syncthreads();
    const Told t = told;
    if (t.d == 0.0f) {
        clear();
        return;
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        if (k * LANES + lane < pieces) {
            keep(v[k]);
            out.put(k, gradients<T>(t, v[k]));
        }
        __builtin_amdgcn_sched_barrier(0);   /* (a piece after the other: in each other's midst they take more registers) */
    }
    if (lane < layout.rest) to[layout.edge(lane)] = gradients<T>(t, edge)[0];
    /* the target's own, by the lane that has just left it as another's */
    if (lane == layout.owner((int)target, LANES)) to[target] = (T)t.at_target;
}

/* A row per workgroup, AHEAD pieces for each lane on their way while as many are worked on.  8 rows of 200,000 in bfloat16 19.6 us, 1,225 97, 5.1 TB/s (256 lanes: 22.9 and
 * 97; 1,024: 20.5 and 121). */
constexpr int AHEAD = 4;
template <class T, int LANES, bool POLICY> __global__ void __launch_bounds__(LANES) loss_rows(const Loss a, int64_t first) {
    __shared__ float tops[LANES / 64];
    __shared__ double sums[LANES / 64];
    const float inf = __builtin_inff();
    const int lane = threadIdx.x;
    const int64_t row = first + blockIdx.x, target = target_of(a, row);
    if (!there(a, target)) {
        if (lane == 0) settle_none<POLICY>(a, row);
        return;
    }
    const T *z = (const T *)a.logits + row * a.stride;
    const float taken = (float)z[target];
    const Layout<T> layout(z, a.vocab);
    const int pieces = layout.pieces;
    const RowPieces<T, LANES> from(z + layout.before, pieces);
    auto ask = [&](piece<T> (&v)[AHEAD], int k) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if ((k + i) * LANES + lane < pieces) v[i] = from.get(k + i);
            else
#pragma unroll
                for (int e = 0; e < PIECE<T>; ++e) v[i][e] = (T)-inf;
        }
    };
    float top = lane < layout.rest ? (float)z[layout.edge(lane)] : -inf;
    /* (a lane has up to half a million elements: their sum is of 64 bits, that of the pieces of a turn of 32) */
    double total = lane < layout.rest ? (double)power(top - around(top)) : 0.0;
    auto use = [&](piece<T> (&v)[AHEAD]) {
        float most = -inf;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int e = 0; e < PIECE<T>; ++e) most = fmaxf(most, (float)v[i][e]);
        if (most > top) total *= (double)power(top - most), top = most;
        const float base = around(top);
        float turn = 0.0f;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            keep(v[i]);
#pragma unroll
            for (int e = 0; e < PIECE<T>; ++e) turn += power((float)v[i][e] - base);
        }
        total += (double)turn;
    };
    piece<T> x[AHEAD], y[AHEAD];
    ask(x, 0);
    for (int k = 0; k * LANES < pieces; k += 2 * AHEAD) {
        ask(y, k + AHEAD);
        use(x);
        ask(x, k + 2 * AHEAD);
        use(y);
    }
    const Row r = join<LANES>(top, total, tops, sums);
    if (lane == 0) settle<POLICY>(a, row, r, taken);
}

/* Gradients of a row's logits, from its statistics: BACK_HELD pieces for each of a workgroup's lanes. */
constexpr int BACK_LANES = 256, BACK_HELD = 4;
/* (a row that begins anywhere has as many whole pieces or one fewer than one that does not) */
template <class T> __host__ __device__ inline int parts_of(int vocab) { return vocab < PIECE<T> ? 1 : (vocab / PIECE<T> + BACK_LANES * BACK_HELD - 1) / (BACK_LANES * BACK_HELD); }
template <class T> __global__ void __launch_bounds__(BACK_LANES) loss_back(const Loss a, bool policy) {
    const int parts = parts_of<T>(a.vocab), lane = threadIdx.x;
    const int64_t items = a.rows * parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t row = item / parts, target = target_of(a, row);
        const int part = (int)(item - row * parts), begin = part * BACK_LANES * BACK_HELD;
        const T *z = (const T *)a.logits + row * a.stride;
        T *to = (T *)a.d_logits + row * a.out_stride;
        const Layout<T> layout(z, a.vocab);
        const int pieces = layout.pieces - begin;
        const RowPieces<T, BACK_LANES> from(z + layout.before + (int64_t)begin * PIECE<T>, pieces), out(to + layout.before + (int64_t)begin * PIECE<T>, pieces);
        const float d = !there(a, target) ? 0.0f : policy ? a.d_logp[row] * (a.g ? *a.g : 1.0f) : a.g[row], top = a.stats[2 * row], by = 1.0f / a.stats[2 * row + 1];
        if (d == 0.0f) {   /* (of a row that takes no part nothing is read) */
#pragma unroll
            for (int k = 0; k < BACK_HELD; ++k)
                if (k * BACK_LANES + lane < pieces) out.put(k, piece<T>{});
            if (part == 0 && lane < layout.rest) to[layout.edge(lane)] = (T)0.0f;
            continue;
        }
        auto grad = [&](float x) { return (T)(-d * (power(x - top) * by)); };
        /* (read before anything is written: the gradient may go where the logits are) */
        const bool mine = lane == layout.owner((int)target, BACK_LANES) && layout.piece_of((int)target) / (BACK_LANES * BACK_HELD) == part;
        const float logp = mine && a.logp ? a.logp[row] : 0.0f, taken = mine && !a.logp ? (float)z[target] : 0.0f, edge = part == 0 && lane < layout.rest ? (float)z[layout.edge(lane)] : 0.0f;
        piece<T> v[BACK_HELD];
#pragma unroll
        for (int k = 0; k < BACK_HELD; ++k)
            if (k * BACK_LANES + lane < pieces) v[k] = from.get(k);
#pragma unroll
        for (int k = 0; k < BACK_HELD; ++k) {
            if (k * BACK_LANES + lane >= pieces) continue;
            piece<T> r;
#pragma unroll
            for (int i = 0; i < PIECE<T>; ++i) r[i] = grad((float)v[k][i]);
            out.put(k, r);
        }
        if (part == 0 && lane < layout.rest) to[layout.edge(lane)] = grad(edge);
        /* the target's own, by the lane that has just left it as another's.  (Next to 1 a probability has no digits left for what it lacks; its logarithm
         * has them all.) */
        if (mine) to[target] = (T)(a.logp ? -d * expm1f(logp) : d * (1.0f - power(taken - top) * by));
    }
}

/* the sum of the rows' losses */
constexpr int SUM_LANES = 1024;
__global__ void __launch_bounds__(SUM_LANES) loss_sum(const double *each, int64_t rows, float *loss) {
    __shared__ double sums[SUM_LANES / 64];
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += SUM_LANES) x += each[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x > 0) return;
    x = 0.0;
    for (int w = 0; w < SUM_LANES / 64; ++w) x += sums[w];
    *loss = (float)x;
}

int check(const ace_token_loss_t *a, bool policy) {
    if (!a || a->rows < 0 || a->vocab < 1 || a->dtype < ACE_T_F32 || a->dtype > ACE_T_F16 || (a->target_bits != 32 && a->target_bits != 64)) return ACE_EINVAL;
    if (a->vocab > ACE_LOSS_MAX_VOCAB || a->rows > (int64_t)1 << 40) return ACE_ETOOBIG;
    if (policy && !(a->ratio_low >= 0.0 && a->ratio_low <= 1.0 && a->ratio_high >= 1.0 && a->kl_weight >= 0.0)) return ACE_EINVAL;
    if (a->rows == 0) return ACE_OK;
    if (!a->d_logits || !a->d_targets || (a->rows > 1 && a->row_stride < a->vocab) || (policy && (!a->d_old || !a->d_advantage))) return ACE_EINVAL;
    if (((uintptr_t)a->d_logits & (a->dtype == ACE_T_F32 ? 3 : 1)) || ((uintptr_t)a->d_targets & (a->target_bits / 8 - 1))) return ACE_EINVAL;
    return ACE_OK;
}

Loss args_of(const ace_token_loss_t *a) {
    Loss k = {};
    k.rows = a->rows, k.stride = a->row_stride, k.vocab = a->vocab, k.wide = a->target_bits == 64, k.logits = a->d_logits, k.targets = a->d_targets;
    k.old = a->d_old, k.advantage = a->d_advantage, k.ref = a->d_ref, k.weight = a->d_weight;
    k.low = a->ratio_low, k.high = a->ratio_high, k.kl_weight = a->kl_weight, k.even_weight = a->even_weight;
    return k;
}

constexpr int64_t MOST_GROUPS = (int64_t)1 << 21;   /* of a launch: 2^31 lanes */
uint32_t groups(int64_t n) { return (uint32_t)(n < MOST_GROUPS ? n : MOST_GROUPS); }

/* go(one of the type's values) */
template <class Go> auto by_type(int dtype, Go go) { return dtype == ACE_T_F32 ? go(float()) : dtype == ACE_T_BF16 ? go(bf16()) : go(f16()); }

/* whether a workgroup's lanes hold a row, and the launch: as many lanes and pieces for each as the row needs */
template <int WHAT, class T> bool held(const Loss &k, hipStream_t s, int *rc) {
    const int pieces = k.vocab / PIECE<T>;
    auto go = [&](auto lanes, auto vecs) {
        constexpr int LANES = decltype(lanes)::value, HELD = decltype(vecs)::value;
        *rc = ACE_OK;
        for (int64_t first = 0; first < k.rows && *rc == ACE_OK; first += MOST_GROUPS) {
            held_rows<T, LANES, HELD, WHAT><<<groups(k.rows - first), LANES, 0, s>>>(k, first);
            *rc = layer_launched();
        }
        return true;
    };
    if (pieces <= 64 * 1) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (pieces <= 64 * 2) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    if (pieces <= 64 * 4) return go(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    if (pieces <= 256 * 2) return go(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (pieces <= 256 * 4) return go(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
    if (pieces <= 512 * 4) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
    if (pieces <= 512 * 8) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 8>());
    if (pieces <= 512 * 13) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 13>());
    if (pieces <= 512 * 16) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 16>());
    if (pieces <= 512 * 24) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 24>());
    if (pieces <= 512 * 32) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 32>());
    if constexpr (sizeof(T) == 4)
        if (pieces <= 512 * 48) return go(std::integral_constant<int, 512>(), std::integral_constant<int, 48>());
    return false;
}

template <bool POLICY> int forward(const Loss &k, int dtype, hipStream_t s) {
    if (k.rows == 0) return ACE_OK;
    return by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        int rc = ACE_OK;
        if (held<(POLICY ? POLICY_LOSS : LOGPROBS), T>(k, s, &rc)) return rc;
        for (int64_t first = 0; first < k.rows && rc == ACE_OK; first += MOST_GROUPS) {
            loss_rows<T, 512, POLICY><<<groups(k.rows - first), 512, 0, s>>>(k, first);
            rc = layer_launched();
        }
        return rc;
    });
}
int backward(const Loss &k, int dtype, bool policy, hipStream_t s) {
    if (k.rows == 0) return ACE_OK;
    return by_type(dtype, [&](auto t) {
        loss_back<decltype(t)><<<groups(k.rows * parts_of<decltype(t)>(k.vocab)), BACK_LANES, 0, s>>>(k, policy);
        return layer_launched();
    });
}
int check_out(const ace_token_loss_t *a, const void *out, int64_t stride) {
    if (a->rows == 0) return ACE_OK;
    if (!out || ((uintptr_t)out & (a->dtype == ACE_T_F32 ? 3 : 1)) || (a->rows > 1 && stride < a->vocab)) return ACE_EINVAL;
    return out == a->d_logits && a->rows > 1 && stride != a->row_stride ? ACE_EINVAL : ACE_OK;
}

}  // namespace

extern "C" int ace_token_logprobs(const ace_token_loss_t *a, float *d_logp, float *d_stats, void *stream) {
    const int rc = check(a, false);
    if (rc != ACE_OK || a->rows == 0) return rc;
    if (!d_logp || !d_stats) return ACE_EINVAL;
    Loss k = args_of(a);
    k.logp = d_logp, k.stats = d_stats;
    return forward<false>(k, a->dtype, (hipStream_t)stream);
}

extern "C" int ace_token_logprobs_gradient(const ace_token_loss_t *a, const float *g_logp, const float *d_logp, const float *d_stats, void *d_dlogits, int64_t out_stride,
                                           void *stream) {
    int rc = check(a, false);
    if (rc != ACE_OK || a->rows == 0) return rc;
    if (!g_logp || !d_stats || (rc = check_out(a, d_dlogits, out_stride)) != ACE_OK) return ACE_EINVAL;
    Loss k = args_of(a);
    k.logp = (float *)d_logp, k.g = g_logp, k.stats = (float *)d_stats, k.d_logits = d_dlogits, k.out_stride = out_stride;
    return backward(k, a->dtype, false, (hipStream_t)stream);
}

extern "C" int ace_token_logprobs_backward(const ace_token_loss_t *a, const float *g_logp, const float *d_stats, void *d_dlogits, int64_t out_stride, void *stream) {
    return ace_token_logprobs_gradient(a, g_logp, nullptr, d_stats, d_dlogits, out_stride, stream);
}

extern "C" size_t ace_policy_loss_workspace_bytes(const ace_token_loss_t *a) { return check(a, true) == ACE_OK ? (size_t)a->rows * sizeof(double) : 0; }

static int policy(const ace_token_loss_t *a, Loss &k, float *d_loss, float *d_logp, float *d_stats, float *d_dlogp, void *d_workspace, size_t workspace_bytes) {
    const int rc = check(a, true);
    if (rc != ACE_OK) return rc;
    if (!d_loss || (a->rows > 0 && (!d_logp || !d_stats || !d_dlogp || !d_workspace))) return ACE_EINVAL;
    if (((uintptr_t)d_workspace & 7) || workspace_bytes < ace_policy_loss_workspace_bytes(a)) return ACE_EINVAL;
    k = args_of(a);
    k.logp = d_logp, k.stats = d_stats, k.d_logp = d_dlogp, k.row_loss = (double *)d_workspace, k.loss = d_loss;
    return ACE_OK;
}
static int sum(const Loss &k, hipStream_t s) {
    loss_sum<<<1, SUM_LANES, 0, s>>>(k.row_loss, k.rows, k.loss);
    return layer_launched();
}

extern "C" int ace_policy_loss(const ace_token_loss_t *a, float *d_loss, float *d_logp, float *d_stats, float *d_dlogp, void *d_workspace, size_t workspace_bytes,
                               void *stream) {
    Loss k;
    int rc = policy(a, k, d_loss, d_logp, d_stats, d_dlogp, d_workspace, workspace_bytes);
    if (rc != ACE_OK || (rc = forward<true>(k, a->dtype, (hipStream_t)stream)) != ACE_OK) return rc;
    return sum(k, (hipStream_t)stream);
}

extern "C" int ace_policy_loss_gradient(const ace_token_loss_t *a, const float *g_loss, float *d_loss, float *d_logp, float *d_stats, float *d_dlogp, void *d_dlogits,
                                        int64_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream) {
    Loss k;
    int rc = policy(a, k, d_loss, d_logp, d_stats, d_dlogp, d_workspace, workspace_bytes);
    if (rc != ACE_OK || (rc = check_out(a, d_dlogits, out_stride)) != ACE_OK) return rc;
    k.g = g_loss, k.d_logits = d_dlogits, k.out_stride = out_stride;
    bool once = false;
    if (k.rows > 0) once = by_type(a->dtype, [&](auto t) { return held<POLICY_GRADIENT, decltype(t)>(k, (hipStream_t)stream, &rc); });
    if (once) return rc != ACE_OK ? rc : sum(k, (hipStream_t)stream);
    if ((rc = forward<true>(k, a->dtype, (hipStream_t)stream)) != ACE_OK) return rc;
    if ((rc = backward(k, a->dtype, true, (hipStream_t)stream)) != ACE_OK) return rc;
    return sum(k, (hipStream_t)stream);
}
