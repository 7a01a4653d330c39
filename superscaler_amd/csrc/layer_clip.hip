/*
 * The norm of many gradients, and clipping in place (ace_gradient_norm, ace_gradient_scale).
 *
 *     norm_t = |s| sqrt(sum g^2),   norm = sqrt(sum norm_t^2),   scale = s min(1, max_norm / (norm + 1e-6))
 *
 * A workgroup takes a chunk of one tensor and leaves the sum of its squares; a second launch has a workgroup per tensor, which adds up
 * its chunks' sums, and the last of them to end adds up the tensors'. Every sum is taken in an order that the sizes alone decide.
 *
 * Squares and sums are of 64 bits: a gradient of 1e20 counts (its square passes the range of 32 bits), one of 1e-25 does too, and a sum over
 * 10^9 elements loses nothing. Beside the loads that costs little: a conversion and a multiply-add per element.
 *
 * Tensors travel as a kernel argument: address, elements of the last chunk, chunks before it (TENSORS of them fill the 4 KB that an
 * argument block holds); a workgroup finds its tensor by halving.
 */
#include "layer_common.h"

namespace {

constexpr int LANES = 256, TENSORS = 240, UNIT = LANES * 8;

struct List {
    uint64_t grad[TENSORS];
    uint32_t chunks_before[TENSORS];   /* of those of this launch */
    uint32_t last[TENSORS];            /* elements of the last chunk, less one; type in the upper two bits */
};
struct Launch {
    List list;
    double *sums;                      /* of this launch's first chunk */
    uint32_t *ticket;                  /* NULL but in the first launch, which clears it */
    const float *scale;                /* (clipping) */
    uint32_t chunks, units;            /* a chunk: that many times UNIT elements */
    int32_t tensors;
};
static_assert(sizeof(Launch) <= 4096, "an argument block holds 4 KB");

struct Chunk {
    uint64_t at;
    uint32_t count, type;
};
__device__ inline Chunk chunk_of(const Launch &a, uint32_t chunk) {
    int lo = 0, hi = a.tensors;        /* the last tensor with no more than `chunk` chunks before it */
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.list.chunks_before[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    const uint32_t end = lo + 1 < a.tensors ? a.list.chunks_before[lo + 1] : a.chunks, own = chunk - a.list.chunks_before[lo], last = a.list.last[lo];
    const uint32_t type = last >> 30, size = type == ACE_T_F32 ? 4 : 2;
    return {a.list.grad[lo] + (uint64_t)own * a.units * UNIT * size, chunk + 1 == end ? (last & 0x3fffffff) + 1 : a.units * UNIT, type};
}

/* sum over a workgroup, for its first lane; `scratch`: one for each wavefront */
__device__ inline double sum_lanes(double x, double *scratch) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) x += scratch[w];
    return x;
}

template <class T> __device__ inline double squares(const T *g, uint32_t count) {
    double x = 0.0, y = 0.0;
    for (uint32_t at = threadIdx.x * 8; at < count; at += UNIT) {
        const vec8<T> v = load_some(g + at, (int)(count - at));
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const double a = (double)(float)v[i], b = (double)(float)v[i + 1];
            x = __builtin_fma(a, a, x), y = __builtin_fma(b, b, y);
        }
    }
    return x + y;
}

__global__ void __launch_bounds__(LANES) square_sums(const Launch a) {
    __shared__ double scratch[LANES / 64];
    if (a.ticket && blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
    if (blockIdx.x >= a.chunks) return;
    const Chunk c = chunk_of(a, blockIdx.x);
    double x = c.type == ACE_T_F32 ? squares((const float *)c.at, c.count) : c.type == ACE_T_BF16 ? squares((const bf16 *)c.at, c.count) : squares((const f16 *)c.at, c.count);
    x = sum_lanes(x, scratch);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = x;
}

struct Join {
    uint32_t chunks_before[TENSORS + 1];
    const double *sums;                /* of this launch's first chunk */
    double *tensor_sums;               /* of all tensors */
    uint32_t *ticket;
    float *norms;                      /* of this launch's first tensor */
    float *result;
    const float *grad_scale;
    double max_norm;
    int64_t first, tensors;            /* this launch's first tensor; how many there are in all */
};

/* The sums of tensors go from workgroup to workgroup through memory: the last one to take a number from `ticket` sees them all. */
__global__ void __launch_bounds__(LANES) join_sums(const Join a) {
    __shared__ double scratch[2][LANES / 64];
    __shared__ bool end;
    const double s = a.grad_scale ? (double)*a.grad_scale : 1.0;
    double x = 0.0;
    const uint32_t end_chunk = a.chunks_before[blockIdx.x + 1];
    for (uint32_t c = a.chunks_before[blockIdx.x] + threadIdx.x; c < end_chunk; c += 8 * LANES) {
        double each[8];      /* (asked for together: a matrix of 5,120 x 20,480 has 6,400) */
#pragma unroll
        for (int k = 0; k < 8; ++k) each[k] = c + k * LANES < end_chunk ? a.sums[c + k * LANES] : 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) x += each[k];
    }
    x = sum_lanes(x, scratch[0]);
    if (threadIdx.x == 0) {
        a.norms[blockIdx.x] = (float)(__builtin_sqrt(x) * __builtin_fabs(s));
        __hip_atomic_store(a.tensor_sums + a.first + blockIdx.x, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        end = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1 == (uint32_t)a.tensors;
    }
    __syncthreads();
    if (!end) return;
    x = 0.0;
    for (int64_t t = threadIdx.x; t < a.tensors; t += LANES) x += __hip_atomic_load(a.tensor_sums + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = sum_lanes(x, scratch[1]);
    if (threadIdx.x == 0) {
        const double norm = __builtin_sqrt(x) * __builtin_fabs(s), by = a.max_norm / (norm + 1e-6);
        a.result[0] = (float)norm, a.result[1] = (float)(a.max_norm > 0.0 && !(by >= 1.0) ? s * by : s);   /* (a norm that is no number makes the factor none) */
    }
}

template <class T> __device__ inline void scale_chunk(T *g, uint32_t count, float by) {
    for (uint32_t at = threadIdx.x * 8; at < count; at += UNIT) {
        vec8<T> v = load_some(g + at, (int)(count - at));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float x = (float)v[i] * by;
            asm volatile("" : "+v"(x));   /* (a product of 32 bits, rounded from there: of half precision the compiler would make one operation) */
            v[i] = (T)x;
        }
        store_some(g + at, v, (int)(count - at));
    }
}
__global__ void __launch_bounds__(LANES) scale_chunks(const Launch a) {
    const float by = *a.scale;
    if (by == 1.0f) return;
    const Chunk c = chunk_of(a, a.chunks - 1 - blockIdx.x);   /* (from the end: what the norm has just read is in the card's cache) */
    if (c.type == ACE_T_F32) scale_chunk((float *)c.at, c.count, by);
    else if (c.type == ACE_T_BF16) scale_chunk((bf16 *)c.at, c.count, by);
    else scale_chunk((f16 *)c.at, c.count, by);
}

constexpr int64_t UNITS = 8, MOST_CHUNKS = (int64_t)1 << 23, MOST_TENSORS = (int64_t)1 << 20;   /* (a launch of chunks: 2^31 lanes) */

int64_t chunks_of(int64_t n) { return (n + UNITS * UNIT - 1) / (UNITS * UNIT); }

int check(const ace_gradient_t *grads, int64_t n) {
    if (n < 0 || (n > 0 && !grads)) return ACE_EINVAL;
    if (n > MOST_TENSORS) return ACE_ETOOBIG;
    for (int64_t t = 0; t < n; ++t) {
        if (grads[t].n < 0 || grads[t].dtype < ACE_T_F32 || grads[t].dtype > ACE_T_F16 || (grads[t].n > 0 && !grads[t].d_grad)) return ACE_EINVAL;
        if ((uintptr_t)grads[t].d_grad & (grads[t].dtype == ACE_T_F32 ? 3 : 1)) return ACE_EINVAL;
        if (chunks_of(grads[t].n) > MOST_CHUNKS) return ACE_ETOOBIG;
    }
    return ACE_OK;
}

/* go(launch, its first tensor, its first chunk): the tensors in runs that a launch holds */
template <class Go> int in_runs(const ace_gradient_t *grads, int64_t n, Go go) {
    Launch l = {};
    l.units = (uint32_t)UNITS;
    int64_t first = 0, before = 0;
    for (int64_t t = 0; t < n; ++t) {
        const int64_t chunks = chunks_of(grads[t].n);
        if (l.tensors == TENSORS || l.chunks + chunks > MOST_CHUNKS) {
            const int rc = go(l, first, before);
            if (rc != ACE_OK) return rc;
            first = t, before += l.chunks, l.tensors = 0, l.chunks = 0;
        }
        /* (an empty tensor has as many chunks before it as the next one, which is the one that is found) */
        l.list.grad[l.tensors] = (uint64_t)(uintptr_t)grads[t].d_grad;
        l.list.chunks_before[l.tensors] = l.chunks;
        l.list.last[l.tensors] = (uint32_t)(chunks ? grads[t].n - (chunks - 1) * UNITS * UNIT - 1 : 0) | (uint32_t)grads[t].dtype << 30;
        l.tensors++, l.chunks += (uint32_t)chunks;
    }
    return l.tensors > 0 ? go(l, first, before) : ACE_OK;
}

int64_t all_chunks(const ace_gradient_t *grads, int64_t n) {
    int64_t chunks = 0;
    for (int64_t t = 0; t < n; ++t) chunks += chunks_of(grads[t].n);
    return chunks;
}

}  // namespace

extern "C" size_t ace_gradient_norm_workspace_bytes(const ace_gradient_t *grads, int64_t n_tensors) {
    if (check(grads, n_tensors) != ACE_OK) return 0;
    return (size_t)(all_chunks(grads, n_tensors) + n_tensors + 1) * sizeof(double);
}

extern "C" int ace_gradient_norm(const ace_gradient_t *grads, int64_t n_tensors, double max_norm, const float *d_grad_scale, float *d_result, float *d_norms,
                                 void *d_workspace, size_t workspace_bytes, void *stream) {
    const int rc = check(grads, n_tensors);
    if (rc != ACE_OK) return rc;
    if (n_tensors == 0 || !d_result || !d_norms || !(max_norm >= 0.0) || !d_workspace || ((uintptr_t)d_workspace & 7)) return ACE_EINVAL;
    if (workspace_bytes < ace_gradient_norm_workspace_bytes(grads, n_tensors)) return ACE_EINVAL;
    uint32_t *ticket = (uint32_t *)d_workspace;
    double *tensor_sums = (double *)d_workspace + 1, *sums = tensor_sums + n_tensors;
    return in_runs(grads, n_tensors, [&](Launch &l, int64_t first, int64_t before) {
        l.sums = sums + before, l.ticket = first == 0 ? ticket : nullptr;
        square_sums<<<l.chunks > 0 ? l.chunks : 1, LANES, 0, (hipStream_t)stream>>>(l);
        const int rc = layer_launched();
        if (rc != ACE_OK) return rc;
        Join j = {};
        for (int t = 0; t < l.tensors; ++t) j.chunks_before[t] = l.list.chunks_before[t];
        j.chunks_before[l.tensors] = l.chunks;
        j.sums = l.sums, j.tensor_sums = tensor_sums, j.ticket = ticket, j.norms = d_norms + first, j.result = d_result, j.grad_scale = d_grad_scale;
        j.max_norm = max_norm, j.first = first, j.tensors = n_tensors;
        join_sums<<<(uint32_t)l.tensors, LANES, 0, (hipStream_t)stream>>>(j);
        return layer_launched();
    });
}

extern "C" int ace_gradient_scale(const ace_gradient_t *grads, int64_t n_tensors, const float *d_scale, void *stream) {
    const int rc = check(grads, n_tensors);
    if (rc != ACE_OK) return rc;
    if (n_tensors > 0 && !d_scale) return ACE_EINVAL;
    return in_runs(grads, n_tensors, [&](Launch &l, int64_t, int64_t) {
        if (l.chunks == 0) return (int)ACE_OK;
        l.scale = d_scale;
        scale_chunks<<<l.chunks, LANES, 0, (hipStream_t)stream>>>(l);
        return layer_launched();
    });
}
