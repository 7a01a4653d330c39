/*
 * AdamW over many tensors in one launch (ace_adamw_step), and the values that 8-bit moments stand for (ace_adamw_moments).
 *
 * A workgroup of 256 lanes takes a chunk of 8,192 elements of one tensor, eight elements per lane and pass, so that every
 * stream is read and written once with 8- to 32-byte accesses.  The gradients' addresses, which a training step may change
 * from call to call, travel as a kernel argument (400 of them: 3.2 of the 4 KB that an argument block holds); everything
 * that stays is in the caller's device tables.  With 8-bit moments the 32 lanes of half a wavefront hold one block of 256
 * elements, whose two maxima are five exchanges between lanes.
 *
 * The moments' arithmetic is unfused, with correctly rounded square roots and quotients: the codes are then the same on every
 * machine that rounds like IEEE 754, and so are runs that are repeated elsewhere.
 *
 * Bound by memory: 630 million weights with copies in bfloat16 and moments of 32 bits, 28 bytes each: 3.39 ms, 5.2 TB/s, as a large copy
 * does; 1.2 billion with moments of 8 bits, 16 bytes each: 3.80 ms, 5.1 TB/s, and 2.25 ms for the values that they stand for, 5.4 TB/s.
 * (Two or four passes of the loop at once change nothing.)
 */
#include "layer_common.h"

#pragma clang fp contract(off)

namespace {

struct Launch {
    const ace_adamw_tensor_t *tensors;
    const int32_t *chunk_tensor;
    int64_t first_chunk;
    int32_t first_tensor;
    float beta1, one_minus_beta1, beta2, one_minus_beta2, decay, step_size, root_scale, eps;
    void *m, *v;
    float *m_scale, *v_scale;
    const float *grad_scale;
    const void *grads[ACE_ADAMW_MAX_TENSORS];
};
static_assert(sizeof(Launch) <= 4096, "an argument block holds 4 KB");

constexpr int LANES = 256, PASS = LANES * 8;

__device__ inline uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

/* the largest magnitude in half a wavefront, as bits: those of a NaN are larger than any number's */
__device__ inline uint32_t half_wave_max(uint32_t bits) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) bits = larger(bits, (uint32_t)__shfl_xor((int)bits, d));
    return bits;
}

struct None {};
template <class C> __device__ inline void store_copy(C *to, int64_t at, const float *p, int n) {
    vec8<C> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (C)p[i];
    store_some(to + at, r, n);
}
template <> __device__ inline void store_copy<None>(None *, int64_t, const float *, int) {}

template <int BITS, class G, class C> __global__ void __launch_bounds__(LANES) adamw_kernel(const Launch a) {
    const int64_t chunk = a.first_chunk + blockIdx.x;
    const int tensor = a.chunk_tensor[chunk];
    const ace_adamw_tensor_t t = a.tensors[tensor];
    const G *grad = (const G *)a.grads[tensor - a.first_tensor];
    C *copy = (C *)t.d_copy;
    const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
    const int64_t base = (chunk - t.first_chunk) * ACE_ADAMW_CHUNK;
#pragma unroll 1
    for (int pass = 0; pass < ACE_ADAMW_CHUNK / PASS; ++pass) {
        const int64_t at = base + pass * PASS + threadIdx.x * 8;
        const int64_t left = t.n - at;
        /* (a block with no element of the tensor is nobody's: nothing of it is read or written) */
        if (BITS == 8 ? left + (threadIdx.x & 31) * 8 <= 0 : left <= 0) break;
        const int n = left > 8 ? 8 : (int)left;
        const vec8<float> p0 = load_some(t.d_param + at, n);
        const vec8<G> g0 = load_some(grad + at, n);
        float m[8], v[8], u[8], p[8];
        if (BITS == 32) {
            const vec8<float> m0 = load_some((const float *)a.m + t.state_at + at, n), v0 = load_some((const float *)a.v + t.state_at + at, n);
#pragma unroll
            for (int i = 0; i < 8; ++i) m[i] = m0[i], v[i] = v0[i];
        } else {
            /* (whole blocks: the moments' storage is padded to them) */
            const vec8<int8_t> mc = load8((const int8_t *)a.m + t.state_at + at);
            const vec8<uint8_t> vc = load8((const uint8_t *)a.v + t.state_at + at);
            const float ms = a.m_scale[(t.state_at + at) / ACE_ADAMW_BLOCK], vs = a.v_scale[(t.state_at + at) / ACE_ADAMW_BLOCK];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m[i] = (float)mc[i] * ms;
                const float root = (float)vc[i] * vs;
                v[i] = root * root;
                if (i >= n) m[i] = v[i] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = (float)g0[i] * gs;
            m[i] = m[i] * a.beta1 + g * a.one_minus_beta1;
            v[i] = v[i] * a.beta2 + (g * g) * a.one_minus_beta2;
            if (BITS == 8 && i >= n) m[i] = v[i] = 0.0f;
            u[i] = __builtin_sqrtf(v[i]);
            /* (the parameter is rounded once more anyway: a reciprocal that is right to its last bit or the one before it) */
            p[i] = p0[i] * a.decay - m[i] * a.step_size * __builtin_amdgcn_rcpf(u[i] * a.root_scale + a.eps);
        }
        vec8<float> out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = p[i];
        store_some(t.d_param + at, out, n);
        store_copy(copy, at, p, n);
        if (BITS == 32) {
            vec8<float> mo, vo;
#pragma unroll
            for (int i = 0; i < 8; ++i) mo[i] = m[i], vo[i] = v[i];
            store_some((float *)a.m + t.state_at + at, mo, n);
            store_some((float *)a.v + t.state_at + at, vo, n);
        } else {
            uint32_t m_bits = 0, u_bits = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m_bits = larger(m_bits, __float_as_uint(m[i]) & 0x7fffffffu);
                u_bits = larger(u_bits, __float_as_uint(u[i]) & 0x7fffffffu);
            }
            const float m_top = __uint_as_float(half_wave_max(m_bits)), u_top = __uint_as_float(half_wave_max(u_bits));
            const bool m_fine = m_top < __builtin_inff(), u_fine = u_top < __builtin_inff();
            /* (a block whose largest m is below 1e-30, whose reciprocal would pass the range's end, goes in steps of that one's; a root
             * that is not zero is never so small) */
            const float m_unit = m_top > 0.0f ? fmaxf(m_top, 1e-30f) : 0.0f;
            const float m_by = m_fine ? 1.0f / fmaxf(m_top, 1e-30f) * 127.0f : 0.0f, u_by = u_fine ? 1.0f / fmaxf(u_top, 1e-30f) * 255.0f : 0.0f;
            vec8<int8_t> mc;
            vec8<uint8_t> vc;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mc[i] = m_fine ? (int8_t)(int)__builtin_rintf(m[i] * m_by) : (int8_t)0;
                const int code = u_fine ? (int)__builtin_rintf(u[i] * u_by) : 0;
                vc[i] = (uint8_t)(u[i] > 0.0f && code < 1 ? 1 : code);
            }
            store8((int8_t *)a.m + t.state_at + at, mc);
            store8((uint8_t *)a.v + t.state_at + at, vc);
            if ((threadIdx.x & 31) == 0) {
                a.m_scale[(t.state_at + at) / ACE_ADAMW_BLOCK] = m_fine ? m_unit * (float)(1.0 / 127) : __builtin_nanf("");
                a.v_scale[(t.state_at + at) / ACE_ADAMW_BLOCK] = u_fine ? u_top * (float)(1.0 / 255) : __builtin_nanf("");
            }
        }
    }
}

/* A lane per eight codes of each moment. */
__global__ void __launch_bounds__(LANES) moments_kernel(const int8_t *m, const uint8_t *v, const float *m_scale, const float *v_scale, int64_t vectors, float *m_out,
                                                        float *v_out) {
    for (int64_t k = (int64_t)blockIdx.x * LANES + threadIdx.x; k < vectors; k += (int64_t)gridDim.x * LANES) {
        const vec8<int8_t> mc = load8(m + k * 8);
        const vec8<uint8_t> vc = load8(v + k * 8);
        const float ms = m_scale[k / (ACE_ADAMW_BLOCK / 8)], vs = v_scale[k / (ACE_ADAMW_BLOCK / 8)];
        vec8<float> mo, vo;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mo[i] = (float)mc[i] * ms;
            const float root = (float)vc[i] * vs;
            vo[i] = root * root;
        }
        store8(m_out + k * 8, mo);
        store8(v_out + k * 8, vo);
    }
}

template <int BITS, class G> int launch_copy(int copy_type, const Launch &l, int64_t chunks, hipStream_t stream) {
    const dim3 grid((uint32_t)chunks);
    if (copy_type == ACE_T_NONE) adamw_kernel<BITS, G, None><<<grid, LANES, 0, stream>>>(l);
    else if (copy_type == ACE_T_BF16) adamw_kernel<BITS, G, bf16><<<grid, LANES, 0, stream>>>(l);
    else adamw_kernel<BITS, G, f16><<<grid, LANES, 0, stream>>>(l);
    return layer_launched();
}

template <int BITS> int launch(int grad_type, int copy_type, const Launch &l, int64_t chunks, hipStream_t stream) {
    if (grad_type == ACE_T_F32) return launch_copy<BITS, float>(copy_type, l, chunks, stream);
    if (grad_type == ACE_T_BF16) return launch_copy<BITS, bf16>(copy_type, l, chunks, stream);
    return launch_copy<BITS, f16>(copy_type, l, chunks, stream);
}

constexpr int64_t MOST_CHUNKS = (int64_t)1 << 23;   /* of one launch: 2^31 lanes */

}  // namespace

extern "C" int ace_adamw_step(const ace_adamw_t *a, const void *const *grads, const int64_t *first_chunks, const float *d_grad_scale, float beta1,
                              float one_minus_beta1, float beta2, float one_minus_beta2, float decay, float step_size, float root_scale, float eps,
                              void *stream) {
    if (!a || a->n_tensors < 0 || a->n_chunks < 0 || (a->state_bits != 8 && a->state_bits != 32)) return ACE_EINVAL;
    if (a->grad_type < ACE_T_F32 || a->grad_type > ACE_T_F16 || a->copy_type < ACE_T_BF16 || a->copy_type > ACE_T_NONE) return ACE_EINVAL;
    if (a->n_tensors == 0 || a->n_chunks == 0) return ACE_OK;
    if (!grads || !first_chunks || !a->d_tensors || !a->d_chunk_tensor || !a->d_m || !a->d_v || (a->state_bits == 8 && (!a->d_m_scale || !a->d_v_scale))) return ACE_EINVAL;
    if (first_chunks[0] != 0 || first_chunks[a->n_tensors] != a->n_chunks) return ACE_EINVAL;
    for (int t = 0; t < a->n_tensors; ++t)
        if (first_chunks[t + 1] < first_chunks[t] || (first_chunks[t + 1] > first_chunks[t] && !grads[t])) return ACE_EINVAL;
    Launch l;
    l.tensors = a->d_tensors;
    l.chunk_tensor = a->d_chunk_tensor;
    l.beta1 = beta1, l.one_minus_beta1 = one_minus_beta1, l.beta2 = beta2, l.one_minus_beta2 = one_minus_beta2;
    l.decay = decay, l.step_size = step_size, l.root_scale = root_scale, l.eps = eps;
    l.m = a->d_m, l.v = a->d_v, l.m_scale = a->d_m_scale, l.v_scale = a->d_v_scale, l.grad_scale = d_grad_scale;
    for (int t = 0; t < a->n_tensors; t += ACE_ADAMW_MAX_TENSORS) {
        const int end = t + ACE_ADAMW_MAX_TENSORS < a->n_tensors ? t + ACE_ADAMW_MAX_TENSORS : a->n_tensors;
        l.first_tensor = t;
        for (int k = t; k < end; ++k) l.grads[k - t] = grads[k];
        for (int64_t chunk = first_chunks[t]; chunk < first_chunks[end]; chunk += MOST_CHUNKS) {
            const int64_t count = first_chunks[end] - chunk < MOST_CHUNKS ? first_chunks[end] - chunk : MOST_CHUNKS;
            l.first_chunk = chunk;
            const int rc = a->state_bits == 8 ? launch<8>(a->grad_type, a->copy_type, l, count, (hipStream_t)stream)
                                              : launch<32>(a->grad_type, a->copy_type, l, count, (hipStream_t)stream);
            if (rc != ACE_OK) return rc;
        }
    }
    return ACE_OK;
}

extern "C" int ace_adamw_moments(const int8_t *d_m, const uint8_t *d_v, const float *d_m_scale, const float *d_v_scale, int64_t n_blocks, float *d_m_out,
                                 float *d_v_out, void *stream) {
    if (n_blocks < 0) return ACE_EINVAL;
    if (n_blocks == 0) return ACE_OK;
    if (!d_m || !d_v || !d_m_scale || !d_v_scale || !d_m_out || !d_v_out) return ACE_EINVAL;
    const int64_t vectors = n_blocks * (ACE_ADAMW_BLOCK / 8), groups = (vectors + LANES - 1) / LANES;
    const uint32_t grid = (uint32_t)(groups < MOST_CHUNKS ? groups : MOST_CHUNKS);
    moments_kernel<<<grid, LANES, 0, (hipStream_t)stream>>>(d_m, d_v, d_m_scale, d_v_scale, vectors, d_m_out, d_v_out);
    return layer_launched();
}
