/* What the kernels of the training-layer operators share: loads of eight elements, conversions, sums over lanes, errors. */
#ifndef LAYER_COMMON_H
#define LAYER_COMMON_H

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>
#include <atomic>
#include "ace_layer.h"

/* (in layer_norm.hip) remembers a HIP error for ace_layer_last_hip_error; ACE_OK or ACE_EHIP */
int layer_hip_status(hipError_t e);

/* (in layer_norm.hip) lets a kernel have `bytes` of LDS on the current device: asked for once per device, whose bits `done` keeps, and
 * again after a failure */
int layer_allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> &done);

static inline int layer_launched() { return layer_hip_status(hipGetLastError()); }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16;
typedef _Float16 f16;

/* Eight consecutive elements as they lie in memory.  Addresses are multiples of the element's size only: the loads and stores
 * below, and those through buffer descriptors of the norms' rows, are full-width at any alignment (unaligned access is on for every
 * process of this platform). */
template <class T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };
template <class T> using vec8 = typename Vec8<T>::type;
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <class T> __device__ inline vec8<T> load8(const T *p) {
    vec8<T> r;
    __builtin_memcpy(&r, p, sizeof r);
    return r;
}
template <class T> __device__ inline void store8(T *p, vec8<T> r) { __builtin_memcpy(p, &r, sizeof r); }

/* of a row's last vector only the first n elements are there; the rest is zero */
template <class T> __device__ inline vec8<T> load_some(const T *p, int n) {
    if (n >= 8) return load8(p);
    vec8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = i < n ? p[i] : (T)0;
    return r;
}
template <class T> __device__ inline void store_some(T *p, vec8<T> r, int n) {
    if (n >= 8) {
        store8(p, r);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = r[i];
}

#endif
