/* What the two passes of the norms around a block share: a row's lanes, sums over them, the launches' arguments. */
#ifndef LAYER_NORM_H
#define LAYER_NORM_H

#include "layer_common.h"

struct NormArgs {
    int64_t rows, rows_per_gate, run, gates, runs;
    int width, layer, token_gate;
    float alpha, eps;
    const void *x, *f, *gate, *w2, *b2, *w1, *b1;
    void *r, *y;
    const void *dr, *dy;
    void *dx, *df, *dgate, *dw2, *db2, *dw1, *db1;
    float *stats;
    float *sum_a, *sum_b, *sum_w1, *sum_b1;
};

/* (in layer_norm_back.hip) */
int norm_backward_launch(const NormArgs &a, int dtype, hipStream_t stream);

/* A row's lanes hold NV vectors of eight elements each, at distances of the workgroup: as few vectors and lanes as hold the row.
 * Up to 12,288 elements of 16 bits (7,680 of 32) the parameters lie in LDS beside the row and its sums in a lane's registers: one
 * vector per lane of up to 1,024, two of up to 768 lanes, whose 168 registers the backward pass needs.  Longer rows read the
 * parameters where they are and ask for no row ahead: at 12,288 that takes 161 us instead of 155 forward and 737 instead of 285 backward
 * (8,192 rows of bfloat16; at 7,680 of float32 223 and 195, 830 and 314).  Their kernels are compiled for 1,024 lanes of 128 registers, which
 * the backward pass overruns: 16,384 elements of bfloat16 take 1,060 us backward, 12,288 of float32 1,375, 1.5 and 1.8 TB/s of six rows,
 * where shorter ones reach 4.2 to 4.7.  So do two vectors per lane of rows that do not end with a whole one: 8,193 elements of bfloat16
 * in 179 and 426 us (8,192 in 104 and 178), 12,289 in 321 and 1,552.  Forward, two vectors per lane begin where one would need
 * more than 768 lanes, of which a CU holds one workgroup: 16,384 rows of 8,192 in 201 us instead of 231, of 6,656 in 177 instead of 216, of
 * 6,144 in 171 against 156.  Backward the sums of a second vector cost more than that: 379 us against 320 at 8,192. */
struct NormShape { int nv, lanes; };
inline NormShape norm_shape(int width, int bytes, bool forward) {
    const int v = (width + 7) / 8, one = forward ? 768 : 1024;
    const int nv = bytes == 2 ? (v <= one ? 1 : v <= 1536 ? 2 : v <= 3 * 1024 ? 3 : 4) : (v <= 960 ? 1 : v <= 3 * 1024 ? 3 : 4);
    return {nv, ((v + nv - 1) / nv + 63) / 64 * 64};
}
template <int NV> constexpr bool norm_params_in_lds() { return NV <= 2; }
/* a parameter's elements in LDS: a vector for every lane, whether the row reaches it or not */
inline int norm_pitch(const NormShape &s) { return s.lanes * s.nv * 8; }

/* CALL(CAP, NV, EVEN), CAP: the most lanes that a variant is launched with */
#define NORM_FOR_SHAPE(CALL, FORWARD)                                     \
    const NormShape shape = norm_shape(a.width, sizeof(T), FORWARD);      \
    if (shape.nv == 1) NORM_EVEN(CALL, 1024, 1)                           \
    else if (shape.nv == 2) NORM_TWO(CALL)                                \
    else if (shape.nv == 3) NORM_EVEN(CALL, 1024, 3)                      \
    else NORM_EVEN(CALL, 1024, 4)
/* rows of whole vectors need no looking at single elements */
#define NORM_EVEN(CALL, CAP, NV)                                          \
    {                                                                     \
        if (a.width % 8 == 0) CALL(CAP, NV, true)                         \
        else CALL(CAP, NV, false)                                         \
    }
#define NORM_TWO(CALL)                                                    \
    {                                                                     \
        if constexpr (sizeof(T) == 2) NORM_EVEN(CALL, 768, 2)             \
    }

/* Sums over the lanes of a wavefront, in every lane, in one fixed order: neighbours, then pairs, fours and eights, then sixteens and
 * halves, all between registers. */
template <int CTRL> __device__ inline float with_lane(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ inline float row_sum(float v) { return with_lane<0x140>(with_lane<0x141>(with_lane<0x4e>(with_lane<0xb1>(v)))); }
__device__ inline float wave_sum(float v) {
    v = row_sum(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}

typedef float2 NormExchange[2][16];

/* over the workgroup's wavefronts; `slot` alternates, so that a later exchange never writes what a slow lane still reads */
__device__ inline float2 sum_all(float2 s, NormExchange &lds, int slot) {
    s.x = wave_sum(s.x), s.y = wave_sum(s.y);
    const int waves = blockDim.x >> 6;
    if (waves > 1) {
        if ((threadIdx.x & 63) == 0) lds[slot][threadIdx.x >> 6] = s;
        __syncthreads();
        const int w = threadIdx.x & 15;
        s = lds[slot][w < waves ? w : 0];
        s.x = row_sum(w < waves ? s.x : 0.0f), s.y = row_sum(w < waves ? s.y : 0.0f);
    }
    return s;
}
__device__ inline float sum_all(float v, NormExchange &lds, int slot) { return sum_all(float2{v, 0.0f}, lds, slot).x; }

/* Eight elements as a lane keeps them: two to a register where they have 16 bits (a vector of such elements would be kept one to a
 * register from one loop iteration to the next). */
template <class T> struct Packed { typedef u32x4 type; };
template <> struct Packed<float> { typedef f32x8 type; };
template <class T> using packed8 = typename Packed<T>::type;

template <class T> __device__ inline f32x8 open8(packed8<T> v) {
    if constexpr (__is_same(T, float)) return v;
    else if constexpr (__is_same(T, bf16)) {
        f32x8 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[2 * i] = __uint_as_float(v[i] << 16), r[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        return r;
    } else
        return __builtin_convertvector(__builtin_bit_cast(vec8<T>, v), f32x8);
}
/* half of them: what is computed at a time where registers are few */
template <class T> __device__ inline f32x4 open4(packed8<T> v, int half) {
    if constexpr (__is_same(T, float)) return half ? v.hi : v.lo;
    else if constexpr (__is_same(T, bf16))
        return f32x4{__uint_as_float(v[2 * half] << 16), __uint_as_float(v[2 * half] & 0xffff0000u), __uint_as_float(v[2 * half + 1] << 16),
                     __uint_as_float(v[2 * half + 1] & 0xffff0000u)};
    else {
        const vec8<T> e = __builtin_bit_cast(vec8<T>, v);
        return f32x4{(float)e[4 * half], (float)e[4 * half + 1], (float)e[4 * half + 2], (float)e[4 * half + 3]};
    }
}
template <class T> __device__ inline packed8<T> pack8(f32x8 v) { return __builtin_bit_cast(packed8<T>, __builtin_convertvector(v, vec8<T>)); }

/* A row's address is the same for the whole workgroup, a lane adds its element's 32-bit place. */
template <class T> __device__ inline const T *row_at(const void *p, int64_t row, int width) { return (const T *)p + row * width; }
template <class T> __device__ inline T *row_at(void *p, int64_t row, int width) { return (T *)p + row * width; }
/* Rows of whole vectors go through a buffer descriptor of the row (scalar registers): one 32-bit place per vector and lane, and lanes
 * past the row's end read zero and write nothing, without a branch. */
template <class T> __device__ inline __amdgpu_buffer_rsrc_t row_buffer(const T *row, int width) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)row, 0, width * (int)sizeof(T), 0x00027000);
}
template <class T, bool EVEN> __device__ inline packed8<T> row_load(const T *row, int width, uint32_t at, int n) {
    packed8<T> r = 0;
    if constexpr (!EVEN) {
        if (n > 0) r = __builtin_bit_cast(packed8<T>, load_some(row + at, n));
    } else {
        const __amdgpu_buffer_rsrc_t b = row_buffer(row, width);
        if constexpr (sizeof(T) == 2) r = __builtin_bit_cast(packed8<T>, __builtin_amdgcn_raw_buffer_load_b128(b, at * 2, 0, 0));
        else {
            r.lo = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b, at * 4, 0, 0));
            r.hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b, at * 4 + 16, 0, 0));
        }
    }
    return r;
}
template <class T, bool EVEN> __device__ inline void row_store(T *row, int width, uint32_t at, packed8<T> v, int n) {
    if constexpr (!EVEN) {
        if (n > 0) store_some(row + at, __builtin_bit_cast(vec8<T>, v), n);
    } else {
        const __amdgpu_buffer_rsrc_t b = row_buffer(row, width);
        if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), b, at * 2, 0, 0);
        else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, (f32x4)v.lo), b, at * 4, 0, 0);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, (f32x4)v.hi), b, at * 4 + 16, 0, 0);
        }
    }
}

/* The same elements, to be widened anew: keeps a lane from holding them in 32 bits as well. */
template <class T> __device__ inline void again(packed8<T> &v) {
    if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(v));
}

/* The parameters as a row's lanes read them: from LDS, where lane and vector find at place `at` what the lane itself has put there
 * (`otherwise` where there is no such parameter, zero past the row's end), or from memory.  A gate's row is put there when a row
 * of x with another gate begins. */
template <class T, int NV, bool EVEN> struct NormParams {
    static constexpr bool IN_LDS = norm_params_in_lds<NV>();
    T *lds;
    int pitch, width;
    __device__ inline void put(int which, const void *p, const uint32_t *at, const int *n, float otherwise) {
        if (!IN_LDS) return;
#pragma unroll
        for (int k = 0; k < NV; ++k) *(packed8<T> *)(lds + which * pitch + at[k]) = from(p, at[k], n[k], otherwise);
    }
    __device__ inline packed8<T> from(const void *p, uint32_t at, int n, float otherwise) const {
        packed8<T> r = 0;
        if (p) r = row_load<T, EVEN>((const T *)p, width, at, n);
        else if (n > 0) {
            f32x8 v = otherwise;
            if (!EVEN)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : 0.0f;
            r = pack8<T>(v);
        }
        return r;
    }
    __device__ inline f32x8 get(int which, const void *p, uint32_t at, int n, float otherwise) const {
        return open8<T>(IN_LDS ? *(const packed8<T> *)(lds + which * pitch + at) : from(p, at, n, otherwise));
    }
    __device__ inline f32x4 get4(int which, const void *p, uint32_t at, int n, float otherwise, int half) const {
        if (!IN_LDS) return open4<T>(from(p, at, n, otherwise), half);
        const T *e = lds + which * pitch + at + 4 * half;
        if constexpr (__is_same(T, bf16)) {
            const u32x2 v = *(const u32x2 *)e;
            return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
        } else {
            typedef T vec4 __attribute__((ext_vector_type(4)));
            return __builtin_convertvector(*(const vec4 *)e, f32x4);
        }
    }
};

#endif
