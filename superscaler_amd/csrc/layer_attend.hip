/*
 * Attention over a window of keys and a few first ones: forward for prompts (attend_forward), forward for few queries over long
 * caches (attend_split, attend_join), backward (attend_dq, attend_dkv).
 *
 * All products run on 32x32x16 matrix instructions.  With A a 32 x 16 and B a 16 x 32 operand, lane l holds row (column) l % 32
 * and the eight k of half h = l / 32; of the result it holds column l % 32 and the sixteen rows 8 (i / 4) + 4 h + i % 4.  The kernels
 * compute S^T = K Q^T, so that a lane's results belong to ONE query: its running maximum and sum need one exchange with the
 * lane 32 further, and a query's factor is a scalar of its lane.  The rows that a lane holds of S^T, eight at a time, are
 * 4 h + {0..3} and 8 + 4 h + {0..3} of sixteen keys: taken as the k of the next product (k is summed over, so any order will do
 * that both operands share) they are its B operand as they stand, P^T or dS^T, and the A operand V^T (K^T, Q^T, dO^T) comes from
 * row-major tiles by transposing LDS reads of four rows each.  No value passes through LDS on its way from one product to the
 * next.
 *
 * Tiles go from memory to LDS without registers between, 16 bytes per lane.  A tile's 16-byte pieces are exchanged within
 * their row, piece c of row r at c ^ swizzle(r): both kinds of reads, eight rows at one piece and four rows at two pieces, then
 * fall on different banks.  Rows past the sequence's length (and pieces past the head's size) are read from a page of zeros:
 * whatever stands there in memory, a number or not, takes no part.
 */
#include "layer_common.h"

namespace {

struct Args {
    int batch, queries, keys, heads, kv_heads, dim, shared, window, sinks;
    float scale, scale2;                 /* scale2 = scale / ln 2: exponentials are powers of two */
    const int *start, *length;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3], g_stride[3];
    const void *q, *k, *v, *g;
    void *out;
    float *lse, *delta;
    void *dq, *dk, *dv;
    float *part_o, *part_ml;             /* attend_split: [splits][rows][width], [splits][rows][2] */
    int splits, row_blocks;
};

__device__ uint4 zero_page[1];

typedef __attribute__((address_space(3))) char *lds_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 *lds_tr_ptr;

template <class T> struct Mma;
template <> struct Mma<bf16> {
    typedef bf16x8 frag;
    static __device__ inline f32x16 go(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<f16> {
    typedef f16x8 frag;
    static __device__ inline f32x16 go(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

constexpr float LOG2E = 1.4426950408889634f;

__device__ inline int swizzle(int row) { return 2 * (row & 3) + ((row >> 2) & 1); }

__device__ inline uint32_t lds_offset(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

/* 16 bytes per lane from `from` to LDS at `to` + 16 lane (`to`: the same for the wavefront).  The LDS write is complete when the
 * wavefront's vector-memory counter says so (wait_tiles).  m0, the destination, needs one state before it is used; nothing else in
 * these kernels uses it. */
__device__ inline void to_lds16(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
__device__ inline void to_lds4(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory");
}
template <int LEFT> __device__ inline void wait_tiles() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }
__device__ inline void meet() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

/* ROWS rows of a tile by LANES lanes; rows at or past `end` and elements past `dim` come from the page of zeros. */
template <class T, int PITCH, int ROWS, int LANES> __device__ inline void load_tile(uint32_t to, const T *base, int64_t stride, int row0, int end, int dim, int lane) {
    constexpr int PER = PITCH / 8;
    static_assert(ROWS * PER % LANES == 0, "whole loads");
    const uint32_t wave_at = __builtin_amdgcn_readfirstlane(to + (lane & ~63) * 16);
#pragma unroll
    for (int i = 0; i < ROWS * PER / LANES; ++i) {
        const int p = i * LANES + lane, row = p / PER, piece = (p % PER) ^ (swizzle(row) & (PER - 1));
        const bool there = row0 + row < end && piece * 8 < dim;
        const void *from = there ? (const void *)(base + (int64_t)(row0 + row) * stride + piece * 8) : (const void *)zero_page;
        to_lds16(from, wave_at + i * LANES * 16);
    }
}

/* Where a lane reads its part of an operand whose rows are the tile's rows: row `row`, pieces 2 s + h. */
template <class T, int PITCH> __device__ inline typename Mma<T>::frag row_frag(const char *tile, int row0, int s, int lane) {
    const int row = row0 + (lane & 31), piece = (2 * s + (lane >> 5)) ^ (swizzle(lane & 31) & (PITCH / 8 - 1));
    return *(const typename Mma<T>::frag *)(tile + row * PITCH * 2 + piece * 16);
}

/* The transposed operand: rows are elements 32 t + lane % 32 of the head, k the sixteen tile rows from row0 on. */
template <class T, int PITCH> __device__ inline typename Mma<T>::frag column_frag(const char *tile, int row0, int t, int lane) {
    const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2);
    const int piece = (4 * t + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ (swizzle(r) & (PITCH / 8 - 1));
    const char *at = tile + (row0 + r) * PITCH * 2 + piece * 16 + (i & 1) * 8;
    union { s16x4 half[2]; typename Mma<T>::frag whole; } u;
    u.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(lds_ptr)at);
    u.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(lds_ptr)(at + 8 * PITCH * 2));
    return u.whole;
}

template <class T> __device__ inline typename Mma<T>::frag pack8(const float *p) {
    typename Mma<T>::frag r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)p[i];
    return r;
}

/* Eight elements of a row in memory; zero where the row or the elements are not there. */
template <class T> __device__ inline typename Mma<T>::frag global_frag(const T *row, int element, int dim, bool there) {
    typename Mma<T>::frag r = {};
    if (there && element < dim) r = *(const typename Mma<T>::frag *)(row + element);
    return r;
}

__device__ inline int result_row(int i, int half) { return 8 * (i / 4) + 4 * half + i % 4; }

struct Sequence { int start, length; };
__device__ inline Sequence sequence(const Args &a, int b) {
    const int length = a.length ? a.length[b] : a.keys;
    const int start = a.start ? a.start[b] : a.keys - a.queries, far = 1 << 30;   /* (positions as far off as that keep their order) */
    return {start < -far ? -far : start > far ? far : start, length < 0 ? 0 : length > a.keys ? a.keys : length};
}

/* The keys that positions lo..hi see, in tiles of SIZE: `first` tiles from 0 on (first keys), then those from `at` to `to`. */
struct Tiles {
    int first, at, count;
    __device__ inline int tile(int t) const { return t < first ? t : at + t - first; }
};
template <int SIZE> __device__ inline Tiles tiles_of(const Args &a, const Sequence &s, int lo, int hi) {
    const int end = s.length < hi + 1 ? s.length : hi + 1;
    if (end <= 0) return {0, 0, 0};
    const int from = a.window > 0 && lo - a.window + 1 > 0 ? lo - a.window + 1 : 0;
    const int to = (end + SIZE - 1) / SIZE, at = from / SIZE < to ? from / SIZE : to;
    const int sinks = a.window > 0 ? (a.sinks < end ? a.sinks : end) : 0;
    const int first = (sinks + SIZE - 1) / SIZE < at ? (sinks + SIZE - 1) / SIZE : at;
    return {first, at, first + to - at};
}

__device__ inline bool sees(const Args &a, int length, int p, int key) {
    return key < length && key <= p && (a.window == 0 || p - key < a.window || key < a.sinks);
}
/* whether positions lo..hi all see (or all do not see) keys from..to - 1 */
__device__ inline bool all_see(const Args &a, int length, int lo, int hi, int from, int to) {
    return to <= length && to - 1 <= lo && (a.window == 0 || hi - from < a.window || to <= a.sinks);
}
__device__ inline bool none_see(const Args &a, int length, int lo, int hi, int from, int to) {
    return from >= length || from > hi || (a.window > 0 && lo - (to - 1) >= a.window && from >= a.sinks);
}

/* Work in an order that keeps a head's blocks, which read the same keys, on one of the eight dies and its cache: workgroups go to
 * the dies in turn, so die d gets the d-th eighth of the work.  Returns count where a workgroup has nothing to do. */
__device__ inline int place(int count) {
    const int per = (count + 7) / 8;
    const int at = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    return blockIdx.x / 8 < (unsigned)per && at < count ? at : count;
}
inline int places(int64_t count) { return (int)((count + 7) / 8 * 8); }

/* What a query's keys have come to: maximum, sum of exponentials (of this lane's keys), weighted sum of values. */
template <int DT> struct Running {
    float top, total;
    f32x16 o[DT];
    __device__ inline void clear() {
        top = -__builtin_inff(), total = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    }
};

__device__ inline float other_half(float x) { return __shfl_xor(x, 32); }

/* One block of 32 keys times NB more for 32 queries: scores, softmax, weighted values.  The maximum that exponentials are taken
 * around moves only when a score passes it by 8 powers of two: the sums stay far from their range's end, and most blocks
 * need no rescaling. */
template <class T, int DP, int PITCH, int NB> __device__ inline void block_step(Running<DP / 32> &run, const typename Mma<T>::frag *qf, const char *ktile, const char *vtile,
                                                                                const Args &a, int length, int p, int key0, bool masked, int lane) {
    const int half = lane >> 5;
    float s[NB][16];
    float top = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        f32x16 acc = {};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) acc = Mma<T>::go(row_frag<T, PITCH>(ktile, n * 32, k, lane), qf[k], acc);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = acc[i];
    }
    if (masked) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!sees(a, length, p, key0 + n * 32 + result_row(i, half))) s[n][i] = -__builtin_inff();
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
    top = fmaxf(top, other_half(top));
    const bool more = (top - run.top) * a.scale2 > 8.0f;   /* (also from no key at all, -inf, to any) */
    if (__any(more)) {
        const float to = more ? top : run.top;
        const float by = to == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((run.top - to) * a.scale2);
        run.top = to;
        run.total *= by;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) run.o[t][i] *= by;
    }
    const float around = run.top == -__builtin_inff() ? 0.0f : run.top * a.scale2;
    typename Mma<T>::frag pf[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], a.scale2, -around));
            sum += s[n][i];
        }
        run.total += sum;
        pf[n][0] = pack8<T>(s[n]), pf[n][1] = pack8<T>(s[n] + 8);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int t = 0; t < DP / 32; ++t) run.o[t] = Mma<T>::go(column_frag<T, PITCH>(vtile, n * 32 + k * 16, t, lane), pf[n][k], run.o[t]);
}

/* Four neighbouring elements of a result, rounded. */
template <class T> __device__ inline void store4(T *to, float a, float b, float c, float d) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *(vec *)to = vec{(T)a, (T)b, (T)c, (T)d};
}

template <int DP> struct Shape { static constexpr int PITCH = DP <= 64 ? 64 : 128; };

constexpr int WAVES = 4, LANES = WAVES * 64, QUERIES = WAVES * 32, KEYS = 64;

/* Prompts: a workgroup takes 128 queries of a head, 32 per wavefront, and walks over its keys in tiles of 64, the next tile on its
 * way while one is worked on. */
template <class T, int DP> __global__ void __launch_bounds__(LANES) attend_forward(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = KEYS * PITCH * 2;
    const int blocks = (a.queries + QUERIES - 1) / QUERIES, count = a.batch * a.heads * blocks;
    const int work = place(count);
    if (work >= count) return;
    const int block = blocks - 1 - work % blocks, head = work / blocks % a.heads, b = work / blocks / a.heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = sequence(a, b);
    const int q0 = block * QUERIES, mine = q0 + wave * 32, query = mine + (lane & 31);
    const int last = (q0 + QUERIES < a.queries ? q0 + QUERIES : a.queries) - 1;
    const T *k = (const T *)a.k + b * a.k_stride[0] + head / a.shared * a.k_stride[2], *v = (const T *)a.v + b * a.v_stride[0] + head / a.shared * a.v_stride[2];
    const Tiles tiles = tiles_of<KEYS>(a, seq, seq.start + q0, seq.start + last);
    const uint32_t lds0 = lds_offset(lds);
    auto ask = [&](int t) {
        const uint32_t to = lds0 + (t & 1) * 2 * TILE;
        const int at = tiles.tile(t) * KEYS;
        load_tile<T, PITCH, KEYS, LANES>(to, k, a.k_stride[1], at, seq.length, a.dim, threadIdx.x);
        load_tile<T, PITCH, KEYS, LANES>(to + TILE, v, a.v_stride[1], at, seq.length, a.dim, threadIdx.x);
    };
    if (tiles.count > 0) ask(0);
    const T *qrow = (const T *)a.q + b * a.q_stride[0] + (int64_t)query * a.q_stride[1] + head * a.q_stride[2];
    typename Mma<T>::frag qf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = global_frag<T>(qrow, s * 16 + half * 8, a.dim, query < a.queries);
    Running<DP / 32> run;
    run.clear();
    const int lo = seq.start + mine, hi = seq.start + (mine + 31 < a.queries ? mine + 31 : a.queries - 1);
    for (int t = 0; t < tiles.count; ++t) {
        wait_tiles<0>();
        meet();
        if (t + 1 < tiles.count) ask(t + 1);
        const int at = tiles.tile(t) * KEYS;
        if (mine >= a.queries || none_see(a, seq.length, lo, hi, at, at + KEYS)) continue;
        const char *ktile = lds + (t & 1) * 2 * TILE;
        block_step<T, DP, PITCH, KEYS / 32>(run, qf, ktile, ktile + TILE, a, seq.length, seq.start + query, at, !all_see(a, seq.length, lo, hi, at, at + KEYS), lane);
    }
    const float total = run.total + other_half(run.total);
    if (query >= a.queries) return;
    const float by = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;   /* (nothing visible: zero; not a number: that) */
    T *to = (T *)a.out + b * a.out_stride[0] + (int64_t)query * a.out_stride[1] + head * a.out_stride[2];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = t * 32 + result_row(i, half);
            if (d < a.dim) store4(to + d, run.o[t][i] * by, run.o[t][i + 1] * by, run.o[t][i + 2] * by, run.o[t][i + 3] * by);
        }
    if (half == 0) a.lse[((int64_t)b * a.heads + head) * a.queries + query] = total == 0.0f ? -__builtin_inff() : run.top * a.scale + __logf(total);
}

/* Few queries: the queries of a key head's heads are the columns of one block of 32; every wavefront walks over tiles of 32 keys
 * of its own, with its own two buffers and no barrier, and the wavefronts' and then the workgroups' results are joined. */
constexpr int SPLIT_KEYS = 32;
template <class T, int DP> __global__ void __launch_bounds__(LANES) attend_split(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = SPLIT_KEYS * PITCH * 2, LOADS = 2 * TILE / 1024;
    const int split = blockIdx.x, rb = blockIdx.y % a.row_blocks, kv = blockIdx.y / a.row_blocks, b = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = sequence(a, b);
    const int rows = a.queries * a.shared, row = rb * 32 + (lane & 31);
    const int query = row / a.shared, head = kv * a.shared + row % a.shared;
    const int lo = seq.start + rb * 32 / a.shared, hi = seq.start + ((rb * 32 + 31 < rows ? rb * 32 + 31 : rows - 1) / a.shared);
    const T *k = (const T *)a.k + b * a.k_stride[0] + kv * a.k_stride[2], *v = (const T *)a.v + b * a.v_stride[0] + kv * a.v_stride[2];
    const Tiles tiles = tiles_of<SPLIT_KEYS>(a, seq, lo, hi);
    const int worker = split * WAVES + wave, workers = a.splits * WAVES;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_offset(lds) + wave * 4 * TILE);
    char *own = lds + wave * 4 * TILE;
    auto ask = [&](int t, int buffer) {
        const uint32_t to = lds0 + buffer * 2 * TILE;
        const int at = tiles.tile(t) * SPLIT_KEYS;
        load_tile<T, PITCH, SPLIT_KEYS, 64>(to, k, a.k_stride[1], at, seq.length, a.dim, lane);
        load_tile<T, PITCH, SPLIT_KEYS, 64>(to + TILE, v, a.v_stride[1], at, seq.length, a.dim, lane);
    };
    const T *qrow = (const T *)a.q + b * a.q_stride[0] + (int64_t)query * a.q_stride[1] + head * a.q_stride[2];
    typename Mma<T>::frag qf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = global_frag<T>(qrow, s * 16 + half * 8, a.dim, row < rows);
    Running<DP / 32> run;
    run.clear();
    int buffer = 0;
    if (worker < tiles.count) ask(worker, 0);
    for (int t = worker; t < tiles.count; t += workers, buffer ^= 1) {
        if (t + workers < tiles.count) {
            /* (the other buffer's last reads have returned: their results went into the products before this) */
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            ask(t + workers, buffer ^ 1);
            wait_tiles<LOADS>();
        } else
            wait_tiles<0>();
        const int at = tiles.tile(t) * SPLIT_KEYS;
        const char *ktile = own + buffer * 2 * TILE;
        block_step<T, DP, PITCH, 1>(run, qf, ktile, ktile + TILE, a, seq.length, seq.start + query, at, !all_see(a, seq.length, lo, hi, at, at + SPLIT_KEYS), lane);
    }
    run.total += other_half(run.total);
    /* join the wavefronts: element d of a row's sum lies at [wave][d][row] */
    float *sums = (float *)lds, *tops = sums + WAVES * DP * 32;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(wave * DP + t * 32 + result_row(i, half)) * 32 + (lane & 31)] = run.o[t][i];
    if (half == 0) tops[(wave * 2) * 32 + lane] = run.top, tops[(wave * 2 + 1) * 32 + lane] = run.total;
    __syncthreads();
    const int r = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int at_row = rb * 32 + r;
    if (at_row >= rows) return;
    float top = -__builtin_inff(), total = 0.0f, by[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w * 2 * 32 + r]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float t = tops[w * 2 * 32 + r];
        by[w] = t == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((t - top) * a.scale2);
        total += by[w] * tops[(w * 2 + 1) * 32 + r];
    }
    const int q = at_row / a.shared, h = kv * a.shared + at_row % a.shared;
    const int64_t flat = ((int64_t)b * a.heads + h) * a.queries + q;
    const float scale = a.splits > 1 ? 1.0f : total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;
    T *out = (T *)a.out + b * a.out_stride[0] + (int64_t)q * a.out_stride[1] + h * a.out_stride[2];
    const int64_t rows_all = (int64_t)a.batch * a.heads * a.queries;
    for (int d = part * 4; d < a.dim; d += LANES / 32 * 4) {
        float x[4] = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += by[w] * sums[(w * DP + d + i) * 32 + r];
        if (a.splits > 1) *(f32x4 *)(a.part_o + (split * rows_all + flat) * a.dim + d) = f32x4{x[0], x[1], x[2], x[3]};
        else store4(out + d, x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale);
    }
    if (part == 0) {
        if (a.splits > 1) a.part_ml[(split * rows_all + flat) * 2] = top, a.part_ml[(split * rows_all + flat) * 2 + 1] = total;
        else a.lse[flat] = total == 0.0f ? -__builtin_inff() : top * a.scale + __logf(total);
    }
}

/* Joins the workgroups' parts of a row: one wavefront each. */
template <class T> __global__ void __launch_bounds__(LANES) attend_join(const Args a) {
    const int64_t rows = (int64_t)a.batch * a.heads * a.queries, row = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    float top = -__builtin_inff(), total = 0.0f, x[2] = {0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[(s * rows + row) * 2]);
    for (int s = 0; s < a.splits; ++s) {
        const float t = a.part_ml[(s * rows + row) * 2];
        const float by = t == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((t - top) * a.scale2);
        total += by * a.part_ml[(s * rows + row) * 2 + 1];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + i * 64 < a.dim) x[i] += by * a.part_o[(s * rows + row) * a.dim + lane + i * 64];
    }
    const int q = (int)(row % a.queries), h = (int)(row / a.queries % a.heads), b = (int)(row / a.queries / a.heads);
    const float by = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;
    T *out = (T *)a.out + b * a.out_stride[0] + (int64_t)q * a.out_stride[1] + h * a.out_stride[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + i * 64 < a.dim) out[lane + i * 64] = (T)(x[i] * by);
    if (lane == 0) a.lse[row] = total == 0.0f ? -__builtin_inff() : top * a.scale + __logf(total);
}

/* dQ: queries in registers, keys in tiles as in attend_forward; per block of 32 keys S^T = K Q^T, dP^T = V dO^T,
 * dQ^T += K^T dS^T.  It also leaves delta = sum dO O of every query for attend_dkv. */
template <class T, int DP> __global__ void __launch_bounds__(LANES) attend_dq(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = KEYS * PITCH * 2;
    const int blocks = (a.queries + QUERIES - 1) / QUERIES, count = a.batch * a.heads * blocks;
    const int work = place(count);
    if (work >= count) return;
    const int block = blocks - 1 - work % blocks, head = work / blocks % a.heads, b = work / blocks / a.heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = sequence(a, b);
    const int q0 = block * QUERIES, mine = q0 + wave * 32, query = mine + (lane & 31);
    const int last = (q0 + QUERIES < a.queries ? q0 + QUERIES : a.queries) - 1;
    const T *k = (const T *)a.k + b * a.k_stride[0] + head / a.shared * a.k_stride[2], *v = (const T *)a.v + b * a.v_stride[0] + head / a.shared * a.v_stride[2];
    const Tiles tiles = tiles_of<KEYS>(a, seq, seq.start + q0, seq.start + last);
    const uint32_t lds0 = lds_offset(lds);
    auto ask = [&](int t) {
        const uint32_t to = lds0 + (t & 1) * 2 * TILE;
        const int at = tiles.tile(t) * KEYS;
        load_tile<T, PITCH, KEYS, LANES>(to, k, a.k_stride[1], at, seq.length, a.dim, threadIdx.x);
        load_tile<T, PITCH, KEYS, LANES>(to + TILE, v, a.v_stride[1], at, seq.length, a.dim, threadIdx.x);
    };
    if (tiles.count > 0) ask(0);
    const bool there = query < a.queries;
    const T *qrow = (const T *)a.q + b * a.q_stride[0] + (int64_t)query * a.q_stride[1] + head * a.q_stride[2];
    const T *grow = (const T *)a.g + b * a.g_stride[0] + (int64_t)query * a.g_stride[1] + head * a.g_stride[2];
    const T *orow = (const T *)a.out + b * a.out_stride[0] + (int64_t)query * a.out_stride[1] + head * a.out_stride[2];
    typename Mma<T>::frag qf[DP / 16], gf[DP / 16];
    float delta = 0.0f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        qf[s] = global_frag<T>(qrow, s * 16 + half * 8, a.dim, there);
        gf[s] = global_frag<T>(grow, s * 16 + half * 8, a.dim, there);
        const typename Mma<T>::frag of = global_frag<T>(orow, s * 16 + half * 8, a.dim, there);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta += (float)gf[s][i] * (float)of[i];
    }
    delta += other_half(delta);
    const int64_t flat = ((int64_t)b * a.heads + head) * a.queries + query;
    if (there && half == 0) a.delta[flat] = delta;
    const float lse2 = there ? a.lse[flat] * LOG2E : 0.0f;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) dq[t] = f32x16{};
    const int lo = seq.start + mine, hi = seq.start + (mine + 31 < a.queries ? mine + 31 : a.queries - 1), p = seq.start + query;
    for (int t = 0; t < tiles.count; ++t) {
        wait_tiles<0>();
        meet();
        if (t + 1 < tiles.count) ask(t + 1);
        const int at = tiles.tile(t) * KEYS;
        if (mine >= a.queries) continue;
        const char *ktile = lds + (t & 1) * 2 * TILE, *vtile = ktile + TILE;
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n) {
            const int key0 = at + n * 32;
            if (none_see(a, seq.length, lo, hi, key0, key0 + 32)) continue;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) s = Mma<T>::go(row_frag<T, PITCH>(ktile, n * 32, j, lane), qf[j], s);
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) dp = Mma<T>::go(row_frag<T, PITCH>(vtile, n * 32, j, lane), gf[j], dp);
            const bool masked = !all_see(a, seq.length, lo, hi, key0, key0 + 32);
            float ds[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float prob = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse2));
                ds[i] = prob * (dp[i] - delta);
            }
            if (masked)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!there || !sees(a, seq.length, p, key0 + result_row(i, half))) ds[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const typename Mma<T>::frag f = pack8<T>(ds + 8 * j);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) dq[d] = Mma<T>::go(column_frag<T, PITCH>(ktile, n * 32 + j * 16, d, lane), f, dq[d]);
            }
        }
    }
    if (!there) return;
    T *to = (T *)a.dq + (((int64_t)b * a.queries + query) * a.heads + head) * a.dim;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = t * 32 + result_row(i, half);
            if (d < a.dim) store4(to + d, dq[t][i] * a.scale, dq[t][i + 1] * a.scale, dq[t][i + 2] * a.scale, dq[t][i + 3] * a.scale);
        }
}

/* dK and dV: a workgroup takes 128 keys of a key head, 32 per wavefront in registers, and walks over the queries that see them, of
 * every head that shares the key head, in tiles of 64: S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.  A key's sums stay
 * with one workgroup: no atomic additions, the same bits every time. */
template <class T, int DP> __global__ void __launch_bounds__(LANES) attend_dkv(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = KEYS * PITCH * 2, STAGE = 2 * TILE + 512;
    const int blocks = (a.keys + QUERIES - 1) / QUERIES, count = a.batch * a.kv_heads * blocks;
    const int work = place(count);
    if (work >= count) return;
    const int block = work % blocks, kv = work / blocks % a.kv_heads, b = work / blocks / a.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = sequence(a, b);
    const int k0 = block * QUERIES, mine = k0 + wave * 32, key = mine + (lane & 31);
    const bool there = key < seq.length;
    const T *krow = (const T *)a.k + b * a.k_stride[0] + (int64_t)key * a.k_stride[1] + kv * a.k_stride[2];
    const T *vrow = (const T *)a.v + b * a.v_stride[0] + (int64_t)key * a.v_stride[1] + kv * a.v_stride[2];
    typename Mma<T>::frag kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) kf[s] = global_frag<T>(krow, s * 16 + half * 8, a.dim, there), vf[s] = global_frag<T>(vrow, s * 16 + half * 8, a.dim, there);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) dk[t] = f32x16{}, dv[t] = f32x16{};
    /* queries that see one of the keys: from position k0 on, and up to the last key's window unless one of them is a first key */
    int from = k0 - seq.start, to = a.queries;
    if (a.window > 0 && k0 >= a.sinks) {
        const int64_t most = (int64_t)k0 + QUERIES - 1 + a.window - seq.start;
        to = most < to ? (int)most : to;
    }
    from = from < 0 ? 0 : from;
    const int first = from / KEYS, per_head = k0 < seq.length && to > from ? (to + KEYS - 1) / KEYS - first : 0, steps = per_head * a.shared;
    const uint32_t lds0 = lds_offset(lds);
    auto ask = [&](int t) {
        const uint32_t at = lds0 + (t & 1) * STAGE;
        const int head = kv * a.shared + t / per_head, q = (first + t % per_head) * KEYS;
        load_tile<T, PITCH, KEYS, LANES>(at, (const T *)a.q + b * a.q_stride[0] + head * a.q_stride[2], a.q_stride[1], q, a.queries, a.dim, threadIdx.x);
        load_tile<T, PITCH, KEYS, LANES>(at + TILE, (const T *)a.g + b * a.g_stride[0] + head * a.g_stride[2], a.g_stride[1], q, a.queries, a.dim, threadIdx.x);
        if (wave < 2) {
            const float *row = (wave == 0 ? a.lse : a.delta) + ((int64_t)b * a.heads + head) * a.queries;
            to_lds4(q + lane < a.queries ? (const void *)(row + q + lane) : (const void *)zero_page, __builtin_amdgcn_readfirstlane(at + 2 * TILE + wave * 256));
        }
    };
    if (steps > 0) ask(0);
    for (int t = 0; t < steps; ++t) {
        wait_tiles<0>();
        meet();
        if (t + 1 < steps) ask(t + 1);
        if (mine >= seq.length) continue;
        const char *qtile = lds + (t & 1) * STAGE, *gtile = qtile + TILE;
        const float *lse = (const float *)(gtile + TILE), *delta = lse + 64;
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n) {
            const int q = (first + t % per_head) * KEYS + n * 32;
            const int lo = seq.start + q, hi = seq.start + (q + 31 < a.queries ? q + 31 : a.queries - 1);
            if (q >= a.queries || none_see(a, seq.length, lo, hi, mine, mine + 32)) continue;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) s = Mma<T>::go(row_frag<T, PITCH>(qtile, n * 32, j, lane), kf[j], s);
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) dp = Mma<T>::go(row_frag<T, PITCH>(gtile, n * 32, j, lane), vf[j], dp);
            const bool masked = q + 32 > a.queries || !all_see(a, seq.length, lo, hi, mine, mine + 32);
            float prob[16], ds[16];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 l = *(const f32x4 *)(lse + n * 32 + result_row(i, half)), d = *(const f32x4 *)(delta + n * 32 + result_row(i, half));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    prob[i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + e], a.scale2, -l[e] * LOG2E));
                    ds[i + e] = prob[i + e] * (dp[i + e] - d[e]);
                }
            }
            if (masked)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int at = q + result_row(i, half);
                    if (at >= a.queries || !sees(a, seq.length, seq.start + at, key)) prob[i] = ds[i] = 0.0f;
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const typename Mma<T>::frag pf = pack8<T>(prob + 8 * j), df = pack8<T>(ds + 8 * j);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) {
                    dv[d] = Mma<T>::go(column_frag<T, PITCH>(gtile, n * 32 + j * 16, d, lane), pf, dv[d]);
                    dk[d] = Mma<T>::go(column_frag<T, PITCH>(qtile, n * 32 + j * 16, d, lane), df, dk[d]);
                }
            }
        }
    }
    if (key >= a.keys) return;
    T *dkrow = (T *)a.dk + (((int64_t)b * a.keys + key) * a.kv_heads + kv) * a.dim, *dvrow = (T *)a.dv + (((int64_t)b * a.keys + key) * a.kv_heads + kv) * a.dim;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = t * 32 + result_row(i, half);
            if (d >= a.dim) continue;
            store4(dkrow + d, dk[t][i] * a.scale, dk[t][i + 1] * a.scale, dk[t][i + 2] * a.scale, dk[t][i + 3] * a.scale);
            store4(dvrow + d, dv[t][i], dv[t][i + 1], dv[t][i + 2], dv[t][i + 3]);
        }
}

int check(const ace_attend_t *a) {
    if (!a || a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return ACE_EINVAL;
    if (a->dim < 8 || a->dim % 8 || a->window < 0 || a->sinks < 0 || (a->dtype != ACE_T_BF16 && a->dtype != ACE_T_F16)) return ACE_EINVAL;
    if (!(a->scale > 0.0f) || a->scale > 1e30f) return ACE_EINVAL;
    if (a->dim > 128 || a->queries > (1 << 30) || a->keys > (1 << 30)) return ACE_ETOOBIG;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8 || a->k_stride[i] % 8 || a->v_stride[i] % 8 || a->out_stride[i] % 8) return ACE_EINVAL;
    if (a->batch == 0 || a->queries == 0) return ACE_OK;
    if (!a->d_q || !a->d_out || !a->d_lse || (a->keys > 0 && (!a->d_k || !a->d_v))) return ACE_EINVAL;
    if (((uintptr_t)a->d_q | (uintptr_t)a->d_k | (uintptr_t)a->d_v | (uintptr_t)a->d_out) & 15) return ACE_EINVAL;
    const int64_t blocks = (a->queries + QUERIES - 1) / QUERIES, kblocks = (a->keys + QUERIES - 1) / QUERIES;
    if ((int64_t)a->batch * a->heads * (blocks + 1) > (1 << 22) || (int64_t)a->batch * a->kv_heads * (kblocks + 1) > (1 << 22)) return ACE_ETOOBIG;
    return ACE_OK;
}

Args args_of(const ace_attend_t *a) {
    Args k = {};
    k.batch = a->batch, k.queries = a->queries, k.keys = a->keys, k.heads = a->heads, k.kv_heads = a->kv_heads, k.dim = a->dim;
    k.shared = a->heads / a->kv_heads, k.window = a->window, k.sinks = a->sinks, k.scale = a->scale, k.scale2 = a->scale * LOG2E;
    k.start = a->d_start, k.length = a->d_length;
    for (int i = 0; i < 3; ++i) k.q_stride[i] = a->q_stride[i], k.k_stride[i] = a->k_stride[i], k.v_stride[i] = a->v_stride[i], k.out_stride[i] = a->out_stride[i];
    k.q = a->d_q, k.k = a->d_k, k.v = a->d_v, k.out = a->d_out, k.lse = a->d_lse;
    return k;
}

/* Few queries go to attend_split. */
constexpr int SPLIT_QUERIES = 16;
bool few(const ace_attend_t *a) { return a->queries <= SPLIT_QUERIES; }

int row_blocks(const ace_attend_t *a) { return (a->queries * (a->heads / a->kv_heads) + 31) / 32; }

int splits_of(const ace_attend_t *a) {
    int64_t seen = a->window > 0 ? (int64_t)a->window + a->queries + a->sinks : a->keys;
    seen = seen < a->keys ? seen : a->keys;
    const int64_t groups = (int64_t)a->batch * a->kv_heads * row_blocks(a), most = (seen + SPLIT_KEYS * WAVES * 2 - 1) / (SPLIT_KEYS * WAVES * 2);
    int64_t splits = (512 + groups - 1) / groups;
    splits = splits < most ? splits : most;
    return splits < 1 ? 1 : splits > 64 ? 64 : (int)splits;
}

template <class K> int with_lds(K kernel, int bytes) { return layer_hip_status(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)); }

template <class T, int DP> int forward(Args &k, const ace_attend_t *a, hipStream_t stream) {
    constexpr int PITCH = Shape<DP>::PITCH;
    if (!few(a)) {
        constexpr int LDS = 4 * KEYS * PITCH * 2;
        static const int ready = with_lds(attend_forward<T, DP>, LDS);
        if (ready != ACE_OK) return ready;
        attend_forward<T, DP><<<places((int64_t)k.batch * k.heads * ((k.queries + QUERIES - 1) / QUERIES)), LANES, LDS, stream>>>(k);
        return layer_launched();
    }
    constexpr int TILES = WAVES * 4 * SPLIT_KEYS * PITCH * 2, JOIN = (WAVES * DP * 32 + WAVES * 2 * 32) * 4, LDS = TILES > JOIN ? TILES : JOIN;
    static const int ready = with_lds(attend_split<T, DP>, LDS);
    if (ready != ACE_OK) return ready;
    if (k.batch > 65535 || (int64_t)k.kv_heads * k.row_blocks > 65535) return ACE_ETOOBIG;
    attend_split<T, DP><<<dim3(k.splits, k.kv_heads * k.row_blocks, k.batch), LANES, LDS, stream>>>(k);
    int rc = layer_launched();
    if (rc != ACE_OK || k.splits == 1) return rc;
    const int64_t rows = (int64_t)k.batch * k.heads * k.queries;
    attend_join<T><<<(uint32_t)((rows + WAVES - 1) / WAVES), LANES, 0, stream>>>(k);
    return layer_launched();
}

template <class T, int DP> int backward(const Args &k, hipStream_t stream) {
    constexpr int PITCH = Shape<DP>::PITCH, LDS = 4 * KEYS * PITCH * 2, LDS2 = LDS + 1024;
    static const int ready = with_lds(attend_dq<T, DP>, LDS), ready2 = with_lds(attend_dkv<T, DP>, LDS2);
    if (ready != ACE_OK || ready2 != ACE_OK) return ACE_EHIP;
    if (k.queries > 0) {
        attend_dq<T, DP><<<places((int64_t)k.batch * k.heads * ((k.queries + QUERIES - 1) / QUERIES)), LANES, LDS, stream>>>(k);
        const int rc = layer_launched();
        if (rc != ACE_OK) return rc;
    }
    if (k.keys == 0) return ACE_OK;
    attend_dkv<T, DP><<<places((int64_t)k.batch * k.kv_heads * ((k.keys + QUERIES - 1) / QUERIES)), LANES, LDS2, stream>>>(k);
    return layer_launched();
}

}  // namespace

extern "C" size_t ace_attend_workspace_bytes(const ace_attend_t *a) {
    if (check(a) != ACE_OK || a->batch == 0 || a->queries == 0 || !few(a) || splits_of(a) == 1) return 0;
    return (size_t)splits_of(a) * a->batch * a->heads * a->queries * (a->dim + 2) * sizeof(float);
}

extern "C" int ace_attend_forward(const ace_attend_t *a, void *d_workspace, size_t workspace_bytes, void *stream) {
    const int rc = check(a);
    if (rc != ACE_OK || a->batch == 0 || a->queries == 0) return rc;
    Args k = args_of(a);
    k.row_blocks = row_blocks(a), k.splits = few(a) ? splits_of(a) : 1;
    if (k.splits > 1) {
        if (!d_workspace || workspace_bytes < ace_attend_workspace_bytes(a)) return ACE_EINVAL;
        k.part_o = (float *)d_workspace;
        k.part_ml = k.part_o + (int64_t)k.splits * k.batch * k.heads * k.queries * k.dim;
    }
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == ACE_T_BF16) return a->dim <= 64 ? forward<bf16, 64>(k, a, s) : a->dim <= 96 ? forward<bf16, 96>(k, a, s) : forward<bf16, 128>(k, a, s);
    return a->dim <= 64 ? forward<f16, 64>(k, a, s) : a->dim <= 96 ? forward<f16, 96>(k, a, s) : forward<f16, 128>(k, a, s);
}

extern "C" int ace_attend_backward(const ace_attend_t *a, const void *d_gout, const int64_t gout_stride[3], float *d_delta, void *d_dq, void *d_dk,
                                   void *d_dv, void *stream) {
    const int rc = check(a);
    if (rc != ACE_OK || a->batch == 0) return rc;
    if ((a->queries > 0 && (!d_gout || !gout_stride || !d_delta || !d_dq)) || (a->keys > 0 && (!d_dk || !d_dv))) return ACE_EINVAL;
    if (((uintptr_t)d_gout | (uintptr_t)d_dq | (uintptr_t)d_dk | (uintptr_t)d_dv) & 15) return ACE_EINVAL;
    Args k = args_of(a);
    k.g = d_gout, k.delta = d_delta, k.dq = d_dq, k.dk = d_dk, k.dv = d_dv;
    for (int i = 0; gout_stride && i < 3; ++i) {
        if (gout_stride[i] % 8) return ACE_EINVAL;
        k.g_stride[i] = gout_stride[i];
    }
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == ACE_T_BF16) return a->dim <= 64 ? backward<bf16, 64>(k, s) : a->dim <= 96 ? backward<bf16, 96>(k, s) : backward<bf16, 128>(k, s);
    return a->dim <= 64 ? backward<f16, 64>(k, s) : a->dim <= 96 ? backward<f16, 96>(k, s) : backward<f16, 128>(k, s);
}
