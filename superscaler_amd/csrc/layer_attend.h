/*
 * Attention over a window of keys and a few first ones: forward for prompts (attend_forward), forward for few queries over long
 * caches (attend_split, attend_join), backward (attend_dq, attend_dkv).  What is PACKED has its sequences one after the other and a table of
 * their blocks; otherwise they are a padded batch.
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
 * Tiles go from memory to LDS without registers between, 16 bytes per lane, through a buffer descriptor of the tile's rows: a lane's
 * place in a tile is the same for every tile, and rows past the sequence's length (and pieces past the head's size) are out of
 * the descriptor's range and arrive as zeros.  Whatever stands there in memory, a number or not, takes no part.  A tile's
 * 16-byte pieces are exchanged within their row, piece c of row r at c ^ swizzle(r), so that what LDS serves at a time in
 * either kind of read, sixteen rows at one piece or four rows at four pieces, lies in all of its 64 banks.
 */
#ifndef LAYER_ATTEND_H
#define LAYER_ATTEND_H

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
    float *far;                          /* attend_far: [far_slots][kv_heads][far_parts][2][width][32], a slot for a sequence's block of 32 first keys */
    int far_blocks, far_parts, far_slots;
    int far_times, far_per;              /* PACKED: a sequence's slots begin at its first token times far_times / far_per; far_per 0: at its number times far_blocks */
    /* PACKED: queries and keys are all tokens, batch the sequences */
    const ace_packed_block_t *query_blocks, *key_blocks;
    const ace_packed_sequence_t *sequences;
    int blocks;
};

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

/* LDS serves a 16-byte read of a wavefront by sixteen lanes at a time (0-3, 12-15, 20-23, 24-27; then the others alike), an 8-byte
 * read by lanes 0-31 and 32-63.  Rows of 256 bytes lie in all banks: the sixteen rows need sixteen places, the four rows of a
 * transposing read four groups of four.  Rows of 128 bytes: two rows share the banks, the rest alike. */
template <int PITCH> __device__ inline int swizzle(int row) { return PITCH == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3); }

__device__ inline uint32_t lds_offset(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

/* 16 bytes per lane from place `at` of the rows to LDS at `to` + 16 lane (`to`: the same for the wavefront).  The LDS write is complete
 * when the wavefront's vector-memory counter says so (wait_tiles).  m0, the destination, needs one state before it is used; nothing
 * else in these kernels uses it. */
__device__ inline void to_lds16(u32x4 rows, uint32_t at, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(rows) : "memory");
}
__device__ inline void to_lds4(u32x4 rows, uint32_t at, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(rows) : "memory");
}
template <int LEFT> __device__ inline void wait_tiles() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }
__device__ inline void meet() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
/* The registers of a value, whole, here: loads that fill them are complete (nothing later waits for them together with what was asked
 * for since), and sums leave a loop in the registers that they have in it. */
template <class V> __device__ inline void arrived(V &v) { asm volatile("" : "+v"(v)); }

/* A buffer descriptor of `bytes` bytes from `p` on, both the same for the wavefront. */
__device__ inline u32x4 buffer(const void *p, uint32_t bytes) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xffff),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00027000u};
}

/* A tile's rows in memory and where the lanes find their pieces of them: ROWS rows of PITCH elements by LANES lanes.  A lane keeps a
 * place per load; with ONE, for kernels without registers for that, one for all of them (a load takes a multiple of sixteen
 * rows then, after which swizzles repeat) and each load has a descriptor of its own rows, some ten scalar operations (which cost
 * attend_forward 15%). */
template <class T, int PITCH, int ROWS, int LANES, bool ONE = false> struct Tile {
    static constexpr int PER = PITCH / 8, LOADS = ROWS * PER / LANES, STEP = LANES / PER, PLACES = ONE ? 1 : LOADS;
    static_assert(ROWS * PER % LANES == 0 && (!ONE || STEP % 16 == 0), "whole loads");
    const T *base;
    uint32_t stride, dim;   /* (tokens are up to 2^23 elements apart) */
    uint32_t at[PLACES], to;
    __device__ inline Tile(const T *b, int64_t s, int d, int lane) : base(b), stride((uint32_t)s), dim(d) {
#pragma unroll
        for (int i = 0; i < PLACES; ++i) {
            const int p = i * LANES + lane, row = p / PER, piece = (p % PER) ^ (swizzle<PITCH>(row) & (PER - 1));
            at[i] = piece * 8 < d ? (uint32_t)(row * (int)s + piece * 8) * 2u : 0x80000000u;   /* (past every descriptor's end) */
        }
        to = __builtin_amdgcn_readfirstlane((lane & ~63) * 16);
    }
    __device__ inline u32x4 rows(int row0, int end, int most) const {
        const int n = end - row0 < most ? end - row0 : most;
        return buffer(base + (uint64_t)(uint32_t)row0 * stride, n > 0 ? ((uint32_t)(n - 1) * stride + dim) * 2 : 0);
    }
    __device__ inline void ask(uint32_t lds, int row0, int end) const {
        const uint32_t at_lds = __builtin_amdgcn_readfirstlane(lds) + to;
        u32x4 b;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (i == 0 || ONE) b = ONE ? rows(row0 + i * STEP, end, STEP) : rows(row0, end, ROWS);
            to_lds16(b, at[ONE ? 0 : i], at_lds + i * LANES * 16);
        }
    }
};

template <class V> __device__ inline V lds_load(uint32_t at) { return *(const __attribute__((address_space(3))) V *)at; }

/* Where a lane finds its part of operands in a tile of rows of PITCH elements; a tile begins at a multiple of a row.  Pieces of other
 * steps differ in bits that are exchanged, never carried, so a place is one base with bits flipped, plus a constant. */
template <class T, int PITCH> struct Operands {
    typedef typename Mma<T>::frag frag;
    uint32_t row, column;
    __device__ inline explicit Operands(int lane) {
        const int half = lane >> 5, i = lane & 15, r = 4 * half + (i >> 2);
        row = (lane & 31) * PITCH * 2 + (half ^ (swizzle<PITCH>(lane & 31) & (PITCH / 8 - 1))) * 16;
        column = r * PITCH * 2 + ((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ (swizzle<PITCH>(r) & (PITCH / 8 - 1))) * 16 + (i & 1) * 8;
    }
    /* rows are the tile's rows row0 + lane % 32, k the elements 16 s to 16 s + 15 */
    __device__ inline frag rows(uint32_t tile, int row0, int s) const { return lds_load<frag>(((tile + row) ^ (s << 5)) + row0 * PITCH * 2); }
    /* rows are the elements 32 t + lane % 32, k the tile's rows row0 to row0 + 15 (row0: a multiple of sixteen) */
    __device__ inline frag columns(uint32_t tile, int row0, int t) const {
        union { s16x4 half[2]; frag whole; } u;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            u.half[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(lds_ptr)(((tile + column) ^ (t << 6 | k << 5)) + (row0 + 8 * k) * PITCH * 2));
        return u.whole;
    }
};

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

/* Queries and keys number up to MOST.  A sequence that begins further before the first key than that has no query that sees one; past
 * LATEST positions are taken as beginning there, and a window as the first that holds every key from there on: no sum or difference of
 * positions, lengths and a window leaves 32 bits. */
constexpr int MOST = 1 << 28, LATEST = 1 << 30, WIDEST = LATEST + MOST;
struct Sequence { int start, length; };

/* Where a sequence lies: that of a batch, or, PACKED, the `tokens` from `first` on, of which number `index` of the sequences sees itself (tokens
 * of no sequence, index -1, see nothing). */
template <bool PACKED> struct Span {
    int b;
    __device__ inline int queries(const Args &a) const { return a.queries; }
    __device__ inline int keys(const Args &a) const { return a.keys; }
    __device__ inline int64_t lead(const int64_t (&stride)[3]) const { return b * stride[0]; }
    __device__ inline int64_t first_query(const Args &a) const { return (int64_t)b * a.queries; }
    __device__ inline int64_t first_key(const Args &a) const { return (int64_t)b * a.keys; }
    __device__ inline int64_t values(const Args &a, int head) const { return ((int64_t)b * a.heads + head) * a.queries; }   /* log-sums and deltas */
    __device__ inline Sequence sequence(const Args &a) const {
        const int length = a.length ? a.length[b] : a.keys, start = a.start ? a.start[b] : a.keys - a.queries;
        return {start < -MOST ? -MOST : start > LATEST ? LATEST : start, length < 0 ? 0 : length > a.keys ? a.keys : length};
    }
    __device__ inline bool has_far(const Args &, int) const { return true; }
    __device__ inline int far_slot(const Args &a) const { return b * a.far_blocks; }
};
template <> struct Span<true> {
    int first, tokens, index;
    __device__ inline int queries(const Args &) const { return tokens; }
    __device__ inline int keys(const Args &) const { return tokens; }
    __device__ inline int64_t lead(const int64_t (&stride)[3]) const { return first * stride[1]; }
    __device__ inline int64_t first_query(const Args &) const { return first; }
    __device__ inline int64_t first_key(const Args &) const { return first; }
    __device__ inline int64_t values(const Args &a, int head) const { return (int64_t)head * a.queries + first; }
    __device__ inline Sequence sequence(const Args &) const { return {0, index < 0 ? 0 : tokens}; }
    __device__ inline bool has_far(const Args &a, int key) const { return index >= 0 && tokens - a.window > key; }   /* queries beyond a key's window */
    __device__ inline int far_slot(const Args &a) const { return a.far_per ? (int)((int64_t)first * a.far_times / a.far_per) : index * a.far_blocks; }
};

/* The order of a run of PRODUCTS matrix products whose operands come from LDS in READS reads each: operands of LEAD products are on
 * their way before the first, and those of one more are asked for with each.  (Left to itself the compiler waits for every
 * operand right behind its read, four times as long as the product takes.) */
template <int PRODUCTS, int READS, int LEAD> __device__ inline void in_step() {
    __builtin_amdgcn_sched_group_barrier(0x100, LEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < PRODUCTS - LEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, LEAD, 0);
    __builtin_amdgcn_sched_barrier(0);
}

/* The keys that positions lo..hi see, in tiles of SIZE: `first` tiles from 0 on (first keys), then those from `at` to `to`. */
struct Tiles {
    int first, at, count;
    __device__ inline int tile(int t) const { return t < first ? t : at + t - first; }
    /* how many of them begin before key `end` */
    template <int SIZE> __device__ inline int upto(int end) const {
        const int last = (end + SIZE - 1) / SIZE, some = first + (last > at ? last - at : 0);
        return end <= 0 ? 0 : some < count ? some : count;
    }
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

/* Numbers from `from` to `end` - 1, asked for by one comparison. */
struct Range {
    int from;
    uint32_t count;
    __device__ inline Range(int f, int end) : from(f), count(end > f ? end - f : 0) {}
    __device__ inline bool has(int i) const { return (uint32_t)(i - from) < count; }
};
__device__ inline int lesser(int a, int b) { return a < b ? a : b; }
/* Where a block of 32 keys begins that positions lo..hi all see by their window, and one that any of them sees. */
__device__ inline Range all_see(const Args &a, int length, int lo, int hi) {
    return Range(a.window > 0 && hi >= a.window ? hi - a.window + 1 : 0, lesser(length, lo + 1) - 31);
}
__device__ inline Range any_see(const Args &a, int length, int lo, int hi) {
    return Range((a.window > 0 && lo >= a.window ? lo - a.window + 1 : 0) - 31, lesser(length, hi + 1));
}

/* What a query sees: `count` keys from `from` on, and those below `first`. */
struct Sight {
    int from, first;
    uint32_t count;
    __device__ inline Sight(const Args &a, int length, int p) {
        const int end = p + 1 < length ? p + 1 : length;
        from = a.window > 0 && p >= a.window ? p - a.window + 1 : 0;
        count = end > from ? end - from : 0;
        first = a.window > 0 ? (a.sinks < end ? a.sinks : end) : 0;
    }
};
/* Values of keys key0 + result_row(i) that are not seen become `otherwise`.  `sinks`: some of the keys are first ones. */
template <class V> __device__ inline void hide(V &s, const Sight &sight, int key0, int half, bool sinks, float otherwise) {
    const int t = key0 + 4 * half - sight.from, u = key0 + 4 * half;
    if (sinks) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((uint32_t)(t + 8 * (i / 4) + i % 4) >= sight.count && u + 8 * (i / 4) + i % 4 >= sight.first) s[i] = otherwise;
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((uint32_t)(t + 8 * (i / 4) + i % 4) >= sight.count) s[i] = otherwise;
    }
}

/* Ones where keys key0 + result_row(i) are seen, zeros elsewhere. */
__device__ inline void show(float (&see)[16], const Sight &sight, int key0, int half) {
#pragma unroll
    for (int i = 0; i < 16; ++i) see[i] = 1.0f;
    hide(see, sight, key0, half, true, 0.0f);
}

/* Work in an order that keeps a head's blocks, which read the same keys, on one of the eight dies and its cache: workgroups go to
 * the dies in turn, so die d gets the d-th eighth of the work.  On a die they go to its 32 CUs in turn: every other 32 are
 * taken in reverse, so that a CU's second workgroup is short where its first is long (blocks at the beginning of a sequence see few
 * keys).  Returns count where a workgroup has nothing to do.  In launch order, by dies, and with every other 32 in reverse: forward, 4 x 40
 * heads of 2,048 tokens, a window of 512: 165, 141 and 138 us, backward 516, 476 and 471; 8 x 16 heads of 512, backward: 54, 49 and 44;
 * 16 heads on 4 of 8,192, no window, backward: 1,470, 1,147 and 1,155. */
__device__ inline int in_turn(int turn, int per) {
    const int begin = turn / 32 * 32, left = per - begin < 32 ? per - begin : 32;
    return begin & 32 ? begin + left - 1 - turn % 32 : turn;
}
__device__ inline int place(int count, int group) {
    const int per = (count + 7) / 8, turn = group / 8, at = group % 8 * per + in_turn(turn, per);
    return turn < per && at < count ? at : count;
}
/* Which rows of a block a wavefront takes: the other way round in the second of two workgroups on a CU.  The wavefronts of the first rows see the least,
 * and wavefronts of one number share a SIMD. */
__device__ inline int in_pairs(int wave) { return blockIdx.x >> 8 & 1 ? 3 - wave : wave; }
inline int places(int64_t count) { return (int)((count + 7) / 8 * 8); }

/* PACKED: the table's blocks come with the longest walks first, and a die takes the same blocks of each of its heads, longest first, in turn
 * over its CUs as above.  Where heads are no multiple of eight, a head's blocks are dealt out in so many classes that dies have equally many
 * pairs of a head and a class. */
struct Deal {
    int classes, pairs, ranks;   /* ranks: blocks of a class */
    __host__ __device__ inline Deal(int heads, int blocks) {
        classes = heads % 8 == 0 ? 1 : heads % 4 == 0 ? 2 : heads % 2 == 0 ? 4 : 8;
        pairs = heads * classes / 8, ranks = (blocks + classes - 1) / classes;
    }
    __host__ __device__ inline int64_t groups() const { return (int64_t)8 * pairs * ranks; }
};

/* What a workgroup works on: a block of a sequence's queries or keys, and a head. */
template <bool PACKED> struct Job {
    Span<PACKED> span;
    int block, head;
    bool some;
};
/* one of PARTS parts, SIZE rows each, of the table's blocks, parts dealt like blocks */
template <int PARTS, int SIZE> __device__ inline Job<true> dealt(const ace_packed_block_t *table, int blocks, int heads, int group) {
    const Deal deal(heads, blocks * PARTS);
    const int per = deal.pairs * deal.ranks, at = in_turn(group / 8, per);
    const int pair = group % 8 * deal.pairs + at % deal.pairs, rank = at / deal.pairs * deal.classes + pair % deal.classes;
    if (rank >= blocks * PARTS) return {{0, 0, -1}, 0, 0, false};
    const ace_packed_block_t b = table[rank / PARTS];
    const int first = __builtin_amdgcn_readfirstlane(b.first), tokens = __builtin_amdgcn_readfirstlane(b.tokens), index = __builtin_amdgcn_readfirstlane(b.sequence);
    const int block = __builtin_amdgcn_readfirstlane(b.block) * PARTS + rank % PARTS;
    return {{first, tokens, index}, block, pair / deal.classes, block * SIZE < tokens};
}
/* SIZE queries of a head */
template <bool PACKED, int SIZE> __device__ inline Job<PACKED> query_job(const Args &a, int group) {
    if constexpr (PACKED) return dealt<1, SIZE>(a.query_blocks, a.blocks, a.heads, group);
    else {
        const int blocks = (a.queries + SIZE - 1) / SIZE, count = a.batch * a.heads * blocks;
        const int work = place(count, group);
        if (work >= count) return {{0}, 0, 0, false};
        return {{work / blocks / a.heads}, blocks - 1 - work % blocks, work / blocks % a.heads, true};
    }
}
/* SIZE keys of a key head; a block of the table has WHOLE */
template <bool PACKED, int SIZE, int WHOLE> __device__ inline Job<PACKED> key_job(const Args &a, int group) {
    if constexpr (PACKED) return dealt<WHOLE / SIZE, SIZE>(a.key_blocks, a.blocks, a.kv_heads, group);
    else {
        const int blocks = (a.keys + SIZE - 1) / SIZE, count = a.batch * a.kv_heads * blocks;
        const int work = place(count, group);
        if (work >= count) return {{0}, 0, 0, false};
        return {{work / blocks / a.kv_heads}, work % blocks, work / blocks % a.kv_heads, true};
    }
}

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

/* of a lane's value and that of the lane 32 further on, the other half of its query's keys */
__device__ inline float sum_halves(float x) {
    const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t a = two[0], b = two[1];
    return __uint_as_float(a) + __uint_as_float(b);
}
__device__ inline float max_halves(float x) {
    const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t a = two[0], b = two[1];
    return fmaxf(__uint_as_float(a), __uint_as_float(b));
}

/* One block of 32 keys for 32 queries: scores, softmax, weighted values.  The maximum that exponentials are taken around moves only when a
 * score passes it by 8 powers of two: the sums stay far from their range's end, and most blocks need no rescaling. */
template <class T, int DP, int PITCH> __device__ inline void block_step(Running<DP / 32> &run, const typename Mma<T>::frag *qf, const Operands<T, PITCH> &ops, uint32_t ktile, uint32_t vtile,
                                                                        const Args &a, const Sight &sight, int key0, bool masked, int lane) {
    const int half = lane >> 5;
    float s[16];
    float top = -__builtin_inff();
    __builtin_amdgcn_s_setprio(1), __builtin_amdgcn_sched_barrier(0);
    f32x16 acc = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) acc = Mma<T>::go(ops.rows(ktile, 0, k), qf[k], acc);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = acc[i];
    in_step<DP / 16, 1, 4>();
    __builtin_amdgcn_s_setprio(0);
    if (masked) hide(s, sight, key0, half, key0 < a.sinks, -__builtin_inff());
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
    top = max_halves(top);
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
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -around));
        sum += s[i];
    }
    run.total += sum;
    const typename Mma<T>::frag pf[2] = {pack8<T>(s), pack8<T>(s + 8)};
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) run.o[t] = Mma<T>::go(ops.columns(vtile, k * 16, t), pf[k], run.o[t]);
    in_step<2 * DP / 32, 2, 3>();
    __builtin_amdgcn_s_setprio(0);
}

/* Half precision has five bits of exponent, and gradients of scores go with those of the answer, of any size, and with weights that a
 * long sequence makes small.  So they meet their products with a power of two of the lane's query or key, which moves only when a
 * gradient would pass 2^15 (the largest is 2^4 to 2^5 then: what is 2^18 times smaller still has all its bits) and takes the sums along.
 * It begins so high that any gradient above 2^-49 moves it.  Normalized weights, 1 at most, meet theirs with 2^12.  The backward pass of 2 x 16
 * heads of 2,048 tokens and size 128, a window of 1,024, takes 154 us with this and 149 without. */
template <class T> struct Fit {
    static constexpr bool FITS = __is_same(T, f16);
    static constexpr int FIRST = FITS ? 64 : 0, WEIGHTS = FITS ? 12 : 0;
    int power;
    __device__ inline void start() { power = FIRST; }
    /* of gradients that have been multiplied: the change of the power, 0 or less */
    template <int DT> __device__ inline int check(float (&ds)[16], f32x16 (&sums)[DT]) {
        if (!FITS) return 0;
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, __builtin_fabsf(ds[i]));
        if (!__any(most > 32768.0f)) return 0;
        most = max_halves(most);
        const int change = most > 32768.0f && most < __builtin_inff() ? 127 + 4 - (int)(__float_as_uint(most) >> 23) : 0;
        power += change;
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] = __builtin_amdgcn_ldexpf(ds[i], change);
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[t][i] = __builtin_amdgcn_ldexpf(sums[t][i], change);
        return change;
    }
    template <int DT> __device__ inline void apply(float (&ds)[16], f32x16 (&sums)[DT]) {
        if (!FITS) return;
        const float by = __uint_as_float((uint32_t)(127 + power) << 23);
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] *= by;
        check(ds, sums);
    }
    template <int DT> static __device__ inline void undo(f32x16 (&sums)[DT], int by) {
        if (!FITS) return;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[t][i] = __builtin_amdgcn_ldexpf(sums[t][i], -by);
    }
};

/* Four neighbouring elements of a result, rounded. */
template <class T> __device__ inline void store4(T *to, float a, float b, float c, float d) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *(vec *)to = vec{(T)a, (T)b, (T)c, (T)d};
}

/* A row's sums as two lanes hold them, times `by`, to `to`: the halves exchange every other four, so that a lane has eight neighbours, 16 bytes, and a
 * row's two lanes 32. */
template <class T, int DT> __device__ inline void store_row(T *to, const f32x16 (&sum)[DT], float by, int dim, int half) {
    typedef T four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            u32x2 x[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                x[k] = __builtin_bit_cast(u32x2, four{(T)(sum[t][i + 4 * k] * by), (T)(sum[t][i + 4 * k + 1] * by), (T)(sum[t][i + 4 * k + 2] * by), (T)(sum[t][i + 4 * k + 3] * by)});
            const auto a = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false), b = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
            const int d = t * 32 + 2 * i + 8 * half;
            if (d < dim) *(u32x4 *)(to + d) = u32x4{a[0], b[0], a[1], b[1]};
        }
}

/* A kernel's arguments and a value as if not known so far: what a rare path computes from these is computed there, and not kept in
 * registers through the loops before it. */
__device__ inline const Args &args_again() {
    auto p = (const __attribute__((address_space(4))) Args *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Args *)p;
}
__device__ inline int again(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

/* Weights of keys that a query does not see are zero, and zero times a value that is no finite number is none: such a value in a block
 * of which others see a part spoils sums that it is no part of.  The kernels look at their sums at the end, and a wavefront that
 * finds one takes its walk once more, with operands from memory: what is not finite meets its products as zero, and counts for those that
 * see it.  (Looking costs an operation per sum, once.  8 heads of 16,384 tokens, a window of 2,048, forward and backward: 159 and 519 us;
 * with one value that is no number in the middle 304 and 3,525, with nothing else 1,280 and 7,110.) */
template <int DT> __device__ inline bool any_odd(const f32x16 (&x)[DT]) {
    float z[4] = {};
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i % 4] = __builtin_fmaf(x[t][i], 0.0f, z[i % 4]);
    return !(z[0] + z[1] + z[2] + z[3] == 0.0f);
}
/* 32 rows from row0 on of a head's q, k, v or gradient, through a buffer descriptor: what is at or past `end`, and past a row's size, reads zero. */
template <class T> struct Rows {
    __amdgpu_buffer_rsrc_t rows;
    int stride, dim;
    __device__ inline Rows(const T *base, int64_t s, int row0, int end, int d) : stride((int)s), dim(d) {
        const int n = end - row0 < 32 ? end - row0 : 32;
        rows = __builtin_amdgcn_make_buffer_rsrc((void *)(base + row0 * s), 0, n > 0 ? ((n - 1) * stride + dim) * 2 : 0, 0x00027000);
    }
    /* the products of the rows and the columns `other` */
    template <int N> __device__ inline f32x16 times(const typename Mma<T>::frag (&other)[N], int lane) const {
        int at = (lane & 31) * stride + (lane >> 5) * 8;
        arrived(at);   /* (places are computed here: kept through a walk, they would take the registers of its sums) */
        f32x16 acc = {};
#pragma unroll
        for (int s = 0; s < N; ++s) {
            const auto f = __builtin_amdgcn_raw_buffer_load_b128(rows, s * 16 + (lane >> 5) * 8 < dim ? (at + s * 16) * 2 : -1, 0, 0);
            acc = Mma<T>::go(__builtin_bit_cast(typename Mma<T>::frag, f), other[s], acc);
        }
        return acc;
    }
    /* element 32 t + lane % 32 of the eight rows result_row(8 k) to result_row(8 k + 7), as `of` makes them */
    template <class F> __device__ inline typename Mma<T>::frag column(int t, int k, int lane, F of) const {
        int d = t * 32 + (lane & 31);
        arrived(d);
        const int at = (lane >> 5) * 4 * stride + d;
        typename Mma<T>::frag r;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t x = __builtin_amdgcn_raw_buffer_load_b16(rows, d < dim ? (at + result_row(8 * k + e, 0) * stride) * 2 : -1, 0, 0);
            r[e] = (T)of((float)__builtin_bit_cast(T, x));
        }
        return r;
    }
};
/* sum += (the rows, transposed) times `weights`; `sees`: ones for the rows that result_row numbers and the lane's column sees, zeros for others.  SIGNED:
 * weights are positive, so that an infinite element leaves its sign. */
template <bool SIGNED, class T, int DT, class Sees> __device__ inline void careful_columns(f32x16 (&sum)[DT], const Rows<T> &rows, const typename Mma<T>::frag (&weights)[2], Sees sees,
                                                                                           int lane) {
    const float inf = __builtin_inff();
    bool some = false;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            sum[t] = Mma<T>::go(rows.column(t, k, lane,
                                            [&](float x) {
                                                const bool fine = __builtin_fabsf(x) < inf;
                                                some = some || !fine;
                                                return fine ? x : 0.0f;
                                            }),
                                weights[k], sum[t]);
            __builtin_amdgcn_sched_barrier(0);   /* (one operand at a time: these kernels' registers are in use) */
        }
    if (!__any(some)) return;
    float see[16];
    sees(see);
    const typename Mma<T>::frag seen[2] = {pack8<T>(see), pack8<T>(see + 8)};
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int sign = 1; sign >= -1; sign -= 2) {
            f32x16 many = {};
#pragma unroll
            for (int k = 0; k < 2; ++k) many = Mma<T>::go(rows.column(t, k, lane, [&](float x) { return !(sign * x < inf) ? 1.0f : 0.0f; }), seen[k], many);
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[t][i] += many[i] > 0.0f ? (SIGNED ? sign * inf : __builtin_nanf("")) : 0.0f;
            __builtin_amdgcn_sched_barrier(0);
        }
}
/* one block of 32 keys for 32 queries whose weights are taken around `around` */
template <class T, int DP> __device__ inline void careful_block(f32x16 (&o)[DP / 32], const typename Mma<T>::frag (&qf)[DP / 16], const T *k, const T *v, const Args &a, int length,
                                                                const Sight &sight, float around, int key0, int lane) {
    float s[16];
    const f32x16 acc = Rows<T>(k, a.k_stride[1], key0, length, a.dim).times(qf, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i], a.scale2, -around));
    hide(s, sight, key0, lane >> 5, key0 < a.sinks, 0.0f);
    const typename Mma<T>::frag pf[2] = {pack8<T>(s), pack8<T>(s + 8)};
    careful_columns<true, T>(o, Rows<T>(v, a.v_stride[1], key0, length, a.dim), pf, [&](float (&see)[16]) { show(see, sight, key0, lane >> 5); }, lane);
}

template <int DP> struct Shape { static constexpr int PITCH = DP <= 64 ? 64 : 128; };

/* How many wavefronts of a SIMD a kernel is scheduled for: exactly as many as its registers allow, so that what is left of them goes to
 * operands on their way.  Without it, forward and backward: 4 x 40 heads of 2,048 tokens, a window of 512, 142 and 638 us instead of 139 and
 * 475; 8 heads on 2 of 16,384, 2,048: 147 and 841 instead of 141 and 507; 2 x 16 heads of 2,048, 1,024: 42 and 208 instead of 40 and 148. */
#define RESIDENT(DP) __attribute__((amdgpu_waves_per_eu((DP) <= 64 ? 3 : 2, (DP) <= 64 ? 3 : 2)))

constexpr int WAVES = 4, LANES = WAVES * 64, QUERIES = WAVES * 32, KEYS = 64;

/* f(0) to f(END - 1), each with its number as a constant */
template <int I> struct Number { static constexpr int value = I; };
template <int I, int END, class F> __device__ __attribute__((always_inline)) inline void each(F f) {
    if constexpr (I < END) f(Number<I>()), each<I + 1, END>(f);
}

/* A wavefront's walk over blocks of 32 keys, three of them in work at a time: scores of one are taken and the weights of another meet
 * its values, matrix instructions that do not depend on each other, and between them softmax turns the scores of the block in the
 * middle into weights, a few vector instructions to each matrix instruction.  The maximum that exponentials are taken around moves only
 * when a score passes it by 8 powers of two: the sums stay far from their range's end, and most blocks need no rescaling. */
template <class T, int DP, int PITCH> struct Walk {
    typedef typename Mma<T>::frag frag;
    typedef T pair __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    static constexpr int N = DP / 16, DT = DP / 32;
    uint32_t row[N], column[2 * DT];   /* where a lane finds operands in a tile at 0 */
    frag qf[N];
    f32x16 o[DT], s;                   /* weighted values; scores of the last block */
    union { uint32_t two[8]; frag whole[2]; } p;   /* weights of the one before it */
    float top, total, around, limit, scale2;   /* around: top as an exponent; past `limit` a score moves it */
    __device__ inline void start(const Operands<T, PITCH> &ops, uint32_t lds, float scale) {
#pragma unroll
        for (int i = 0; i < N; ++i) row[i] = (lds + ops.row) ^ (i << 5);
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) column[i] = (lds + ops.column) ^ (i << 5);
        top = limit = -__builtin_inff(), total = around = 0.0f, scale2 = scale;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = f32x16{};
    }
    __device__ inline frag keys(uint32_t at, int i) const { return lds_load<frag>(row[i] + at); }
    __device__ inline frag values(uint32_t at, int i) const {
        union { s16x4 half[2]; frag whole; } u;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            u.half[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(lds_ptr)(column[2 * (i % DT) + k] + at + (i / DT * 16 + 8 * k) * PITCH * 2));
        return u.whole;
    }
    struct Soft { float by, last; bool moved; uint32_t two[8]; };
    /* the maximum of s, and whether it moves the one that exponentials are taken around (also from no key at all, -inf, to any) */
    __device__ inline void look(Soft &f) {
        float most = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[i]);
        f.moved = __any(most > limit), f.by = 1.0f;
        if (f.moved) {
            most = max_halves(most);
            if (most > limit) {
                f.by = __builtin_amdgcn_exp2f((top - most) * scale2);
                total *= f.by, top = most, around = most * scale2, limit = most + 8.0f / scale2;
            }
        }
    }
    /* the weight of key i */
    __device__ inline void weight(Soft &f, int i) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale2, -around));
        total += w;
        if (i % 2) f.two[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{f.last, w}, pair)), arrived(f.two[i / 2]);
        else f.last = w, arrived(f.last);
        arrived(total);   /* here, not where they are used */
    }
    __device__ inline void finish(const Soft &f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p.two[i] = f.two[i];
        if (f.moved)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= f.by;
    }
    __device__ inline f32x16 scores(uint32_t at) const {
        f32x16 acc = {};
#pragma unroll
        for (int i = 0; i < N; ++i) acc = Mma<T>::go(keys(at, i), qf[i], acc);
        in_step<N, 1, 4>();
        return acc;
    }
    __device__ inline void weigh(uint32_t at) {
#pragma unroll
        for (int i = 0; i < N; ++i) o[i % DT] = Mma<T>::go(values(at, i), p.whole[i / DT], o[i % DT]);
        in_step<N, 2, 3>();
    }
    __device__ inline void softmax() {
        Soft f;
        look(f);
#pragma unroll
        for (int i = 0; i < 16; ++i) weight(f, i);
        finish(f);
    }
    /* the scores of the block at k_at, the weights of the last one, and p times the values at v_at */
    __device__ inline void step(uint32_t k_at, uint32_t v_at) {
        constexpr int AHEAD = 3, PRODUCTS = 2 * N;
        f32x16 acc = {};
        frag kf[N], vf[N];
        Soft f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kf[i] = keys(k_at, i), vf[i] = values(v_at, i);
        each<0, PRODUCTS>([&](auto at) __attribute__((always_inline)) {
            constexpr int m = decltype(at)::value, i = m / 2;
            __builtin_amdgcn_sched_barrier(0);
            if (m % 2 == 0) {
                if (i + AHEAD < N) kf[i + AHEAD] = keys(k_at, i + AHEAD), vf[i + AHEAD] = values(v_at, i + AHEAD);
                acc = Mma<T>::go(kf[i], qf[i], acc);
            } else
                o[i % DT] = Mma<T>::go(vf[i], p.whole[i / DT], o[i % DT]);
            __builtin_amdgcn_sched_barrier(0);
            if (m == 1) look(f);
            if (m >= 2)
#pragma unroll
                for (int j = (m - 2) * 16 / (PRODUCTS - 2); j < (m - 1) * 16 / (PRODUCTS - 2); ++j) weight(f, j);
        });
        __builtin_amdgcn_sched_barrier(0);
        finish(f);
        s = acc;
    }
};

/* Prompts: a workgroup takes 128 queries of a head, 32 per wavefront, and walks over its keys in tiles of 64, the next tile on its
 * way while one is worked on, up to the last tile that the wavefront sees; blocks before that which it does not see are masked like others, but for the second
 * and the last two (passing over the rest took 1% off where a window is 512 and added 3% where it is 2,048).  Tiles of 32 keys, which leave registers for a
 * third wavefront per SIMD, took 3% off with a window of 512 and added 6% with 2,048.
 *
 * 4 x 40 heads of 2,048 tokens and size 128, a window of 512: 122 us, 620 TFLOP/s of the pairs that are seen; 8 heads of 16,384, 2,048:
 * 137 us, 945 (a large product of the matrix library: 1,250), the least of three runs; 143 to 156 and 142 in another process.  The card lowers its clock
 * under this load: on zeros these take 17 to 23% less, whole prompts of 32,768 31%, the library's product 25%; how operands and softmax are ordered further makes no difference.  Short walks are bound by memory: 128 sequences of 128
 * tokens, 40 heads, read and write their 674 MB in 126 us; in between, times are near the sum of both: of 1,024 tokens 227 us, 130 of which the bytes alone and 140 the products
 * alone would take.  LDS has no conflicts and is at work for less than a quarter of the time. */
template <class T, int DP, bool PACKED> __global__ void __launch_bounds__(LANES) RESIDENT(DP) attend_forward(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = KEYS * PITCH * 2;
    const Job<PACKED> job = query_job<PACKED, QUERIES>(a, blockIdx.x);
    if (!job.some) return;
    const Span<PACKED> span = job.span;
    const int head = job.head, queries = span.queries(a);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = span.sequence(a);
    const int q0 = job.block * QUERIES, mine = q0 + in_pairs(wave) * 32, query = mine + (lane & 31);
    const int last = (q0 + QUERIES < queries ? q0 + QUERIES : queries) - 1;
    const T *k = (const T *)a.k + span.lead(a.k_stride) + head / a.shared * a.k_stride[2], *v = (const T *)a.v + span.lead(a.v_stride) + head / a.shared * a.v_stride[2];
    const Tiles tiles = tiles_of<KEYS>(a, seq, seq.start + q0, seq.start + last);
    /* in LDS: what of the queries' tile is not in the first buffer, and two buffers, which hold the values of a tile and the keys of the tile after it */
    const uint32_t qtile = lds_offset(lds), lds0 = qtile + QUERIES * PITCH * 2 - TILE;
    const Tile<T, PITCH, KEYS, LANES> ktiles(k, a.k_stride[1], a.dim, threadIdx.x), vtiles(v, a.v_stride[1], a.dim, threadIdx.x);
    auto ask = [&](int t) {
        const uint32_t to = lds0 + (t & 1) * 2 * TILE;
        if (t < tiles.count) ktiles.ask(to + TILE, tiles.tile(t) * KEYS, seq.length);
        if (t > 0) vtiles.ask(to, tiles.tile(t - 1) * KEYS, seq.length);
    };
    /* the queries, the first keys, and the first values and second keys are on their way together */
    if (tiles.count > 0) {
        const T *q = (const T *)a.q + span.lead(a.q_stride) + head * a.q_stride[2];
        Tile<T, PITCH, QUERIES, LANES>(q, a.q_stride[1], a.dim, threadIdx.x).ask(qtile, q0, queries);
        ask(0), ask(1);
    }
    const T *qrow = (const T *)a.q + span.lead(a.q_stride) + (int64_t)query * a.q_stride[1] + head * a.q_stride[2];
    Walk<T, DP, PITCH> walk;
    const Operands<T, PITCH> ops(lane);
    walk.start(ops, lds0, a.scale2);
    const Sight sight(a, seq.length, seq.start + query);
    const int lo = seq.start + mine, hi = seq.start + (mine + 31 < queries ? mine + 31 : queries - 1);
    const Range clear = all_see(a, seq.length, lo, hi), seen = any_see(a, seq.length, lo, hi);
    const int sinks = a.window > 0 ? a.sinks : 0;
    auto mask = [&](int key0) {
        if (!clear.has(key0)) hide(walk.s, sight, key0, half, key0 < a.sinks, -__builtin_inff());
    };
    auto arrive = [&](int t) {
        wait_tiles<0>();
        meet();
        if (t < tiles.count) ask(t + 1);
    };
    constexpr int BLOCK = 32 * PITCH * 2, LOADS = Tile<T, PITCH, KEYS, LANES>::LOADS;
    const int own = mine < queries ? tiles.upto<KEYS>(lesser(hi + 1, seq.length)) : 0;   /* (the wavefront sees none of the later ones) */
    if (tiles.count > 0) {
        if (tiles.count > 1) wait_tiles<2 * LOADS>();
        else wait_tiles<LOADS>();
        meet();
    }
    int t = 0;
    if (own > 0) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) walk.qf[s] = ops.rows(qtile, mine - q0, s);
        walk.s = walk.scores(TILE);
        mask(tiles.tile(0) * KEYS);
        walk.softmax();
        /* (a tile of first keys is often one block only, and the last tile's blocks are not seen by the first wavefronts) */
        if (seen.has(tiles.tile(0) * KEYS + 32) || tiles.tile(0) * KEYS + 32 < sinks) walk.s = walk.scores(TILE + BLOCK);
        mask(tiles.tile(0) * KEYS + 32);
        auto middle = [&](int t, uint32_t at) {
            arrive(t);
            const int key0 = tiles.tile(t) * KEYS;
            walk.step(at + TILE, at);
            mask(key0);
            walk.step(at + TILE + BLOCK, at + BLOCK);
            mask(key0 + 32);
        };
        for (t = 1; t + 1 < own; t += 2) middle(t, 2 * TILE), middle(t + 1, 0);
        if (t < own) middle(t, 2 * TILE), ++t;
        arrive(t);
        const uint32_t at = (t & 1) * 2 * TILE;
        const int key0 = tiles.tile(t - 1) * KEYS;
        if (seen.has(key0) || key0 < sinks) walk.weigh(at);
        if (seen.has(key0 + 32) || key0 + 32 < sinks) {
            walk.softmax();
            walk.weigh(at + BLOCK);
        }
    }
    while (t < tiles.count) arrive(++t);   /* (its part of the others' tiles) */
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) arrived(walk.o[t]);
    const float total = sum_halves(walk.total);
    const float by = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;   /* (nothing visible: zero; not a number: that) */
    T *to = (T *)a.out + span.lead(a.out_stride) + (int64_t)query * a.out_stride[1] + head * a.out_stride[2];
    auto leave = [&] { store_row(to, walk.o, by, a.dim, half); };
    if (query < queries) {
        leave();
        if (half == 0) a.lse[span.values(a, head) + query] = total == 0.0f ? -__builtin_inff() : walk.top * a.scale + __logf(total);
    }
    const bool odd = query < queries && total < __builtin_inff() && any_odd(walk.o);
    if (__builtin_expect(!__any(odd), 1)) return;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) walk.qf[s] = global_frag<T>(qrow, s * 16 + half * 8, a.dim, query < queries);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) walk.o[t] = f32x16{};
    for (int t = 0; t < tiles.count; ++t)
        for (int key0 = tiles.tile(t) * KEYS, n = 0; n < KEYS / 32; ++n, key0 += 32)
            if (seen.has(key0) || key0 < sinks) careful_block<T, DP>(walk.o, walk.qf, k, v, a, seq.length, sight, walk.around, key0, lane);
    /* (a query and its sums are with two lanes, of which one may have found nothing) */
    if (query < queries && max_halves(odd ? 1.0f : 0.0f) > 0.0f) leave();
}

/* Few queries: the queries of a key head's heads are the columns of one block of 32; every wavefront walks over tiles of 32 keys
 * of its own, with its own two buffers and no barrier, and the wavefronts' and then the workgroups' results are joined.  Bound by
 * memory: 32 x 8 heads of 8,192 keys of size 128, one query of 4 heads each: 180 us, 6.0 TB/s (a large copy reaches 5.2, half of it
 * writes). */
constexpr int SPLIT_KEYS = 32;
template <class T, int DP> __global__ void __launch_bounds__(LANES) attend_split(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = SPLIT_KEYS * PITCH * 2, LOADS = 2 * TILE / 1024;
    const int split = blockIdx.x, rb = blockIdx.y % a.row_blocks, kv = blockIdx.y / a.row_blocks, b = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = Span<false>{b}.sequence(a);
    const int rows = a.queries * a.shared, row = rb * 32 + (lane & 31);
    const int query = row / a.shared, head = kv * a.shared + row % a.shared;
    const int lo = seq.start + rb * 32 / a.shared, hi = seq.start + ((rb * 32 + 31 < rows ? rb * 32 + 31 : rows - 1) / a.shared);
    const T *k = (const T *)a.k + b * a.k_stride[0] + kv * a.k_stride[2], *v = (const T *)a.v + b * a.v_stride[0] + kv * a.v_stride[2];
    const Tiles tiles = tiles_of<SPLIT_KEYS>(a, seq, lo, hi);
    const int worker = split * WAVES + wave, workers = a.splits * WAVES;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_offset(lds) + wave * 4 * TILE);
    const Operands<T, PITCH> ops(lane);
    const Tile<T, PITCH, SPLIT_KEYS, 64> ktiles(k, a.k_stride[1], a.dim, lane), vtiles(v, a.v_stride[1], a.dim, lane);
    auto ask = [&](int t, int buffer) {
        const uint32_t to = lds0 + buffer * 2 * TILE;
        const int at = tiles.tile(t) * SPLIT_KEYS;
        ktiles.ask(to, at, seq.length), vtiles.ask(to + TILE, at, seq.length);
    };
    const T *qrow = (const T *)a.q + b * a.q_stride[0] + (int64_t)query * a.q_stride[1] + head * a.q_stride[2];
    typename Mma<T>::frag qf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = global_frag<T>(qrow, s * 16 + half * 8, a.dim, row < rows);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) arrived(qf[s]);
    Running<DP / 32> run;
    run.clear();
    const Sight sight(a, seq.length, seq.start + query);
    const Range clear = all_see(a, seq.length, lo, hi);
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
        const uint32_t ktile = lds0 + buffer * 2 * TILE;
        block_step<T, DP, PITCH>(run, qf, ops, ktile, ktile + TILE, a, sight, at, !clear.has(at), lane);
    }
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) arrived(run.o[t]);
    run.total = sum_halves(run.total);
    if (__builtin_expect(__any(row < rows && run.total < __builtin_inff() && any_odd(run.o)), 0)) {
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) run.o[t] = f32x16{};
        const float around = run.top == -__builtin_inff() ? 0.0f : run.top * a.scale2;
        for (int t = worker; t < tiles.count; t += workers) careful_block<T, DP>(run.o, qf, k, v, a, seq.length, sight, around, tiles.tile(t) * SPLIT_KEYS, lane);
    }
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

/* Of how many tiles a walk counts as short (attend_dq takes delta differently there): with up to three 64s of keys (150 tokens) the error of
 * dQ and dK in half precision is 2.9e-4 of their norm, 3.2e-4 without; at most 0.8% of the backward pass's time (4 x 40 heads of
 * 2,048, a window of 512: 475 us and 471). */
constexpr int FEW_TILES = 3;

/* dQ: queries in registers, keys in tiles as in attend_forward; per block of 32 keys S^T = K Q^T, dP^T = V dO^T,
 * dQ^T += K^T dS^T.  It also leaves delta = sum dO O of every query for attend_dkv.  2 x 16 heads of 2,048 tokens and size 128, a window of
 * 1,024: 63 us, 616 TFLOP/s of the pairs that are seen, the matrix units at work a third of the time. */
template <class T, int DP, bool PACKED> __global__ void __launch_bounds__(LANES) RESIDENT(DP) attend_dq(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH, TILE = KEYS * PITCH * 2;
    const Job<PACKED> job = query_job<PACKED, QUERIES>(a, blockIdx.x);
    if (!job.some) return;
    const Span<PACKED> span = job.span;
    const int head = job.head, queries = span.queries(a);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Sequence seq = span.sequence(a);
    const int q0 = job.block * QUERIES, mine = q0 + wave * 32, query = mine + (lane & 31);
    const int last = (q0 + QUERIES < queries ? q0 + QUERIES : queries) - 1;
    const T *k = (const T *)a.k + span.lead(a.k_stride) + head / a.shared * a.k_stride[2], *v = (const T *)a.v + span.lead(a.v_stride) + head / a.shared * a.v_stride[2];
    const Tiles tiles = tiles_of<KEYS>(a, seq, seq.start + q0, seq.start + last);
    const uint32_t lds0 = lds_offset(lds);
    const Operands<T, PITCH> ops(lane);
    const Tile<T, PITCH, KEYS, LANES> ktiles(k, a.k_stride[1], a.dim, threadIdx.x), vtiles(v, a.v_stride[1], a.dim, threadIdx.x);
    auto ask = [&](int t) {
        const uint32_t to = lds0 + (t & 1) * 2 * TILE;
        const int at = tiles.tile(t) * KEYS;
        ktiles.ask(to, at, seq.length), vtiles.ask(to + TILE, at, seq.length);
    };
    if (tiles.count > 0) ask(0);
    const bool there = query < queries;
    const T *qrow = (const T *)a.q + span.lead(a.q_stride) + (int64_t)query * a.q_stride[1] + head * a.q_stride[2];
    const T *grow = (const T *)a.g + span.lead(a.g_stride) + (int64_t)query * a.g_stride[1] + head * a.g_stride[2];
    const T *orow = (const T *)a.out + span.lead(a.out_stride) + (int64_t)query * a.out_stride[1] + head * a.out_stride[2];
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
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) arrived(qf[s]), arrived(gf[s]);
    delta = sum_halves(delta);
    const int64_t flat = span.values(a, head) + query;
    float lse2 = there ? a.lse[flat] * LOG2E : 0.0f;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) dq[t] = f32x16{};
    arrived(lse2);
    const int lo = seq.start + mine, hi = seq.start + (mine + 31 < queries ? mine + 31 : queries - 1);
    const Sight sight(a, seq.length, seq.start + query);
    const Range clear = all_see(a, seq.length, lo, hi), seen = any_see(a, seq.length, lo, hi);
    const int first = a.window > 0 ? a.sinks : 0;
    /* With few keys the rounding of the forward pass's answer, which delta goes by, is no small part of dS: there delta is the sum of
     * P dP itself, in a walk before the walk. */
    const bool few = tiles.count <= FEW_TILES;
    float sum = 0.0f;
    Fit<T> fit;
    fit.start();
    auto walk = [&](auto number) {
        constexpr int WALK = decltype(number)::value;
        for (int t = 0; t < tiles.count; ++t) {
            wait_tiles<0>();
            meet();
            if (t + 1 < tiles.count) ask(t + 1);
            const int at = tiles.tile(t) * KEYS;
            if (mine >= queries) continue;
            const uint32_t buffer_at = lds0 + (t & 1) * 2 * TILE;
#pragma unroll 1
            for (int n = 0; n < KEYS / 32; ++n) {
                const int key0 = at + n * 32;
                const uint32_t ktile = buffer_at + n * 32 * PITCH * 2, vtile = ktile + TILE;
                if (!seen.has(key0) && key0 >= first) continue;
                __builtin_amdgcn_s_setprio(1);
                __builtin_amdgcn_sched_barrier(0);
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) s = Mma<T>::go(ops.rows(ktile, 0, j), qf[j], s);
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) dp = Mma<T>::go(ops.rows(vtile, 0, j), gf[j], dp);
                in_step<DP / 8, 1, 4>();
                __builtin_amdgcn_s_setprio(0);
                float ds[16];
                const float less = WALK == 0 ? 0.0f : delta;
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse2)) * (dp[i] - less);
                if (!clear.has(key0)) hide(ds, sight, key0, half, key0 < a.sinks, 0.0f);
                if constexpr (WALK == 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum += ds[i];
                    continue;
                }
                lse2 -= (float)fit.check(ds, dq);
                const typename Mma<T>::frag df[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
                __builtin_amdgcn_s_setprio(1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) dq[d] = Mma<T>::go(ops.columns(ktile, j * 16, d), df[j], dq[d]);
                in_step<DP / 16, 2, 3>();
                __builtin_amdgcn_s_setprio(0);
            }
        }
    };
    if (few) {
        walk(Number<0>());
        delta = sum_halves(sum);
        meet();   /* (every wavefront is through with the first walk's last tile) */
        if (tiles.count > 0) ask(0);
    }
    lse2 -= (float)fit.power;   /* (weights of the first walk are as they are; here their exponent is rounded to 2^-18) */
    if (there && half == 0) a.delta[flat] = delta;
    walk(Number<1>());
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) arrived(dq[t]);
    fit.undo(dq, fit.power);
    if (__builtin_expect(__any(there && any_odd(dq)), 0)) {
        const Args &r = args_again();
        const Job<PACKED> job = query_job<PACKED, QUERIES>(r, __builtin_amdgcn_readfirstlane(again(blockIdx.x)));
        const Span<PACKED> span = job.span;
        const int head = job.head, q0 = job.block * QUERIES, lane = again(threadIdx.x) & 63, queries = span.queries(r);
        const int mine = q0 + __builtin_amdgcn_readfirstlane(again(threadIdx.x) >> 6) * 32, query = mine + (lane & 31), half = lane >> 5;
        const Sequence seq = span.sequence(r);
        const bool there = query < queries;
        const T *k = (const T *)r.k + span.lead(r.k_stride) + head / r.shared * r.k_stride[2], *v = (const T *)r.v + span.lead(r.v_stride) + head / r.shared * r.v_stride[2];
        const T *qrow = (const T *)r.q + span.lead(r.q_stride) + (int64_t)query * r.q_stride[1] + head * r.q_stride[2];
        const T *grow = (const T *)r.g + span.lead(r.g_stride) + (int64_t)query * r.g_stride[1] + head * r.g_stride[2];
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) qf[s] = global_frag<T>(qrow, s * 16 + half * 8, r.dim, there), gf[s] = global_frag<T>(grow, s * 16 + half * 8, r.dim, there);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) dq[t] = f32x16{};
        fit.start();
        const int64_t flat = span.values(r, head) + query;
        lse2 = (there ? r.lse[flat] * LOG2E : 0.0f) - (float)fit.power;
        const Sight sight(r, seq.length, seq.start + query);
        const Tiles tiles = tiles_of<KEYS>(r, seq, seq.start + q0, seq.start + lesser(q0 + QUERIES, queries) - 1);
        const Range seen = any_see(r, seq.length, seq.start + mine, seq.start + lesser(mine + 32, queries) - 1);
        const int first = r.window > 0 ? r.sinks : 0;
        for (int t = 0; t < tiles.count; ++t)
            for (int key0 = tiles.tile(t) * KEYS, n = 0; n < KEYS / 32; ++n, key0 += 32) {
                if (!seen.has(key0) && key0 >= first) continue;
                const Rows<T> krows(k, r.k_stride[1], key0, seq.length, r.dim);
                const f32x16 s = krows.times(qf, lane), dp = Rows<T>(v, r.v_stride[1], key0, seq.length, r.dim).times(gf, lane);
                float ds[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], r.scale2, -lse2)) * (dp[i] - delta);
                hide(ds, sight, key0, half, key0 < r.sinks, 0.0f);
                lse2 -= (float)fit.check(ds, dq);
                const typename Mma<T>::frag df[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
                careful_columns<false, T>(dq, krows, df, [&](float (&see)[16]) { show(see, sight, key0, half); }, lane);
            }
        fit.undo(dq, fit.power);
    }
    if (!there) return;
    store_row((T *)a.dq + ((span.first_query(a) + query) * a.heads + head) * a.dim, dq, a.scale, a.dim, half);
}

/* dK and dV: 32 keys of a key head in a wavefront's registers, 32 queries at a time: S = Q K^T, dP = dO V^T, dV^T += dO^T P,
 * dK^T += Q^T dS.  A key's sums stay with one wavefront: no atomic additions, the same bits every time. */
template <class T, int DP> struct KeyGrads {
    static constexpr int PITCH = Shape<DP>::PITCH;
    typename Mma<T>::frag kf[DP / 16], vf[DP / 16];
    f32x16 dk[DP / 32], dv[DP / 32];
    Fit<T> fit;
    __device__ inline void start(const T *krow, const T *vrow, int dim, bool there, int half) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) kf[s] = global_frag<T>(krow, s * 16 + half * 8, dim, there), vf[s] = global_frag<T>(vrow, s * 16 + half * 8, dim, there);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) arrived(kf[s]), arrived(vf[s]);
        clear();
    }
    __device__ inline void clear() {
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) dk[t] = f32x16{}, dv[t] = f32x16{};
        fit.start();
    }
    __device__ inline void stop() {
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) arrived(dk[t]), arrived(dv[t]);
        fit.undo(dk, fit.power + Fit<T>::WEIGHTS), fit.undo(dv, Fit<T>::WEIGHTS);
    }
    /* `t`: the first query's position from the first one that sees this lane's key; the `count` from there on see it */
    __device__ inline void step(const Operands<T, PITCH> &ops, uint32_t qtile, uint32_t gtile, uint32_t lse, uint32_t delta, float scale2, int t, uint32_t count, bool masked,
                                int half) {
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int j = 0; j < DP / 16; ++j) s = Mma<T>::go(ops.rows(qtile, 0, j), kf[j], s);
#pragma unroll
        for (int j = 0; j < DP / 16; ++j) dp = Mma<T>::go(ops.rows(gtile, 0, j), vf[j], dp);
        in_step<DP / 8, 1, 4>();
        __builtin_amdgcn_s_setprio(0);
        float prob[16], ds[16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f32x4 l = lds_load<f32x4>(lse + 16 * half + 8 * i), d = lds_load<f32x4>(delta + 16 * half + 8 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float lse2 = Fit<T>::FITS ? __builtin_fmaf(l[e], -LOG2E, (float)Fit<T>::WEIGHTS) : -l[e] * LOG2E;
                prob[i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + e], scale2, lse2));
                ds[i + e] = prob[i + e] * (dp[i + e] - d[e]);
            }
        }
        if (masked)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((uint32_t)(t + result_row(i, half)) >= count) prob[i] = ds[i] = 0.0f;
        fit.apply(ds, dk);
        const typename Mma<T>::frag pf[2] = {pack8<T>(prob), pack8<T>(prob + 8)}, df[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                dv[d] = Mma<T>::go(ops.columns(gtile, j * 16, d), pf[j], dv[d]);
                dk[d] = Mma<T>::go(ops.columns(qtile, j * 16, d), df[j], dk[d]);
            }
        in_step<DP / 8, 2, 2>();
        __builtin_amdgcn_s_setprio(0);
    }
    /* the same with a head's queries from row0 on and what is not finite among them counted for those that see it only */
    template <bool PACKED> __device__ inline void careful_step(const Args &a, const Span<PACKED> &span, int head, int row0, int t, uint32_t count, int lane) {
        const int half = lane >> 5, queries = span.queries(a);
        const int64_t flat = span.values(a, head) + row0;
        const Rows<T> q((const T *)a.q + span.lead(a.q_stride) + head * a.q_stride[2], a.q_stride[1], row0, queries, a.dim);
        const Rows<T> g((const T *)a.g + span.lead(a.g_stride) + head * a.g_stride[2], a.g_stride[1], row0, queries, a.dim);
        auto sees = [&](int i) { return row0 + result_row(i, half) < queries && (uint32_t)(t + result_row(i, half)) < count; };
        float prob[16], ds[16];
        const f32x16 s = q.times(kf, lane);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            prob[i] = 0.0f;
            if (sees(i)) prob[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, __builtin_fmaf(a.lse[flat + result_row(i, half)], -LOG2E, (float)Fit<T>::WEIGHTS)));
        }
        __builtin_amdgcn_sched_barrier(0);
        const f32x16 dp = g.times(vf, lane);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            ds[i] = 0.0f;
            if (sees(i)) ds[i] = prob[i] * (dp[i] - a.delta[flat + result_row(i, half)]);
        }
        __builtin_amdgcn_sched_barrier(0);
        fit.apply(ds, dk);
        const typename Mma<T>::frag pf[2] = {pack8<T>(prob), pack8<T>(prob + 8)}, df[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
        auto show = [&](float (&see)[16]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) see[i] = sees(i) ? 1.0f : 0.0f;
        };
        careful_columns<true, T>(dv, g, pf, show, lane);
        careful_columns<false, T>(dk, q, df, show, lane);
    }
    __device__ inline bool odd() const { return any_odd(dk) || any_odd(dv); }
};

/* Tiles of queries: rows of q and of the answer's gradient, then log-sums and deltas, by LANES lanes. */
template <class T, int PITCH, int ROWS, int LANES> struct QueryTiles {
    static constexpr int BYTES = ROWS * PITCH * 2, ROW_VALUES = ROWS > 64 ? ROWS * 4 : 256, STAGE = 2 * BYTES + 2 * ROW_VALUES;
    static constexpr int LOADS = 2 * Tile<T, PITCH, ROWS, LANES, LANES != 64>::LOADS + (LANES == 64 ? 2 : 1);
    static_assert(ROWS <= 64 || (ROWS == 128 && LANES == 256), "a row's values by one or two wavefronts");
    Tile<T, PITCH, ROWS, LANES, LANES != 64> q, g;
    const float *lse, *delta;
    int queries;
    template <bool PACKED> __device__ inline QueryTiles(const Args &a, const Span<PACKED> &span, int lane)
        : q((const T *)a.q + span.lead(a.q_stride), a.q_stride[1], a.dim, lane), g((const T *)a.g + span.lead(a.g_stride), a.g_stride[1], a.dim, lane),
          lse(a.lse + span.values(a, 0)), delta(a.delta + span.values(a, 0)), queries(span.queries(a)) {}
    /* (a workgroup's four wavefronts: each asks for as many loads, the last two for the second 64 rows' or, of 64, for those of the first two
     * again) */
    __device__ inline void ask(const Args &a, uint32_t lds, int head, int row, int wave, int lane) const {
        Tile<T, PITCH, ROWS, LANES, LANES != 64> qh = q, gh = g;
        qh.base += head * a.q_stride[2], gh.base += head * a.g_stride[2];
        qh.ask(lds, row, queries), gh.ask(lds + BYTES, row, queries);
        const int second = ROWS > 64 ? wave >> 1 : 0, left = queries - row - 64 * second;
        const int64_t at = (int64_t)head * a.queries + row + 64 * second, last = left < 0 ? 0 : left < 64 && left < ROWS ? left : ROWS < 64 ? ROWS : 64;
        const uint32_t to = lds + 2 * BYTES + 256 * second;
        if (LANES == 64 || (wave & 1) == 0) to_lds4(buffer(lse + at, (uint32_t)last * 4), lane * 4, __builtin_amdgcn_readfirstlane(to));
        if (LANES == 64 || (wave & 1) == 1) to_lds4(buffer(delta + at, (uint32_t)last * 4), lane * 4, __builtin_amdgcn_readfirstlane(to + ROW_VALUES));
    }
};

/* The pairs of a window: a workgroup takes 128 keys and walks over the queries whose window they are in, of every head that shares the
 * key head, in tiles of 64.  With SHARE 2 or 4 it takes 64 or 32 keys, and so many wavefronts share 32 keys and a tile's queries (128 of
 * them with SHARE 4): more workgroups, for calls that would leave CUs without one.  2 x 16 heads of 2,048 tokens and size 128, a window of
 * 1,024: 79 us, 654 TFLOP/s of the pairs that are seen, the matrix units at work a third of the time: all 256 registers of a wavefront are
 * in use, and the four products of a block of 32 x 32 wait for each other. */
constexpr int query_rows(int share) { return share == 4 ? 128 : 64; }
/* a wavefront's keys, of a workgroup's from k0 on, and the queries that see them */
template <int SHARE> struct WaveKeys {
    static constexpr int OWN = QUERIES / SHARE, OWNERS = WAVES / SHARE, ROWS = query_rows(SHARE);
    Sequence seq;
    int mine, key, first, per_head;   /* in tiles of ROWS: the first that the workgroup walks over, and how many of each head */
    uint32_t sight;                   /* how many queries see this lane's key: from its own position on, for a window's length, those that there are */
    Range seen, clear;                /* where a block of 32 queries begins of which any sees one of the wavefront's keys, and one of which all see all */
    __device__ inline WaveKeys(const Args &a, Sequence s, int queries, int k0, int wave, int lane) : seq(s), mine(k0 + wave % OWNERS * 32), key(mine + (lane & 31)), seen(0, 0), clear(0, 0) {
        /* queries from the first key's position on, up to the last key's window */
        int from = k0 - seq.start, to = queries;
        if (a.window > 0) {
            const int64_t most = (int64_t)k0 + OWN - 1 + a.window - seq.start;
            to = most < to ? (int)most : to;
        }
        from = from < 0 ? 0 : from;
        first = from / ROWS, per_head = k0 < seq.length && to > from ? (to + ROWS - 1) / ROWS - first : 0;
        const int64_t left = (int64_t)seq.start + queries - key;
        sight = key >= seq.length || left <= 0 ? 0 : a.window > 0 && a.window < left ? a.window : (uint32_t)left;
        const int begin = mine - seq.start;
        seen = Range(begin - 31, mine < seq.length ? a.window > 0 ? lesser(begin + 31 + a.window, queries) : queries : begin - 31);
        clear = Range(begin + 31, mine + 32 <= seq.length ? a.window > 0 ? lesser(begin - 31 + a.window, queries - 31) : queries - 31 : begin);
    }
};
template <class T, int DP, int SHARE, bool PACKED> __global__ void __launch_bounds__(LANES) RESIDENT(DP) attend_dkv(const Args a) {
    extern __shared__ char lds[];
    typedef WaveKeys<SHARE> Mine;
    constexpr int PITCH = Shape<DP>::PITCH, OWN = Mine::OWN, OWNERS = Mine::OWNERS, ROWS = Mine::ROWS;
    typedef QueryTiles<T, PITCH, ROWS, LANES> Queries;
    const Job<PACKED> job = key_job<PACKED, OWN, QUERIES>(a, blockIdx.x);
    if (!job.some) return;
    const Span<PACKED> span = job.span;
    const int kv = job.head;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Mine m(a, span.sequence(a), span.queries(a), job.block * OWN, wave, lane);
    const Sequence seq = m.seq;
    const int mine = m.mine, key = m.key, first = m.first, per_head = m.per_head, steps = per_head * a.shared;
    const uint32_t sight = m.sight;
    const Range seen = m.seen, clear = m.clear;
    const T *krow = (const T *)a.k + span.lead(a.k_stride) + (int64_t)key * a.k_stride[1] + kv * a.k_stride[2];
    const T *vrow = (const T *)a.v + span.lead(a.v_stride) + (int64_t)key * a.v_stride[1] + kv * a.v_stride[2];
    const uint32_t lds0 = lds_offset(lds);
    const Operands<T, PITCH> ops(lane);
    const Queries queries(a, span, threadIdx.x);
    int head = kv * a.shared, tile = first;      /* of the next step to be asked for */
    auto ask = [&](int t) {
        queries.ask(a, lds0 + (t & 1) * Queries::STAGE, head, tile * ROWS, wave, lane);
        if (++tile == first + per_head) tile = first, ++head;
    };
    KeyGrads<T, DP> grads;
    grads.start(krow, vrow, a.dim, key < seq.length, half);
    if (steps > 0) ask(0);
    int q = first * ROWS;
    for (int t = 0; t < steps; ++t) {
        wait_tiles<0>();
        meet();
        if (t + 1 < steps) ask(t + 1);
        const uint32_t buffer_at = lds0 + (t & 1) * Queries::STAGE;
        auto half_tile = [&](int n) {
            const int q0 = q + n * 32;
            if (!seen.has(q0)) return;
            const uint32_t qtile = buffer_at + n * 32 * PITCH * 2, lse = buffer_at + 2 * Queries::BYTES + n * 32 * 4;
            grads.step(ops, qtile, qtile + Queries::BYTES, lse, lse + Queries::ROW_VALUES, a.scale2, seq.start + q0 - key, sight, !clear.has(q0), half);
        };
        if (SHARE > 1) half_tile(wave / OWNERS);
        else
#pragma unroll 1
            for (int n = 0; n < ROWS / 32; ++n) half_tile(n);
        q = q + ROWS < (first + per_head) * ROWS ? q + ROWS : first * ROWS;
    }
    grads.stop();
    if (__builtin_expect(__any(key < span.keys(a) && grads.odd()), 0)) {
        const Args &r = args_again();
        const Job<PACKED> job = key_job<PACKED, OWN, QUERIES>(r, __builtin_amdgcn_readfirstlane(again(blockIdx.x)));
        const Span<PACKED> span = job.span;
        const int kv = job.head, lane = again(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(again(threadIdx.x) >> 6);
        const Mine m(r, span.sequence(r), span.queries(r), job.block * OWN, wave, lane);
        grads.start((const T *)r.k + span.lead(r.k_stride) + (int64_t)m.key * r.k_stride[1] + kv * r.k_stride[2],
                    (const T *)r.v + span.lead(r.v_stride) + (int64_t)m.key * r.v_stride[1] + kv * r.v_stride[2], r.dim, m.key < m.seq.length, lane >> 5);
        for (int t = 0; t < m.per_head * r.shared; ++t)
            for (int n = SHARE > 1 ? wave / OWNERS : 0; n < (SHARE > 1 ? wave / OWNERS + 1 : ROWS / 32); ++n) {
                const int q0 = (m.first + t % m.per_head) * ROWS + n * 32;
                if (m.seen.has(q0)) grads.careful_step(r, span, kv * r.shared + t / m.per_head, q0, m.seq.start + q0 - m.key, m.sight, lane);
            }
        grads.stop();
    }
    if (SHARE > 1) {
        /* the other wavefronts' sums go to those of the first one or two, in order, dK and then dV */
        float *sums = (float *)lds + (lane & 31);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            meet();
            if (wave >= OWNERS)
#pragma unroll
                for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sums[((wave - OWNERS) * DP + t * 32 + result_row(i, half)) * 32] = which ? grads.dv[t][i] : grads.dk[t][i];
            meet();
            if (wave < OWNERS)
                for (int from = wave; from < WAVES - OWNERS; from += OWNERS)
#pragma unroll
                    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) (which ? grads.dv : grads.dk)[t][i] += sums[(from * DP + t * 32 + result_row(i, half)) * 32];
        }
        if (wave >= OWNERS) return;
    }
    if (key >= span.keys(a)) return;
    /* what queries beyond the window have left for a first key */
    if (a.far_parts > 0 && mine < a.sinks && span.has_far(a, mine)) {
        const float *part = a.far + ((int64_t)(span.far_slot(a) + mine / 32) * a.kv_heads + kv) * a.far_parts * (2 * 32 * DP) + (lane & 31);
        for (int c = 0; c < a.far_parts; ++c, part += 2 * 32 * DP)
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int d = t * 32 + result_row(i, half);
                    grads.dk[t][i] += part[d * 32], grads.dv[t][i] += part[(DP + d) * 32];
                }
    }
    const int64_t row = ((span.first_key(a) + key) * a.kv_heads + kv) * a.dim;
    store_row((T *)a.dk + row, grads.dk, a.scale, a.dim, half);
    store_row((T *)a.dv + row, grads.dv, 1.0f, a.dim, half);
}

/* The first keys and the queries beyond their window: every later query of every head sees those few keys, so the work is split
 * over the queries.  A wavefront walks over tiles of 32 queries with buffers of its own; a workgroup's sums, element d of key j at
 * [dk, dv][d][j], are one part, and attend_dkv adds the parts in order.  4 first keys of 2 x 16 heads, 1,024 queries beyond their window: 13 us,
 * two or three tiles for each wavefront, from launch to end a chain of loads, one tile and the sums. */
template <class T, int DP, bool PACKED> __global__ void __launch_bounds__(LANES) __attribute__((amdgpu_waves_per_eu((DP) <= 64 ? 2 : 1))) attend_far(const Args a) {
    extern __shared__ char lds[];
    constexpr int PITCH = Shape<DP>::PITCH;
    typedef QueryTiles<T, PITCH, 32, 64> Queries;
    /* (in one dimension, which holds what check() lets through: fewer than 2^24 blocks, or 256 workgroups) */
    const int part = blockIdx.x % a.far_parts, item = blockIdx.x / a.far_parts, block = item % a.far_blocks, kv = item / a.far_blocks % a.kv_heads, b = item / a.far_blocks / a.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    Span<PACKED> span;
    if constexpr (PACKED) span = {__builtin_amdgcn_readfirstlane(a.sequences[b].first), __builtin_amdgcn_readfirstlane(a.sequences[b].tokens), b};
    else span = {b};
    const int k0 = block * 32, key = k0 + (lane & 31);
    if (!span.has_far(a, k0)) return;
    const Sequence seq = span.sequence(a);
    const int all = span.queries(a);
    const T *krow = (const T *)a.k + span.lead(a.k_stride) + (int64_t)key * a.k_stride[1] + kv * a.k_stride[2];
    const T *vrow = (const T *)a.v + span.lead(a.v_stride) + (int64_t)key * a.v_stride[1] + kv * a.v_stride[2];
    KeyGrads<T, DP> grads;
    grads.start(krow, vrow, a.dim, key < seq.length, half);
    const int64_t begin = (int64_t)k0 + a.window - seq.start;      /* the first query beyond the first key's window */
    const int first = begin <= 0 ? 0 : begin < all ? (int)begin / 32 : 0;
    const int per_head = k0 < seq.length && begin < all ? (all + 31) / 32 - first : 0, items = per_head * a.shared;
    const int worker = part * WAVES + wave, workers = a.far_parts * WAVES;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_offset(lds) + wave * 2 * Queries::STAGE);
    const Operands<T, PITCH> ops(lane);
    const Queries queries(a, span, lane);
    auto ask = [&](int i, int buffer) { queries.ask(a, lds0 + buffer * Queries::STAGE, kv * a.shared + i / per_head, (first + i % per_head) * 32, 0, lane); };
    const int64_t left = (int64_t)seq.start + all - key - a.window;
    const uint32_t sight = key >= seq.length || key >= a.sinks || left <= 0 ? 0 : (uint32_t)left;
    int buffer = 0;
    if (worker < items) ask(worker, 0);
    for (int i = worker; i < items; i += workers, buffer ^= 1) {
        if (i + workers < items) {
            /* (the other buffer's last reads have returned: their results went into the products before this) */
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            ask(i + workers, buffer ^ 1);
            wait_tiles<Queries::LOADS>();
        } else
            wait_tiles<0>();
        const uint32_t qtile = lds0 + buffer * Queries::STAGE, lse = qtile + 2 * Queries::BYTES;
        grads.step(ops, qtile, qtile + Queries::BYTES, lse, lse + Queries::ROW_VALUES, a.scale2, seq.start + (first + i % per_head) * 32 - key - a.window, sight, true, half);
    }
    grads.stop();
    if (__builtin_expect(__any(grads.odd()), 0)) {
        grads.clear();
        for (int i = worker; i < items; i += workers) {
            const int q0 = (first + i % per_head) * 32;
            grads.careful_step(a, span, kv * a.shared + i / per_head, q0, seq.start + q0 - key - a.window, sight, lane);
        }
        grads.stop();
    }
    float *sums = (float *)lds;
    constexpr int HALF = DP * 32;
    float *to = a.far + (((int64_t)(span.far_slot(a) + block) * a.kv_heads + kv) * a.far_parts + part) * (2 * HALF);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[wave * HALF + (t * 32 + result_row(i, half)) * 32 + (lane & 31)] = which ? grads.dv[t][i] : grads.dk[t][i];
        __syncthreads();
        for (int e = threadIdx.x; e < HALF; e += LANES) to[which * HALF + e] = sums[e] + sums[HALF + e] + sums[2 * HALF + e] + sums[3 * HALF + e];
    }
}

/* whether a call's numbers, layout and tensors are such that the kernels take them (rows and batch aside) */
int check_call(const ace_attend_t *a) {
    if (!a || a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return ACE_EINVAL;
    if (a->dim < 8 || a->dim % 8 || a->window < 0 || a->sinks < 0 || (a->dtype != ACE_T_BF16 && a->dtype != ACE_T_F16)) return ACE_EINVAL;
    if (!(a->scale > 0.0f) || a->scale > 1e30f) return ACE_EINVAL;
    if (a->dim > 128 || a->queries > MOST || a->keys > MOST) return ACE_ETOOBIG;
    /* (a tile of 64 rows is named by 32-bit places) */
    const int64_t widest = (int64_t)1 << 23;
    if (a->q_stride[1] >= widest || a->k_stride[1] >= widest || a->v_stride[1] >= widest || a->q_stride[1] < 0 || a->k_stride[1] < 0 || a->v_stride[1] < 0) return ACE_ETOOBIG;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8 || a->k_stride[i] % 8 || a->v_stride[i] % 8 || a->out_stride[i] % 8) return ACE_EINVAL;
    if (a->batch == 0 || a->queries == 0) return ACE_OK;
    if (!a->d_q || !a->d_out || !a->d_lse || (a->keys > 0 && (!a->d_k || !a->d_v))) return ACE_EINVAL;
    if (((uintptr_t)a->d_q | (uintptr_t)a->d_k | (uintptr_t)a->d_v | (uintptr_t)a->d_out) & 15) return ACE_EINVAL;
    return ACE_OK;
}

Args args_of(const ace_attend_t *a) {
    Args k = {};
    k.batch = a->batch, k.queries = a->queries, k.keys = a->keys, k.heads = a->heads, k.kv_heads = a->kv_heads, k.dim = a->dim;
    k.shared = a->heads / a->kv_heads, k.window = a->window < WIDEST ? a->window : WIDEST, k.sinks = a->sinks, k.scale = a->scale, k.scale2 = a->scale * LOG2E;
    k.start = a->d_start, k.length = a->d_length;
    for (int i = 0; i < 3; ++i) k.q_stride[i] = a->q_stride[i], k.k_stride[i] = a->k_stride[i], k.v_stride[i] = a->v_stride[i], k.out_stride[i] = a->out_stride[i];
    k.q = a->d_q, k.k = a->d_k, k.v = a->d_v, k.out = a->d_out, k.lse = a->d_lse;
    return k;
}

/* Blocks of 32 first keys, and over how many workgroups the queries beyond their window go: `workgroups` in all, as many as there are CUs, at least four
 * tiles of queries for a wavefront.  (4 x 40 heads of 2,048 queries, all of the backward pass: 475 us; with two workgroups for every CU
 * 479.  4 heads on 1 of 16,384, a window of 2,048: 344 us in up to 32 parts, 354 in up to 16; 8 on 1 of 32,768, 1,024: 623 and 731.) */
void far_of(const ace_attend_t *a, int64_t batch, int64_t queries, int64_t keys, int64_t workgroups, Args &k) {
    const int64_t sinks = a->window > 0 ? (a->sinks < keys ? a->sinks : keys) : 0;
    k.far_blocks = (int)((sinks + 31) / 32), k.far_parts = 0, k.far_slots = 0, k.far_times = k.far_per = 0;
    if (sinks == 0 || batch == 0 || queries == 0) return;
    k.far_slots = (int)(batch * k.far_blocks);
    const int64_t groups = batch * a->kv_heads * k.far_blocks, tiles = (int64_t)(a->heads / a->kv_heads) * ((queries + 31) / 32);
    int64_t parts = workgroups / groups;
    const int64_t most = (tiles + WAVES * 4 - 1) / (WAVES * 4);
    parts = parts < most ? parts : most;
    k.far_parts = parts < 1 ? 1 : parts > 32 ? 32 : (int)parts;
}
int width_of(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }
int64_t delta_floats(const ace_attend_t *a) { return ((int64_t)a->batch * a->heads * a->queries + 3) / 4 * 4; }

size_t backward_workspace(const ace_attend_t *a, const Args &k) {
    return (size_t)(delta_floats(a) + (int64_t)k.far_slots * a->kv_heads * k.far_parts * 2 * 32 * width_of(a->dim)) * sizeof(float);
}
/* the gradients' part of the arguments */
int backward_args(const ace_attend_t *a, const void *d_gout, const int64_t *gout_stride, void *d_dq, void *d_dk, void *d_dv, void *d_workspace, Args &k) {
    if ((a->queries > 0 && (!d_gout || !gout_stride || !d_dq || !d_workspace)) || (a->keys > 0 && (!d_dk || !d_dv))) return ACE_EINVAL;
    if (((uintptr_t)d_gout | (uintptr_t)d_dq | (uintptr_t)d_dk | (uintptr_t)d_dv | (uintptr_t)d_workspace) & 15) return ACE_EINVAL;
    k.g = d_gout, k.delta = (float *)d_workspace, k.far = k.delta + delta_floats(a), k.dq = d_dq, k.dk = d_dk, k.dv = d_dv;
    for (int i = 0; gout_stride && i < 3; ++i) {
        if (gout_stride[i] % 8) return ACE_EINVAL;
        k.g_stride[i] = gout_stride[i];
    }
    return k.g_stride[1] < 0 || k.g_stride[1] >= (int64_t)1 << 23 ? ACE_ETOOBIG : ACE_OK;
}

template <auto KERNEL> int with_lds(int bytes) {
    static std::atomic<uint64_t> done;
    return layer_allow_lds((const void *)KERNEL, bytes, done);
}

/* workgroups for blocks of SIZE rows of that many heads */
template <bool PACKED> uint32_t grid(const Args &k, int heads, int rows, int size) {
    return PACKED ? (uint32_t)Deal(heads, k.blocks * (QUERIES / size)).groups() : (uint32_t)places((int64_t)k.batch * heads * ((rows + size - 1) / size));
}

template <class T, int DP, bool PACKED> int forward_blocks(const Args &k, hipStream_t stream) {
    constexpr int LDS = (QUERIES + 3 * KEYS) * Shape<DP>::PITCH * 2;
    const int ready = with_lds<attend_forward<T, DP, PACKED>>(LDS);
    if (ready != ACE_OK) return ready;
    attend_forward<T, DP, PACKED><<<grid<PACKED>(k, k.heads, k.queries, QUERIES), LANES, LDS, stream>>>(k);
    return layer_launched();
}

/* Fewer workgroups of 128 keys than this: half as many keys for each, or a quarter.  Measured, all of the backward pass, with 128, 64
 * and 32 keys, at 512 workgroups of 128 (2 x 16 heads of 2,048 tokens, a window of 512): 110, 118 and 190 us; at 384 (8 x 4 heads
 * of 1,531 tokens and size 64, 256): 49, 49 and 63; at 256 (16 heads): 81, 75 and 115; at 128 (8 heads): 75, 68 and 81; at 64 (16 heads
 * on 4): 155, 115 and 105; at 8 (2 heads of 512 tokens and size 64, no window): 33, 28 and 25. */
constexpr int SHARED_BELOW = 448, SHARED_BY_4_BELOW = 96;
template <class T, int DP, int SHARE, bool PACKED> int key_grads(const Args &k, hipStream_t stream) {
    constexpr int LDS = 2 * QueryTiles<T, Shape<DP>::PITCH, query_rows(SHARE), LANES>::STAGE, OWN = QUERIES / SHARE;
    static_assert(LDS >= (WAVES - WAVES / SHARE) * DP * 32 * 4, "the wavefronts' sums");
    const int ready = with_lds<attend_dkv<T, DP, SHARE, PACKED>>(LDS);
    if (ready != ACE_OK) return ready;
    attend_dkv<T, DP, SHARE, PACKED><<<grid<PACKED>(k, k.kv_heads, k.keys, OWN), LANES, LDS, stream>>>(k);
    return layer_launched();
}

template <class T, int DP, bool PACKED> int backward(const Args &k, hipStream_t stream) {
    constexpr int PITCH = Shape<DP>::PITCH, DQ = 4 * KEYS * PITCH * 2;
    constexpr int FAR_TILES = WAVES * 2 * QueryTiles<T, PITCH, 32, 64>::STAGE, FAR_JOIN = WAVES * DP * 32 * 4, FAR = FAR_TILES > FAR_JOIN ? FAR_TILES : FAR_JOIN;
    const int ready = with_lds<attend_dq<T, DP, PACKED>>(DQ), ready2 = with_lds<attend_far<T, DP, PACKED>>(FAR);
    if (ready != ACE_OK || ready2 != ACE_OK) return ACE_EHIP;
    int rc = ACE_OK;
    if (k.queries > 0) {
        attend_dq<T, DP, PACKED><<<grid<PACKED>(k, k.heads, k.queries, QUERIES), LANES, DQ, stream>>>(k);
        if ((rc = layer_launched()) != ACE_OK) return rc;
    }
    if (k.keys == 0) return ACE_OK;
    if (k.far_parts > 0) {
        attend_far<T, DP, PACKED><<<(uint32_t)((int64_t)k.far_parts * k.far_blocks * k.kv_heads * k.batch), LANES, FAR, stream>>>(k);
        if ((rc = layer_launched()) != ACE_OK) return rc;
    }
    const int64_t groups = PACKED ? (int64_t)k.kv_heads * k.blocks : (int64_t)k.batch * k.kv_heads * ((k.keys + QUERIES - 1) / QUERIES);
    return groups < SHARED_BY_4_BELOW ? key_grads<T, DP, 4, PACKED>(k, stream) : groups < SHARED_BELOW ? key_grads<T, DP, 2, PACKED>(k, stream) : key_grads<T, DP, 1, PACKED>(k, stream);
}

}  // namespace

#endif
