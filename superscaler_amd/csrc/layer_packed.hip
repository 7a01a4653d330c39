/*
 * Attention over sequences that lie one after the other (ace_packed_attend_forward, ace_packed_attend_backward): the kernels of layer_attend.h
 * over a table of the sequences' blocks, which the host makes once for all the layers that see them (ace_packing_table).
 *
 * Nothing is padded: a workgroup takes a block of 128 tokens of one sequence, whichever comes next by the length of its walk, so that what
 * is dispatched last is short. A sequence's rows are a range of a buffer descriptor: what stands behind them, the next sequence's rows, is
 * out of range and arrives as zeros.
 */
#include <algorithm>
#include "layer_attend.h"

namespace {

int check(const ace_attend_t *a, const ace_packing_t *p) {
    if (!p || !a || a->batch != 1 || a->queries != a->keys || a->queries != p->tokens || a->d_start || a->d_length) return ACE_EINVAL;
    const int rc = check_call(a);
    if (rc != ACE_OK || p->tokens == 0) return rc;
    if (p->blocks < 1 || p->sequences < 0 || p->longest < 0 || p->longest > p->tokens || !p->d_table || ((uintptr_t)p->d_table & 15)) return ACE_EINVAL;
    return (int64_t)a->heads * ((int64_t)p->blocks + 1) > (1 << 22) ? ACE_ETOOBIG : ACE_OK;
}

/* Walks from the longest to the shortest, so that what is dispatched last is short: of queries the longest are those that have the most keys before them,
 * of keys those that have the most queries behind them.  But blocks of one sequence read the same rows, which a die's cache holds for a while: in
 * the first order those of them whose walks differ by a few blocks stay together, in the second all of them do, the longest sequence first.  That is for
 * calls of many workgroups, which end together anyway.  Strictly by their walks, and in the two orders, forward and backward: 16,384 tokens in 24 sequences, 40
 * heads (5,720 workgroups): 299 and 975, 285 and 972, 280 and 947 us; in 128, 16 heads (3,056): 64 and 256, 58 and 252, 58 and 249; in 8, 16 heads on 4, a window of
 * 1,024 (2,112): 132 and 502, 133 and 497, 138 and 508; 8,192 in 12, 16 heads (1,088): 51 and 179, 50 and 177, 52 and 192. */
constexpr int64_t BY_SEQUENCE = 2560;
Args packed_args(const ace_attend_t *a, const ace_packing_t *p) {
    Args k = args_of(a);
    k.batch = p->sequences, k.blocks = p->blocks;
    const ace_packed_block_t *table = (const ace_packed_block_t *)p->d_table;
    k.sequences = (const ace_packed_sequence_t *)(table + 4 * (int64_t)p->blocks);
    k.query_blocks = table + ((int64_t)p->blocks * a->heads < BY_SEQUENCE ? 0 : 2 * (int64_t)p->blocks), k.key_blocks = k.query_blocks + p->blocks;
    return k;
}

/* attend_far's part of the arguments: none where no sequence is longer than the window.
 *
 * Slots for what it leaves: a block of first keys has one where a query stands beyond its first key's window, so a sequence of w + 1 + 32 (j - 1) tokens
 * or more has j, up to far_blocks.  Which sequences are that long is not known here; the most slots per token that any has are the largest of
 * j / (w + 1 + 32 (j - 1)), which is that of the first or the last j.  With a sequence's slots from its first token times that on, rounded down, no two
 * sequences' meet (n tokens times it are no fewer than the slots that n tokens need, a whole number).  Where sequences are few, or about as long as first keys and window
 * together, far_blocks for each are fewer.  (256 sequences of 128 tokens on average, 20 key heads of 128, a window of 256: with 37 first keys 148 MB, for each the same
 * number 336; with 1,024 first keys and a sequence as long 550 MB and 5.4 GB.) */
int packed_far(const ace_attend_t *a, const ace_packing_t *p, Args &k) {
    if (p->longest <= a->window) return ACE_OK;
    /* (Of many groups most are short sequences' and end at once: 40 sequences, 4 key heads of 64, 6,143 tokens, a window of 256, all of the backward pass: 74.5 us
     * in one part, 67.6 in three.  Of few, more parts than that are more for attend_dkv to add up: 8 sequences, 4 key heads, 8,192 tokens, a window of 512:
     * 184 in 8 parts, 193 in 16.) */
    far_of(a, p->sequences, p->longest, p->longest, (int64_t)p->sequences * a->kv_heads > 64 ? 512 : 256, k);
    if ((int64_t)p->sequences * a->kv_heads * k.far_blocks > (1 << 22)) return ACE_ETOOBIG;
    if (k.far_blocks == 0) return ACE_OK;
    int64_t times = 1, per = (int64_t)a->window + 1;
    if (k.far_blocks * per > per + 32 * ((int64_t)k.far_blocks - 1)) times = k.far_blocks, per += 32 * ((int64_t)k.far_blocks - 1);
    const int64_t slots = (int64_t)p->tokens * times / per;
    if (slots < k.far_slots) k.far_slots = (int)slots, k.far_times = (int)times, k.far_per = (int)per;
    return ACE_OK;
}

}  // namespace

extern "C" int ace_packing_table(const int64_t *lengths, int64_t n, int64_t tokens, ace_packing_t *p, void *table, size_t table_bytes) {
    if (n < 0 || (n > 0 && !lengths) || tokens < 0 || !p) return ACE_EINVAL;
    if (tokens > MOST) return ACE_ETOOBIG;
    static_assert(ACE_PACKED_BLOCK == QUERIES, "a workgroup's queries");
    int64_t used = 0, blocks = 0, longest = 0, sequences = 0;
    for (int64_t i = 0; i < n; ++i) {
        if (lengths[i] < 0 || lengths[i] > tokens - used) return ACE_EINVAL;
        used += lengths[i], blocks += (lengths[i] + QUERIES - 1) / QUERIES, sequences += lengths[i] > 0;
        longest = lengths[i] > longest ? lengths[i] : longest;
    }
    blocks += (tokens - used + QUERIES - 1) / QUERIES;
    *p = {(int32_t)tokens, (int32_t)sequences, (int32_t)blocks, (int32_t)longest, nullptr};
    if (!table) return ACE_OK;
    if (table_bytes < (size_t)blocks * 4 * sizeof(ace_packed_block_t) + (size_t)sequences * sizeof(ace_packed_sequence_t)) return ACE_EINVAL;
    ace_packed_block_t *q = (ace_packed_block_t *)table, *k = q + blocks, *at = q;
    ace_packed_sequence_t *s = (ace_packed_sequence_t *)(k + 3 * blocks);
    int32_t first = 0, index = 0;
    for (int64_t i = 0; i <= n; ++i) {
        const int32_t length = (int32_t)(i < n ? lengths[i] : tokens - used);
        for (int32_t b = 0; b * QUERIES < length; ++b) *at++ = {first, length, b, i < n ? index : -1};
        if (i < n && length > 0) s[index++] = {first, length};
        first += length;
    }
    for (ace_packed_block_t *to = k; to < (ace_packed_block_t *)s; to += blocks) std::copy(q, k, to);
    const auto order = [](const bool keys, const int run) {
        return [keys, run](const ace_packed_block_t &x, const ace_packed_block_t &y) {
            if ((x.sequence < 0) != (y.sequence < 0)) return y.sequence < 0;
            const int walk_x = keys ? (x.tokens - 1) / QUERIES - x.block : x.block, walk_y = keys ? (y.tokens - 1) / QUERIES - y.block : y.block;
            if (run > 0 && walk_x / run != walk_y / run) return walk_x > walk_y;
            if (x.first != y.first) return x.tokens != y.tokens ? x.tokens > y.tokens : x.first < y.first;
            return walk_x > walk_y;
        };
    };
    std::sort(q, q + blocks, order(false, 3));
    std::sort(k, k + blocks, order(true, 2));
    std::sort(k + blocks, k + 2 * blocks, order(false, 0));
    std::sort(k + 2 * blocks, k + 3 * blocks, order(true, 0));
    return ACE_OK;
}

extern "C" int ace_packed_attend_forward(const ace_attend_t *a, const ace_packing_t *p, void *stream) {
    const int rc = check(a, p);
    if (rc != ACE_OK || p->tokens == 0) return rc;
    const Args k = packed_args(a, p);
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == ACE_T_BF16)
        return a->dim <= 64 ? forward_blocks<bf16, 64, true>(k, s) : a->dim <= 96 ? forward_blocks<bf16, 96, true>(k, s) : forward_blocks<bf16, 128, true>(k, s);
    return a->dim <= 64 ? forward_blocks<f16, 64, true>(k, s) : a->dim <= 96 ? forward_blocks<f16, 96, true>(k, s) : forward_blocks<f16, 128, true>(k, s);
}

extern "C" size_t ace_packed_attend_backward_workspace_bytes(const ace_attend_t *a, const ace_packing_t *p) {
    Args k = {};
    return check(a, p) != ACE_OK || p->tokens == 0 || packed_far(a, p, k) != ACE_OK ? 0 : backward_workspace(a, k);
}

extern "C" int ace_packed_attend_backward(const ace_attend_t *a, const ace_packing_t *p, const void *d_gout, const int64_t gout_stride[3], void *d_dq, void *d_dk,
                                          void *d_dv, void *d_workspace, size_t workspace_bytes, void *stream) {
    int rc = check(a, p);
    if (rc != ACE_OK || p->tokens == 0) return rc;
    Args k = packed_args(a, p);
    if ((rc = packed_far(a, p, k)) != ACE_OK) return rc;
    if (workspace_bytes < backward_workspace(a, k)) return ACE_EINVAL;
    if ((rc = backward_args(a, d_gout, gout_stride, d_dq, d_dk, d_dv, d_workspace, k)) != ACE_OK) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == ACE_T_BF16) return a->dim <= 64 ? backward<bf16, 64, true>(k, s) : a->dim <= 96 ? backward<bf16, 96, true>(k, s) : backward<bf16, 128, true>(k, s);
    return a->dim <= 64 ? backward<f16, 64, true>(k, s) : a->dim <= 96 ? backward<f16, 96, true>(k, s) : backward<f16, 128, true>(k, s);
}
