/* Attention over a window of keys and a few first ones, of a padded batch: the kernels of layer_attend.h. */
#include "layer_attend.h"

namespace {

int check(const ace_attend_t *a) {
    const int rc = check_call(a);
    if (rc != ACE_OK || a->batch == 0 || a->queries == 0) return rc;
    const int64_t blocks = (a->queries + QUERIES - 1) / QUERIES, kblocks = (a->keys + QUERIES - 1) / QUERIES;
    if ((int64_t)a->batch * a->heads * (blocks + 1) > (1 << 22) || (int64_t)a->batch * a->kv_heads * (kblocks + 1) > (1 << 22)) return ACE_ETOOBIG;
    return ACE_OK;
}

int row_blocks(const ace_attend_t *a) { return (int)(((int64_t)a->queries * (a->heads / a->kv_heads) + 31) / 32); }

/* the most keys that a query's block can see */
int64_t most_seen(const ace_attend_t *a) {
    const int64_t seen = (int64_t)a->window + a->queries + a->sinks;
    return a->window > 0 && seen < a->keys ? seen : a->keys;
}

/* How many workgroups attend_split takes for a key head's block of rows: no more than there are CUs for (LDS holds one of these
 * workgroups), and two tiles or more for a wavefront.  32 x 8 heads of 8,192 keys (256 blocks) in one part each: 180 us, in two:
 * 187; 24 x 4 heads of 4,096 (96 blocks) in two: 38, in three, some CUs with a second one: 47; 4 x 40 heads of 2,048 (160 blocks)
 * in one: 29, in two: 39, in four: 40. */
int splits_of(const ace_attend_t *a) {
    const int64_t groups = (int64_t)a->batch * a->kv_heads * row_blocks(a), most = (most_seen(a) + SPLIT_KEYS * WAVES * 2 - 1) / (SPLIT_KEYS * WAVES * 2);
    int64_t splits = 256 / groups;
    splits = splits < most ? splits : most;
    return splits < 1 ? 1 : splits > 64 ? 64 : (int)splits;
}

/* Whether few queries go to attend_split, which reads a key once for all the heads that share it and splits the keys, or to
 * attend_forward, which reads them once per head: by what each would take.  While a CU waits for memory more than it computes, a step of
 * a workgroup of attend_split, 128 keys, takes about 2.4 us and its join 6, one of attend_forward, 64 keys, 1.3 us.  Measured, split
 * and forward: 32 x 32 heads on 8 of 8,192 keys, 1 query: 187 and 342 us, 16: 301 and 339, 24: 481 and 342, 64: 1,227 and 489; 40 heads of
 * 2,048 keys, 1: 26 and 42, 128: 38 and 45; 32 heads on 4 of 32,768, 128: 166 and 625; 16 x 16 heads, a window of 512, 64: 32 and 21. */
bool few(const ace_attend_t *a) {
    if (a->queries > QUERIES || a->batch > 65535 || (int64_t)a->kv_heads * row_blocks(a) > 65535) return false;
    const int64_t groups = (int64_t)a->batch * a->kv_heads * row_blocks(a), heads = (int64_t)a->batch * a->heads, splits = splits_of(a), seen = most_seen(a);
    const int64_t split = (groups * splits + 255) / 256 * ((seen + SPLIT_KEYS * WAVES * splits - 1) / (SPLIT_KEYS * WAVES * splits)) * 24 + (splits > 1 ? 60 : 0);
    const int64_t whole = (heads + 511) / 512 * ((seen + KEYS - 1) / KEYS) * 13;
    return split < whole;
}

template <class T, int DP> int forward(Args &k, const ace_attend_t *a, hipStream_t stream) {
    constexpr int PITCH = Shape<DP>::PITCH;
    if (!few(a)) return forward_blocks<T, DP, false>(k, stream);
    constexpr int TILES = WAVES * 4 * SPLIT_KEYS * PITCH * 2, JOIN = (WAVES * DP * 32 + WAVES * 2 * 32) * 4, LDS = TILES > JOIN ? TILES : JOIN;
    const int ready = with_lds<attend_split<T, DP>>(LDS);
    if (ready != ACE_OK) return ready;
    attend_split<T, DP><<<dim3(k.splits, k.kv_heads * k.row_blocks, k.batch), LANES, LDS, stream>>>(k);
    int rc = layer_launched();
    if (rc != ACE_OK || k.splits == 1) return rc;
    const int64_t rows = (int64_t)k.batch * k.heads * k.queries;
    attend_join<T><<<(uint32_t)((rows + WAVES - 1) / WAVES), LANES, 0, stream>>>(k);
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

extern "C" size_t ace_attend_backward_workspace_bytes(const ace_attend_t *a) {
    if (check(a) != ACE_OK || a->batch == 0) return 0;
    Args k = {};
    far_of(a, a->batch, a->queries, a->keys, 256, k);
    return backward_workspace(a, k);
}

extern "C" int ace_attend_backward(const ace_attend_t *a, const void *d_gout, const int64_t gout_stride[3], void *d_dq, void *d_dk, void *d_dv, void *d_workspace,
                                   size_t workspace_bytes, void *stream) {
    int rc = check(a);
    if (rc != ACE_OK || a->batch == 0) return rc;
    if (workspace_bytes < ace_attend_backward_workspace_bytes(a)) return ACE_EINVAL;
    Args k = args_of(a);
    far_of(a, a->batch, a->queries, a->keys, 256, k);
    if ((rc = backward_args(a, d_gout, gout_stride, d_dq, d_dk, d_dv, d_workspace, k)) != ACE_OK) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == ACE_T_BF16) return a->dim <= 64 ? backward<bf16, 64, false>(k, s) : a->dim <= 96 ? backward<bf16, 96, false>(k, s) : backward<bf16, 128, false>(k, s);
    return a->dim <= 64 ? backward<f16, 64, false>(k, s) : a->dim <= 96 ? backward<f16, 96, false>(k, s) : backward<f16, 128, false>(k, s);
}
