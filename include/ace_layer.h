/*
 * ace_layer.h -- C ABI of the training-layer operators (libace_layer.so): what a profile database of a transformer
 * layer is taken of on an MI355X, beside plain matrix products, and the optimizer step whose state bytes the memory
 * model counts.
 *
 * Conventions as in ace_eval.h: plain pointers and sizes, every "d_" pointer is DEVICE memory owned by the caller and is
 * read or written by work on the hipStream_t the caller passes (as void*); 0 or a negative ACE_E* code comes back
 * (ace_layer_strerror names it, ace_layer_last_hip_error says which HIP call failed); nothing is allocated, nothing
 * waits for the device, and nothing is kept between calls.  The device whose memory is passed must be current.
 */
#ifndef ACE_LAYER_H
#define ACE_LAYER_H

#include <stddef.h>
#include <stdint.h>
#include "ace_eval.h" /* the codes ACE_OK ... */

#ifdef __cplusplus
extern "C" {
#endif

#define ACE_LAYER_ABI_VERSION 2

enum { ACE_T_F32 = 0, ACE_T_BF16 = 1, ACE_T_F16 = 2, ACE_T_NONE = 3 };

int ace_layer_abi_version(void);
const char *ace_layer_strerror(int code);
const char *ace_layer_last_hip_error(void);

/* ---- norms around a block --------------------------------------------------------------------------------------------
 * Rows of `width` elements, one after the other; for every row
 *     N(u) = (u - mean u) / sqrt(var u + eps)   (layer != 0)   or   u / sqrt(mean u^2 + eps)
 *     z = N(block) * exit_weight + exit_bias    (block itself where exit_weight is NULL)
 *     r = residual_scale * x + gate * z         (x where block is NULL)
 *     y = N(r) * entry_weight + entry_bias      (not computed where entry_weight is NULL)
 * Every tensor is of one type; arithmetic in 32 bits, one rounding per result. */
#define ACE_NORM_MAX_WIDTH 32768
typedef struct ace_block_norm {
    int64_t rows;
    int64_t rows_per_gate;      /* consecutive rows that share one row of `gate` */
    int32_t width, dtype;       /* ACE_T_* */
    int32_t layer;
    float residual_scale, eps;
    const void *d_x, *d_block;  /* [rows][width]; d_block may be NULL */
    const void *d_gate;         /* NULL, or [ceil(rows / rows_per_gate)][width] */
    const void *d_exit_weight, *d_exit_bias, *d_entry_weight, *d_entry_bias;   /* [width] or NULL */
} ace_block_norm_t;

/* d_residual: r (unused where block is NULL), d_normed: y (unused without entry_weight), d_stats: float[rows][4] =
 * mean and 1 / sqrt of the exit norm, then of the entry norm. */
int ace_block_norm_forward(const ace_block_norm_t *a, void *d_residual, void *d_normed, float *d_stats, void *stream);

/* Gradients.  g_residual and g_normed: of r and y (either may be NULL: zero).  Results that are not wanted are NULL; d_dgate has
 * the shape of the gate.  Sums over rows are taken in an order that depends on the sizes alone.
 * d_workspace: ace_block_norm_workspace_bytes(a) bytes. */
size_t ace_block_norm_workspace_bytes(const ace_block_norm_t *a);
int ace_block_norm_backward(const ace_block_norm_t *a, const void *g_residual, const void *g_normed, const float *d_stats,
                            void *d_dx, void *d_dblock, void *d_dgate, void *d_dexit_weight, void *d_dexit_bias,
                            void *d_dentry_weight, void *d_dentry_bias, void *d_workspace, size_t workspace_bytes, void *stream);

/* ---- attention over a window and a few first keys ----------------------------------------------------------------------
 * Query i of sequence b stands at position p = start[b] + i and sees key j where
 *     j < length[b], j <= p and (p - j < window or j < sinks).
 * out = softmax(scale q k^T) v over the keys it sees, lse = log sum exp of the scaled products; a query that sees none has
 * out = 0 and lse = -inf.  Keys at or past length[b] are not read.  Up to 2^28 queries and keys, and up to 2^22 of batch * heads *
 * (ceil(queries / 128) + 1) and of batch * kv_heads * (ceil(keys / 128) + 1); a start past 2^30 is taken as 2^30. */
typedef struct ace_attend {
    int32_t batch, queries, keys, heads, kv_heads, dim;   /* heads a multiple of kv_heads; dim a multiple of 8 up to 128 */
    int32_t dtype;                                        /* ACE_T_BF16 or ACE_T_F16 */
    int32_t window, sinks;                                /* window 0: all earlier keys */
    float scale;
    const int32_t *d_start, *d_length;                    /* int32[batch]; NULL: keys - queries, keys */
    /* elements between consecutive sequences, tokens and heads (a head's elements are adjacent); all multiples of 8, between
     * tokens 0 to 2^23 - 8, and every tensor starts at a multiple of 16 bytes */
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
    const void *d_q, *d_k, *d_v;
    void *d_out;                                          /* [batch][queries][heads][dim] by out_stride */
    float *d_lse;                                         /* [batch][heads][queries] */
} ace_attend_t;

size_t ace_attend_workspace_bytes(const ace_attend_t *a);
int ace_attend_forward(const ace_attend_t *a, void *d_workspace, size_t workspace_bytes, void *stream);

/* dq [batch][queries][heads][dim], dk and dv [batch][keys][kv_heads][dim], contiguous; d_gout: gradient of out, by
 * gout_stride.  d_out and d_lse of `a` are read.  d_workspace: ace_attend_backward_workspace_bytes(a) bytes. */
size_t ace_attend_backward_workspace_bytes(const ace_attend_t *a);
int ace_attend_backward(const ace_attend_t *a, const void *d_gout, const int64_t gout_stride[3], void *d_dq, void *d_dk, void *d_dv,
                        void *d_workspace, size_t workspace_bytes, void *stream);

/* ---- the same over sequences that lie one after the other ---------------------------------------------------------------
 * Tokens [tokens][heads][dim]; a sequence is a run of them, and its queries see its own keys only, query i key j where j <= i and
 * (i - j < window or j < sinks).  Tokens behind the last sequence are of none: out 0, lse -inf, gradients 0.
 *
 * A table says where sequences lie and in which order their blocks of ACE_PACKED_BLOCK tokens are worked on; it is made once on the host
 * (ace_packing_table) and copied to the device by the caller: the blocks of queries, `blocks` of them, those of keys, both in another order, and the
 * sequences. */
#define ACE_PACKED_BLOCK 128
typedef struct ace_packed_block {
    int32_t first, tokens;         /* of the sequence */
    int32_t block;                 /* tokens block * 128 to block * 128 + 127 of it */
    int32_t sequence;              /* its number, or -1: tokens of none */
} ace_packed_block_t;
typedef struct ace_packed_sequence { int32_t first, tokens; } ace_packed_sequence_t;
typedef struct ace_packing {
    int32_t tokens, sequences;     /* all tokens, those of no sequence among them; sequences that are not empty */
    int32_t blocks, longest;
    const void *d_table;           /* at a multiple of 16 bytes */
} ace_packing_t;

/* lengths: HOST int64[n], 0 and more, `tokens` at most in all, which is 2^28 at most.  Fills in *p but d_table; table: HOST memory of
 * table_bytes bytes, or NULL (then only *p is filled in).  The table takes 64 blocks + 8 sequences bytes. */
int ace_packing_table(const int64_t *lengths, int64_t n, int64_t tokens, ace_packing_t *p, void *table, size_t table_bytes);

/* As ace_attend_forward and ace_attend_backward: batch is 1, queries and keys are all tokens, d_start and d_length NULL; lse is
 * [heads][tokens].  Up to 2^22 of heads * (blocks + 1), and for gradients of sequences * kv_heads * (blocks of 32 first keys) where a sequence is
 * longer than the window. */
int ace_packed_attend_forward(const ace_attend_t *a, const ace_packing_t *p, void *stream);
size_t ace_packed_attend_backward_workspace_bytes(const ace_attend_t *a, const ace_packing_t *p);
int ace_packed_attend_backward(const ace_attend_t *a, const ace_packing_t *p, const void *d_gout, const int64_t gout_stride[3], void *d_dq, void *d_dk, void *d_dv,
                               void *d_workspace, size_t workspace_bytes, void *stream);

/* ---- AdamW over many tensors -------------------------------------------------------------------------------------------
 *     g = grad_scale * grad;  m = m b1 + g (1 - b1);  v = v b2 + g^2 (1 - b2)
 *     p = p decay - m step_size / (sqrt(v) root_scale + eps);  copy = p rounded
 * with decay = 1 - lr * weight_decay, step_size = lr / (1 - b1^t), root_scale = 1 / sqrt(1 - b2^t).
 * Moments of 32 bits: d_m, d_v float.  Of 8 bits: blocks of 256 elements of a tensor, d_m int8 codes of m in steps of max|m| / 127 (1e-30 / 127 at least),
 * d_v uint8 codes of sqrt(v) in steps of its maximum / 255; a code of d_v is 0 only where sqrt(v) is, so no divisor
 * vanishes that was not zero.  A block whose largest value is not finite comes back as NaN as a whole. */
#define ACE_ADAMW_BLOCK 256
#define ACE_ADAMW_CHUNK 8192       /* elements of a tensor that one workgroup takes */
#define ACE_ADAMW_MAX_TENSORS 400  /* of one launch */
typedef struct ace_adamw_tensor {  /* device array, one per tensor */
    float *d_param;
    void *d_copy;                  /* or NULL */
    int64_t n;                     /* elements */
    int64_t state_at;              /* first element of its moments: a multiple of ACE_ADAMW_BLOCK */
    int64_t first_chunk;           /* chunks of the tensors before it */
} ace_adamw_tensor_t;

typedef struct ace_adamw {
    const ace_adamw_tensor_t *d_tensors;   /* [n_tensors] */
    const int32_t *d_chunk_tensor;         /* [n_chunks]: which tensor a chunk belongs to */
    int32_t n_tensors;
    int64_t n_chunks;
    int32_t state_bits, grad_type, copy_type;   /* 32 or 8; ACE_T_*; ACE_T_BF16, _F16 or _NONE */
    void *d_m, *d_v;
    float *d_m_scale, *d_v_scale;          /* 8 bits: one per block */
} ace_adamw_t;

/* grads: HOST array of n_tensors device pointers, read during the call; first_chunks: HOST copy of the tensors' first_chunk with
 * n_chunks behind it, int64[n_tensors + 1].  d_grad_scale: device float or NULL. */
int ace_adamw_step(const ace_adamw_t *a, const void *const *grads, const int64_t *first_chunks, const float *d_grad_scale, float beta1, float one_minus_beta1, float beta2,
                   float one_minus_beta2, float decay, float step_size, float root_scale, float eps, void *stream);

/* The values that 8-bit moments stand for: float[n_blocks * 256] each. */
int ace_adamw_moments(const int8_t *d_m, const uint8_t *d_v, const float *d_m_scale, const float *d_v_scale, int64_t n_blocks, float *d_m_out,
                      float *d_v_out, void *stream);

/* ---- the norm of many gradients, and clipping --------------------------------------------------------------------------
 *     norms[t] = |s| sqrt(sum g^2 over tensor t);  norm = sqrt(sum of norms[t]^2);  scale = s min(1, max_norm / (norm + 1e-6))
 * with s = *d_grad_scale (1 where it is NULL) and max_norm 0: no limit.  Squares and sums in 64 bits, in an order that the sizes alone
 * decide.  A norm that is no number makes scale none, an infinite one makes it 0, where there is a limit. */
typedef struct ace_gradient {      /* HOST array, read during the call */
    void *d_grad;                  /* elements one after the other */
    int64_t n;
    int32_t dtype;                 /* ACE_T_F32, _BF16 or _F16 */
    int32_t reserved;
} ace_gradient_t;

/* d_result: norm and scale; d_norms: float[n_tensors].  d_workspace: ace_gradient_norm_workspace_bytes(...) bytes, a multiple of 8.  Up to 2^20
 * tensors of up to 2^37 elements. */
size_t ace_gradient_norm_workspace_bytes(const ace_gradient_t *grads, int64_t n_tensors);
int ace_gradient_norm(const ace_gradient_t *grads, int64_t n_tensors, double max_norm, const float *d_grad_scale, float *d_result, float *d_norms,
                      void *d_workspace, size_t workspace_bytes, void *stream);
/* g = g scale, in place, rounded to g's type; nothing is written where scale is 1.  No two tensors may overlap. */
int ace_gradient_scale(const ace_gradient_t *grads, int64_t n_tensors, const float *d_scale, void *stream);

/* ---- log-probabilities of taken tokens, and the clipped policy loss ----------------------------------------------------------
 * Of every row z of `vocab` logits, with its target t:
 *     top = max z;  total = sum exp(z - top);  logp = z_t - top - log total
 *     ratio = exp(logp - old);  gain = min(ratio A, clamp(ratio, ratio_low, ratio_high) A);  away = ref - logp
 *     loss += w (kl_weight (exp(away) - away - 1) - gain)                     (without d_ref: no term of it)
 *     d_logp = w (kl_weight (1 - exp(away)) - ratio A where the gain is not clipped)
 *     d_z = g d_logp ([it is the target] - exp(z - top) / total)
 * A row whose target is not in [0, vocab) has none: logp 0, no loss, gradients 0, statistics 0; its logits may be anything.  Nor does a row
 * of weight 0 take part in the loss, whatever its numbers are; where d_logp is 0, d_z is.
 * Exponentials in 32 bits, sums over lanes and what follows from them for a row in 64. */
#define ACE_LOSS_MAX_VOCAB (1 << 28)
typedef struct ace_token_loss {
    int64_t rows, row_stride;      /* row_stride: elements between consecutive rows of d_logits, at least vocab */
    int32_t vocab, dtype;          /* ACE_T_* */
    int32_t target_bits;           /* 32 or 64 */
    int32_t reserved;
    const void *d_logits;
    const void *d_targets;         /* int32 or int64 [rows] */
    /* for the policy's loss: float [rows] each; d_ref and d_weight may be NULL (every row's weight is even_weight then) */
    const float *d_old, *d_advantage, *d_ref, *d_weight;
    double ratio_low, ratio_high, kl_weight, even_weight;
} ace_token_loss_t;

/* d_logp: float[rows]; d_stats: float[rows][2] = top and total. */
int ace_token_logprobs(const ace_token_loss_t *a, float *d_logp, float *d_stats, void *stream);
/* d_dlogits: of the logits' type, rows out_stride elements apart; may be the logits themselves, row for row.  g_logp: float[rows]. */
int ace_token_logprobs_backward(const ace_token_loss_t *a, const float *g_logp, const float *d_stats, void *d_dlogits, int64_t out_stride, void *stream);
/* The same with the d_logp of ace_token_logprobs, or NULL: the target's d_z keeps its digits where its probability is next to 1 (without, it is off by up to
 * 2^-22 g). */
int ace_token_logprobs_gradient(const ace_token_loss_t *a, const float *g_logp, const float *d_logp, const float *d_stats, void *d_dlogits, int64_t out_stride,
                                void *stream);
/* d_loss: one float; d_dlogp: float[rows], for g = 1.  d_workspace: ace_policy_loss_workspace_bytes(a) bytes, a multiple of 8. */
size_t ace_policy_loss_workspace_bytes(const ace_token_loss_t *a);
int ace_policy_loss(const ace_token_loss_t *a, float *d_loss, float *d_logp, float *d_stats, float *d_dlogp, void *d_workspace, size_t workspace_bytes, void *stream);
/* The same with the gradient of the logits, for a gradient of the loss of *g_loss (1 where it is NULL). */
int ace_policy_loss_gradient(const ace_token_loss_t *a, const float *g_loss, float *d_loss, float *d_logp, float *d_stats, float *d_dlogp, void *d_dlogits,
                             int64_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ACE_LAYER_H */
