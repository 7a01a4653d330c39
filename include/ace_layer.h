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

#define ACE_LAYER_ABI_VERSION 1

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

#ifdef __cplusplus
}
#endif
#endif /* ACE_LAYER_H */
