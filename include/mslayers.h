/* C ABI of the training-layer operators (libmsdecode.so): attention, rotary positions, RMSNorm with the
 * residual's addition and SwiGLU, each forward and backward.
 *
 * Entry points and the reference interface each replaces (zahlmann/transformer):
 *   msd_attn_forward, msd_attn_backward
 *                      <- model.py:122-147 causal_attention's dot_product_attention (q (T, n_heads, d_head), k and v
 *                         (T, n_kv, d_head)) and its gradient
 *   msd_rotary         <- model.py:110-119 apply_rope on q and k, and (sign -1) its gradient
 *   msd_rms_forward, msd_rms_backward
 *                      <- model.py:94-98 rms_norm and :157 the residual's addition, and their gradients
 *   msd_swiglu_forward, msd_swiglu_backward
 *                      <- model.py:159 silu(x W_gate) * (x W_up) between the projections, and its gradient
 *
 * All calls are asynchronous on `stream` (a hipStream_t of the current device), allocate nothing and return MSD_OK or
 * a negative MSD_E_* code (msdecode.h): MSD_E_ARG for a null or misaligned pointer, MSD_E_CONFIG for a shape outside
 * the limits below.  Every result is deterministic: sums are taken in a fixed order, without atomics.
 */
#ifndef MSLAYERS_H
#define MSLAYERS_H

#include <stdint.h>

#include "msdecode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One attention call.  bf16 tensors, addressed by (sequence, row, head) strides in elements, the d_head values of a
 * head contiguous; every pointer 16-byte aligned and every stride a multiple of 8.  out, dq, dk and dv are contiguous
 * (rows, heads, d_head).
 *
 * seqs == NULL: n_seqs sequences of q_len query rows and k_len key rows each; q_rows = n_seqs * q_len and k_rows =
 * n_seqs * k_len.  seqs != NULL: a device array of n_seqs (q_start, q_len, k_start, k_len), rows of one flat tensor of
 * q_rows (k_rows) rows (the sequence strides are not used), 16-byte aligned, with q_len and k_len here the longest.
 * The ranges must lie inside the rows and not overlap one another; rows outside every range are neither read nor
 * written.
 *
 * causal: query i of a sequence sees keys 0 .. k_len - q_len + i (the last query sees the last key).  A query that
 * sees nothing has output 0 and contributes to no gradient.
 *
 * Limits: d_head a multiple of 8 up to 128; n_heads a multiple of n_kv_heads; scale > 0; rows and heads such that
 * q_rows * n_heads and k_rows * n_kv_heads are below 2^31; 64 consecutive rows of one head (and the heads of one
 * group) span less than 2^30 elements. */
typedef struct msd_attn {
  int32_t n_seqs, q_len, k_len;
  int32_t n_heads, n_kv_heads, d_head;
  int32_t causal;
  float scale;
  int64_t q_rows, k_rows;
  int64_t q_stride[3], k_stride[3], v_stride[3], dout_stride[3];   /* sequence, row, head */
  const int32_t* seqs;
} msd_attn;

/* Bytes of device workspace of a forward (backward != 0: of a backward) call, 0 or more.  Needs no initialisation;
 * belongs to one call at a time. */
int64_t msd_attn_workspace_bytes(const msd_attn* a, int32_t backward);

/* out = softmax(scale q k^T) v.  lse: device f32 (q_rows * n_heads), kept for the backward (its layout is the
 * library's own); may be NULL when no backward follows. */
int32_t msd_attn_forward(const msd_attn* a, const void* q, const void* k, const void* v, void* out, float* lse,
                         void* workspace, void* stream);

/* dq, dk, dv of the forward's arguments, `out` and `lse` its results and dout the gradient of `out`. */
int32_t msd_attn_backward(const msd_attn* a, const void* q, const void* k, const void* v, const void* out,
                          const float* lse, const void* dout, void* dq, void* dk, void* dv, void* workspace,
                          void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MSLAYERS_H */
