/* C ABI of the training-layer operators (libmsdecode.so): attention, rotary positions, RMSNorm with the
 * residual's addition and SwiGLU, each forward and backward.
 *
 * Entry points and the reference interface each replaces (zahlmann/transformer):
 *   msd_attn_forward, msd_attn_backward
 *                      <- model.py:122-147 causal_attention's dot_product_attention (q (T, n_heads, d_head), k and v
 *                         (T, n_kv, d_head)) and its gradient
 *   msd_rope_apply     <- model.py:110-119 apply_rope on q and k, and (sign -1) its gradient
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
 * q_rows (k_rows) rows (the sequence strides are not used), 16-byte aligned, and seqs_host the same numbers on the host,
 * read during the call; q_len and k_len here are the longest.  The ranges must lie inside the rows and not overlap one
 * another; rows outside every range are neither read nor written.  A device entry that leaves the rows or the longest
 * lengths (it then differs from its host copy, which is checked) counts as an empty sequence.  The longest sequences first run
 * fastest.
 *
 * causal: query i of a sequence sees keys 0 .. k_len - q_len + i (the last query sees the last key).  A query that
 * sees nothing has output 0 and, where its dout is finite, contributes to no gradient.
 *
 * Limits: d_head a multiple of 8 up to 128; n_heads a multiple of n_kv_heads, up to 4096; scale in [2^-60, 2^60]; q_rows and
 * k_rows below 2^30, q_rows * n_heads and k_rows * n_kv_heads below 2^31; 128 consecutive rows of one head and the heads of
 * one group together span less than 2^30 elements; q_len times the heads of a group below 2^30 - 256; n_seqs up to 65535,
 * n_seqs * n_kv_heads below 2^20; a launch's workgroups (of up to 256 sequences, or of more whose lengths are alike) below
 * 2^24. */
typedef struct msd_attn {
  int32_t n_seqs, q_len, k_len;
  int32_t n_heads, n_kv_heads, d_head;
  int32_t causal;
  float scale;
  int64_t q_rows, k_rows;
  int64_t q_stride[3], k_stride[3], v_stride[3], dout_stride[3];   /* sequence, row, head */
  const int32_t *seqs, *seqs_host;
} msd_attn;

/* Bytes of device workspace of a forward (backward != 0: of a backward) call, 0 or more.  Needs no initialisation;
 * belongs to one call at a time. */
int64_t msd_attn_workspace_bytes(const msd_attn* a, int32_t backward);

/* out = softmax(scale q k^T) v.  lse: device f32 (q_rows * n_heads), kept for the backward (its layout is the
 * library's own); out_low: a byte (q_rows * n_heads * d_head, 8-byte aligned) for what the rounding to bf16 took off each
 * value of out, from which the backward forms rowsum(dout * out) with values of out to 2^-15 rather than bf16's 2^-8 (dq and dk
 * then lie a tenth nearer the exact ones).  Either may be NULL: no backward follows, or out itself will do. */
int32_t msd_attn_forward(const msd_attn* a, const void* q, const void* k, const void* v, void* out, void* out_low,
                         float* lse, void* workspace, void* stream);

/* dq, dk, dv of the forward's arguments; `out`, `out_low` (or NULL) and `lse` are its results and dout the gradient of
 * `out`. */
int32_t msd_attn_backward(const msd_attn* a, const void* q, const void* k, const void* v, const void* out,
                          const void* out_low, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                          void* workspace, void* stream);

/* Value types of the calls below. */
enum { MSD_BF16 = 0, MSD_F32 = 1 };

/* Rotary positions applied to q and k: batch x tokens rows of n_heads (n_kv_heads) heads of d_head contiguous values,
 * by (batch, token, head) strides in elements; outputs contiguous, of the same type (MSD_BF16 or MSD_F32).  The first
 * d_rot (even) values of a head are pairs, (i, i + d_rot / 2) or, interleaved, (2 i, 2 i + 1), i < d_rot / 2; pair i at
 * position p becomes amplitude times itself turned by 2 pi p turns[i] (sign -1: back, which is the gradient).  The
 * others are copied.  p: positions (device, 4- or 8-byte integers by position_bytes, (batch, token) strides), or, with
 * position_bytes 0, start + token. */
typedef struct msd_rope {
  int32_t batch, tokens, n_heads, n_kv_heads, d_head, d_rot;
  int32_t interleaved, type, sign, position_bytes;
  float amplitude;
  int64_t start;
  int64_t q_stride[3], k_stride[3], position_stride[2];
} msd_rope;

/* turns: device f64 (d_rot / 2); the angle is formed in f64 and reduced to less than a turn before it is rounded.
 * k and k_out may be NULL with n_kv_heads 0.  batch * tokens * (n_heads + n_kv_heads) * d_head < 2^40, batch * tokens < 2^27,
 * d_head <= 4096, n_heads + n_kv_heads <= 4096. */
int32_t msd_rope_apply(const msd_rope* r, const void* q, const void* k, const void* positions, const double* turns,
                       void* q_out, void* k_out, void* stream);

/* Bytes of an 8-bit checkpoint of rows x d values (16-byte aligned device memory): int8 rows padded to 128 columns,
 * then one f32 scale per row and 128 columns.  For the block's largest magnitude m, a value x is kept as
 * rint(x * (127 / m)) and stands for that times (m / 127), all in f32; a block below 2^-100 is kept as zeros; a block
 * that holds a NaN or an infinity stands for NaN. */
int64_t msd_checkpoint_bytes(int64_t rows, int32_t d);

/* y = s / sqrt(mean(s^2) + eps) * scale per row of d values, s = x + residual rounded to their type (x itself without a
 * residual).  x, residual: rows of d contiguous values, `*_stride` elements apart, of `type`; y and sum (= s; NULL
 * without a residual) contiguous, of the same type; scale (d) of scale_type.  rstd: f32 (rows), or NULL when no backward
 * follows; checkpoint: NULL, or msd_checkpoint_bytes(rows, d) for s * rstd in 8 bits.  1 <= d <= 16384;
 * rows below 2^26, beyond 1024 values a row 2^24, beyond 4096 values 2^22. */
int32_t msd_rms_forward(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                        const void* scale, int32_t scale_type, int64_t rows, int32_t d, int32_t type, float eps, void* y,
                        void* sum, float* rstd, void* checkpoint, void* stream);

/* Bytes of msd_rms_backward's workspace (needs no initialisation; belongs to one call at a time). */
int64_t msd_rms_workspace_bytes(int64_t rows, int32_t d);

/* dx (contiguous): the gradient of x, and of the residual: rstd (dy scale - n mean(dy scale n)) + dsum with n = s rstd;
 * dsum NULL or the gradient of `sum`.  dscale (of scale_type; NULL: not wanted): sum over the rows of dy n, the rows'
 * f32 partial sums added in a fixed order.  From s (the forward's sum, or x) or, when checkpoint is not NULL, from the
 * forward's checkpoint in place of n. */
int32_t msd_rms_backward(const void* s, int64_t s_stride, const float* rstd, const void* checkpoint, const void* scale,
                         int32_t scale_type, const void* dy, int64_t dy_stride, const void* dsum, int64_t dsum_stride,
                         int64_t rows, int32_t d, int32_t type, void* dx, void* dscale, void* workspace, void* stream);

/* y = gate / (1 + exp(-gate)) * up, rows of d contiguous values `*_stride` elements apart, y contiguous.  checkpoint:
 * NULL, or 2 msd_checkpoint_bytes(rows, d): gate's, then up's.  1 <= d < 2^24, rows times d rounded up to a multiple of 128
 * below 2^35. */
int32_t msd_swiglu_forward(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, int64_t rows,
                           int32_t d, int32_t type, void* y, void* checkpoint, void* stream);

/* dgate, dup (contiguous) from gate and up or, when checkpoint is not NULL, from the forward's checkpoint. */
int32_t msd_swiglu_backward(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride,
                            const void* checkpoint, const void* dy, int64_t dy_stride, int64_t rows, int32_t d,
                            int32_t type, void* dgate, void* dup, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MSLAYERS_H */
