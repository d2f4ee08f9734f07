/* C ABI of the paged cache's operators (libmsdecode.so): appending a step's keys and values, attention of the newest
 * tokens over their sequences' pages, with or without the weight that each position receives, and eviction.
 *
 * Entry points and the reference interface each stands for (zahlmann/transformer describes the paged cache without
 * shipping it, knowledge/program.md:214-216, 245-250):
 *   msd_paged_append   <- model.py:212-215 prefill_with_kv's and multi_sm_decode.py:194-208's writes to the cache
 *   msd_paged_attn     <- model.py:122-147 causal_attention of new tokens (one, or a chunk) over cached keys and values
 *   msd_paged_evict    (no counterpart: a bounded cache)
 *
 * All calls but msd_paged_plan are asynchronous on `stream` (a hipStream_t of the current device), allocate nothing and return
 * MSD_OK or a negative MSD_E_* code (msdecode.h): MSD_E_ARG for a null or misaligned pointer or a plan that msd_paged_plan has
 * not made, MSD_E_CONFIG for a shape outside the limits below.  Every result is deterministic: sums of floating-point numbers are
 * taken in a fixed order.
 */
#ifndef MSPAGED_H
#define MSPAGED_H

#include <stdint.h>

#include "msdecode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Positions of a page.  Keys and values lie in pages of a pool: bf16 (n_kv_heads, positions, d_head) by (head, position) strides
 * in elements, position p of a sequence in the pool's position 16 table[p / 16] + p % 16. */
enum { MSD_PAGE = 16 };

/* The first words of a plan, in int32. */
enum {
  MSD_PLAN_MAGIC, MSD_PLAN_WORDS, MSD_PLAN_SEQS, MSD_PLAN_HEADS, MSD_PLAN_KV_HEADS, MSD_PLAN_WIDTH, MSD_PLAN_LONGEST,
  MSD_PLAN_Q_END, MSD_PLAN_Q_COUNT, MSD_PLAN_PAGES, MSD_PLAN_SHARED, MSD_PLAN_RESERVED, MSD_PLAN_HEADER = 40
};

/* The plan of a step: how `n_seqs` sequences' work is shared out, in int32 words that the calls below read on the host and, from
 * a copy of the caller's, on the device.  seqs: (q_start, q_len, length) of each: its new tokens are rows q_start ..
 * q_start + q_len of flat tensors (the ranges do not overlap; one without new tokens has none and starts anywhere), the last q_len of
 * its `length` positions.  tables: n_seqs rows of table_width page numbers (those behind a sequence's length are not read).  longest 0:
 * for these lengths, launches as large as they need.  Otherwise lengths up to `longest`: plans of the same n_seqs, q_starts, q_lens,
 * heads, width and longest have the same words but for the numbers that the device reads, and the same launches, so that a captured
 * graph goes on with a new plan in the same memory.
 * words NULL: returns how many there are; otherwise writes them (`room` of them are there) and returns that.  Word MSD_PLAN_Q_END:
 * one past the last row; Q_COUNT: rows of all sequences; PAGES: one past the largest page in use; SHARED: whether a page
 * that takes new rows is in use elsewhere too.
 * Limits: 0 <= q_len <= length <= longest <= 16 table_width, below 2^31 - 2^16; n_heads a multiple of n_kv_heads, up to 4096; n_seqs
 * up to 65535, rows and pool positions below 2^31; q_len times the heads of a group below 2^30 - 256; the words below 2^28, the
 * pages that take new rows and the pieces of work below 2^24. */
int64_t msd_paged_plan(int32_t n_seqs, const int32_t* seqs, const int32_t* tables, int32_t table_width, int32_t n_heads,
                       int32_t n_kv_heads, int32_t longest, int32_t* words, int64_t room);

/* One call on a plan (on the device, 16-byte aligned, and on the host, read during the call).  q_rows: rows of the flat tensors;
 * positions: of the pool, a multiple of 16; strides in elements, multiples of 8 and not negative, the d_head values of a head
 * contiguous; every pointer 16-byte aligned.  Heads and positions of pages that are only read may lie over one another (stride 0: one
 * for all).  A page number outside the pool that only the device's words hold reads as rows of zeros and is not written.
 * Limits: d_head a multiple of 8 up to 128; scale in [2^-60, 2^60]; 128 consecutive rows of one head and the heads of one group
 * together span less than 2^30 elements, as do 16 positions of a page; q_rows times n_heads below 2^31. */
typedef struct msd_paged {
  int32_t d_head;
  float scale;
  int64_t q_rows, positions;
  int64_t q_stride[2];                 /* row, head */
  int64_t k_stride[2], v_stride[2];    /* head, position */
  const int32_t *plan, *plan_host;
} msd_paged;

/* k_new, v_new (q_rows, n_kv_heads, d_head by (row, head) strides) to the positions of their rows.  No two places of k and v are one, and
 * none that is written is one of the new rows'. */
int32_t msd_paged_append(const msd_paged* a, const void* k_new, const int64_t* k_new_stride, const void* v_new,
                         const int64_t* v_new_stride, void* k, void* v, void* stream);

/* Bytes of msd_paged_attn's workspace, 0 or more (needs no initialisation; belongs to one call at a time); weighted: whether
 * weights are counted. */
int64_t msd_paged_attn_workspace_bytes(const msd_paged* a, int32_t weighted);

/* out = softmax(scale q k^T) v of every new token over the positions up to its own, (q_rows, n_heads, d_head) contiguous; rows of
 * no sequence are left as they are.
 * weights_out: NULL, or f32 (n_seqs, n_kv_heads, longest): per position the sum, over the sequence's new tokens and the heads of
 * the group, of the probabilities that it has in the softmax, plus what `weights` (n_seqs, n_kv_heads, weights_width; NULL
 * with a width of 0) has for it, if it is not a new token's and lies inside weights_width; zeros behind the length.  It may be
 * `weights` itself where weights_width is longest.
 * Limits of a call with weights: the sequences of more than 32 rows of a group, times the K/V heads, times longest / 128 rounded up, below 2^22;
 * the others times the K/V heads times longest / 1024 rounded up, and with them what joins pieces, below 2^24.  Nothing has been launched
 * where a call is refused. */
int32_t msd_paged_attn(const msd_paged* a, const void* q, const void* k, const void* v, void* out, const float* weights,
                       int32_t weights_width, float* weights_out, void* workspace, void* stream);

/* Of each sequence, layer and K/V head: the newest `recent` of its positions and, of the others, those with the largest weights
 * (of equal ones the lower position; a NaN counts as larger than any number and comes back as one of no particular bits),
 * min(length, keep) in all, copied in their order to positions 0, 1, .. of the pages that `to` (n_seqs rows of to_width page
 * numbers, on the device) names, which are none that the sequences use and different from one another.  Layers of k (v) are
 * k_layer (v_layer) elements apart.  weights: f32 (n_layers, n_seqs, n_kv_heads, weights_width), positions from weights_width on
 * have weight 0; weights_out (.., keep) those of the kept ones, kept (.., keep) int32 their positions; 0 and -1 behind the last.
 * Limits: 0 <= recent <= keep <= 16 to_width; n_layers times n_kv_heads below 65536, times n_seqs times keep below 2^40. */
int32_t msd_paged_evict(const msd_paged* a, int32_t n_layers, int64_t k_layer, int64_t v_layer, void* k, void* v, const float* weights,
                        int32_t weights_width, int32_t keep, int32_t recent, const int32_t* to, int32_t to_width, float* weights_out,
                        int32_t* kept, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MSPAGED_H */
