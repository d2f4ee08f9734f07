// Attention with its gradient (gfx950): O = softmax(scale Q K^T) V for grouped heads, and the backward pass that
// recomputes the probabilities.
//
// Reference: model.py:122-147 (causal_attention's dot_product_attention; q (T, n_heads, d_head), k, v (T, n_kv,
// d_head)).
//
// For a query row i and a key row j that it sees, with c = scale log2(e):
//   P_ij = 2^(c q_i.k_j - L_i), L_i = log2 sum_j 2^(c q_i.k_j);   O_i = sum_j P_ij v_j
//   D_i = dO_i.O_i;   dS_ij = P_ij (dO_i.v_j - D_i)
//   dV_j = sum_i P_ij dO_i;   dK_j = scale sum_i dS_ij q_i;   dQ_i = scale sum_j dS_ij k_j
//
// Rows.  The g query heads that share a K/V head are rows of one problem: row r is position r / g, head r % g.  A tile of
// rows then covers g times fewer positions (less of the diagonal's masked area is computed, and one token of g heads
// is a tile already), and every K/V tile in LDS serves all g heads.
//
// Matrix products.  v_mfma_f32_32x32x16_bf16 gives lane l column l % 32 and rows 8 (i / 4) + 4 (l / 32) + i % 4 of its
// 32 x 32 result (i < 16).  Each product is oriented so that its result is, register by register, the operand of the
// next one: the forward and dQ take S^T = K Q^T (a lane holds one query's scores, so maxima and sums stay in the lane),
// dK/dV take S = Q K^T (a lane holds one key's).  The contraction index of the next product then runs, for half h = l /
// 32, over 4 h + {0..3} and 8 + 4 h + {0..3} of each 16: the other operand, which lies in LDS row by row, is read with
// the transposing read ds_read_b64_tr_b16 in that same order, so the probabilities are never moved between lanes.
//
// LDS tiles.  Rows of 128 bytes (d_head <= 64) or 256 bytes, in 16-byte pieces; row r holds piece c at position c ^
// f(r), with f chosen (swizzle()) so that both the plain reads (32 rows, one piece each) and the transposing reads (4
// rows, 64 bytes each) touch every bank once.  Tiles go from memory to LDS directly, the next one or two on their way while this
// one is worked on, one barrier a tile (through registers, at the long case below as the kernels were then: 318 us in
// place of 300 forward, 445 in place of 390 for dQ).  Rows and columns that do not exist are zeros (buffer loads outside the
// descriptor), so what lies behind a sequence's rows is never read.
//
// The backward is two kernels: attn_dq (like the forward, rows outside, keys inside) and attn_dkv (keys outside, all
// rows of the group inside).  Each recomputes S and dP: 7 products instead of the 5 of one kernel, which would have to
// add dQ across workgroups with atomics, in no fixed order.
//
// A workgroup is four waves of 32 rows (or keys) at every size: with one wave of 32 rows for few of them one token against
// a cache took 7.0 us in place of 6.3, 333 rows against 1021 keys 23 in place of 14, and many rows twice as long (the
// tile's fetch serves a quarter of them).
//
// What bounds it: the matrix cores where there are many rows.  Measured, bf16, us and the rate of the products that the
// mask leaves (a large library product reaches 1,262 TFLOP/s on this card):
//   rows x keys, heads / kv, d, mask          forward        dQ             dK and dV, their parts' sum
//   8192 x 8192, 16 / 4, 128, causal          318-352 (865)  403-440 (1020) 542-579 (1014), 24     clocks fall to 2.0 GHz
//   4096 x 4096, 32 / 32, 64, none            180 (763)      221 (933)      273 (1007)
//   24 documents in 8191, 16 / 4, 64, causal  38             45             54, 8.0
//   8 x 512 x 512, 16 / 4, 64, causal         16.7           19.8           22.6, 7.4
//   3 x 333 x 1021, 6 / 2, 96, none           13.2, 7.3 join 15.8, 4.2 join 20.0, 4.9
//   4 x 1 x 2000, 16 / 4, 64                  6.2, 4.4 join
// At d_head 64 the exponentials and the other vector work fill half of the issue slots beside the products (matrix cores
// busy 56 % of attn_dkv's time, vector units 51 %).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mslayers.h"
#include "attn_tiles.h"
#include "internal.h"

namespace msa {

// Rows of an LDS tile of q and dout
template <int DP>
constexpr int tile_rows() { return DP <= 64 ? 64 : 32; }

struct View {
  const uint16_t* p;
  int64_t seq, row, head;   // strides in elements
};

struct Args {
  View q, k, v, dout;
  const uint16_t* o;
  const int32_t* seqs;
  int n_seqs, q_len, k_len;
  int H, KV, g, D, causal;
  uint32_t g_magic;         // r / g = umulhi(2 r, g_magic) >> g_shift for r < 2^30 (see magic())
  int g_shift;
  float c, scale;
  int splits;               // forward: of the keys
  int64_t groups, blocks;   // workgroups of rows; blocks of 128 keys of all sequences (see Parts)
  int row_slots, key_slots;
  int tile_rows, head_parts, row_parts, chunk;   // dK and dV: see KeyPart
  int64_t q_rows, k_rows;
  uint16_t *out, *dq, *dk, *dv;
  uint8_t* low;             // what the rounding to bf16 took off each value of out (low_byte()), or null
  float* lse;
  float* stats;             // backward: (-lse / c, -D) of every row, in the order of lse
  float* part;              // see Parts
};

// Parts.  What the splits of the keys leave of a row, and what the parts of a key block leave of its dK and dV, lies workgroup by
// workgroup: row r of workgroup x at x row_slots + r % 128, key k of block i (as attn_sum_parts counts them) at i key_slots +
// k % 128; the slots are 128, or as many as the longest sequence has.  So they take the memory of what the sequences hold, not
// of the tensors' rows: 1 MB for a new row in each of 16 x 4096 padded ones, 32 / 8 heads of 128 over 4096 keys (4.3 GB by the
// tensors' rows).  The rows' take 68 MB at most, as splits times workgroups stay below 4 kCus, the keys' 1 GB (plan()).
//   forward: [splits][groups row_slots][D], then [splits][groups row_slots] logsumexps; dQ: [splits][groups row_slots][D]
//   dK and dV: [2][parts][blocks key_slots][KV][D]

struct Seq {
  int qs, qn, ks, kn;
};

// Which sequence a workgroup works on.  Sequences of one shape: the same number of jobs each, a sequence's in a stride of `n_seqs`
// (the jobs of all sequences with the most work come first).  Otherwise the first job of each of up to kMostSeqs sequences, as
// the host has counted them (it has their lengths; 1 KB of kernel arguments): the longest's number of jobs for each, of which
// the others' are empty, takes 60, 73 and 109 us for the three kernels in place of 37, 44 and 62 at 24 documents of 3 to 1596
// rows (with the parts of that time).  More sequences: launches of that many, and one of the longest's jobs for each from where that
// leaves few empty (uniform_from()).
constexpr int kMostSeqs = 256;
struct Jobs {
  int counted;              // sequences in `first`, or 0
  int32_t first[kMostSeqs];
};

__device__ __forceinline__ Seq sequence(const Args& p, int b) {
  if (!p.seqs) return {b * p.q_len, p.q_len, b * p.k_len, p.k_len};
  const int4 x = reinterpret_cast<const int4*>(p.seqs)[b];
  const Seq s = {__builtin_amdgcn_readfirstlane(x.x), __builtin_amdgcn_readfirstlane(x.y), __builtin_amdgcn_readfirstlane(x.z),
                 __builtin_amdgcn_readfirstlane(x.w)};
  // (the host has checked its own numbers; a device table that has been overwritten since must not lead out of the rows)
  const bool ok = s.qs >= 0 && s.qn >= 0 && s.ks >= 0 && s.kn >= 0 && s.qn <= p.q_len && s.kn <= p.k_len &&
                  s.qs <= p.q_rows - s.qn && s.ks <= p.k_rows - s.kn;
  return ok ? s : Seq{0, 0, 0, 0};
}

// The first element of row 0, head `head` of sequence b, whose rows start at `start`.
__device__ __forceinline__ const uint16_t* origin(const Args& p, const View& v, int b, int start, int head) {
  return v.p + (p.seqs ? int64_t(start) * v.row : int64_t(b) * v.seq) + int64_t(head) * v.head;
}

__device__ __forceinline__ int div_g(const Args& p, int r) {
  return div_by(r, p.g_magic, p.g_shift);
}

// x is to 2^-15 what a = bf16(x) and this byte say together: the upper eight of the sixteen bits by which x's differ from a's.
// The rounding is to nearest, so the difference lies in [-0x8000, 0x8000] and its upper byte is a signed one but for the
// upper end, a tie that is rounded down (means of two or four values often are one): that takes the largest byte, which is
// off by 0x100 of x's bits as any other may be.
__device__ __forceinline__ uint32_t low_byte(float x, uint32_t a) {
  return uint32_t(min(int32_t(__float_as_uint(x) - (a << 16)), 0x7fff)) >> 8 & 0xff;
}
__device__ __forceinline__ float with_low(uint32_t a, uint32_t byte) {
  return __uint_as_float((a << 16) + uint32_t(int32_t(byte << 24) >> 16));
}
// the bytes of four values and their two bf16 pairs
__device__ __forceinline__ uint32_t low_bytes(float x0, float x1, float x2, float x3, uint32_t a01, uint32_t a23) {
  return low_byte(x0, a01 & 0xffff) | low_byte(x1, a01 >> 16) << 8 | low_byte(x2, a23 & 0xffff) << 16 | low_byte(x3, a23 >> 16) << 24;
}

template <int DP, class F>
__device__ __forceinline__ void store_low(uint8_t* stage, const f32x16 (&acc)[DP / 32], float by, int D, int lane, F dst) {
  constexpr int P = DP + 8, C = DP / 8;   // (the eight spread the rows over the banks)
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x0 = acc[b][4 * q] * by, x1 = acc[b][4 * q + 1] * by, x2 = acc[b][4 * q + 2] * by, x3 = acc[b][4 * q + 3] * by;
      *reinterpret_cast<uint32_t*>(stage + (lane & 31) * P + 32 * b + 8 * q + 4 * (lane >> 5)) =
          low_bytes(x0, x1, x2, x3, pack2(x0, x1), pack2(x2, x3));
    }
  wave_lds_order();
#pragma unroll
  for (int u = 0; u < 32 * C / 64; ++u) {
    const int i = lane + 64 * u, r = i / C, c = i % C;
    const u32x2 x = *reinterpret_cast<const u32x2*>(stage + r * P + 8 * c);
    uint8_t* to = dst(r);
    if (to && 8 * c < D) *reinterpret_cast<u32x2*>(to + 8 * c) = x;
  }
  wave_lds_order();
}

// The sequence that job i belongs to, and its number among that sequence's jobs
__device__ __forceinline__ int job_sequence(const Args& p, const Jobs& jobs, int i, int& local, int lane) {
  if (!jobs.counted) {
    local = i / p.n_seqs;
    return i % p.n_seqs;
  }
  int b = -1;   // one less than the number of sequences that begin at or before i
#pragma unroll
  for (int k = 0; k < kMostSeqs; k += 64)
    if (k < jobs.counted) b += __popcll(__ballot(k + lane < jobs.counted && jobs.first[k + lane] <= i));
  b = __builtin_amdgcn_readfirstlane(b);
  local = i - jobs.first[b];
  return b;
}

// (P and dS are rounded to bf16 as operands of the next product, to nearest: what f32 sums of bf16 operands allow.)

// What a workgroup of row tiles works on: 32 rows a wave, the keys in tiles
struct RowJob {
  Seq s;
  int b, kvh, rows, r;      // r: this lane's row
  bool ok;                  // it exists
  int pos, head;            // its position and query head
  int seen;                 // keys it sees
  int wave_full, wave_end;  // keys that every row of the wave sees, that some row sees
  int t0, t1;               // key tiles of this split
};

__device__ __forceinline__ bool row_job(const Args& p, const Jobs& jobs, RowJob& j, int lane, int wv) {
  j.kvh = blockIdx.x % p.KV;
  int local;
  j.b = job_sequence(p, jobs, blockIdx.x / p.KV, local, lane);
  j.s = sequence(p, j.b);
  j.rows = j.s.qn * p.g;
  constexpr int kRowsWg = 32 * kWaves;
  const int r0 = ((j.rows + kRowsWg - 1) / kRowsWg - 1 - local) * kRowsWg;   // the longest key ranges first
  if (r0 < 0) return false;
  j.r = r0 + 32 * wv + (lane & 31);
  j.ok = j.r < j.rows;
  j.pos = div_g(p, min(j.r, j.rows - 1));
  j.head = j.kvh * p.g + (j.ok ? j.r - j.pos * p.g : 0);
  const int last = j.s.kn - j.s.qn + 1;   // keys that position 0 sees
  j.seen = p.causal ? min(max(last + j.pos, 0), j.s.kn) : j.s.kn;
  const int w0 = min(r0 + 32 * wv, j.rows - 1), w1 = min(r0 + 32 * wv + 31, j.rows - 1), wg = min(r0 + kRowsWg, j.rows) - 1;
  auto seen_by = [&](int r) { return p.causal ? min(max(last + div_g(p, r), 0), j.s.kn) : j.s.kn; };
  j.wave_full = seen_by(w0);
  j.wave_end = seen_by(w1);
  const int n = (seen_by(wg) + kKeys - 1) / kKeys;
  const int per = n / p.splits, more = n % p.splits, y = blockIdx.y;
  j.t0 = per * y + min(y, more);
  j.t1 = j.t0 + per + (y < more);
  return true;
}

// Where a row's statistics lie: sequence by sequence, head by head
__device__ __forceinline__ int64_t stat_index(const Args& p, const RowJob& j) {
  return int64_t(j.s.qs) * p.H + int64_t(j.head) * j.s.qn + j.pos;
}

// Row `row` of a sequence's H qn, by K/V heads: where it lies and where its parts do
struct JoinRow {
  bool ok;
  int pos, head;
  int64_t slot;
};
__device__ __forceinline__ JoinRow join_row(const Args& p, const Jobs& jobs, const Seq& s, int b, int64_t row) {
  const int n = s.qn * p.g;
  JoinRow j{};
  if (row >= int64_t(n) * p.KV) return j;
  const int kvh = int(row) / n, r = int(row) - kvh * n, local = (n - 1) / (32 * kWaves) - r / (32 * kWaves);   // (see row_job)
  j.pos = div_g(p, r);
  j.head = kvh * p.g + r - j.pos * p.g;
  const int64_t x = (jobs.counted ? jobs.first[b] + local : int64_t(local) * p.n_seqs + b) * p.KV + kvh;
  j.ok = x < p.groups;   // (else a device table that has been overwritten: the host has counted fewer rows)
  j.slot = x * p.row_slots + r % (32 * kWaves);
  return j;
}

// ---- forward ----
// Per 32 keys: the scores' maximum; the probabilities, while the matrix cores form the next 32 keys' scores; then their
// product with V.  So the scores run 32 keys ahead, K one tile ahead of V: three K buffers and two of V, one barrier a tile.
// The running maximum may lag by 2^8 before the sums are rescaled: most tiles then need no pass over the output.
template <int DP>
__global__ __launch_bounds__(64 * kWaves, DP <= 64 ? 3 : 2) void attn_fwd(Args p, Jobs jobs) {
  constexpr int P = pitch<DP>(), TILE = kKeys * P;
  __shared__ __attribute__((aligned(16))) uint8_t lds[5 * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  RowJob j;
  if (!row_job(p, jobs, j, lane, wv)) return;
  const uint16_t* kb = origin(p, p.k, j.b, j.s.ks, j.kvh);
  const uint16_t* vb = origin(p, p.v, j.b, j.s.ks, j.kvh);
  Tile<DP, kKeys> kt, vt;
  kt.init(p.k.row, p.D, lane, wv);
  vt.init(p.v.row, p.D, lane, wv);
  auto load_k = [&](uint8_t* to, int t) { kt.load(to, kb + int64_t(t) * kKeys * p.k.row, j.s.kn - t * kKeys, wv); };
  auto load_v = [&](uint8_t* to, int t) { vt.load(to, vb + int64_t(t) * kKeys * p.v.row, j.s.kn - t * kKeys, wv); };
  uint8_t *k0 = lds, *k1 = lds + TILE, *k2 = lds + 2 * TILE, *v0 = lds + 3 * TILE, *v1 = lds + 4 * TILE;
  if (j.t0 < j.t1) {
    load_k(k0, j.t0);
    load_v(v0, j.t0);
    load_k(k1, j.t0 + 1);
  }
  bf16x8 q[DP / 16];
  row_operands<DP>(q, origin(p, p.q, j.b, j.s.qs, 0), int64_t(j.pos) * p.q.row + int64_t(j.head) * p.q.head, j.ok, p.D, lane);

  f32x16 o[DP / 32] = {};
  float m = -INFINITY, l = 0;   // running maximum of c s, up to 2^8 too small; sum of 2^(c s - m) over this lane's keys

  auto scores = [&](const uint8_t* K, int row0) {
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = mfma(rows_operand<P>(K, row0, ks, lane), q[ks], s);
    return s;
  };
  // s: the scores of 32 keys from key0, which lie from row0 of V; next: where the next 32 keys' K rows lie
  auto step = [&](f32x16& s, f32x16& ahead, const uint8_t* V, int row0, int key0, const uint8_t* next, int next_row0) {
    if (key0 + 32 > j.wave_full) {   // the diagonal or the end
      const int left = j.seen - key0 - 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + (i & 3) >= left) s[i] = -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top = fmaxf(top, swap_halves(top)) * p.c;
    if (__any(top > m + 8.0f)) {   // rescaling by less than 2^8 can wait: f32 sums and bf16 P keep their precision
      const float mn = fmaxf(m, top), by = mn == -INFINITY ? 1.0f : exp2_hw(m - mn);
      m = mn;
      l *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) o[d] *= by;
    }
    const float sub = m == -INFINITY ? 0.0f : m;
    ahead = scores(next, next_row0);
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2_hw(fmaf(s[i], p.c, -sub));
      sum += s[i];
    }
    l += sum;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x8 pr = pack8(s, 8 * h);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) o[d] = mfma(cols_operand<P>(V, row0 + 16 * h, d, lane), pr, o[d]);
    }
  };

  f32x16 s0, s1;
  dma_wait();
  __syncthreads();
  if (j.t0 < j.t1) s0 = scores(k0, 0);
  for (int t = j.t0; t < j.t1; ++t) {
    if (t + 1 < j.t1) {
      load_k(k2, t + 2);
      load_v(v1, t + 1);
    }
    const int key0 = t * kKeys;
    if (key0 < j.wave_end) {
      step(s0, s1, v0, 0, key0, k0, 32);
      step(s1, s0, v0, 32, key0 + 32, k1, 0);
    }
    uint8_t* k = k0;
    k0 = k1;
    k1 = k2;
    k2 = k;
    uint8_t* v = v0;
    v0 = v1;
    v1 = v;
    dma_wait();
    __syncthreads();
  }
  l += swap_halves(l);
  const float by = l == 0 ? 0.0f : 1.0f / l;   // (a NaN sum stays one)
  const float lse = l == 0 ? INFINITY : m + __log2f(l);   // +inf: 2^(c s - lse) is 0 for a row that sees nothing
  if (p.splits > 1) {   // normalised part and its weight, joined by attn_join
    if (j.ok) {
      const int64_t slots = p.groups * p.row_slots, row = blockIdx.y * slots + int64_t(blockIdx.x) * p.row_slots + 32 * wv + (lane & 31);
      float* to = p.part + row * p.D;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = 32 * d + 8 * u + 4 * (lane >> 5);
          if (c < p.D)
            *reinterpret_cast<f32x4*>(to + c) = f32x4{o[d][4 * u] * by, o[d][4 * u + 1] * by, o[d][4 * u + 2] * by, o[d][4 * u + 3] * by};
        }
      if (lane < 32) p.part[p.splits * slots * p.D + row] = lse;
    }
    return;
  }
  if (p.lse && j.ok && lane < 32) p.lse[stat_index(p, j)] = lse;
  const int r0 = j.r - (lane & 31);
  auto at = [&](int r) -> int64_t {
    if (r0 + r >= j.rows) return -1;
    const int pos = div_g(p, r0 + r);
    return (int64_t(j.s.qs + pos) * p.H + j.kvh * p.g + (r0 + r - pos * p.g)) * p.D;
  };
  store_rows<DP>(lds + wv * 32 * P, o, by, p.D, lane, [&](int r) { return at(r) < 0 ? nullptr : p.out + at(r); });
  if (p.low) store_low<DP>(lds + wv * 32 * P, o, by, p.D, lane, [&](int r) { return at(r) < 0 ? nullptr : p.low + at(r); });
}

// A row from its parts over the splits, weighted by 2^(lse_z - lse).  16 lanes a row's 8-value pieces (as many as it has), G
// of them in turn over the splits, joined through LDS in order; 16 / G rows a workgroup.  A few rows are bound by latency, and
// more lanes share a row's splits: 16 for more than 8 splits (32 rows of 64 splits, d_head 128: 8.9 us, with 4 lanes
// 20), 4 for more than 4 (2400 x 16 rows: 15 us, with 16 lanes 43), else 1 (3200 x 16 rows of two splits: 13.8 us, with 4 lanes 20).
constexpr int kJoinLanes = 256;
template <int G>
__global__ __launch_bounds__(kJoinLanes) void attn_join(Args p, Jobs jobs) {
  __shared__ float lds[kJoinLanes][11];
  const int tid = threadIdx.x, c = tid % 16, zg = tid / 16 % G;
  const Seq s = sequence(p, blockIdx.y);
  const int64_t n = p.groups * p.row_slots;
  const JoinRow j = join_row(p, jobs, s, blockIdx.y, int64_t(blockIdx.x) * (kJoinLanes / 16 / G) + tid / 16 / G);
  const bool ok = j.ok && 8 * c < p.D;
  const float* w = p.part + p.splits * n * p.D;
  float m = -INFINITY, l = 0, acc[8] = {};
  if (ok)
#pragma unroll 2
    for (int z = zg; z < p.splits; z += G) {
      const float x = w[z * n + j.slot];
      const float* from = p.part + (z * n + j.slot) * p.D + 8 * c;
      const f32x4 a = *reinterpret_cast<const f32x4*>(from), b = *reinterpret_cast<const f32x4*>(from + 4);
      if (x == INFINITY) continue;   // nothing seen in this part
      const float mn = fmaxf(m, x), old = exp2_hw(m - mn), e = exp2_hw(x - mn);   // (a NaN stays one through e)
      m = mn;
      l = fmaf(l, old, e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i] = fmaf(acc[i], old, e * a[i]);
        acc[4 + i] = fmaf(acc[4 + i], old, e * b[i]);
      }
    }
  lds[tid][0] = m;
  lds[tid][1] = l;
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[tid][2 + i] = acc[i];
  __syncthreads();
  if (zg || !ok) return;
  m = -INFINITY;
#pragma unroll
  for (int g = 0; g < G; ++g) m = fmaxf(m, lds[tid + 16 * g][0]);
  l = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float* x = lds[tid + 16 * g];
    const float e = x[1] == 0 ? 0.0f : exp2_hw(x[0] - m);
    l = fmaf(e, x[1], l);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(e, x[2 + i], acc[i]);
  }
  const float by = l == 0 ? 0.0f : 1.0f / l;
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2(acc[2 * i] *= by, acc[2 * i + 1] *= by);
  const int64_t to = (int64_t(s.qs + j.pos) * p.H + j.head) * p.D + 8 * c;
  *reinterpret_cast<u32x4*>(p.out + to) = x;
  if (p.low)
    *reinterpret_cast<u32x2*>(p.low + to) = u32x2{low_bytes(acc[0], acc[1], acc[2], acc[3], x[0], x[1]),
                                                  low_bytes(acc[4], acc[5], acc[6], acc[7], x[2], x[3])};
  if (p.lse && c == 0) p.lse[int64_t(s.qs) * p.H + int64_t(j.head) * s.qn + j.pos] = l == 0 ? INFINITY : m + __log2f(l);
}

// ---- backward ----
// dQ of 32 rows a wave; also D_i = dO_i.O_i, which attn_dkv reads beside lse.  Two workgroups a CU; operands read ahead by
// hand, as attn_dkv does, cost a wave's registers here and were slower.
template <int DP>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_dq(Args p, Jobs jobs) {
  constexpr int P = pitch<DP>(), TILE = kKeys * P;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  RowJob j;
  if (!row_job(p, jobs, j, lane, wv)) return;
  const uint16_t* kb = origin(p, p.k, j.b, j.s.ks, j.kvh);
  const uint16_t* vb = origin(p, p.v, j.b, j.s.ks, j.kvh);

  Tile<DP, kKeys> kt, vt;
  kt.init(p.k.row, p.D, lane, wv);
  vt.init(p.v.row, p.D, lane, wv);
  auto load = [&](uint8_t* to, int t) {
    kt.load(to, kb + int64_t(t) * kKeys * p.k.row, j.s.kn - t * kKeys, wv);
    vt.load(to + TILE, vb + int64_t(t) * kKeys * p.v.row, j.s.kn - t * kKeys, wv);
  };
  if (j.t0 < j.t1) load(lds, j.t0);
  bf16x8 q[DP / 16], dO[DP / 16];
  row_operands<DP>(q, origin(p, p.q, j.b, j.s.qs, 0), int64_t(j.pos) * p.q.row + int64_t(j.head) * p.q.head, j.ok, p.D, lane);
  row_operands<DP>(dO, origin(p, p.dout, j.b, j.s.qs, 0), int64_t(j.pos) * p.dout.row + int64_t(j.head) * p.dout.head, j.ok,
                   p.D, lane);
  float delta = 0;
  {
    const int64_t at = (int64_t(j.s.qs + j.pos) * p.H + j.head) * p.D;
    bf16x8 o[DP / 16];
    row_operands<DP>(o, p.o, at, j.ok, p.D, lane);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int c = 16 * ks + 8 * (lane >> 5);
      u32x2 low{};
      if (p.low && j.ok && c < p.D) low = *reinterpret_cast<const u32x2*>(p.low + at + c);
      const u32x4 bits = __builtin_bit_cast(u32x4, o[ks]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        delta = fmaf(with_low(bits[i >> 1] >> (16 * (i & 1)) & 0xffff, low[i >> 2] >> (8 * (i & 3)) & 0xff), float(dO[ks][i]), delta);
    }
  }
  delta += swap_halves(delta);
  const float lse = j.ok ? p.lse[stat_index(p, j)] : INFINITY;
  if (j.ok && lane < 32 && blockIdx.y == 0) *reinterpret_cast<f32x2*>(p.stats + 2 * stat_index(p, j)) = f32x2{-lse / p.c, -delta};

  f32x16 dq[DP / 32] = {};
  dma_wait();
  __syncthreads();
  for (int t = j.t0; t < j.t1; ++t) {
    uint8_t* K = lds + ((t - j.t0) & 1) * 2 * TILE;
    const uint8_t* V = K + TILE;
    uint8_t* next = lds + ((t - j.t0 + 1) & 1) * 2 * TILE;
    if (t + 1 < j.t1) load(next, t + 1);
    const int key0 = t * kKeys;
    if (key0 < j.wave_end) {
      const bool edge = key0 + kKeys > j.wave_full;
      const int left = j.seen - key0 - 4 * (lane >> 5);
#pragma unroll
      for (int b = 0; b < kKeys / 32; ++b) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          s = mfma(rows_operand<P>(K, 32 * b, ks, lane), q[ks], s);
          dp = mfma(rows_operand<P>(V, 32 * b, ks, lane), dO[ks], dp);
        }
        if (edge)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * b + 8 * (i >> 2) + (i & 3) >= left) s[i] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = exp2_hw(fmaf(s[i], p.c, -lse)) * (dp[i] - delta);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 ds = pack8(s, 8 * h);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) dq[d] = mfma(cols_operand<P>(K, 32 * b + 16 * h, d, lane), ds, dq[d]);
        }
      }
    }
    dma_wait();
    __syncthreads();
  }
  if (p.splits > 1) {   // a part, joined by attn_join_dq
    float* to = p.part + ((blockIdx.y * p.groups + blockIdx.x) * p.row_slots + 32 * wv + (lane & 31)) * p.D;
    if (j.ok)
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = 32 * d + 8 * u + 4 * (lane >> 5);
          if (c < p.D) *reinterpret_cast<f32x4*>(to + c) = f32x4{dq[d][4 * u], dq[d][4 * u + 1], dq[d][4 * u + 2], dq[d][4 * u + 3]};
        }
    return;
  }
  const int r0 = j.r - (lane & 31);
  store_rows<DP>(lds + wv * 32 * P, dq, p.scale, p.D, lane, [&](int r) -> uint16_t* {
    if (r0 + r >= j.rows) return nullptr;
    const int pos = div_g(p, r0 + r);
    return p.dq + (int64_t(j.s.qs + pos) * p.H + j.kvh * p.g + (r0 + r - pos * p.g)) * p.D;
  });
}

// dQ as the sum of its parts over the splits, in order: 8 values a thread, of the rows of a sequence
__global__ __launch_bounds__(256) void attn_join_dq(Args p, Jobs jobs) {
  const Seq s = sequence(p, blockIdx.y);
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / (uint32_t(p.D) / 8), c = i - row * (uint32_t(p.D) / 8);
  const JoinRow j = join_row(p, jobs, s, blockIdx.y, row);
  if (!j.ok) return;
  const int64_t n = p.groups * p.row_slots;
  const float* from = p.part + j.slot * p.D + 8 * c;
  f32x4 x = {}, y = {};
#pragma unroll 4
  for (int z = 0; z < p.splits; ++z) {
    x += *reinterpret_cast<const f32x4*>(from + z * n * p.D);
    y += *reinterpret_cast<const f32x4*>(from + z * n * p.D + 4);
  }
  x *= p.scale;
  y *= p.scale;
  *reinterpret_cast<u32x4*>(p.dq + (int64_t(s.qs + j.pos) * p.H + j.head) * p.D + 8 * c) =
      u32x4{pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(y[0], y[1]), pack2(y[2], y[3])};
}

// Row tiles of R rows (of one head) that see a key of the 128 of block kb: [first, first + n)
__device__ __forceinline__ int row_tiles(const Args& p, const Seq& s, int kb, int& first) {
  first = p.causal ? min(max(128 * kb - (s.kn - s.qn), 0), s.qn) / p.tile_rows : 0;
  return (s.qn + p.tile_rows - 1) / p.tile_rows - first;
}

// The work on 128 keys: the row tiles of the group's heads, head by head.  The heads are shared out to p.head_parts parts,
// each part's list of tiles to parts of p.chunk of them: at most p.row_parts, here `parts`.
struct KeyPart {
  int n, first;   // row tiles a head
  int t0, t1, parts;
};
__device__ __forceinline__ KeyPart key_part(const Args& p, const Seq& s, int kb, int z, int n_heads) {
  KeyPart k;
  k.n = row_tiles(p, s, kb, k.first);
  const int n = k.n * n_heads;
  k.parts = max((n + p.chunk - 1) / p.chunk, 1);
  k.t0 = min(z * p.chunk, n);
  k.t1 = min(k.t0 + p.chunk, n);
  return k;
}

// Blocks of 128 keys that have a part z (of all heads of a group): the first ones, and every block has part 0
__host__ __device__ inline int blocks_with_part(const Seq& s, int z, int g, int tile_rows, int chunk, bool causal) {
  const int blocks = (s.kn + 127) / 128, tiles = (s.qn + tile_rows - 1) / tile_rows;
  if (z == 0) return blocks;
  const int most = tiles - (int(int64_t(z) * chunk / g) + 1);   // row tiles that may lie before the block's first
  if (most < 0) return 0;
  const int64_t end = int64_t(most + 1) * tile_rows;            // the block's first row lies before it
  if (!causal || end > s.qn) return blocks;
  const int64_t keys = end + s.kn - s.qn;                       // 128 kb - (kn - qn) < end
  return keys <= 0 ? 0 : int(keys + 127) / 128 < blocks ? int(keys + 127) / 128 : blocks;
}

// The way through the row tiles of a part, from the last rows to the first, head by head: where the next tile
// lies.  Workgroups of one K/V head start on the same rows and so share them in L2.
template <int DP>
struct RowStream {
  static constexpr int R = tile_rows<DP>();
  const uint16_t *q, *dout;
  const float* stats;
  int row0, left, before;   // its first row; tiles still to come, it included; tiles of its head before it
  __device__ __forceinline__ void start(const Args& p, const KeyPart& w, const Seq& s, const uint16_t* q0, const uint16_t* d0,
                                        const float* stats0) {
    const int t = w.t0, n = max(w.n, 1), head = t / n;
    left = w.t1 - t;
    before = n - 1 - t % n;
    row0 = (w.first + before) * R;
    q = q0 + int64_t(head) * p.q.head + int64_t(row0) * p.q.row;
    dout = d0 + int64_t(head) * p.dout.head + int64_t(row0) * p.dout.row;
    stats = stats0 + 2 * (int64_t(head) * s.qn + row0);
  }
  __device__ __forceinline__ void advance(const Args& p, const KeyPart& w, const Seq& s) {
    --left;
    row0 -= R;
    q -= R * p.q.row;
    dout -= R * p.dout.row;
    stats -= 2 * R;
    if (--before < 0) {   // to the next head's last rows
      const int n = w.n;
      before += n;
      row0 += n * R;
      q += int64_t(n * R) * p.q.row + p.q.head;
      dout += int64_t(n * R) * p.dout.row + p.dout.head;
      stats += 2 * (n * R + s.qn);
    }
  }
};

// dK and dV of 128 keys, 32 a wave, head by head over the rows that see them, from the last rows: workgroups of one K/V head
// run on one XCD's L2 over the same rows (the group's heads row by row, each workgroup from its own first row: 1079 us in
// place of 675 at the long case, as the kernel was then).  Part by part, block by block, so that whole parts start before the
// rests of blocks (block by block: 97 us in place of 74 at 2400 rows of heads of 128).  Two workgroups a CU, so that one's
// first loads and last stores (8 us together) are behind the other's products; eight waves a workgroup, one a CU, expose
// them.  Heads of 97 to 128 need four registers more than the 256 of two waves a SIMD: three are kept in scratch over the loop; one,
// which the diagonal's mask takes, is read back there, where the wait for it is one for the tile on its way too.
template <int DP>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void attn_dkv(Args p, Jobs jobs, Jobs sums) {
  constexpr int P = pitch<DP>(), R = tile_rows<DP>(), TILE = R * P, STAGE = 2 * TILE + 8 * R, S = DP <= 64 ? 3 : 2, SUB = R / 32;
  constexpr int DB = DP / 32, LOADS = 2 * TILE / 1024 / kWaves + 1;   // of a wave and stage
  __shared__ __attribute__((aligned(16))) uint8_t lds[S * STAGE + 128 * P];
  static_assert(sizeof(lds) <= 80 * 1024 && S * STAGE >= kWaves * 32 * P, "two workgroups a CU; the results' staging");
  uint8_t* vs = lds + S * STAGE;   // the workgroup's V rows: in registers they would spill
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the first keys, which the most rows see, first
  int b, kvh, kb, zh = 0, zr;
  if (jobs.counted) {   // part by part, block by block
    kvh = blockIdx.x % p.KV;
    b = job_sequence(p, jobs, blockIdx.x / p.KV, kb, lane);
  } else {   // likewise; workgroups of the same rows are all = n_seqs * KV * head_parts apart: a multiple of 8 is one XCD
    const int all = p.n_seqs * p.KV * p.head_parts, blocks = (p.k_len + 127) / 128, id = blockIdx.x % all;
    kb = blockIdx.x / all % blocks;
    zr = blockIdx.x / all / blocks;
    zh = id / (p.n_seqs * p.KV);
    b = id / p.KV % p.n_seqs;
    kvh = id % p.KV;
  }
  const Seq s = sequence(p, b);
  if (jobs.counted) {
    zr = 0;
    for (int n; kb >= (n = blocks_with_part(s, zr, p.g, p.tile_rows, p.chunk, p.causal)) && zr < p.row_parts; ++zr) kb -= n;
  }
  const int parts = p.head_parts * p.row_parts, z = zh * p.row_parts + zr;
  const int h0 = zh * p.g / p.head_parts, n_heads = (zh + 1) * p.g / p.head_parts - h0;
  if (128 * kb >= s.kn) return;
  const KeyPart w = key_part(p, s, kb, zr, n_heads);
  if (zr >= w.parts) return;   // (a block that no row sees has one, which writes its zeros)
  const int last = s.kn - s.qn + 1;
  const uint16_t* qb = origin(p, p.q, b, s.qs, kvh * p.g + h0);
  const uint16_t* db = origin(p, p.dout, b, s.qs, kvh * p.g + h0);
  const float* sb = p.stats + 2 * (int64_t(s.qs) * p.H + int64_t(kvh * p.g + h0) * s.qn);
  const int k0 = 128 * kb + 32 * wv, key = k0 + (lane & 31);
  const bool ok = key < s.kn;
  bf16x8 k[DP / 16];
  row_operands<DP>(k, origin(p, p.k, b, s.ks, kvh), int64_t(key) * p.k.row, ok, p.D, lane);
  Tile<DP, 128> vt;
  vt.init(p.v.row, p.D, lane, wv);
  vt.load(vs, origin(p, p.v, b, s.ks, kvh) + int64_t(128 * kb) * p.v.row, s.kn - 128 * kb, wv);
  Tile<DP, R> qt, dt;
  qt.init(p.q.row, p.D, lane, wv);
  dt.init(p.dout.row, p.D, lane, wv);
  // the (-lse / c, -D) pairs of a tile's rows as two rows of R: 64 lanes fetch one of them, or both of 32
  const int stat_row = lane & (R - 1), stat_plane = R == 64 ? wv & 1 : lane >> 5;

  f32x16 dk[DB] = {}, dv[DB] = {};
  RowStream<DP> rs;
  rs.start(p, w, s, qb, db, sb);
  int slot_next = 0, slot = 0;
  auto load = [&]() {   // (past the last tile too, of zeros: every stage is the same number of loads)
    uint8_t* to = lds + slot_next * STAGE;
    const int n = rs.left > 0 ? s.qn - rs.row0 : 0;
    qt.load(to, rs.q, n, wv);
    dt.load(to + TILE, rs.dout, n, wv);
    dma4(rs.stats, stat_row < n ? 8 * stat_row + 4 * stat_plane : kOutside, lds_address(to + 2 * TILE) + (R == 64 ? 256 * (wv & 1) : 0));
    rs.advance(p, w, s);
    slot_next = slot_next + 1 == S ? 0 : slot_next + 1;
  };
  int rows[S - 1];   // the first rows of the tiles on their way
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    rows[i] = rs.row0;
    load();
  }
  dma_wait();   // (for k, so that the compiler does not wait for all loads in the loop)
  for (int t = w.t0; t < w.t1; ++t) {
    // this wave's loads of the tile have landed; behind the barrier everyone's have, and the tile before is done with
    dma_wait<(S - 2) * LOADS>();
    __syncthreads();
    const uint8_t* Q = lds + slot * STAGE;
    const uint8_t* dO = Q + TILE;
    const float* stats = reinterpret_cast<const float*>(Q + 2 * TILE);
    const int row0 = rows[0];
#pragma unroll
    for (int i = 0; i + 1 < S - 1; ++i) rows[i] = rows[i + 1];
    rows[S - 2] = rs.row0;
    load();
    slot = slot + 1 == S ? 0 : slot + 1;

    // The tile's products as a list of steps of W LDS operands; the operands of step n + 1 are on their way while step n
    // multiplies (left to itself the compiler waits for each operand in turn).
    constexpr int W = DP <= 64 ? 4 : 2, KS = DP / 16, SG = KS % W ? 2 : W, PG = W / 2, DG = DB % (W / 2) ? 1 : W / 2;
    constexpr int M1 = KS / SG, M2 = KS / PG, M3 = 2 * DB / DG, N1 = SUB * M1, N2 = N1 + SUB * M2, N3 = N2 + SUB * M3;
    bf16x8 f[2][W], pr[SUB][2], ds[SUB][2];
    f32x16 sc[SUB], dp[SUB];   // they start as -lse / c and -D, row by row
    auto read = [&](int n) {
      bf16x8(&to)[W] = f[n & 1];
      if (n < N1) {
        const int a = n / M1, i0 = n % M1 * SG;
#pragma unroll
        for (int i = 0; i < SG; ++i) to[i] = rows_operand<P>(Q, 32 * a, i0 + i, lane);
      } else if (n < N2) {
        const int a = (n - N1) / M2, i0 = (n - N1) % M2 * PG;
#pragma unroll
        for (int i = 0; i < PG; ++i) {
          to[2 * i] = rows_operand<P>(dO, 32 * a, i0 + i, lane);
          to[2 * i + 1] = rows_operand<P>(vs, 32 * wv, i0 + i, lane);
        }
      } else if (n < N3) {
        const int a = (n - N2) / M3, h = (n - N2) % M3 / (DB / DG), d = (n - N2) % (DB / DG) * DG;
#pragma unroll
        for (int i = 0; i < DG; ++i) {
          to[2 * i] = cols_operand<P>(dO, 32 * a + 16 * h, d + i, lane);
          to[2 * i + 1] = cols_operand<P>(Q, 32 * a + 16 * h, d + i, lane);
        }
      }
    };
    auto begin = [&](f32x16& x, const float* from) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(from + 8 * u + 4 * (lane >> 5));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * u + i] = y[i];
      }
    };
    begin(sc[0], stats);
    read(0);
#pragma unroll
    for (int n = 0; n < N3; ++n) {
      if (n < N2 && n + 1 < N1 && (n + 1) % M1 == 0) begin(sc[(n + 1) / M1], stats + 32 * ((n + 1) / M1));
      if (n + 1 >= N1 && n + 1 < N2 && (n + 1 - N1) % M2 == 0) begin(dp[(n + 1 - N1) / M2], stats + R + 32 * ((n + 1 - N1) / M2));
      read(n + 1);
      order_reads();
      bf16x8(&x)[W] = f[n & 1];
      if (n < N1) {
        const int a = n / M1, i0 = n % M1 * SG;
#pragma unroll
        for (int i = 0; i < SG; ++i) sc[a] = mfma(x[i], k[i0 + i], sc[a]);
      } else if (n < N2) {
        const int a = (n - N1) / M2;
#pragma unroll
        for (int i = 0; i < PG; ++i) dp[a] = mfma(x[2 * i], x[2 * i + 1], dp[a]);
      } else {
        const int a = (n - N2) / M3, h = (n - N2) % M3 / (DB / DG), d = (n - N2) % (DB / DG) * DG;
#pragma unroll
        for (int i = 0; i < DG; ++i) {
          dv[d + i] = mfma(x[2 * i], pr[a][h], dv[d + i]);
          dk[d + i] = mfma(x[2 * i + 1], ds[a][h], dk[d + i]);
        }
      }
      if (n == N1 - 1) {
        // the diagonal (rows that do not exist have q, dout, lse and D of 0 and add nothing; keys that do not exist are
        // not stored)
        if (p.causal && last + row0 < k0 + 32) {
#pragma unroll
          for (int a = 0; a < SUB; ++a) {
            const int hidden = key - last - row0 - 32 * a - 4 * (lane >> 5);   // rows up to here do not see the key
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (8 * (i >> 2) + (i & 3) <= hidden) sc[a][i] = -INFINITY;
          }
        }
#pragma unroll
        for (int a = 0; a < SUB; ++a) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[a][i] = exp2_hw(sc[a][i] * p.c);
          pr[a][0] = pack8(sc[a], 0);
          pr[a][1] = pack8(sc[a], 8);
        }
      }
      if (n >= N1 && n < N2 && (n + 1 - N1) % M2 == 0) {
        const int a = (n - N1) / M2;
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[a][i] *= sc[a][i];
        ds[a][0] = pack8(dp[a], 0);
        ds[a][1] = pack8(dp[a], 8);
      }
    }
  }
  dma_wait();
  __syncthreads();
  if (parts > 1 && (p.head_parts > 1 || w.parts > 1)) {
    const int64_t block = jobs.counted ? sums.first[b] + kb : int64_t(kb) * p.n_seqs + b;
    float* to = p.part + (((z * p.blocks + block) * p.key_slots + 32 * wv + (lane & 31)) * p.KV + kvh) * p.D;
    const int64_t all = parts * p.blocks * p.key_slots * p.KV * p.D;
    if (ok && block < p.blocks)   // (more: a device table that has been overwritten)
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = 32 * d + 8 * u + 4 * (lane >> 5);
          if (c < p.D) {
            *reinterpret_cast<f32x4*>(to + c) = f32x4{dk[d][4 * u], dk[d][4 * u + 1], dk[d][4 * u + 2], dk[d][4 * u + 3]};
            *reinterpret_cast<f32x4*>(to + all + c) = f32x4{dv[d][4 * u], dv[d][4 * u + 1], dv[d][4 * u + 2], dv[d][4 * u + 3]};
          }
        }
    return;
  }
  auto row = [&](uint16_t* base, int r) -> uint16_t* {
    return k0 + r < s.kn ? base + (int64_t(s.ks + k0 + r) * p.KV + kvh) * p.D : nullptr;
  };
  store_rows<DP>(lds + wv * 32 * P, dk, p.scale, p.D, lane, [&](int r) { return row(p.dk, r); });
  store_rows<DP>(lds + wv * 32 * P, dv, 1.0f, p.D, lane, [&](int r) { return row(p.dv, r); });
}

// dK (blockIdx.z 0) and dV of 128 keys as the sum of their parts, in order: 8 values a thread
__global__ __launch_bounds__(256) void attn_sum_parts(Args p, Jobs jobs) {
  int kb;
  const int b = job_sequence(p, jobs, blockIdx.x, kb, threadIdx.x & 63);
  const Seq s = sequence(p, b);
  const int width = p.KV * p.D, i = (blockIdx.y * 256 + threadIdx.x) * 8, row = i / width;
  if (row >= 128 || 128 * kb + row >= s.kn) return;
  const bool v = blockIdx.z;
  const int64_t n = p.blocks * p.key_slots * width, at = int64_t(s.ks + 128 * kb) * width + i;
  const float* from = p.part + (v ? p.head_parts * p.row_parts * n : 0) + int64_t(blockIdx.x) * p.key_slots * width + i;
  f32x4 x = {}, y = {};
  for (int zh = 0; zh < p.head_parts; ++zh) {
    const KeyPart w = key_part(p, s, kb, 0, (zh + 1) * p.g / p.head_parts - zh * p.g / p.head_parts);
    if (p.head_parts == 1 && w.parts == 1) return;   // written as they are
#pragma unroll 4
    for (int z = 0; z < w.parts; ++z) {
      x += *reinterpret_cast<const f32x4*>(from + (zh * p.row_parts + z) * n);
      y += *reinterpret_cast<const f32x4*>(from + (zh * p.row_parts + z) * n + 4);
    }
  }
  const float by = v ? 1.0f : p.scale;
  x *= by;
  y *= by;
  *reinterpret_cast<u32x4*>((v ? p.dv : p.dk) + at) = u32x4{pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(y[0], y[1]), pack2(y[2], y[3])};
}

// ---- host ----
// Row tiles of a part at least, half as many of a part of the heads: its K, V and results are traffic of two or three tiles.
// With 8: 25.1 us and 6.6 for the sum in place of 22.9 and 4.4 (3 x 333 x 1021)
constexpr int kLeast = 16;
// A part's row tiles, of what there is for each of two workgroups a CU.  With 1 all of them would start at once if they were
// alike; larger ones are fewer first loads and sums.  With 1, 1.5 and 2, the sum included: 72, 61 and 72 us (24 documents in
// 8191), 125, 103 and 117 (the same, heads of 128), 571, 571 and 662 (8192 rows), 128, 112 and 119 (3200 rows, heads of 128)
constexpr double kShare = 1.5;

// What a launch works on: the sequences from `first` on, with counted jobs at most kMostSeqs of them
struct Launch {
  int first, n, q_len, k_len;   // the longest of them
  int row_parts;                // of the longest's row tiles
  int64_t groups, blocks, key_groups;
  Jobs rows, keys, sums;
};
struct Plan {
  int splits, dq_splits;     // of the keys, forward and for dQ
  int uniform;               // the sequences from here on are one launch of the longest's jobs for each; those before it are counted
  int64_t groups;            // row tiles of a launch's sequences and K/V heads, at most
  int row_slots, key_slots;  // see Parts
  int64_t key_groups;        // dK and dV: workgroups of a launch, at most
  int tile_rows, head_parts, row_parts, chunk;   // see KeyPart
  int64_t blocks;            // of 128 keys, of a launch's sequences, at most
  Launch one;                // the first
};

constexpr int kCus = 256;
constexpr int64_t kMostGroups = (int64_t(1) << 32) / 256 - 1;   // a launch has fewer than 2^32 threads a dimension

Seq host_seq(const msd_attn& a, int b) {
  if (!a.seqs) return {0, a.q_len, 0, a.k_len};
  const int32_t* s = a.seqs_host + 4 * b;
  return {s[0], s[1], s[2], s[3]};
}

// Jobs of a launch's sequences, f(sequence) each; how many
template <class F>
int64_t count(const msd_attn& a, const Plan& p, const Launch& l, Jobs& jobs, F f) {
  jobs.counted = l.first < p.uniform ? l.n : 0;
  if (!jobs.counted) return int64_t(l.n) * f(Seq{0, l.q_len, 0, l.k_len});
  int64_t all = 0;
  for (int b = 0; b < l.n; ++b) {
    jobs.first[b] = int(std::min<int64_t>(all, INT32_MAX));
    all += f(host_seq(a, l.first + b));
  }
  return all;
}

int64_t row_tiles(const msd_attn& a, int qn) { return cdiv(int64_t(qn) * (a.n_heads / a.n_kv_heads), 32 * kWaves); }

void rows_and_blocks(const msd_attn& a, const Plan& p, int first, Launch& l) {
  l.first = first;
  l.n = first < p.uniform ? std::min(kMostSeqs, a.n_seqs - first) : a.n_seqs - first;
  l.q_len = a.seqs ? 0 : a.q_len;
  l.k_len = a.seqs ? 0 : a.k_len;
  for (int b = 0; a.seqs && b < l.n; ++b) {
    const Seq s = host_seq(a, first + b);
    l.q_len = std::max(l.q_len, s.qn);
    l.k_len = std::max(l.k_len, s.kn);
  }
  l.groups = a.n_kv_heads * count(a, p, l, l.rows, [&](Seq s) { return row_tiles(a, s.qn); });
  l.blocks = count(a, p, l, l.sums, [&](Seq s) { return cdiv(s.kn, 128); });
}

void key_jobs(const msd_attn& a, const Plan& p, Launch& l) {
  const int g = a.n_heads / a.n_kv_heads;
  l.row_parts = int(std::max<int64_t>(1, cdiv(cdiv(l.q_len, p.tile_rows) * cdiv(g, p.head_parts), p.chunk)));
  l.key_groups = a.n_kv_heads * count(a, p, l, l.keys, [&](Seq s) {
    if (l.first >= p.uniform) return cdiv(s.kn, 128) * p.head_parts * l.row_parts;
    int64_t all = 0;
    for (int z = 0, blocks = 1; z < l.row_parts && blocks; ++z)   // (fewer from part to part)
      all += blocks = blocks_with_part(s, z, g, p.tile_rows, p.chunk, a.causal != 0);
    return all;
  });
}

// Jobs of the longest for all sequences from `first` on are up to this many times their own jobs: one such launch then takes
// what counted launches take (512 sequences of 16 to 1024 rows, 4.0 times: 360 us and 1350 with the gradients in place of 340 and
// 1310; 4096 of 16 rows, once: 128 and 667 in place of 235 and 1024; one of 8192 rows before 299 of 64, 57 times: 653 and
// 2306 in place of 186 and 831).
constexpr int kMostEmpty = 4;

int uniform_from(const msd_attn& a) {
  if (!a.seqs) return 0;
  int from = a.n_seqs, q_len = 0, k_len = 0;
  int64_t jobs = 0;
  for (int b = a.n_seqs - 1; b >= 0; --b) {
    const Seq s = host_seq(a, b);
    q_len = std::max(q_len, s.qn);
    k_len = std::max(k_len, s.kn);
    jobs += row_tiles(a, s.qn) + cdiv(s.kn, 128);
    const int n = a.n_seqs - b;
    if (b % kMostSeqs == 0 && n > kMostSeqs && n * (row_tiles(a, q_len) + cdiv(k_len, 128)) <= kMostEmpty * jobs) from = b;
  }
  return from;
}

// f(launch) of every launch of the call, from the first; p.one is the first one's before and the last one's afterwards
template <class F>
void launches(const msd_attn& a, Plan& p, F f) {
  for (int first = 0; first < a.n_seqs; first += p.one.n) {
    if (first) {
      rows_and_blocks(a, p, first, p.one);
      key_jobs(a, p, p.one);
    }
    f(p.one);
  }
}

void plan(const msd_attn& a, Plan& p) {
  const int64_t g = a.n_heads / a.n_kv_heads;
  p.uniform = uniform_from(a);
  auto pairs = [&](Seq s) {   // rows x keys that the mask leaves, about
    const double q = s.qn, k = s.kn;
    return !a.causal ? q * k : q <= k ? q * (k - q / 2) : k * k / 2;
  };
  double all = 0;
  p.groups = p.blocks = p.key_groups = 0;
  rows_and_blocks(a, p, 0, p.one);
  for (int first = 0; first < a.n_seqs; first += p.one.n) {
    if (first) rows_and_blocks(a, p, first, p.one);
    p.groups = std::max(p.groups, p.one.groups);
    p.blocks = std::max(p.blocks, p.one.blocks);
    double sum = a.seqs ? 0 : double(a.n_seqs) * pairs(Seq{0, a.q_len, 0, a.k_len});
    for (int b = first; a.seqs && b < first + p.one.n; ++b) sum += pairs(host_seq(a, b));
    all = std::max(all, sum);
  }
  const bool several = p.one.first > 0;
  // few rows: the keys are split too, into at least 128 each (dQ, whose parts are the larger share of its work: 256), until
  // every CU has two workgroups (four: 54 + 17 us for the join in place of 44 + 8, dQ 70 + 12 in place of 58 + 7 at 2 x 512 rows
  // against 4096 keys, 16 / 4 heads of 128; row tiles for one a CU left whole: 38 us in place of 31 + 10, dQ 44 in place
  // of 38 + 6 at 2400 rows, but 75 in place of 59 + 12, dQ 94 in place of 77 + 11 at 3200 of heads of 128).  Without: one token
  // against 2000 keys 47 us in place of 6.2 and 4.4 for the join, 333 rows against 1021 keys 36 in place of 13 and 7, dQ 33 in
  // place of 16 and 4.
  const int64_t few = p.groups >= 2 * kCus ? 1 : cdiv(2 * kCus, std::max<int64_t>(p.groups, 1));
  p.splits = int(std::max<int64_t>(1, std::min(few, cdiv(a.k_len, 128))));
  p.dq_splits = int(std::max<int64_t>(1, std::min(few, cdiv(a.k_len, 256))));
  p.row_slots = int(std::min<int64_t>(a.q_len * g, 32 * kWaves));
  p.key_slots = std::min(a.k_len, 128);
  // dK and dV: parts of a key block, as many as make kShare: the heads of a group first, whose parts are alike (four heads in
  // two parts, not four: 27.2 + 5.0 us for the sum in place of 22.5 + 7.3 at 8 x 512), then the rows, as long as a part's K,
  // V and results are worth their traffic.  Of sequences in a table the heads are one list.
  p.tile_rows = a.d_head <= 64 ? tile_rows<64>() : tile_rows<128>();
  const int64_t most = cdiv(a.q_len, p.tile_rows);
  const double share = kShare * all * a.n_heads / (128.0 * p.tile_rows * 2 * kCus);
  // (a sequence far longer than the others, or one of few keys, would have more parts than their keys' share of the workspace is
  // worth: up to 8192 blocks of a part and K/V head)
  const int64_t parts = std::max<int64_t>(32 * kCus / std::max<int64_t>(cdiv(p.blocks * p.key_slots, 128) * a.n_kv_heads, 1), 1);
  p.head_parts = a.seqs ? 1 : int(std::min(double(g), std::max(1.0, ceil(double(most * g) / std::max(share, kLeast / 2.0)))));
  while (g % p.head_parts) ++p.head_parts;   // (parts of the heads are alike)
  while (p.head_parts > parts || g % p.head_parts) --p.head_parts;
  const int64_t list = most * cdiv(g, p.head_parts);   // row tiles of a head part
  p.chunk = int(std::max<int64_t>({kLeast, cdiv(list, std::max<int64_t>(parts / p.head_parts, 1)), std::min(list, int64_t(std::min(share, 1e9)) + 1)}));
  p.row_parts = int(std::max<int64_t>(1, cdiv(list, p.chunk)));
  if (several) rows_and_blocks(a, p, 0, p.one);
  key_jobs(a, p, p.one);
  launches(a, p, [&](const Launch& l) { p.key_groups = std::max(p.key_groups, l.key_groups); });
  if (several) {
    rows_and_blocks(a, p, 0, p.one);
    key_jobs(a, p, p.one);
  }
}

bool fits(const int64_t (&s)[3], int64_t heads) {
  for (int64_t x : s)
    if (x < 0 || x % 8) return false;
  constexpr int64_t most = int64_t(1) << 30;
  return s[1] <= most / 128 && s[2] <= most / heads && 128 * s[1] + heads * s[2] < most;   // (a tile of 128 rows)
}

// whether the library takes the call, and how
int32_t check(const msd_attn* a, bool backward, Plan& p) {
  if (!a) return MSD_E_ARG;
  if (a->n_seqs < 0 || a->q_len < 0 || a->k_len < 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->n_heads % a->n_kv_heads ||
      a->d_head <= 0 || a->d_head > 128 || a->d_head % 8 || !(a->scale >= 0x1p-60f) || !(a->scale <= 0x1p60f) || a->q_rows < 0 ||
      a->k_rows < 0)
    return MSD_E_CONFIG;
  const int64_t most = int64_t(1) << 31;
  if (a->q_rows >= most / 2 || a->k_rows >= most / 2 || a->q_rows * a->n_heads >= most || a->k_rows * a->n_kv_heads >= most ||
      int64_t(a->q_len) * (a->n_heads / a->n_kv_heads) >= (1 << 30) - 256 || int64_t(a->n_seqs) * a->n_kv_heads >= (1 << 20) || a->n_heads > 4096 || a->n_seqs > 65535)
    return MSD_E_CONFIG;
  if (!a->seqs && (a->q_rows != int64_t(a->n_seqs) * a->q_len || a->k_rows != int64_t(a->n_seqs) * a->k_len)) return MSD_E_CONFIG;
  if (a->q_len > a->q_rows || a->k_len > a->k_rows) return MSD_E_CONFIG;
  const int64_t g = a->n_heads / a->n_kv_heads;
  if (!fits(a->q_stride, g) || !fits(a->k_stride, 1) || !fits(a->v_stride, 1) || (backward && !fits(a->dout_stride, g)))
    return MSD_E_CONFIG;
  if (a->seqs) {
    if (reinterpret_cast<uintptr_t>(a->seqs) % 16 || !a->seqs_host || reinterpret_cast<uintptr_t>(a->seqs_host) % 4) return MSD_E_ARG;
    for (int b = 0; b < a->n_seqs; ++b) {
      const Seq s = host_seq(*a, b);
      if (s.qs < 0 || s.qn < 0 || s.ks < 0 || s.kn < 0 || s.qn > a->q_len || s.kn > a->k_len || s.qs > a->q_rows - s.qn ||
          s.ks > a->k_rows - s.kn)
        return MSD_E_CONFIG;
    }
  }
  plan(*a, p);
  return std::max(p.groups, p.key_groups) > kMostGroups || p.splits > 65535 ? MSD_E_CONFIG : MSD_OK;
}

bool bad(const void* p) { return !p || reinterpret_cast<uintptr_t>(p) % 16; }

View view(const void* p, const int64_t (&s)[3]) { return {static_cast<const uint16_t*>(p), s[0], s[1], s[2]}; }

Args args(const msd_attn& a, const Plan& pl, const void* q, const void* k, const void* v) {
  Args p{};
  p.row_slots = pl.row_slots;
  p.key_slots = pl.key_slots;
  p.q = view(q, a.q_stride);
  p.k = view(k, a.k_stride);
  p.v = view(v, a.v_stride);
  p.H = a.n_heads;
  p.KV = a.n_kv_heads;
  p.g = a.n_heads / a.n_kv_heads;
  magic(uint32_t(p.g), p.g_magic, p.g_shift);
  p.D = a.d_head;
  p.causal = a.causal != 0;
  p.scale = a.scale;
  p.c = a.scale * kLog2e;
  p.q_rows = a.q_rows;
  p.k_rows = a.k_rows;
  return p;
}

Args args(Args p, const msd_attn& a, const Launch& l) {
  p.seqs = a.seqs ? a.seqs + 4 * l.first : nullptr;
  p.n_seqs = l.n;
  p.q_len = l.q_len;
  p.k_len = l.k_len;
  p.groups = l.groups;
  p.blocks = l.blocks;
  p.row_parts = l.row_parts;
  return p;
}

int32_t launched() { return hipGetLastError() == hipSuccess ? MSD_OK : MSD_E_HIP; }

int64_t up(int64_t x) { return cdiv(x, 256) * 256; }

}  // namespace msa

using namespace msa;

extern "C" int64_t msd_attn_workspace_bytes(const msd_attn* a, int32_t backward) {
  Plan pl;
  const int32_t rc = check(a, false, pl);
  if (rc != MSD_OK) return rc;
  const int64_t slots = pl.groups * pl.row_slots;
  if (!backward) return pl.splits > 1 ? 4 * pl.splits * slots * (a->d_head + 1) : 0;
  const int64_t dq = pl.dq_splits > 1 ? up(4 * pl.dq_splits * slots * a->d_head) : 0;
  const int64_t n = pl.head_parts * pl.row_parts;
  const int64_t parts = n > 1 ? 8 * n * pl.blocks * pl.key_slots * a->n_kv_heads * a->d_head : 0;
  return up(8 * a->q_rows * a->n_heads) + std::max(dq, parts);   // (one after the other)
}

extern "C" int32_t msd_attn_forward(const msd_attn* a, const void* q, const void* k, const void* v, void* out, void* out_low,
                                    float* lse, void* workspace, void* stream) {
  Plan pl;
  const int32_t rc = check(a, false, pl);
  if (rc != MSD_OK) return rc;
  if (a->n_seqs == 0 || a->q_len == 0) return MSD_OK;
  if (bad(q) || bad(out) || (a->k_len && (bad(k) || bad(v))) || reinterpret_cast<uintptr_t>(out_low) % 8 ||
      reinterpret_cast<uintptr_t>(lse) % 16)
    return MSD_E_ARG;
  if (pl.splits > 1 && bad(workspace)) return MSD_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Args p = args(*a, pl, q, k, v);
  p.out = static_cast<uint16_t*>(out);
  p.low = static_cast<uint8_t*>(out_low);
  p.lse = lse;
  p.part = static_cast<float*>(workspace);
  p.splits = pl.splits;
  launches(*a, pl, [&](const Launch& l) {
    if (!l.groups) return;
    const Args x = args(p, *a, l);
    with_head(a->d_head, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      hipLaunchKernelGGL((attn_fwd<DP>), dim3(unsigned(l.groups), pl.splits), dim3(64 * kWaves), 0, s, x, l.rows);
    });
    if (pl.splits == 1) return;
    const int64_t rows = int64_t(l.q_len) * a->n_heads;
    auto join = [&](auto lanes) {
      constexpr int G = decltype(lanes)::value;
      hipLaunchKernelGGL(attn_join<G>, dim3(unsigned(cdiv(rows, 16 / G)), l.n), dim3(kJoinLanes), 0, s, x, l.rows);
    };
    if (pl.splits > 8) join(std::integral_constant<int, 16>());
    else if (pl.splits > 4) join(std::integral_constant<int, 4>());
    else join(std::integral_constant<int, 1>());
  });
  return launched();
}

extern "C" int32_t msd_attn_backward(const msd_attn* a, const void* q, const void* k, const void* v, const void* out,
                                     const void* out_low, const float* lse, const void* dout, void* dq, void* dk, void* dv, void* workspace,
                                     void* stream) {
  Plan pl;
  const int32_t rc = check(a, true, pl);
  if (rc != MSD_OK) return rc;
  if (a->n_seqs == 0 || (a->q_len == 0 && a->k_len == 0)) return MSD_OK;
  if ((a->q_len && (bad(q) || bad(out) || bad(lse) || bad(dout) || bad(dq) ||
                    reinterpret_cast<uintptr_t>(out_low) % 8)) ||
      (a->k_len && (bad(k) || bad(v) || bad(dk) || bad(dv))))
    return MSD_E_ARG;
  if (bad(workspace) && (a->q_len || pl.head_parts * pl.row_parts > 1)) return MSD_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Args p = args(*a, pl, q, k, v);
  p.dout = view(dout, a->dout_stride);
  p.o = static_cast<const uint16_t*>(out);
  p.low = static_cast<uint8_t*>(const_cast<void*>(out_low));
  p.lse = const_cast<float*>(lse);
  p.stats = static_cast<float*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + up(8 * a->q_rows * a->n_heads));
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  p.splits = pl.dq_splits;
  p.tile_rows = pl.tile_rows;
  p.head_parts = pl.head_parts;
  p.chunk = pl.chunk;
  launches(*a, pl, [&](const Launch& l) {
    const Args x = args(p, *a, l);
    with_head(a->d_head, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      if (l.groups) {
        hipLaunchKernelGGL((attn_dq<DP>), dim3(unsigned(l.groups), pl.dq_splits), dim3(64 * kWaves), 0, s, x, l.rows);
        if (pl.dq_splits > 1)
          hipLaunchKernelGGL(attn_join_dq, dim3(unsigned(cdiv(int64_t(l.q_len) * a->n_heads * a->d_head, 2048)), l.n), dim3(256), 0, s, x,
                             l.rows);
      }
      if (l.key_groups)
        hipLaunchKernelGGL((attn_dkv<DP>), dim3(unsigned(l.key_groups)), dim3(64 * kWaves), 0, s, x, l.keys, l.sums);
    });
    if (l.key_groups && pl.head_parts * l.row_parts > 1) {
      const int64_t slices = cdiv(128 * int64_t(a->n_kv_heads) * a->d_head, 2048);
      hipLaunchKernelGGL(attn_sum_parts, dim3(unsigned(l.blocks), unsigned(slices), 2), dim3(256), 0, s, x, l.sums);
    }
  });
  return launched();
}
