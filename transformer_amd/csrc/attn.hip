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
// LDS tiles.  64 rows of 128 bytes (d_head <= 64) or 256 bytes, in 16-byte pieces; row r holds piece c at position c ^
// f(r), with f chosen (swizzle()) so that both the plain reads (32 rows, one piece each) and the transposing reads (4
// rows, 64 bytes each) touch every bank once.  Two buffers: the next tile is loaded to registers while this one is
// worked on.  Rows and columns that do not exist are zeros (buffer loads outside the descriptor), so what lies
// behind a sequence's rows is never read.
//
// The backward is two kernels: attn_dq (like the forward, rows outside, keys inside) and attn_dkv (keys outside, all
// rows of the group inside).  Each recomputes S and dP: 7 products instead of the 5 of one kernel, which would have to
// add dQ across workgroups with atomics, in no fixed order.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mslayers.h"
#include "internal.h"

namespace msa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 64;        // rows of an LDS tile
constexpr uint32_t kOutside = 0x80000000u;   // a buffer offset past every descriptor: the load gives zeros

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
  uint32_t g_magic;         // r / g = umulhi(r, g_magic) for g > 1, r < 2^31 (see magic())
  int g_shift;
  float c, scale;
  int tiles;                // row (or key) tiles of the longest sequence
  int splits;
  int64_t q_rows, k_rows;
  uint16_t *out, *dq, *dk, *dv;
  float *lse, *delta;
  float* part;              // forward: [splits][q_rows * H][D + 1]; backward: [2][splits][k_rows * KV][D]
};

struct Seq {
  int qs, qn, ks, kn;
};

__device__ __forceinline__ Seq sequence(const Args& p, int b) {
  if (!p.seqs) return {b * p.q_len, p.q_len, b * p.k_len, p.k_len};
  const int4 s = reinterpret_cast<const int4*>(p.seqs)[b];
  return {__builtin_amdgcn_readfirstlane(s.x), __builtin_amdgcn_readfirstlane(s.y), __builtin_amdgcn_readfirstlane(s.z),
          __builtin_amdgcn_readfirstlane(s.w)};
}

// The first element of row 0, head `head` of sequence b, whose rows start at `start`.
__device__ __forceinline__ const uint16_t* origin(const Args& p, const View& v, int b, int start, int head) {
  return v.p + (p.seqs ? int64_t(start) * v.row : int64_t(b) * v.seq) + int64_t(head) * v.head;
}

__device__ __forceinline__ int div_g(const Args& p, int r) {
  return p.g_magic ? int(__umulhi(uint32_t(r), p.g_magic) >> p.g_shift) : r >> p.g_shift;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& s, int i) {
  return __builtin_bit_cast(bf16x8, (u32x4{pack2(s[i], s[i + 1]), pack2(s[i + 2], s[i + 3]), pack2(s[i + 4], s[i + 5]),
                                           pack2(s[i + 6], s[i + 7])}));
}

__device__ __forceinline__ float swap_halves(float x) {   // the value of lane l ^ 32
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
#else
  return x;
#endif
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}

// 16 bytes at byte offset `off` of the tensor part at `base` (wave-uniform), zeros for kOutside
__device__ __forceinline__ u32x4 load16(const uint16_t* base, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, 0x7fffffff, 0x00020000);
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
#else
  return u32x4{};
#endif
}

template <int DP>
constexpr int pitch() { return DP <= 64 ? 128 : 256; }

// Piece c of row r of a tile lies at position c ^ swizzle(r).  Plain reads go in groups of 16 lanes whose rows are
// 0-3, 12-15, 20-27 (or the other 16) of 32: with 128-byte rows two rows share the 64 banks, and (r >> 1) & 7 takes all
// 8 values over each group's even (odd) rows; with 256-byte rows r & 15 takes all 16.  A transposing read touches rows
// 4 m .. 4 m + 3, four pieces each: the bits that tell those rows apart are put where they move the group of four.
template <int P>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (P == 128) return ((r & 2) << 1) | ((r & 4) >> 1) | ((r >> 3) & 1);
  return ((r & 3) << 2) | ((r >> 2) & 3);
}

template <int P>
__device__ __forceinline__ int piece_at(int r, int c) { return r * P + ((c ^ swizzle<P>(r)) << 4); }

// The operand of 32 rows row0.. , contraction values 16 ks + 8 h .. + 8 (pieces of the rows)
template <int P>
__device__ __forceinline__ bf16x8 rows_operand(const uint8_t* tile, int row0, int ks, int lane) {
  return *reinterpret_cast<const bf16x8*>(tile + piece_at<P>(row0 + (lane & 31), 2 * ks + (lane >> 5)));
}

// The operand of columns 32 blk .. + 32, contraction over rows row0 + 4 h + {0..3}, row0 + 8 + 4 h + {0..3}
template <int P>
__device__ __forceinline__ bf16x8 cols_operand(const uint8_t* tile, int row0, int blk, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int t = lane & 15, r = row0 + 4 * (lane >> 5) + (t >> 2);
  const int c = 4 * blk + 2 * ((lane >> 4) & 1) + ((t & 3) >> 1);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + piece_at<P>(r, c) + 8 * (t & 1)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + piece_at<P>(r + 8, c) + 8 * (t & 1)));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
  return bf16x8{};
#endif
}

// A 64-row tile of K or V on its way to LDS
template <int DP, int NT>
struct KeyTile {
  static constexpr int P = pitch<DP>(), C = P / 16, N = kKeys * C / NT;
  u32x4 x[N];
  __device__ __forceinline__ void load(const uint16_t* base, int64_t row_stride, int row0, int n_rows, int D, int tid) {
    const uint16_t* at = base + int64_t(row0) * row_stride;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = tid + NT * u, r = i / C, c = i % C;
      x[u] = load16(at, row0 + r < n_rows && 8 * c < D ? uint32_t(r) * uint32_t(row_stride) * 2 + 16 * c : kOutside);
    }
  }
  __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = tid + NT * u, r = i / C, c = i % C;
      *reinterpret_cast<u32x4*>(tile + piece_at<P>(r, c)) = x[u];
    }
  }
};

// A 64-row tile of q or dout rows (position r / g, head r % g)
template <int DP, int NT>
struct RowTile {
  static constexpr int P = pitch<DP>(), C = P / 16, N = kKeys * C / NT;
  u32x4 x[N];
  __device__ __forceinline__ void load(const Args& p, const uint16_t* base, const View& v, int row0, int n_rows,
                                       int tid) {
    const int pos0 = div_g(p, row0);
    const uint16_t* at = base + int64_t(pos0) * v.row;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = tid + NT * u, r = row0 + i / C, c = i % C, pos = div_g(p, r);
      x[u] = load16(at, r < n_rows && 8 * c < p.D ? (uint32_t(pos - pos0) * uint32_t(v.row) +
                                                     uint32_t(r - pos * p.g) * uint32_t(v.head)) * 2 + 16 * c
                                                  : kOutside);
    }
  }
  __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = tid + NT * u, r = i / C, c = i % C;
      *reinterpret_cast<u32x4*>(tile + piece_at<P>(r, c)) = x[u];
    }
  }
};

// The operands of 32 rows of a strided tensor, straight from memory: lane l holds row l % 32 (element offset `at`,
// `ok` whether it exists), contraction values 16 ks + 8 (l / 32) .. + 8
template <int DP>
__device__ __forceinline__ void row_operands(bf16x8 (&f)[DP / 16], const uint16_t* base, int64_t at, bool ok, int D,
                                             int lane) {
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int c = 16 * ks + 8 * (lane >> 5);
    u32x4 x{};
    if (ok && c < D) x = *reinterpret_cast<const u32x4*>(base + at + c);
    f[ks] = __builtin_bit_cast(bf16x8, x);
  }
}

// Keeps the compiler from moving LDS accesses of this wave across (the hardware runs a wave's in order)
__device__ __forceinline__ void wave_lds_order() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#endif
}

// A wave's transposed result (columns = 32 rows of the output, DP of its columns down the registers), times `by` per
// lane, to LDS as bf16 rows; then `dst(row)` gets the rows' 16-byte pieces
template <int DP, class F>
__device__ __forceinline__ void store_rows(uint8_t* stage, const f32x16 (&acc)[DP / 32], float by, int D, int lane, F dst) {
  constexpr int P = pitch<DP>(), C = P / 16;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u32x2 x = {pack2(acc[b][4 * q] * by, acc[b][4 * q + 1] * by), pack2(acc[b][4 * q + 2] * by, acc[b][4 * q + 3] * by)};
      *reinterpret_cast<u32x2*>(stage + piece_at<P>(lane & 31, 4 * b + q) + 8 * (lane >> 5)) = x;
    }
  wave_lds_order();   // one wave writes and reads its own part
#pragma unroll
  for (int u = 0; u < 32 * C / 64; ++u) {
    const int i = lane + 64 * u, r = i / C, c = i % C;
    const u32x4 x = *reinterpret_cast<const u32x4*>(stage + piece_at<P>(r, c));
    uint16_t* to = dst(r);
    if (to && 8 * c < D) *reinterpret_cast<u32x4*>(to + 8 * c) = x;
  }
  wave_lds_order();
}

// What a workgroup of row tiles works on: 32 rows a wave, keys [k_lo, k_hi) in tiles of 64
struct RowJob {
  Seq s;
  int b, kvh, rows, r;      // r: this lane's row
  bool ok;                  // it exists
  int pos, head;            // its position and query head
  int seen;                 // keys it sees
  int wave_full, wave_end;  // keys that every row of the wave sees, that some row sees
  int t0, t1;               // key tiles of this split
};

template <int NW>
__device__ __forceinline__ bool row_job(const Args& p, RowJob& j, int lane, int wv) {
  const int heads = p.n_seqs * p.KV, id = blockIdx.x % heads;
  const int tile = p.tiles - 1 - int(blockIdx.x / heads);   // the longest key ranges first
  j.b = id / p.KV;
  j.kvh = id % p.KV;
  j.s = sequence(p, j.b);
  j.rows = j.s.qn * p.g;
  const int r0 = tile * 32 * NW;
  if (r0 >= j.rows) return false;
  j.r = r0 + 32 * wv + (lane & 31);
  j.ok = j.r < j.rows;
  j.pos = div_g(p, min(j.r, j.rows - 1));
  j.head = j.kvh * p.g + (j.ok ? j.r - j.pos * p.g : 0);
  const int last = j.s.kn - j.s.qn + 1;   // keys that position 0 sees
  j.seen = p.causal ? min(max(last + j.pos, 0), j.s.kn) : j.s.kn;
  const int w0 = min(r0 + 32 * wv, j.rows - 1), w1 = min(r0 + 32 * wv + 31, j.rows - 1), wg = min(r0 + 32 * NW, j.rows) - 1;
  auto seen_by = [&](int r) { return p.causal ? min(max(last + div_g(p, r), 0), j.s.kn) : j.s.kn; };
  j.wave_full = seen_by(w0);
  j.wave_end = seen_by(w1);
  const int n = (seen_by(wg) + kKeys - 1) / kKeys;
  j.t0 = int(int64_t(n) * blockIdx.y / p.splits);
  j.t1 = int(int64_t(n) * (blockIdx.y + 1) / p.splits);
  return true;
}

__device__ __forceinline__ int64_t stat_index(const Args& p, const RowJob& j) {
  return int64_t(j.s.qs) * p.H + int64_t(j.kvh) * j.rows + j.r;
}

// ---- forward ----
template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 64 ? 3 : 2) void attn_fwd(Args p) {
  constexpr int P = pitch<DP>(), TILE = kKeys * P, NT = 64 * NW;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  RowJob j;
  if (!row_job<NW>(p, j, lane, wv)) return;
  const uint16_t* kb = origin(p, p.k, j.b, j.s.ks, j.kvh);
  const uint16_t* vb = origin(p, p.v, j.b, j.s.ks, j.kvh);

  bf16x8 q[DP / 16];
  row_operands<DP>(q, origin(p, p.q, j.b, j.s.qs, 0), int64_t(j.pos) * p.q.row + int64_t(j.head) * p.q.head, j.ok, p.D, lane);

  f32x16 o[DP / 32] = {};
  float m = -INFINITY, l = 0;   // running maximum of c s, up to 2^8 too small; sum of 2^(c s - m) over this lane's keys

  KeyTile<DP, NT> kt, vt;
  if (j.t0 < j.t1) {
    kt.load(kb, p.k.row, j.t0 * kKeys, j.s.kn, p.D, tid);
    vt.load(vb, p.v.row, j.t0 * kKeys, j.s.kn, p.D, tid);
    kt.store(lds, tid);
    vt.store(lds + TILE, tid);
  }
  __syncthreads();
  for (int t = j.t0; t < j.t1; ++t) {
    const uint8_t* K = lds + ((t - j.t0) & 1) * 2 * TILE;
    const uint8_t* V = K + TILE;
    uint8_t* next = lds + ((t - j.t0 + 1) & 1) * 2 * TILE;
    if (t + 1 < j.t1) {
      kt.load(kb, p.k.row, (t + 1) * kKeys, j.s.kn, p.D, tid);
      vt.load(vb, p.v.row, (t + 1) * kKeys, j.s.kn, p.D, tid);
    }
    const int key0 = t * kKeys;
    if (key0 < j.wave_end) {
      f32x16 s[2] = {};
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = mfma(rows_operand<P>(K, 32 * b, ks, lane), q[ks], s[b]);
      if (key0 + kKeys > j.wave_full) {   // the diagonal or the end
        const int left = j.seen - key0 - 4 * (lane >> 5);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * b + 8 * (i >> 2) + (i & 3) >= left) s[b][i] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
      top = fmaxf(top, swap_halves(top)) * p.c;
      if (__any(top > m + 8.0f)) {   // rescaling by less than 2^8 can wait: f32 sums and bf16 P keep their precision
        const float mn = fmaxf(m, top), by = mn == -INFINITY ? 1.0f : exp2_hw(m - mn);
        m = mn;
        l *= by;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] *= by;
      }
      const float sub = m == -INFINITY ? 0.0f : m;
      float sum = 0;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[b][i] = exp2_hw(fmaf(s[b][i], p.c, -sub));
          sum += s[b][i];
        }
      l += sum;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 pr = pack8(s[b], 8 * h);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) o[d] = mfma(cols_operand<P>(V, 32 * b + 16 * h, d, lane), pr, o[d]);
        }
    }
    if (t + 1 < j.t1) {
      kt.store(next, tid);
      vt.store(next + TILE, tid);
    }
    __syncthreads();
  }
  l += swap_halves(l);
  const float by = l == 0 ? 0.0f : 1.0f / l;   // (a NaN sum stays one)
  const float lse = l == 0 ? INFINITY : m + __log2f(l);   // +inf: 2^(c s - lse) is 0 for a row that sees nothing
  if (p.splits > 1) {   // normalised part and its weight, joined by attn_join
    if (j.ok) {
      const int64_t row = stat_index(p, j);
      float* to = p.part + (int64_t(blockIdx.y) * p.q_rows * p.H + row) * p.D;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = 32 * d + 8 * u + 4 * (lane >> 5);
          if (c < p.D)
            *reinterpret_cast<f32x4*>(to + c) = f32x4{o[d][4 * u] * by, o[d][4 * u + 1] * by, o[d][4 * u + 2] * by, o[d][4 * u + 3] * by};
        }
      if (lane < 32) p.part[int64_t(p.splits) * p.q_rows * p.H * p.D + int64_t(blockIdx.y) * p.q_rows * p.H + row] = lse;
    }
    return;
  }
  if (p.lse && j.ok && lane < 32) p.lse[stat_index(p, j)] = lse;
  const int r0 = j.r - (lane & 31);
  store_rows<DP>(lds + wv * 32 * P, o, by, p.D, lane, [&](int r) -> uint16_t* {
    if (r0 + r >= j.rows) return nullptr;
    const int pos = div_g(p, r0 + r);
    return p.out + (int64_t(j.s.qs + pos) * p.H + j.kvh * p.g + (r0 + r - pos * p.g)) * p.D;
  });
}

// The parts of a row over the splits, weighted by 2^(lse_z - lse): one thread for 8 values
__global__ void attn_join(Args p) {
  const int per = p.D / 8;
  const int64_t n = p.q_rows * p.H, id = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int b = blockIdx.y;
  const Seq s = sequence(p, b);
  const int64_t rows = int64_t(s.qn) * p.H, row = id / per;
  if (row >= rows) return;
  const int c = int(id - row * per) * 8;
  const int64_t at = int64_t(s.qs) * p.H + row;   // statistics order: kv head, position, head of the group
  const float* w = p.part + int64_t(p.splits) * n * p.D;
  float m = -INFINITY;
  for (int z = 0; z < p.splits; ++z) {
    const float x = w[z * n + at];
    if (x != INFINITY) m = fmaxf(m, x);
  }
  float acc[8] = {}, l = 0;
  for (int z = 0; z < p.splits; ++z) {
    const float x = w[z * n + at];
    if (x == INFINITY) continue;   // nothing seen in this part
    const float e = exp2_hw(x - m);
    const float* from = p.part + (z * n + at) * p.D + c;
    l += e;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(e, from[i], acc[i]);
  }
  const float by = l == 0 ? 0.0f : 1.0f / l;
  const int kvh = int(row / (int64_t(s.qn) * p.g)), r = int(row - int64_t(kvh) * s.qn * p.g), pos = r / p.g;
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2(acc[2 * i] * by, acc[2 * i + 1] * by);
  *reinterpret_cast<u32x4*>(p.out + (int64_t(s.qs + pos) * p.H + kvh * p.g + (r - pos * p.g)) * p.D + c) = x;
  if (p.lse && c == 0) p.lse[at] = l == 0 ? INFINITY : m + __log2f(l);
}

// ---- backward ----
// dQ of 32 rows a wave; also D_i = dO_i.O_i, which attn_dkv reads
template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_dq(Args p) {
  constexpr int P = pitch<DP>(), TILE = kKeys * P, NT = 64 * NW;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  RowJob j;
  if (!row_job<NW>(p, j, lane, wv)) return;
  const uint16_t* kb = origin(p, p.k, j.b, j.s.ks, j.kvh);
  const uint16_t* vb = origin(p, p.v, j.b, j.s.ks, j.kvh);

  bf16x8 q[DP / 16], dO[DP / 16];
  row_operands<DP>(q, origin(p, p.q, j.b, j.s.qs, 0), int64_t(j.pos) * p.q.row + int64_t(j.head) * p.q.head, j.ok, p.D, lane);
  row_operands<DP>(dO, origin(p, p.dout, j.b, j.s.qs, 0), int64_t(j.pos) * p.dout.row + int64_t(j.head) * p.dout.head, j.ok,
                   p.D, lane);
  float delta = 0;
  {
    bf16x8 o[DP / 16];
    row_operands<DP>(o, p.o, (int64_t(j.s.qs + j.pos) * p.H + j.head) * p.D, j.ok, p.D, lane);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) delta = fmaf(float(o[ks][i]), float(dO[ks][i]), delta);
  }
  delta += swap_halves(delta);
  const float lse = j.ok ? p.lse[stat_index(p, j)] : INFINITY;
  if (j.ok && lane < 32) p.delta[stat_index(p, j)] = delta;

  f32x16 dq[DP / 32] = {};
  KeyTile<DP, NT> kt, vt;
  if (j.t0 < j.t1) {
    kt.load(kb, p.k.row, j.t0 * kKeys, j.s.kn, p.D, tid);
    vt.load(vb, p.v.row, j.t0 * kKeys, j.s.kn, p.D, tid);
    kt.store(lds, tid);
    vt.store(lds + TILE, tid);
  }
  __syncthreads();
  for (int t = j.t0; t < j.t1; ++t) {
    const uint8_t* K = lds + ((t - j.t0) & 1) * 2 * TILE;
    const uint8_t* V = K + TILE;
    uint8_t* next = lds + ((t - j.t0 + 1) & 1) * 2 * TILE;
    if (t + 1 < j.t1) {
      kt.load(kb, p.k.row, (t + 1) * kKeys, j.s.kn, p.D, tid);
      vt.load(vb, p.v.row, (t + 1) * kKeys, j.s.kn, p.D, tid);
    }
    const int key0 = t * kKeys;
    if (key0 < j.wave_end) {
      const bool edge = key0 + kKeys > j.wave_full;
      const int left = j.seen - key0 - 4 * (lane >> 5);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          s = mfma(rows_operand<P>(K, 32 * b, ks, lane), q[ks], s);
          dp = mfma(rows_operand<P>(V, 32 * b, ks, lane), dO[ks], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x = exp2_hw(fmaf(s[i], p.c, -lse)) * (dp[i] - delta);
          if (edge && 32 * b + 8 * (i >> 2) + (i & 3) >= left) x = 0;
          s[i] = x;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 ds = pack8(s, 8 * h);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) dq[d] = mfma(cols_operand<P>(K, 32 * b + 16 * h, d, lane), ds, dq[d]);
        }
      }
    }
    if (t + 1 < j.t1) {
      kt.store(next, tid);
      vt.store(next + TILE, tid);
    }
    __syncthreads();
  }
  const int r0 = j.r - (lane & 31);
  store_rows<DP>(lds + wv * 32 * P, dq, p.scale, p.D, lane, [&](int r) -> uint16_t* {
    if (r0 + r >= j.rows) return nullptr;
    const int pos = div_g(p, r0 + r);
    return p.dq + (int64_t(j.s.qs + pos) * p.H + j.kvh * p.g + (r0 + r - pos * p.g)) * p.D;
  });
}

// dK and dV of 128 keys, 32 a wave; the rows of all heads of the group, 64 at a time
template <int DP>
__global__ __launch_bounds__(256, 2) void attn_dkv(Args p) {
  constexpr int P = pitch<DP>(), TILE = kKeys * P, NT = 256;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TILE];
  __shared__ __attribute__((aligned(16))) float stats[2][3][64];   // lse, D and the keys seen, of a tile's rows
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = p.n_seqs * p.KV, id = blockIdx.x % heads, b = id / p.KV, kvh = id % p.KV;
  const Seq s = sequence(p, b);
  const int kb0 = int(blockIdx.x / heads) * 128;   // (the first keys are seen by the most rows)
  if (kb0 >= s.kn) return;
  const int k0 = kb0 + 32 * wv, key = k0 + (lane & 31);
  const bool ok = key < s.kn;
  const int rows = s.qn * p.g, last = s.kn - s.qn + 1;
  const uint16_t* qb = origin(p, p.q, b, s.qs, kvh * p.g);
  const uint16_t* db = origin(p, p.dout, b, s.qs, kvh * p.g);

  bf16x8 k[DP / 16], v[DP / 16];
  row_operands<DP>(k, origin(p, p.k, b, s.ks, kvh), int64_t(key) * p.k.row, ok, p.D, lane);
  row_operands<DP>(v, origin(p, p.v, b, s.ks, kvh), int64_t(key) * p.v.row, ok, p.D, lane);

  // row tiles that see a key of this workgroup, and this split's part of them
  const int first = p.causal ? min(max(kb0 - last + 1, 0), s.qn) * p.g / 64 : 0;
  const int n = (rows + 63) / 64 - first;
  const int t0 = first + int(int64_t(n) * blockIdx.y / p.splits), t1 = first + int(int64_t(n) * (blockIdx.y + 1) / p.splits);
  const int64_t stat0 = int64_t(s.qs) * p.H + int64_t(kvh) * rows;

  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  RowTile<DP, NT> qt, dt;
  float st = 0;
  auto load = [&](int t) {
    qt.load(p, qb, p.q, 64 * t, rows, tid);
    dt.load(p, db, p.dout, 64 * t, rows, tid);
    const int r = 64 * t + lane;
    if (wv == 0) st = r < rows ? p.lse[stat0 + r] : INFINITY;
    if (wv == 1) st = r < rows ? p.delta[stat0 + r] : 0.0f;
    if (wv == 2) st = __int_as_float(r >= rows ? 0 : p.causal ? min(max(last + div_g(p, r), 0), s.kn) : s.kn);
  };
  auto store = [&](int buf) {
    qt.store(lds + buf * 2 * TILE, tid);
    dt.store(lds + buf * 2 * TILE + TILE, tid);
    if (wv < 3) stats[buf][wv][lane] = st;
  };
  if (t0 < t1) {
    load(t0);
    store(0);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const uint8_t* Q = lds + buf * 2 * TILE;
    const uint8_t* dO = Q + TILE;
    if (t + 1 < t1) load(t + 1);
    // (uniform) whether every row of the tile sees all 32 keys of the wave
    const int r_lo = 64 * t;
    const bool edge = r_lo + 64 > rows || (p.causal && last + div_g(p, r_lo) < k0 + 32) || k0 + 32 > s.kn;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      f32x16 sc = {}, dp = {};
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        sc = mfma(rows_operand<P>(Q, 32 * a, ks, lane), k[ks], sc);
        dp = mfma(rows_operand<P>(dO, 32 * a, ks, lane), v[ks], dp);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = 32 * a + 8 * u + 4 * (lane >> 5);
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&stats[buf][0][r]);
        const f32x4 del = *reinterpret_cast<const f32x4*>(&stats[buf][1][r]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = exp2_hw(fmaf(sc[4 * u + i], p.c, -lse[i]));
          float y = x * (dp[4 * u + i] - del[i]);
          if (edge && key >= __float_as_int(stats[buf][2][r + i])) x = y = 0;
          sc[4 * u + i] = x;
          dp[4 * u + i] = y;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x8 pr = pack8(sc, 8 * h), ds = pack8(dp, 8 * h);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          dv[d] = mfma(cols_operand<P>(dO, 32 * a + 16 * h, d, lane), pr, dv[d]);
          dk[d] = mfma(cols_operand<P>(Q, 32 * a + 16 * h, d, lane), ds, dk[d]);
        }
      }
    }
    if (t + 1 < t1) store((t - t0 + 1) & 1);
    __syncthreads();
  }
  if (p.splits > 1) {
    if (!ok) return;
    const int64_t n = p.k_rows * p.KV * p.D;
    float* to = p.part + int64_t(blockIdx.y) * n + (int64_t(s.ks + key) * p.KV + kvh) * p.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = 32 * d + 8 * u + 4 * (lane >> 5);
        if (c < p.D) {
          *reinterpret_cast<f32x4*>(to + c) = f32x4{dk[d][4 * u], dk[d][4 * u + 1], dk[d][4 * u + 2], dk[d][4 * u + 3]};
          *reinterpret_cast<f32x4*>(to + p.splits * n + c) =
              f32x4{dv[d][4 * u], dv[d][4 * u + 1], dv[d][4 * u + 2], dv[d][4 * u + 3]};
        }
      }
    return;
  }
  auto row = [&](uint16_t* base, int r) -> uint16_t* {
    return k0 + r < s.kn ? base + (int64_t(s.ks + k0 + r) * p.KV + kvh) * p.D : nullptr;
  };
  uint8_t* stage = lds + wv * 32 * P;
  store_rows<DP>(stage, dk, p.scale, p.D, lane, [&](int r) { return row(p.dk, r); });
  store_rows<DP>(stage, dv, 1.0f, p.D, lane, [&](int r) { return row(p.dv, r); });
}

// dK and dV as the sum of their parts, in the order of the splits: 8 values a thread, of the rows of a sequence
__global__ void attn_sum_parts(Args p) {
  const Seq s = sequence(p, blockIdx.y);
  const int64_t n = p.k_rows * p.KV * p.D, own = int64_t(s.kn) * p.KV * p.D;
  const int64_t i = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) * 8;
  if (i >= own) return;
  const int64_t at = int64_t(s.ks) * p.KV * p.D + i;
  const bool v = blockIdx.z;
  const float* from = p.part + (v ? p.splits * n : 0) + at;
  f32x4 a = {}, b = {};
  for (int z = 0; z < p.splits; ++z) {
    a += *reinterpret_cast<const f32x4*>(from + z * n);
    b += *reinterpret_cast<const f32x4*>(from + z * n + 4);
  }
  const float by = v ? 1.0f : p.scale;
  a *= by;
  b *= by;
  *reinterpret_cast<u32x4*>((v ? p.dv : p.dk) + at) = u32x4{pack2(a[0], a[1]), pack2(a[2], a[3]), pack2(b[0], b[1]), pack2(b[2], b[3])};
}

// ---- host ----
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// r / g for 0 <= r < 2^31: a shift for powers of two, else umulhi by ceil(2^(32 + s) / g) with 2^s < g: the error g m -
// 2^(32 + s) is below g <= 2^(s + 1), so r < 2^31 gives the exact quotient
void magic(uint32_t g, uint32_t& m, int& s) {
  s = 31 - __builtin_clz(g);
  m = 0;
  if ((g & (g - 1)) == 0) return;
  m = uint32_t(((uint64_t(1) << (32 + s)) + g - 1) / g);
}

struct Plan {
  int waves;          // of a forward or dQ workgroup
  int tiles, splits;  // forward: row tiles, splits of the keys
  int dq_waves, dq_tiles, key_tiles, row_splits;
};

constexpr int kCus = 256;
constexpr int64_t kMostGroups = (int64_t(1) << 32) / 256 - 1;   // a launch has fewer than 2^32 threads a dimension

Plan plan(const msd_attn& a) {
  Plan p;
  const int64_t heads = int64_t(a.n_seqs) * a.n_kv_heads, rows = int64_t(a.q_len) * (a.n_heads / a.n_kv_heads);
  const int64_t key_tiles = std::max<int64_t>(cdiv(a.k_len, kKeys), 1);
  p.waves = heads * cdiv(rows, 128) >= kCus ? 4 : 1;
  p.tiles = int(cdiv(rows, 32 * p.waves));
  const int64_t groups = heads * p.tiles;
  p.splits = int(groups >= 2 * kCus ? 1 : std::max<int64_t>(1, std::min(cdiv(4 * kCus, std::max<int64_t>(groups, 1)), cdiv(key_tiles, 2))));
  p.dq_waves = p.waves;
  p.dq_tiles = p.tiles;
  p.key_tiles = int(cdiv(a.k_len, 128));
  const int64_t wgs = heads * p.key_tiles;
  p.row_splits = int(wgs >= 2 * kCus ? 1 : std::max<int64_t>(1, std::min(cdiv(2 * kCus, std::max<int64_t>(wgs, 1)), cdiv(rows, 128))));
  return p;
}

bool fits(const int64_t (&s)[3], int64_t heads) {
  for (int64_t x : s)
    if (x < 0 || x % 8) return false;
  constexpr int64_t most = int64_t(1) << 30;
  return s[1] <= most / 64 && s[2] <= most / heads && 64 * s[1] + heads * s[2] < most;
}

int32_t check(const msd_attn* a, bool backward) {
  if (!a) return MSD_E_ARG;
  if (a->n_seqs < 0 || a->q_len < 0 || a->k_len < 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->n_heads % a->n_kv_heads ||
      a->d_head <= 0 || a->d_head > 128 || a->d_head % 8 || !(a->scale > 0) || !isfinite(a->scale) || a->q_rows < 0 ||
      a->k_rows < 0)
    return MSD_E_CONFIG;
  const int64_t most = int64_t(1) << 31;
  if (a->q_rows >= most || a->k_rows >= most || a->q_rows * a->n_heads >= most || a->k_rows * a->n_kv_heads >= most ||
      int64_t(a->q_len) * a->n_heads >= most || int64_t(a->n_seqs) * a->n_kv_heads >= (1 << 20) || a->n_seqs > 65535)
    return MSD_E_CONFIG;
  if (!a->seqs && (a->q_rows != int64_t(a->n_seqs) * a->q_len || a->k_rows != int64_t(a->n_seqs) * a->k_len)) return MSD_E_CONFIG;
  if (a->q_len > a->q_rows || a->k_len > a->k_rows) return MSD_E_CONFIG;
  const int64_t g = a->n_heads / a->n_kv_heads;
  if (!fits(a->q_stride, g) || !fits(a->k_stride, 1) || !fits(a->v_stride, 1) || (backward && !fits(a->dout_stride, g)))
    return MSD_E_CONFIG;
  if (int64_t(a->n_seqs) * a->n_kv_heads * std::max(cdiv(int64_t(a->q_len) * g, 128), cdiv(a->k_len, 128)) > kMostGroups)
    return MSD_E_CONFIG;
  if (a->seqs && reinterpret_cast<uintptr_t>(a->seqs) % 16) return MSD_E_ARG;
  return MSD_OK;
}

bool bad(const void* p) { return !p || reinterpret_cast<uintptr_t>(p) % 16; }

View view(const void* p, const int64_t (&s)[3]) { return {static_cast<const uint16_t*>(p), s[0], s[1], s[2]}; }

Args args(const msd_attn& a, const void* q, const void* k, const void* v) {
  Args p{};
  p.q = view(q, a.q_stride);
  p.k = view(k, a.k_stride);
  p.v = view(v, a.v_stride);
  p.seqs = a.seqs;
  p.n_seqs = a.n_seqs;
  p.q_len = a.q_len;
  p.k_len = a.k_len;
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

// f(integral_constant) for the padded head size
template <class F>
void with_head(int D, F f) {
  if (D <= 32) f(std::integral_constant<int, 32>());
  else if (D <= 64) f(std::integral_constant<int, 64>());
  else if (D <= 96) f(std::integral_constant<int, 96>());
  else f(std::integral_constant<int, 128>());
}

int32_t launched() { return hipGetLastError() == hipSuccess ? MSD_OK : MSD_E_HIP; }

int64_t up(int64_t x) { return cdiv(x, 256) * 256; }

}  // namespace msa

using namespace msa;

extern "C" int64_t msd_attn_workspace_bytes(const msd_attn* a, int32_t backward) {
  const int32_t rc = check(a, false);
  if (rc != MSD_OK) return rc;
  const Plan pl = plan(*a);
  if (!backward) return pl.splits > 1 ? 4 * pl.splits * a->q_rows * a->n_heads * (a->d_head + 1) : 0;
  const int64_t parts = pl.row_splits > 1 ? 8 * pl.row_splits * a->k_rows * a->n_kv_heads * a->d_head : 0;
  return up(4 * a->q_rows * a->n_heads) + parts;
}

extern "C" int32_t msd_attn_forward(const msd_attn* a, const void* q, const void* k, const void* v, void* out, float* lse,
                                    void* workspace, void* stream) {
  const int32_t rc = check(a, false);
  if (rc != MSD_OK) return rc;
  if (a->n_seqs == 0 || a->q_len == 0) return MSD_OK;
  if (bad(q) || bad(out) || (a->k_len && (bad(k) || bad(v)))) return MSD_E_ARG;
  const Plan pl = plan(*a);
  if (pl.splits > 1 && bad(workspace)) return MSD_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Args p = args(*a, q, k, v);
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  p.part = static_cast<float*>(workspace);
  p.tiles = pl.tiles;
  p.splits = pl.splits;
  const dim3 grid(unsigned(pl.tiles) * a->n_seqs * a->n_kv_heads, pl.splits);
  with_head(a->d_head, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (pl.waves == 4) hipLaunchKernelGGL((attn_fwd<DP, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((attn_fwd<DP, 1>), grid, dim3(64), 0, s, p);
  });
  if (pl.splits > 1) {
    const int64_t n = int64_t(a->q_len) * a->n_heads * (a->d_head / 8);
    hipLaunchKernelGGL(attn_join, dim3(unsigned(cdiv(n, 128)), a->n_seqs), dim3(128), 0, s, p);
  }
  return launched();
}

extern "C" int32_t msd_attn_backward(const msd_attn* a, const void* q, const void* k, const void* v, const void* out,
                                     const float* lse, const void* dout, void* dq, void* dk, void* dv, void* workspace,
                                     void* stream) {
  const int32_t rc = check(a, true);
  if (rc != MSD_OK) return rc;
  if (a->n_seqs == 0 || (a->q_len == 0 && a->k_len == 0)) return MSD_OK;
  if ((a->q_len && (bad(q) || bad(out) || bad(lse) || bad(dout) || bad(dq))) ||
      (a->k_len && (bad(k) || bad(v) || bad(dk) || bad(dv))))
    return MSD_E_ARG;
  const Plan pl = plan(*a);
  if (bad(workspace) && (a->q_len || pl.row_splits > 1)) return MSD_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Args p = args(*a, q, k, v);
  p.dout = view(dout, a->dout_stride);
  p.o = static_cast<const uint16_t*>(out);
  p.lse = const_cast<float*>(lse);
  p.delta = static_cast<float*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + up(4 * a->q_rows * a->n_heads));
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  const unsigned heads = unsigned(a->n_seqs) * a->n_kv_heads;
  with_head(a->d_head, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (a->q_len) {
      p.tiles = pl.dq_tiles;
      p.splits = 1;
      const dim3 grid(unsigned(pl.dq_tiles) * heads);
      if (pl.dq_waves == 4) hipLaunchKernelGGL((attn_dq<DP, 4>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((attn_dq<DP, 1>), grid, dim3(64), 0, s, p);
    }
    if (a->k_len) {
      p.tiles = pl.key_tiles;
      p.splits = pl.row_splits;
      hipLaunchKernelGGL((attn_dkv<DP>), dim3(unsigned(pl.key_tiles) * heads, pl.row_splits), dim3(256), 0, s, p);
    }
  });
  if (a->k_len && pl.row_splits > 1) {
    const int64_t n = int64_t(a->k_len) * a->n_kv_heads * (a->d_head / 8);
    hipLaunchKernelGGL(attn_sum_parts, dim3(unsigned(cdiv(n, 256)), a->n_seqs, 2), dim3(256), 0, s, p);
  }
  return launched();
}
