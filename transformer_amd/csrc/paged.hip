// The paged cache's operators (gfx950): a step's keys and values into their pages, attention of each sequence's newest tokens
// over its pages with or without the weight that each position receives, and eviction.
//
// Reference: model.py:122-147 (attention), :212-215 (the cache); the paged cache itself is only described there.
//
// New token i of a sequence of length L with n of them stands at position L - n + i and sees positions j <= L - n + i.  With
// c = scale log2(e), for every query head and its K/V head:
//   P_ij = 2^(c q_i.k_j - L_i), L_i = log2 sum_j 2^(c q_i.k_j);   O_i = sum_j P_ij v_j;   W'_j = W_j + sum_i P_ij
//
// Work is shared out on the host (msd_paged_plan), which has the lengths: lists of jobs that the device reads, with all that a
// job needs beside the pages, so that none of the attention's workgroups is empty or counts sequences.  (What follows it, joins and the
// weights of pieces and of chunks, is launched for the most rows, parts and positions that a sequence has, and ends where one has less.)  Row r of a sequence's group is position r / g,
// head r % g (see attn.hip, whose tiles these kernels use).
//   few rows (up to 32 of a group: a token, a few drafts): paged_few, then paged_finish where the keys are split or weights counted
//                                                   or, of few short sequences, paged_whole alone
//   more (a chunk of a prompt): paged_many, paged_finish where the keys are split, paged_weights where weights are counted
//
// Measured (us, kernels under a tracer):
//   paged_few       memory.  64 tokens over up to 16000 positions, 8 K/V heads of 128: 418, 6.4 TB/s of reads (24 over up to 8000, 16 heads, with
//                   weights: 187, 5.8 TB/s); 4 over up to 2000, 4 heads of 64: 4.9, a chain of plan, pages, rows
//   paged_whole     latency, then a CU's own rate of loads.  8 tokens over up to 512 positions, 4 K/V heads of 64, weights: 6.9 a pass; 32 over up
//                   to 1000, 8 heads of 128: 16
//   paged_many      the matrix cores' power.  2048 rows at 16384, 32 / 8 heads of 128: 477-526 by card, 980-1080 TFLOP/s of the products under
//                   the mask (a library's 8192^3 product: 1215-1242); 8 x 128 over up to 512, 16 / 4 heads of 64: 12, one round, a chain of tiles
//   paged_finish    latency: 4.4-8
//   paged_weights   LDS reads, and first loads where rows are few.  511 rows at 8191, 16 / 4 heads of 128: 27, 610 TFLOP/s
//   paged_append    memory.  28665 tokens, 8 heads of 128: 46 with pages out of the caches, a copy's rate and above
//   paged_select, paged_move   30000 positions of 64 heads: 25, latency of counts in LDS; 8000 rows each of 128: 93, a copy's rate
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <vector>

#include "../../include/mspaged.h"
#include "attn_tiles.h"
#include "internal.h"

namespace msp {
using namespace msa;

constexpr int kPage = MSD_PAGE;
constexpr int kFewRows = 32;      // of a group: paged_few
constexpr int kFewKeys = 32;      // keys of its tiles
constexpr int kManyRows = 32 * kWaves;
constexpr int kLongest = INT32_MAX - 65536;
constexpr int32_t kMagic = 0x70616731;

// Words of a plan behind the public ones: launches' sizes, then where the lists lie
enum {
  N_MANY = MSD_PLAN_RESERVED + 1, N_FEWS, N_TILES, N_MANYS, N_APPENDS, MANY_PARTS, FEW_ROWS, SCORES,
  AT_SEQS, AT_MANY, AT_TILES, AT_MANYS, AT_APPENDS, AT_TABLES,
  N_FEW, FEW_PARTS = N_FEW + 2, AT_FEW = FEW_PARTS + 2, AT_FEWS = AT_FEW + 2, END = AT_FEWS + 2   // two each: without, with weights
};
static_assert(END <= MSD_PLAN_HEADER, "the header's words");

// A piece of a sequence's keys against 32 of its rows (few) or 128 (many): tiles t0 .. t1 of 32 or 64 keys
struct Job {
  int q0, n, len, seq;
  int row0, t0, t1, slot;         // slot: where its part lies; paged_few: the lowest bit of row0 says whether it is the only one,
};                                // the others where the sequence's scores lie; paged_many: row0 < 0: the only one, of row -row0 - 1
struct SeqOf { int q0, n, len, zero; };
struct Few { int q0, n, len, seq, slot, parts, scores, zero; };
struct RowTile { int q0, n, len, seq, row0, slot, parts, tiles; };
struct Append { int row, count, position, zero; };   // rows `row` .. to the pool's positions `position` ..
static_assert(sizeof(Job) == 32 && sizeof(Few) == 32 && sizeof(RowTile) == 32 && sizeof(Append) == 16 && sizeof(SeqOf) == 16, "");

struct Pages {
  const uint16_t* p;
  int64_t head, row;              // strides in elements
};

struct Args {
  const uint16_t* q;
  int64_t q_row, q_head;
  Pages k, v;
  int D, H, KV, g;
  uint32_t g_magic;
  int g_shift;
  float c;
  int64_t q_rows;
  int n_seqs, width, longest, n_pages;
  const int32_t* tables;
  const Job *few, *many;
  int n_few, n_many;
  uint16_t* out;
  float *few_part, *few_lse;      // [slot][kv head][32] rows of D, logsumexps
  float *many_part, *many_lse;    // [slot][kv head][128]
  float* lse;                     // -L_i / c of every row of many, sequence by sequence, head by head, or null
  float* scores;                  // c q.k of few rows, [sequence][kv head][tile of 32 keys][row][key], or null
  int64_t score_words;
  const float* weights;
  int weights_width;
  float* weights_out;
};

// Scalar loads of what a plan says (it does not change while a kernel runs)
template <class T>
__device__ __forceinline__ T scalar_load(const T* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef const __attribute__((address_space(4))) uint32_t word;
  T x;
  uint32_t w[sizeof(T) / 4];
  word* from = (word*)(uintptr_t)p;
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(from[i]);
  __builtin_memcpy(&x, w, sizeof(T));
  return x;
#else
  return *p;
#endif
}

__device__ __forceinline__ int pick(int i, int a, int b, int c, int d) {   // (of values: of members it would become an array in memory)
  const int low = i & 1 ? b : a, high = i & 1 ? d : c;
  return i & 2 ? high : low;
}

// The host has checked its own numbers; device words that have been overwritten since must not lead out of anything.  (A sequence without
// new tokens has no rows and may start anywhere, behind the last row too.)
__device__ __forceinline__ bool sound(const Args& p, int q0, int n, int len, int seq) {
  return n >= 0 && (n == 0 || (q0 >= 0 && q0 <= p.q_rows - n)) && len >= n && len <= p.longest && seq >= 0 && seq < p.n_seqs;
}

__device__ __forceinline__ int tiles_of(int len, int keys) { return len / keys + (len % keys != 0); }

__device__ __forceinline__ int div_g(const Args& p, int r) { return div_by(r, p.g_magic, p.g_shift); }

__device__ __forceinline__ const uint16_t* row_at(const Args& p, int q0, int kvh, int pos, int of_group) {
  return p.q + int64_t(q0 + pos) * p.q_row + int64_t(kvh * p.g + of_group) * p.q_head;
}

// As dma(), of what is read once
__device__ __forceinline__ void dma_once(const uint16_t* base, uint32_t off, uint32_t to) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, 0x7fffffff, 0x00020000);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(to), "v"(off), "s"(r) : "m0");
#endif
}

// A tile of R positions on its way from pages to LDS, NW waves: an instruction's rows are 8 (or 4) of one page.
template <int DP, int R, int NW>
struct PagedTile {
  static constexpr int P = pitch<DP>(), C = P / 16, N = R * P / 1024 / NW, ROWS = 64 / C;   // rows of an instruction
  static constexpr int KINDS = NW * ROWS >= kPage ? 1 : kPage / (NW * ROWS);                // of offsets: the same rows of a page
  int row;               // of the first instruction
  uint32_t off[KINDS];   // from the page's start
  __device__ __forceinline__ void init(int64_t row_stride, int D, int lane, int wv) {
    row = ROWS * wv + lane / C;
#pragma unroll
    for (int u = 0; u < KINDS; ++u) {
      const int r = row + ROWS * NW * u, c = lane % C ^ swizzle<P>(r);
      off[u] = 8 * c < D ? uint32_t(r % kPage) * uint32_t(row_stride) * 2 + 16 * c : kOutside;
    }
  }
  // page(i): the tile's page i, of a head's pages at `head`; `left` of the tile's rows exist, the others are zeros
  template <class F>
  __device__ __forceinline__ void load(uint32_t to, int left, int wv, const uint16_t* head, int64_t row_stride, int n_pages, F page) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint32_t at = page((ROWS * wv + ROWS * NW * u) / kPage);
      const bool there = at < uint32_t(n_pages);
      dma_once(head + int64_t(there ? at : 0) * (kPage * row_stride), row + ROWS * NW * u < (there ? left : 0) ? off[u % KINDS] : kOutside,
          to + 1024 * (wv + NW * u));
    }
  }
};

// LDS reads of this wave are done (their memory may be written)
__device__ __forceinline__ void reads_done() {
#if defined(__HIP_DEVICE_COMPILE__)
  wave_lds_order();
  __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt 0
  wave_lds_order();
#endif
}
template <int N>
__device__ __forceinline__ void landed() {
  wave_lds_order();
  dma_wait<N>();
  wave_lds_order();
}

// One tile of 32 keys against 32 rows: scores, running maximum and sum, product with V.  The running maximum may lag by 2^8
// before the sums are rescaled.
template <int DP>
struct Rows {
  f32x16 o[DP / 32];
  float m, l;
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = f32x16{};
    m = -INFINITY;
    l = 0;
  }
  // s: c-scaled or raw scores of this lane's row against 16 keys
  __device__ __forceinline__ float new_maximum(const f32x16& s, float c) {
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top = fmaxf(top, swap_halves(top)) * c;
    if (__any(top > m + 8.0f)) {
      const float mn = fmaxf(m, top), by = mn == -INFINITY ? 1.0f : exp2_hw(m - mn);
      m = mn;
      l *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) o[d] *= by;
    }
    return m == -INFINITY ? 0.0f : m;
  }
  __device__ __forceinline__ void probabilities(f32x16& s, float c, float sub) {
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2_hw(fmaf(s[i], c, -sub));
      sum += s[i];
    }
    l += sum;
  }
  // The probabilities as two bf16, of which the second is what the first's rounding has taken off: to 2^-17.  A few rows wait for
  // memory, so the second product costs nothing; the output's own rounding is what is left (relative errors against 64 bits
  // 0.0017, with one product 0.0023 to 0.0026).
  __device__ __forceinline__ void add(const f32x16& s, const uint8_t* V, int row0, int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x8 pr = pack8(s, 8 * h);
      f32x16 off;
#pragma unroll
      for (int i = 0; i < 8; ++i) off[i] = s[8 * h + i] - float(pr[i]);
      const bf16x8 rest = pack8(off, 0);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        const bf16x8 v = cols_operand<pitch<DP>()>(V, row0 + 16 * h, d, lane);
        o[d] = mfma(v, pr, o[d]);
        o[d] = mfma(v, rest, o[d]);
      }
    }
  }
};

template <int DP>
__device__ __forceinline__ f32x16 scores_of(const uint8_t* K, int row0, const bf16x8 (&q)[DP / 16], int lane) {
  f32x16 s = {};
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) s = mfma(rows_operand<pitch<DP>()>(K, row0, ks, lane), q[ks], s);
  return s;
}

// ---- few rows ----
// The waves of a workgroup take a job's tiles in turn, each with LDS of its own that it fills itself, so that none waits for
// another before the end, where they are joined.
template <int DP, int W>
constexpr int few_lds() { return W * (4 * kFewKeys * pitch<DP>() + 256); }   // and two statistics of 32 rows a wave

// Workgroup `group` of few rows by W of its NW waves; the others take no tiles and meet them at the barrier
template <int DP, int W, int NW = W>
__device__ __forceinline__ void few_rows(const Args& p, int group, uint8_t* lds) {
  constexpr int P = pitch<DP>(), TILE = kFewKeys * P, OROW = DP + 4;
  float(*stats)[2][32] = reinterpret_cast<float(*)[2][32]>(lds + W * 4 * TILE);
  static_assert(4 * TILE >= 4 * 32 * OROW, "a wave's part of the output");
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = group % p.KV;
  const Job j = scalar_load(p.few + group / p.KV);
  const int R = j.n * p.g;
  if (!sound(p, j.q0, j.n, j.len, j.seq) || R > kFewRows || j.t0 < 0 || j.t1 < j.t0 || j.t1 > tiles_of(j.len, kFewKeys) || j.slot < 0 || j.slot >= p.n_few)
    return;
  const bool works = W == NW || wv < W;
  uint8_t* mine = lds + (works ? wv : 0) * 4 * TILE;
  const uint32_t to = lds_address(mine);
  const uint16_t *kb = p.k.p + kvh * p.k.head, *vb = p.v.p + kvh * p.v.head;
  const int32_t* table = p.tables + int64_t(j.seq) * p.width;
  PagedTile<DP, kFewKeys, 1> kt, vt;
  kt.init(p.k.row, p.D, lane, 0);
  vt.init(p.v.row, p.D, lane, 0);
  constexpr int HALF = decltype(kt)::N;
  auto pages_of = [&](int t) { return scalar_load(reinterpret_cast<const int2*>(table) + min(t, j.t1 - 1)); };
  auto load = [&](int2 pages, int t, int stage) {
    const int left = j.len - t * kFewKeys;
    auto page = [&](int i) { return pick(i, pages.x, pages.y, 0, 0); };
    kt.load(to + stage * 2 * TILE, left, 0, kb, p.k.row, p.n_pages, page);
    vt.load(to + stage * 2 * TILE + TILE, left, 0, vb, p.v.row, p.n_pages, page);
  };
  int t = works ? j.t0 + wv : j.t1;
  int2 pages{};   // of the next tile: asked for a tile ahead, as nothing can be fetched before they are there
  if (t < j.t1) {
    const int2 now = pages_of(t);
    pages = pages_of(t + W);
    load(now, t, 0);
  }
  const int r = lane & 31, pos = div_g(p, min(r, R - 1));
  const bool ok = works && r < R;
  bf16x8 q[DP / 16];
  row_operands<DP>(q, p.q, row_at(p, j.q0, kvh, pos, ok ? r - pos * p.g : 0) - p.q, ok, p.D, lane);
  const int first = j.len - j.n + 1, seen = first + pos;   // keys that the first row sees, that this one sees
  const int padded = tiles_of(j.len, kFewKeys) * kFewKeys;
  const int64_t scores_at = int64_t(j.row0 >> 1) * kFewKeys * p.KV + int64_t(kvh) * R * padded;
  const bool keep = p.scores && scores_at >= 0 && scores_at + int64_t(R) * padded <= p.score_words;
  float* scores = keep ? p.scores + scores_at + r * kFewKeys + 4 * (lane >> 5) : nullptr;

  Rows<DP> x;
  x.start();
  dma_wait();   // (for q, so that the compiler does not wait for all loads in the loop)
  for (int stage = 0; t < j.t1; t += W, stage ^= 1) {
    const uint8_t *K = mine + stage * 2 * TILE, *V = K + TILE;
    const bool more = t + W < j.t1;
    if (more) {
      reads_done();
      load(pages, t + W, stage ^ 1);
      pages = pages_of(t + 2 * W);
      landed<3 * HALF>();
    } else {
      landed<HALF>();
    }
    f32x16 s = scores_of<DP>(K, 0, q, lane);
    const int key0 = t * kFewKeys;
    if (key0 + kFewKeys > first) {
      const int left = seen - key0 - 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + (i & 3) >= left) s[i] = -INFINITY;
    }
    const float sub = x.new_maximum(s, p.c);
    if (keep && ok)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<f32x4*>(scores + int64_t(t) * R * kFewKeys + 8 * u) = f32x4{s[4 * u] * p.c, s[4 * u + 1] * p.c, s[4 * u + 2] * p.c, s[4 * u + 3] * p.c};
    x.probabilities(s, p.c, sub);
    if (keep) {   // (its four stores are behind the loads of V: waited for with them they took a quarter of the time)
      if (more) landed<2 * HALF + 4>();
      else landed<4>();
    } else {
      if (more) landed<2 * HALF>();
      else landed<0>();
    }
    x.add(s, V, 0, lane);
  }
  x.l += swap_halves(x.l);
  // the waves' parts, joined
  if (works) {
    reads_done();
    float* part = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<f32x4*>(part + r * OROW + 32 * d + 8 * u + 4 * (lane >> 5)) =
            f32x4{x.o[d][4 * u], x.o[d][4 * u + 1], x.o[d][4 * u + 2], x.o[d][4 * u + 3]};
    if (lane < 32) {
      stats[wv][0][r] = x.m;
      stats[wv][1][r] = x.l;
    }
  }
  __syncthreads();
  const bool only = j.row0 & 1;
  if (!only && !p.few_part) return;   // (overwritten device words)
  const int64_t slot = (int64_t(j.slot) * p.KV + kvh) * kFewRows;
  const int pieces = p.D / 4;
  for (int i = tid; i < R * pieces; i += 64 * NW) {
    const int row = i / pieces, c = i - row * pieces;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, stats[w][0][row]);
    float l = 0;
    f32x4 o = {};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float lw = stats[w][1][row], e = lw == 0 ? 0.0f : exp2_hw(stats[w][0][row] - m);   // (a NaN sum stays one)
      l = fmaf(e, lw, l);
      o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * 4 * TILE) + row * OROW + 4 * c) * e;
    }
    o *= l == 0 ? 0.0f : 1.0f / l;
    if (!only) {
      *reinterpret_cast<f32x4*>(p.few_part + (slot + row) * p.D + 4 * c) = o;
    } else {
      const int at = div_g(p, row);
      *reinterpret_cast<u32x2*>(p.out + (int64_t(j.q0 + at) * p.H + kvh * p.g + row - at * p.g) * p.D + 4 * c) =
          u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
    }
    if (c == 0 && (!only || p.scores)) p.few_lse[slot + row] = l == 0 ? INFINITY : m + __log2f(l);
  }
}

// ---- many rows ----
// 128 rows a workgroup, 32 a wave, tiles of 64 keys, each in two halves.  While the softmax of a half is formed (vector units), the
// matrix cores form the scores of the half behind it and the product of the half before it with V: three independent pieces of
// work in one stretch of code.  A wave issues an instruction every four cycles or more, and two of them share a SIMD, so what is not a
// product counts by its instructions.  Hence: each wave fetches from one page of a tile, whose descriptor ends with the rows that
// exist; LDS places are constants (the loop's body is there for even and odd tiles); addresses within a place are kept.
//
// Wave w fetches page w of a tile, rows r of it with r < 8 to the tile's first half and the others to its second: instruction u of
// ROWS rows lies, in the half, behind those of the waves before it.  So the first half's keys are the first eight of each
// page.  In a half, LDS row x (a score's register and lane half) is key key_of(x) of the tile, plus 8 in the second.
template <int DP>
struct HalfTile {
  static constexpr int P = pitch<DP>(), C = P / 16, ROWS = 64 / C, N = kPage / 2 / ROWS, BYTES = 32 * P;   // N instructions a wave
  uint32_t off, step;   // of this lane in a page, and from one instruction's rows to the next
  __device__ __forceinline__ void init(int64_t row_stride, int D, int lane, int wv) {
    const int i = lane / C, c = lane % C ^ swizzle<P>(ROWS * wv + i);
    step = ROWS * uint32_t(row_stride) * 2;
    off = 8 * c < D ? uint32_t(i) * uint32_t(row_stride) * 2 + 16 * c : kOutside;
  }
  // the key of register i (of a score) of lanes 0 .. 31; those of the others lie kLanes behind
  static constexpr int kLanes = P == 128 ? 4 : kPage;
  static constexpr int key_of(int i) { return P == 128 ? kPage * (i / 4) + i % 4 : kPage * 2 * (i / 4 % 2) + 4 * (i / 8) + i % 4; }
};
// The rows (0 .. 16) of a page's positions of a head that exist, as a buffer
struct PageRows {
  const uint16_t* p;
  uint32_t bytes;
};
template <int DP, int HALF>
__device__ __forceinline__ void load_half(const HalfTile<DP>& x, const PageRows& page, uint32_t to) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(page.p), 0, page.bytes, 0x00020000);
#pragma unroll
  for (int u = 0; u < HalfTile<DP>::N; ++u)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to + 4096 * u),
                 "v"(x.off + (HALF * HalfTile<DP>::N + u) * x.step), "s"(r) : "m0");
#endif
}

// Nothing moves across
__device__ __forceinline__ void order_steps() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// Workgroup `group` of many rows; lds: four halves of K, four of V
template <int DP>
__device__ __forceinline__ void many_rows(const Args& p, int group, uint8_t* lds) {
  using Half = HalfTile<DP>;
  constexpr int P = pitch<DP>(), BYTES = Half::BYTES, KS = DP / 16, DB = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = group % p.KV;
  const Job j = scalar_load(p.many + group / p.KV);
  const int rows = j.n * p.g, row0 = j.row0 < 0 ? -j.row0 - 1 : j.row0;
  const bool only = j.row0 < 0;
  if (!sound(p, j.q0, j.n, j.len, j.seq) || row0 >= rows || j.t0 < 0 || j.t1 <= j.t0 || j.t1 > tiles_of(j.len, kKeys) || j.slot < 0 || j.slot >= p.n_many)
    return;
  const uint16_t *kb = p.k.p + kvh * p.k.head, *vb = p.v.p + kvh * p.v.head;
  const int32_t* table = p.tables + int64_t(j.seq) * p.width;
  Half kt, vt;
  kt.init(p.k.row, p.D, lane, wv);
  vt.init(p.v.row, p.D, lane, wv);
  const uint32_t k_row = uint32_t(p.k.row) * 2, v_row = uint32_t(p.v.row) * 2;   // (16 rows span less than 2^31 bytes)
  auto page_of = [&](int t) { return scalar_load(table + min(t * (kKeys / kPage) + wv, p.width - 1)); };
  // this wave's page of tile t: rows that the job reads
  auto rows_in = [&](int t, int page) {
    return t < j.t0 || t >= j.t1 || uint32_t(page) >= uint32_t(p.n_pages) ? 0 : min(max(j.len - t * kKeys - kPage * wv, 0), kPage);
  };
  // (to the last row's end: rows may be nearer to each other than they are long.  What a row behind the last then reads lies within those
  // that are there, its scores are masked)
  auto page_rows = [&](const uint16_t* head, uint32_t row, int page, int n) {
    return PageRows{head + (uint64_t(uint32_t(n ? page : 0)) * (kPage * row) >> 1), n * row + min(n, 1) * (2 * p.D - row)};
  };
  auto k_page = [&](int t, int page) { return page_rows(kb, k_row, page, rows_in(t, page)); };
  auto v_page = [&](int t, int page) { return page_rows(vb, v_row, page, rows_in(t, page)); };
  const uint32_t mine = lds_address(lds) + 1024 * wv;
  auto k_place = [&](int i) { return mine + (i & 3) * BYTES; };
  auto v_place = [&](int i) { return mine + (4 + (i & 3)) * BYTES; };
  // half i of K and V (counted from the job's first tile) lies in place i % 4; an iteration reads K's halves 2 t + 1 and 2 t + 2, V's
  // 2 t - 1 (zeros before the first) and 2 t, and fetches the next two of each
  int page1 = page_of(j.t0 + 1), page2 = page_of(j.t0 + 2);
  PageRows k1, v0;   // of tile t + 1 and t
  {
    const int page = page_of(j.t0);
    const PageRows k0 = k_page(j.t0, page);
    v0 = v_page(j.t0, page);
    k1 = k_page(j.t0 + 1, page1);
    load_half<DP, 0>(kt, k0, k_place(0));
    load_half<DP, 1>(kt, k0, k_place(1));
    load_half<DP, 0>(kt, k1, k_place(2));
    load_half<DP, 1>(vt, PageRows{vb, 0}, v_place(3));
    load_half<DP, 0>(vt, v0, v_place(0));
  }
  const int r = row0 + 32 * wv + (lane & 31), pos = div_g(p, min(r, rows - 1));
  const bool ok = r < rows;
  bf16x8 q[KS];
  row_operands<DP>(q, p.q, row_at(p, j.q0, kvh, pos, ok ? r - pos * p.g : 0) - p.q, ok, p.D, lane);
  const int first = j.len - j.n + 1, seen = first + pos, wave_full = first + div_g(p, min(row0 + 32 * wv, rows - 1));

  // where this lane reads in a half's rows: the operands of 32 keys (K), of 32 columns (V: the first and the second eight rows)
  uint32_t k_at[KS], v_at[2][DB];
  const uint32_t base = lds_address(lds);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) k_at[ks] = base + piece_at<P>(lane & 31, 2 * ks + (lane >> 5));
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = lane & 15, x = 8 * h + 4 * (lane >> 5) + (t >> 2), c = 4 * d + 2 * ((lane >> 4) & 1) + ((t & 3) >> 1);
      v_at[h][d] = base + 4 * BYTES + piece_at<P>(x, c) + 8 * (t & 1);
    }
#if defined(__HIP_DEVICE_COMPILE__)   // (kept in registers: formed again at each read they cost a quarter of the loop's vector instructions)
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm("" : "+v"(k_at[ks]));
#pragma unroll
  for (int d = 0; d < 2 * DB; ++d) asm("" : "+v"(v_at[d / DB][d % DB]));
#endif
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  typedef __attribute__((address_space(3))) const bf16x8 lds_bf16x8;
#else
  typedef s16x4 lds_s16x4;
  typedef const bf16x8 lds_bf16x8;
#endif
  f32x16 o[DB] = {};
  float m = -INFINITY, l = 0;   // running maximum of c s, up to 2^8 too small; sum of 2^(c s - m) over this lane's keys
  // The half before, as operands: one bf16 of each probability, off by up to 2^-8 of it (outputs 0.0023 from 64 bits where their own rounding
  // leaves 0.0017), as in attn.hip.  A second one, as few rows have it, would be half as many matrix products again, which are what
  // bounds these.  The sums and the weights are of the f32 values.
  bf16x8 pr[2] = {};
  // operand n of a half: K's for the scores, then V's for the product
  auto operand = [&](int n, int k, int v) {
#if defined(__HIP_DEVICE_COMPILE__)
    if (n < KS) return *(lds_bf16x8*)(k_at[n] + k * BYTES);
    const int h = (n - KS) / DB, d = (n - KS) % DB;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v_at[0][d] + v * BYTES + 16 * h * P));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v_at[1][d] + v * BYTES + 16 * h * P));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
    return bf16x8{};
#endif
  };
  auto scores = [&](int place) {
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma(operand(ks, place, 0), q[ks], s);
    return s;
  };
  auto product = [&](int place) {
#pragma unroll
    for (int n = 0; n < 2 * DB; ++n) o[n % DB] = mfma(operand(KS + n, 0, place), pr[n / DB], o[n % DB]);
  };
  // s: the scores of half `second` of tile t; ahead: those of the half behind it, in K's place k; the half before is V's place v.
  // Step by step: a matrix product, the operand of the one after the next, a share of the softmax (left to itself the compiler waits
  // for each operand in turn and forms the softmax after all products).
  constexpr int STEPS = KS + 2 * DB, AHEAD = 2;
  auto half = [&](f32x16& s, f32x16& ahead, int t, int second, int k, int v) {
    if (t * kKeys + kKeys > wave_full) {   // the diagonal or the end
      const int left = seen - t * kKeys - 8 * second - Half::kLanes * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (Half::key_of(i) >= left) s[i] = -INFINITY;
    }
    bf16x8 f[AHEAD + 1], next[2];
    float top = s[0], sum = 0, by = 1, sub = 0;
    bool grown = false;
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) f[n] = operand(n, k, v);
    ahead = f32x16{};
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      if (n + AHEAD < STEPS) f[(n + AHEAD) % (AHEAD + 1)] = operand(n + AHEAD, k, v);
      const bf16x8 x = f[n % (AHEAD + 1)];
      if (n < KS) ahead = mfma(x, q[n], ahead);
      else o[(n - KS) % DB] = mfma(x, pr[(n - KS) / DB], o[(n - KS) % DB]);
      if (n < 2) {
#pragma unroll
        for (int i = 8 * n + (n == 0); i < 8 * n + 8; ++i) top = __builtin_elementwise_maximum(top, s[i]);
      } else if (n == 2) {
        top = __builtin_elementwise_maximum(top, swap_halves(top)) * p.c;
        grown = __any(top > m + 8.0f);   // rescaling by less than 2^8 can wait: f32 sums and bf16 P keep their precision
        const float mn = grown ? fmaxf(m, top) : m;
        by = mn == -INFINITY ? 1.0f : exp2_hw(m - mn);
        sub = mn == -INFINITY ? 0.0f : mn;
        m = mn;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (3 + i * (STEPS - 3) / 16 == n) {
            s[i] = exp2_hw(fmaf(s[i], p.c, -sub));
            sum += s[i];
            if (i == 7) next[0] = pack8(s, 0);
            if (i == 15) next[1] = pack8(s, 8);
          }
      }
      order_steps();
    }
    l = fmaf(l, by, sum);
    pr[0] = next[0];
    pr[1] = next[1];
#if defined(__HIP_DEVICE_COMPILE__)   // (formed above, not behind the branch)
    asm volatile("" : "+v"(pr[0]), "+v"(pr[1]), "+v"(l));
#endif
    if (grown)
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= by;
  };

  f32x16 s0, s1;
  dma_wait();   // (for q too, so that the compiler does not wait for all loads in the loop)
  __syncthreads();
  s0 = scores(0);
  __syncthreads();   // (the first place is fetched to next)
  auto tile = [&](auto odd, int t) {
    constexpr int X = 2 * decltype(odd)::value;
    const PageRows k2 = k_page(t + 2, page2), v1 = v_page(t + 1, page1);
    load_half<DP, 1>(kt, k1, k_place(X + 3));
    load_half<DP, 0>(kt, k2, k_place(X + 4));
    load_half<DP, 1>(vt, v0, v_place(X + 1));
    load_half<DP, 0>(vt, v1, v_place(X + 2));
    k1 = k2;
    v0 = v1;
    page1 = page2;
    page2 = page_of(t + 3);
    half(s0, s1, t, 0, X + 1, (X + 3) & 3);
    half(s1, s0, t, 1, (X + 2) & 3, X);
    dma_wait();
    __syncthreads();
  };
  int t = j.t0;
  for (; t + 1 < j.t1; t += 2) {
    tile(std::integral_constant<int, 0>(), t);
    tile(std::integral_constant<int, 1>(), t + 1);
  }
  if (t < j.t1) {
    tile(std::integral_constant<int, 0>(), t);
    product(1);
  } else {
    product(3);
  }
  __syncthreads();   // (the tiles are read, the rows are staged in their place)
  l += swap_halves(l);
  const float by = l == 0 ? 0.0f : 1.0f / l;   // (a NaN sum stays one)
  const float lse = l == 0 ? INFINITY : m + __log2f(l);
  if (!only) {   // a normalised part and its weight, joined by paged_finish
    if (ok && p.many_part) {
      const int64_t row = (int64_t(j.slot) * p.KV + kvh) * kManyRows + 32 * wv + (lane & 31);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = 32 * d + 8 * u + 4 * (lane >> 5);
          if (c < p.D)
            *reinterpret_cast<f32x4*>(p.many_part + row * p.D + c) =
                f32x4{o[d][4 * u] * by, o[d][4 * u + 1] * by, o[d][4 * u + 2] * by, o[d][4 * u + 3] * by};
        }
      if (lane < 32) p.many_lse[row] = lse;
    }
    return;
  }
  if (p.lse && ok && lane < 32) p.lse[int64_t(j.q0) * p.H + int64_t(kvh * p.g + r - pos * p.g) * j.n + pos] = -lse / p.c;
  const int r0 = r - (lane & 31);
  store_rows<DP>(lds + wv * 32 * P, o, by, p.D, lane, [&](int i) -> uint16_t* {
    if (r0 + i >= rows) return nullptr;
    const int at = div_g(p, r0 + i);
    return p.out + (int64_t(j.q0 + at) * p.H + (kvh * p.g + (r0 + i - at * p.g))) * p.D;
  });
}

// Four waves at every head size (of heads above 64 one workgroup a CU; of two waves each and two a CU, 256 positions of 8 sequences took
// 8.6 us in place of 7.4, 64 sequences of up to 16000 the same)
template <int DP>
__global__ __launch_bounds__(64 * kWaves, DP <= 64 ? 2 : 1) void paged_few(Args p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds<DP, kWaves>()];
  few_rows<DP, kWaves>(p, blockIdx.x, lds);
}
template <int DP>
constexpr int many_lds() { return 8 * HalfTile<DP>::BYTES; }
template <int DP>
__global__ __launch_bounds__(64 * kWaves, DP <= 64 ? 3 : 2) void paged_many(Args p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[many_lds<DP>()];
  many_rows<DP>(p, blockIdx.x, lds);
}
// A step of both: tokens' workgroups, which wait for memory, spread among the chunks', which wait for the matrix cores.  The tokens' LDS is the
// larger: 66,560 bytes where heads are up to 64, of which two workgroups share a CU in place of three of the chunks' 32,768; 66,048 (65,536)
// above.  It pays all the same: chunks of 333 and 248 and six tokens over up to 2900 positions take 33.0 us, in calls of their own 27.2 and 9.9
// (16 / 4 heads of 64); 24.2, 20.4 and 10.5 (6 / 2 heads of 96).
template <int DP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_both(Args p) {
  constexpr int W = DP <= 64 ? kWaves : 2;
  __shared__ __attribute__((aligned(16))) uint8_t lds[std::max(few_lds<DP, W>(), many_lds<DP>())];
  const uint32_t few = p.n_few * p.KV, b = blockIdx.x, before = uint32_t(uint64_t(b) * few / gridDim.x);
  if (uint32_t(uint64_t(b + 1) * few / gridDim.x) > before) {
    few_rows<DP, W, kWaves>(p, before, lds);
  } else {
    many_rows<DP>(p, b - before, lds);
  }
}

// ---- few rows of few short sequences ----
// One workgroup of eight waves a sequence and K/V head, whose waves take up to four tiles each as in few_rows: no pieces to be joined by
// another launch, and the weights at once, from scores that stay in registers.  Latency bound: the plan, the pages, the first tiles,
// two joins in LDS.  (Keys straight into registers as operands, lanes by rows, took 11.5 us where this takes 6.9; 16 waves 11.)
constexpr int kWholeWaves = 8, kWholeTiles = 4;   // tiles of a wave
template <int DP>
constexpr int whole_rows() { return DP <= 64 ? 32 : 16; }   // (by the LDS for their joining)

template <int DP, bool WEIGHTED>
__global__ __launch_bounds__(64 * kWholeWaves) void paged_whole(Args p, const Few* fews) {
  constexpr int W = kWholeWaves, T = kWholeTiles, RS = whole_rows<DP>(), P = pitch<DP>(), TILE = kFewKeys * P, OROW = DP + 4, PROW = kFewKeys + 4;
  constexpr int STAGES = DP <= 64 ? 2 : 1, MINE = 2 * STAGES * TILE;
  static_assert(MINE >= RS * (OROW + PROW) * 4, "a wave's part of the output, and its probabilities");
  __shared__ __attribute__((aligned(16))) uint8_t lds[W * MINE];
  __shared__ __attribute__((aligned(16))) float stats[2][RS][W + 4];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), kvh = blockIdx.x % p.KV;
  const Few f = scalar_load(fews + blockIdx.x / p.KV);
  const int R = f.n * p.g;
  if (!sound(p, f.q0, f.n, f.len, f.seq) || R > RS || f.len > W * T * kFewKeys) return;
  const int tiles = R ? tiles_of(f.len, kFewKeys) : 0, r = lane & 31;
  uint8_t* mine = lds + wv * MINE;
  const int64_t row = int64_t(f.seq) * p.KV + kvh;
  float old[T] = {};
  if constexpr (WEIGHTED)
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int key = kFewKeys * (wv + W * i) + r;
      if (key < f.len - f.n && key < p.weights_width) old[i] = p.weights[row * p.weights_width + key];
    }
  Rows<DP> x;
  x.start();
  f32x16 s[T];
  const int pos = div_g(p, min(r, max(R - 1, 0)));
  const bool ok = r < R;
  if (wv < tiles) {
    const uint16_t *kb = p.k.p + kvh * p.k.head, *vb = p.v.p + kvh * p.v.head;
    const int32_t* table = p.tables + int64_t(f.seq) * p.width;
    const uint32_t to = lds_address(mine);
    PagedTile<DP, kFewKeys, 1> kt, vt;
    kt.init(p.k.row, p.D, lane, 0);
    vt.init(p.v.row, p.D, lane, 0);
    constexpr int HALF = decltype(kt)::N;
    int2 pages[T];
#pragma unroll
    for (int i = 0; i < T; ++i) pages[i] = scalar_load(reinterpret_cast<const int2*>(table) + min(wv + W * i, tiles - 1));
    auto there = [&](int i) { return i < T && wv + W * i < tiles; };
    auto load = [&](const PagedTile<DP, kFewKeys, 1>& tile, const uint16_t* head, int64_t stride, int i, int which) {
      tile.load(to + (i % STAGES * 2 + which) * TILE, f.len - kFewKeys * (wv + W * i), 0, head, stride, p.n_pages,
                [&](int h) { return pick(h, pages[i].x, pages[i].y, 0, 0); });
    };
    auto load_k = [&](int i) { load(kt, kb, p.k.row, i, 0); };
    auto load_v = [&](int i) { load(vt, vb, p.v.row, i, 1); };
    load_k(0);
    load_v(0);
    bf16x8 q[DP / 16];
    row_operands<DP>(q, p.q, row_at(p, f.q0, kvh, pos, ok ? r - pos * p.g : 0) - p.q, ok, p.D, lane);
    if (STAGES == 2 && there(1)) {
      load_k(1);
      load_v(1);
    }
    const int first = f.len - f.n + 1, seen = first + pos;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      if (!there(i)) break;
      const uint8_t *K = mine + i % STAGES * 2 * TILE, *V = K + TILE;
      const bool more = there(i + 1);
      if (STAGES == 2 && more) landed<3 * HALF>();
      else landed<HALF>();
      f32x16 now = scores_of<DP>(K, 0, q, lane);
      if (STAGES == 1 && more) {
        reads_done();
        load_k(i + 1);
      }
      const int key0 = (wv + W * i) * kFewKeys;
      if (key0 + kFewKeys > first) {
        const int left = seen - key0 - 4 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (8 * (e >> 2) + (e & 3) >= left) now[e] = -INFINITY;
      }
      const float sub = x.new_maximum(now, p.c);
      if constexpr (WEIGHTED) s[i] = now;
      x.probabilities(now, p.c, sub);
      if (more) landed<STAGES * HALF>();
      else landed<0>();
      x.add(now, V, 0, lane);
      if (there(i + STAGES)) {
        reads_done();
        if (STAGES == 2) load_k(i + 2);
        load_v(i + STAGES);
      }
    }
    x.l += swap_halves(x.l);
  }
  if (lane < RS) {
    stats[0][r][wv] = x.m;
    stats[1][r][wv] = x.l;
  }
  __syncthreads();
  // the row's statistics, from all waves'; what this wave's part counts
  float m = -INFINITY, l = 0;
  {
    const int of = lane % RS;
    float ms[W], ls[W];
#pragma unroll
    for (int w = 0; w < W; w += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(&stats[0][of][w]), b = *reinterpret_cast<const f32x4*>(&stats[1][of][w]);
#pragma unroll
      for (int i = 0; i < 4; ++i) ms[w + i] = a[i], ls[w + i] = b[i];
    }
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, ms[w]);
#pragma unroll
    for (int w = 0; w < W; ++w) l = fmaf(ls[w] == 0 ? 0.0f : exp2_hw(ms[w] - m), ls[w], l);   // (a NaN sum stays one)
  }
  const float by = (x.l == 0 ? 0.0f : exp2_hw(x.m - m)) * (l == 0 ? 0.0f : 1.0f / l);
  float* part = reinterpret_cast<float*>(mine);
  if (ok)
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<f32x4*>(part + r * OROW + 32 * d + 8 * u + 4 * (lane >> 5)) =
            f32x4{x.o[d][4 * u] * by, x.o[d][4 * u + 1] * by, x.o[d][4 * u + 2] * by, x.o[d][4 * u + 3] * by};
  __syncthreads();
  const int pieces = p.D / 4;
  for (int i = tid; i < R * pieces; i += 64 * W) {
    const int of = i / pieces, c = i - of * pieces;
    f32x4 o = {};
#pragma unroll
    for (int w = 0; w < W; ++w) o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * MINE) + of * OROW + 4 * c);
    const int at = div_g(p, of);
    *reinterpret_cast<u32x2*>(p.out + (int64_t(f.q0 + at) * p.H + kvh * p.g + of - at * p.g) * p.D + 4 * c) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
  }
  if constexpr (WEIGHTED) {
    const float lse = l == 0 ? INFINITY : m + __log2f(l);
    float* here = part + RS * OROW;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int t = wv + W * i, key = kFewKeys * t + r;
      float sum = 0;
      if (t < tiles) {
        if (ok)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            f32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = exp2_hw(fmaf(s[i][4 * u + e], p.c, -lse));
            *reinterpret_cast<f32x4*>(here + r * PROW + 8 * u + 4 * (lane >> 5)) = w;
          }
        reads_done();
#pragma unroll 4
        for (int of = 0; of < R; ++of) sum += here[of * PROW + r];
        reads_done();
      }
      if (lane < 32 && key < p.longest) p.weights_out[row * p.longest + key] = key < f.len ? old[i] + sum : 0.0f;
    }
  }
}

// ---- what is left ----
// Workgroups, in this order: four rows of a row tile of many; four rows of a sequence of few; 1024 positions' weights of such.
constexpr int kFinish = 256, kWeightKeys = 4 * kFinish, kJoinRows = 4;

// Rows `rows` (up to four) from their parts' normalised outputs, weighted by 2^(lse_z - lse): 16 lanes a row's 8-value
// pieces, G of them in turn over the parts, joined through LDS in order.
__device__ __forceinline__ void join(const Args& p, float (*lds)[11], const float* part, const float* lse, int64_t stride, int parts, int rows,
                                     int q0, int n, int row0, int kvh, bool keep) {
  const int tid = threadIdx.x, c = tid % 16;
  const int shift = rows > 2 ? 2 : rows > 1 ? 3 : 4, G = 1 << shift, zg = tid / 16 % G, row = tid / 16 >> shift;
  const bool ok = row < rows && 8 * c < p.D;
  float m = -INFINITY, l = 0, acc[8] = {};
  if (ok)
#pragma unroll 4
    for (int z = zg; z < parts; z += G) {
      const float x = lse[z * stride + row];
      const float* from = part + (z * stride + row) * p.D + 8 * c;
      const f32x4 a = *reinterpret_cast<const f32x4*>(from), b = *reinterpret_cast<const f32x4*>(from + 4);
      // (infinite: nothing seen in this part; no branch, so that the next parts' loads need not wait; a NaN stays one through e)
      const float mn = x == INFINITY ? m : fmaxf(m, x);
      const float old = m == -INFINITY ? 0.0f : exp2_hw(m - mn), e = x == INFINITY ? 0.0f : exp2_hw(x - mn);
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
  for (int g = 0; g < G; ++g) m = fmaxf(m, lds[tid + 16 * g][0]);
  l = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0;
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
  for (int i = 0; i < 4; ++i) x[i] = pack2(acc[2 * i] * by, acc[2 * i + 1] * by);
  const int pos = div_g(p, row0 + row), head = kvh * p.g + row0 + row - pos * p.g;
  *reinterpret_cast<u32x4*>(p.out + (int64_t(q0 + pos) * p.H + head) * p.D + 8 * c) = x;
  if (keep && c == 0) p.lse[int64_t(q0) * p.H + int64_t(head) * n + pos] = l == 0 ? -INFINITY : -(m + __log2f(l)) / p.c;
}

__global__ __launch_bounds__(kFinish) void paged_finish(Args p, const RowTile* tiles, int n_tiles, const Few* fews, int n_fews, int few_joins, int join_rows) {
  __shared__ float lds[kFinish][11];
  __shared__ float row_lse[kFewRows];
  constexpr int kSubs = kManyRows / kJoinRows;
  const int tid = threadIdx.x;
  int id = blockIdx.x;
  if (id < n_tiles * p.KV * kSubs) {
    const int kvh = id % p.KV, sub = id / p.KV % kSubs;
    const RowTile t = scalar_load(tiles + id / p.KV / kSubs);
    const int row0 = t.row0 + kJoinRows * sub, rows = min(t.n * p.g - row0, kJoinRows);
    if (!sound(p, t.q0, t.n, t.len, t.seq) || t.row0 < 0 || t.row0 >= t.n * p.g || rows <= 0 || t.parts < 2 || t.slot < 0 || t.slot > p.n_many - t.parts) return;
    const int64_t at = (int64_t(t.slot) * p.KV + kvh) * kManyRows + kJoinRows * sub;
    join(p, lds, p.many_part + at * p.D, p.many_lse + at, int64_t(p.KV) * kManyRows, t.parts, rows, t.q0, t.n, row0, kvh, p.lse);
    return;
  }
  id -= n_tiles * p.KV * kSubs;
  const int joins = n_fews * p.KV * few_joins;
  const bool weigh = id >= joins;
  if (weigh) id -= joins;
  const int kvh = id % p.KV, nth = id / p.KV / n_fews;
  const Few f = scalar_load(fews + id / p.KV % n_fews);
  const int R = f.n * p.g;
  if (!sound(p, f.q0, f.n, f.len, f.seq) || R > kFewRows || f.parts < 0 || f.slot < 0 || f.slot > p.n_few - f.parts) return;
  const int64_t at = (int64_t(f.slot) * p.KV + kvh) * kFewRows, stride = int64_t(p.KV) * kFewRows;
  if (!weigh) {
    const int row0 = join_rows * nth, rows = min(R - row0, join_rows);
    if (f.parts > 1 && rows > 0)
      join(p, lds, p.few_part + (at + row0) * p.D, p.few_lse + at + row0, stride, f.parts, rows, f.q0, f.n, row0, kvh, false);
    return;
  }
  // the rows' logsumexps, from their parts': eight lanes a row
  {
    const int row = tid / 8;
    float m = -INFINITY, l = 0;
    if (row < R)
      for (int z = tid % 8; z < f.parts; z += 8) {
        const float x = p.few_lse[at + z * stride + row];
        if (x == INFINITY) continue;
        const float mn = fmaxf(m, x);
        l = fmaf(l, exp2_hw(m - mn), exp2_hw(x - mn));
        m = mn;
      }
#pragma unroll
    for (int w = 1; w < 8; w *= 2) {
      const float m2 = __shfl_xor(m, w), l2 = __shfl_xor(l, w), mn = fmaxf(m, m2);
      l = (l == 0 ? 0.0f : l * exp2_hw(m - mn)) + (l2 == 0 ? 0.0f : l2 * exp2_hw(m2 - mn));
      m = mn;
    }
    if (row < kFewRows && tid % 8 == 0) row_lse[row] = l == 0 ? INFINITY : m + __log2f(l);
  }
  __syncthreads();
  const int key = nth * kWeightKeys + 4 * tid;
  if (key >= p.longest) return;
  const int padded = tiles_of(f.len, kFewKeys) * kFewKeys;
  float w[4] = {};
  if (key < f.len) {
    const int64_t row = int64_t(f.seq) * p.KV + kvh;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (key + i < f.len - f.n && key + i < p.weights_width) w[i] = p.weights[row * p.weights_width + key + i];
    const int64_t base = int64_t(f.scores) * kFewKeys * p.KV + int64_t(kvh) * R * padded;
    if (base >= 0 && base + int64_t(R) * padded <= p.score_words) {
      f32x4 sum = {};
#pragma unroll 4
      for (int r = 0; r < R; ++r) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(p.scores + base + (int64_t(key / kFewKeys) * R + r) * kFewKeys + key % kFewKeys);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += exp2_hw(s[i] - row_lse[r]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + i < f.len) w[i] += sum[i];
    }
  }
  float* out = p.weights_out + (int64_t(f.seq) * p.KV + kvh) * p.longest + key;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + i < p.longest) out[i] = w[i];
}

// ---- the weights of many rows ----
// 128 keys a workgroup, 32 a wave in registers, over the group's heads and the rows that see them: S = Q K^T, a lane holds one
// key's scores against 16 rows, so that its sum stays in the lane; a row's scores start as -L_i / c (what p.lse holds here).  Four
// teams of four waves take the tiles of 64 rows in turn.  While the probabilities of 32 rows are formed, the matrix cores form the
// next 32 rows' scores.
constexpr int kHalves = 4;
template <int DP>
__global__ __launch_bounds__(64 * kWaves * kHalves) void paged_weights(Args p, const Job* seqs, int n_seqs) {
  constexpr int P = pitch<DP>(), R = 64, TILE = R * P, STAGE = TILE + 256 * kWaves, STAGES = 2, KS = DP / 16;
  constexpr int LOADS = TILE / 1024 / kWaves + 1;   // of a wave and stage: rows, and their logsumexps, of which each wave has its own
  __shared__ __attribute__((aligned(16))) uint8_t lds[kHalves * STAGES * STAGE];
  __shared__ float other[kHalves][kWaves * 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wv = wave % kWaves, half = wave / kWaves;
  const int kvh = blockIdx.x % p.KV, kb = blockIdx.x / p.KV / n_seqs;
  const Job j = scalar_load(seqs + blockIdx.x / p.KV % n_seqs);
  if (!sound(p, j.q0, j.n, j.len, j.seq) || !j.n) return;   // (without new tokens there is no way through the tiles below)
  const int k0 = 128 * kb + 32 * wv, key = k0 + (lane & 31);
  float sum = 0;
  if (128 * kb < j.len) {
    const uint16_t* kbase = p.k.p + kvh * p.k.head;
    const int page = key < j.len ? p.tables[int64_t(j.seq) * p.width + key / kPage] : -1;
    const int before = j.len - j.n, pos0 = max(128 * kb - before, 0) / R * R, n = (j.n - pos0 + R - 1) / R, all = n * p.g;   // tiles a head, of the group
    Tile<DP, R> qt;
    qt.init(p.q_row, p.D, lane, wv);
    // this half's way through the tiles, head by head
    const uint16_t* q = p.q + int64_t(j.q0 + pos0 + half * R) * p.q_row + int64_t(kvh * p.g) * p.q_head;
    const float* l = p.lse + int64_t(j.q0) * p.H + int64_t(kvh * p.g) * j.n + pos0 + half * R;
    const int64_t q_on = kHalves * R * p.q_row, q_back = p.q_head - n * R * p.q_row;   // to the next tile; from behind a head's last to the next's
    int left = j.n - pos0 - half * R, tiles = (all - half + kHalves - 1) / kHalves;     // rows from the tile on; tiles to be fetched
    const int last = j.n - pos0 - n * R;                                                // (0 or less: of the rows behind the last tile)
    const uint32_t mine = lds_address(lds) + half * STAGES * STAGE;
    auto load = [&](int stage) {   // (past the last tile too, of zeros: every stage is the same number of loads)
      while (left <= last) {
        left += n * R;
        q += q_back;
        l += j.n - n * R;
      }
      const uint32_t to = mine + stage * STAGE + 1024 * wv;
      const int there = tiles > 0 ? left : 0;
      const uint16_t* from = tiles > 0 ? q : p.q;
#pragma unroll
      for (int u = 0; u < LOADS - 1; ++u)
        dma(from, qt.row + 64 * kWaves / (P / 16) * u < there ? qt.off[u] : kOutside, to + 1024 * kWaves * u);
      dma4(tiles > 0 ? l : p.lse, lane < there ? 4 * lane : kOutside, mine + stage * STAGE + TILE + 256 * wv);
      --tiles;
      left -= kHalves * R;
      q += q_on;
      l += kHalves * R;
    };
    bf16x8 k[KS];
    row_operands<DP>(k, kbase, (int64_t(page) * kPage + key % kPage) * p.k.row, uint32_t(page) < uint32_t(p.n_pages), p.D, lane);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) load(i);
    uint32_t q_at[KS], l_at = mine + TILE + 256 * wv + 16 * (lane >> 5);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q_at[ks] = mine + piece_at<P>(lane & 31, 2 * ks + (lane >> 5));
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm("" : "+v"(q_at[ks]));
    asm("" : "+v"(l_at));
    typedef __attribute__((address_space(3))) const bf16x8 lds_bf16x8;
    typedef __attribute__((address_space(3))) const f32x4 lds_f32x4;
#else
    typedef const bf16x8 lds_bf16x8;
    typedef const f32x4 lds_f32x4;
#endif
    dma_wait();   // (for k, so that the compiler does not wait for all loads in the loop)
    f32x16 s0, s1;
#pragma unroll
    for (int i = 0; i < 16; ++i) s1[i] = -INFINITY;
    int pos = pos0 + half * R;   // of the tile that is worked on
    // ahead: the scores of rows 32 a .. of the tile in a stage; s: those before, which are summed
    auto step = [&](f32x16& ahead, const f32x16& s, int stage, int a) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 x = *(lds_f32x4*)(uintptr_t)(l_at + stage * STAGE + 128 * a + 32 * u);
#pragma unroll
        for (int i = 0; i < 4; ++i) ahead[4 * u + i] = x[i];
      }
      bf16x8 f[3];
      auto operand = [&](int ks) { return *(lds_bf16x8*)(uintptr_t)(q_at[ks] + stage * STAGE + 32 * a * P); };
#pragma unroll
      for (int i = 0; i < 2; ++i) f[i] = operand(i);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + 2 < KS) f[(ks + 2) % 3] = operand(ks + 2);
        ahead = mfma(f[ks % 3], k[ks], ahead);
#pragma unroll
        for (int i = 16 * ks / KS; i < 16 * (ks + 1) / KS; ++i) sum += exp2_hw(s[i] * p.c);
        order_steps();
      }
      const int at = pos + 32 * a;
      if (before + at < k0 + 31 || at + 32 > j.n) {   // the diagonal, the last rows
        const int hidden = max(key - before, 0) - at - 4 * (lane >> 5), rows = j.n - at - 4 * (lane >> 5);   // (a row sees the key from `hidden` on)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) < hidden || 8 * (i >> 2) + (i & 3) >= rows) ahead[i] = -INFINITY;
      }
    };
    int work = (all - half + kHalves - 1) / kHalves;
    auto tile = [&](int stage, int next) {
      dma_wait<(STAGES - 2) * LOADS>();
      __syncthreads();
      load(next);
      if (work-- > 0) {
        while (pos - pos0 >= n * R) pos -= n * R;
        step(s0, s1, stage, 0);
        step(s1, s0, stage, 1);
        pos += kHalves * R;
      }
    };
    static_assert(STAGES == 2, "the stages in turn");
    for (int i = (all + kHalves - 1) / kHalves; i > 0;) {
      tile(0, 1);
      if (--i == 0) break;
      tile(1, 0);
      --i;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += exp2_hw(s1[i] * p.c);
    dma_wait();
  }
  sum += swap_halves(sum);
  if (lane < 32) other[half][32 * wv + lane] = sum;
  __syncthreads();
  if (half || lane >= 32 || key >= p.longest) return;
#pragma unroll
  for (int h = 1; h < kHalves; ++h) sum += other[h][32 * wv + lane];
  const int64_t row = int64_t(j.seq) * p.KV + kvh;
  float w = 0;
  if (key < j.len) w = (key < j.len - j.n && key < p.weights_width ? p.weights[row * p.weights_width + key] : 0.0f) + sum;
  p.weights_out[row * p.longest + key] = w;
}

// ---- append ----
struct AppendArgs {
  const uint16_t *k_new, *v_new;
  int64_t k_new_row, k_new_head, v_new_row, v_new_head;
  uint16_t *k, *v;
  int64_t k_head, k_row, v_head, v_row;
  const Append* jobs;
  int KV, pieces;      // 16-byte pieces of a head
  int64_t q_rows, positions;
};

// The rows of one page and sequence, up to 256 16-byte pieces of a head: a thread has one piece of every head (of every second,
// fourth, .. where there are fewer), K's heads, then V's.  Memory bound.  Stores that do not stay in the caches: 28665 tokens of 8
// heads of 128 to pages that are not in them take 46 us, before that and the heads in flight together 58.
__global__ __launch_bounds__(256) void paged_append(AppendArgs p) {
  const Append a = scalar_load(p.jobs + blockIdx.x);
  if (a.row < 0 || a.count <= 0 || a.count > kPage || a.row > p.q_rows - a.count || a.position < 0 || a.position > p.positions - a.count)
    return;
  const int n = a.count * p.pieces, heads = 256 / n, h0 = threadIdx.x / n, i = threadIdx.x - h0 * n, r = i / p.pieces, c = i - r * p.pieces;
  if (h0 >= heads) return;
  const uint16_t *k_from = p.k_new + (a.row + r) * p.k_new_row + 8 * c, *v_from = p.v_new + (a.row + r) * p.v_new_row + 8 * c;
  uint16_t *k_to = p.k + (a.position + r) * p.k_row + 8 * c, *v_to = p.v + (a.position + r) * p.v_row + 8 * c;
  constexpr int U = 4;
  for (int h = h0; h < p.KV; h += U * heads) {
    u32x4 x[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u * heads < p.KV) {
        x[2 * u] = *reinterpret_cast<const u32x4*>(k_from + (h + u * heads) * p.k_new_head);
        x[2 * u + 1] = *reinterpret_cast<const u32x4*>(v_from + (h + u * heads) * p.v_new_head);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u * heads < p.KV) {
        __builtin_nontemporal_store(x[2 * u], reinterpret_cast<u32x4*>(k_to + (h + u * heads) * p.k_head));
        __builtin_nontemporal_store(x[2 * u + 1], reinterpret_cast<u32x4*>(v_to + (h + u * heads) * p.v_head));
      }
  }
}

// ---- eviction ----
struct EvictArgs {
  uint16_t *k, *v;
  int64_t k_layer, k_head, k_row, v_layer, v_head, v_row;
  const float* weights;
  int weights_width, keep, recent;
  const SeqOf* seqs;
  const int32_t *tables, *to;
  int width, to_width, n_pages, longest;
  int n_seqs, KV, pieces;
  float* weights_out;
  int32_t* kept;
};

// Weights in the order of eviction as unsigned numbers: larger is kept first; -0 is 0, a NaN the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f), key = b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);   // (-0 + 0 is 0)
  return x != x ? 0xffffffffu : key;
}
__device__ __forceinline__ float weight_of(uint32_t key) {   // (a NaN, of many)
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// The kept positions of one sequence, layer and head.  The candidates are those before the newest; wave w has them from w S on,
// S a multiple of 64, as keys in IT registers a lane (IT 0: read again each time), 0 where there is none, which no weight's key
// is.  The least kept key comes digit by digit (11, 11 and 10 bits) from counts in LDS; what is above it stays, and of what is
// equal the first ones.  Each wave then counts what stays of its own, and writes it behind what stays of the waves before it.
constexpr int kBins = 2048;
template <int T>
struct SelectLds {
  uint32_t counts[kBins];
  uint32_t state[2];               // key so far, how many equal ones are still to be taken
  uint32_t sums[T / 64][2];
};
// Also to `list`, where there is one
template <int T, int IT>
__device__ __forceinline__ void choose(const EvictArgs& p, SelectLds<T>& lds, int s, int64_t row, int32_t* list) {
  constexpr int W = T / 64, B = kBins / T;
  auto& counts = lds.counts;
  auto& state = lds.state;
  auto& sums = lds.sums;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const SeqOf q = scalar_load(p.seqs + s);
  const int len = q.len < 0 || q.len > p.longest ? 0 : q.len, held = min(len, p.keep);
  const int old = len - min(p.recent, len), heavy = held - (len - old);   // candidates, how many of them stay
  const int read = min(old, p.weights_width);
  const float* w = p.weights + row * p.weights_width;
  const int its = tiles_of(old, T), first = wv * its * 64 + lane;
  // (the loads without branches: one after the other they took 30 us of 30000 positions)
  auto load = [&](int j) { return read > 0 ? w[min(j, read - 1)] : 0.0f; };
  auto key_of = [&](int j, float x) { return j < old ? order_of(j < read ? x : 0.0f) : 0u; };
  uint32_t x[IT ? IT : 1];
  if constexpr (IT) {
    float y[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) y[i] = load(first + 64 * i);
#pragma unroll
    for (int i = 0; i < IT; ++i) x[i] = i < its ? key_of(first + 64 * i, y[i]) : 0;
  }
  auto each = [&](auto f) {   // f(position, key)
    if constexpr (IT) {
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (i < its) f(first + 64 * i, x[i]);
    } else {
      for (int i = 0; i < its; ++i) f(first + 64 * i, key_of(first + 64 * i, load(first + 64 * i)));
    }
  };
  uint32_t key = heavy > 0 ? 0 : 0xffffffffu, need = 0;   // (all candidates, or none, stay)
  if (heavy > 0 && heavy < old) {
    need = heavy;
    auto digit = [&](int shift, uint32_t mask, uint32_t above) {   // above: the key's bits that are settled
#pragma unroll
      for (int i = 0; i < B; ++i) counts[tid + T * i] = 0;
      __syncthreads();
      each([&](int, uint32_t k) {
        if (!above || (k & above) == key) atomicAdd(&counts[k >> shift & mask], 1u);
      });
      __syncthreads();
      uint32_t n[B], mine = 0;   // from the largest digit down
#pragma unroll
      for (int i = 0; i < B; ++i) mine += n[i] = counts[kBins - 1 - B * tid - i];
      uint32_t before = mine;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(before, d);
        if (lane >= d) before += y;
      }
      if (lane == 63) sums[wv][0] = before;
      __syncthreads();
      for (int v = 0; v < wv; ++v) before += sums[v][0];
      before -= mine;
      if (before < need && before + mine >= need) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
          if (before < need && before + n[i] >= need) {
            state[0] = key | uint32_t(kBins - 1 - B * tid - i) << shift;
            state[1] = need - before;
          }
          before += n[i];
        }
      }
      __syncthreads();
      key = state[0];
      need = state[1];
    };
    digit(21, 2047, 0);
    digit(10, 2047, 0xffe00000u);
    digit(0, 1023, 0xfffffc00u);
  }
  uint32_t aboves = 0, equals = 0;
  each([&](int, uint32_t k) {
    aboves += __popcll(__ballot(k > key));
    equals += __popcll(__ballot(k == key));
  });
  __syncthreads();
  if (lane == 0) {
    sums[wv][0] = aboves;
    sums[wv][1] = equals;
  }
  __syncthreads();
  uint32_t at = 0, rank = 0;   // of what stays before, of equal ones before
  for (int v = 0; v < wv; ++v) {
    at += sums[v][0];
    rank += sums[v][1];
  }
  at += min(rank, need);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  each([&](int j, uint32_t k) {
    const uint64_t e = __ballot(k == key);
    const bool stays = k > key || (k == key && rank + __popcll(e & below) < need);
    rank += __popcll(e);
    const uint64_t kept = __ballot(stays);
    const uint32_t to = at + __popcll(kept & below);
    at += __popcll(kept);
    if (stays && to < uint32_t(p.keep)) {
      if (list) list[to] = j;
      p.kept[row * p.keep + to] = j;
      p.weights_out[row * p.keep + to] = weight_of(k);
    }
  });
  for (int i = max(heavy, 0) + tid; i < p.keep; i += T) {   // the newest, and what is behind them
    const int j = len - held + i;
    if (list && i < held) list[i] = j;
    p.kept[row * p.keep + i] = i < held ? j : -1;
    p.weights_out[row * p.keep + i] = i < held && j < p.weights_width ? w[j] : 0.0f;
  }
}

template <int T, int IT>
__global__ __launch_bounds__(T) void paged_select(EvictArgs p) {
  __shared__ SelectLds<T> lds;
  const int s = blockIdx.y, layer = blockIdx.x / p.KV;
  choose<T, IT>(p, lds, s, (int64_t(layer) * p.n_seqs + s) * p.KV + blockIdx.x % p.KV, nullptr);
}

// A row's 16-byte piece from one position of a head's pages to another's, in two steps so that several are on their way
struct Piece {
  const uint16_t* from;   // null: there is none
  uint16_t* to;
};
__device__ __forceinline__ Piece piece_of(const EvictArgs& p, uint16_t* base, int64_t row_stride, const int32_t* table, int s, int from, int row, int c) {
  const int page = from >= 0 ? table[from / kPage] : -1, to = row < p.keep ? p.to[int64_t(s) * p.to_width + row / kPage] : -1;
  if (uint32_t(page) >= uint32_t(p.n_pages) || uint32_t(to) >= uint32_t(p.n_pages)) return {nullptr, nullptr};
  return {base + (int64_t(page) * kPage + from % kPage) * row_stride + 8 * c, base + (int64_t(to) * kPage + row % kPage) * row_stride + 8 * c};
}

// Choice and rows of one sequence, layer and head by one workgroup, where there are enough of them to fill the card: 768 of up to
// 512 positions, 64 KB of rows each, 22.2 us in place of 24.1 by two launches.
constexpr int kShort = 2048, kFills = 512;
__global__ __launch_bounds__(256) void paged_evict_short(EvictArgs p) {
  __shared__ SelectLds<256> lds;
  __shared__ int32_t list[kShort];
  const int s = blockIdx.y, layer = blockIdx.x / p.KV, kvh = blockIdx.x % p.KV;
  choose<256, kShort / 256>(p, lds, s, (int64_t(layer) * p.n_seqs + s) * p.KV + kvh, list);
  __syncthreads();
  const SeqOf q = scalar_load(p.seqs + s);
  const int len = q.len < 0 || q.len > p.longest ? 0 : q.len, n = min(len, p.keep) * p.pieces;
  const int32_t* table = p.tables + int64_t(s) * p.width;
  uint16_t *k = p.k + layer * p.k_layer + kvh * p.k_head, *v = p.v + layer * p.v_layer + kvh * p.v_head;
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * U) {
    Piece a[U], b[U];
    u32x4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u, row = i / p.pieces, c = i - row * p.pieces, from = i < n ? list[row] : -1;
      a[u] = piece_of(p, k, p.k_row, table, s, from, row, c);
      b[u] = piece_of(p, v, p.v_row, table, s, from, row, c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (a[u].from) {
        x[u] = *reinterpret_cast<const u32x4*>(a[u].from);
        y[u] = *reinterpret_cast<const u32x4*>(b[u].from);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (a[u].from) {
        __builtin_nontemporal_store(x[u], reinterpret_cast<u32x4*>(a[u].to));
        __builtin_nontemporal_store(y[u], reinterpret_cast<u32x4*>(b[u].to));
      }
  }
}

// The kept rows to their new places: 16-byte pieces, four in flight a thread; K (blockIdx.z 0) and V.
constexpr int kMove = 4;
__global__ __launch_bounds__(256) void paged_move(EvictArgs p, int blocks) {
  const int s = blockIdx.x / blocks, layer = blockIdx.y / p.KV, kvh = blockIdx.y % p.KV;
  const bool value = blockIdx.z;
  const int64_t row_stride = value ? p.v_row : p.k_row;
  uint16_t* base = value ? p.v + layer * p.v_layer + kvh * p.v_head : p.k + layer * p.k_layer + kvh * p.k_head;
  const int32_t *kept = p.kept + ((int64_t(layer) * p.n_seqs + s) * p.KV + kvh) * p.keep, *table = p.tables + int64_t(s) * p.width;
  const int64_t first = int64_t(blockIdx.x % blocks) * 256 * kMove + threadIdx.x;
  int from[kMove], page[kMove], to[kMove], row[kMove], piece[kMove];
#pragma unroll
  for (int u = 0; u < kMove; ++u) {
    const int64_t i = first + u * 256;
    row[u] = int(i / p.pieces);
    piece[u] = int(i - int64_t(row[u]) * p.pieces);
    from[u] = row[u] < p.keep ? kept[row[u]] : -1;
    to[u] = row[u] < p.keep ? p.to[int64_t(s) * p.to_width + row[u] / kPage] : -1;
  }
#pragma unroll
  for (int u = 0; u < kMove; ++u) page[u] = from[u] >= 0 ? table[from[u] / kPage] : -1;
  u32x4 x[kMove];
#pragma unroll
  for (int u = 0; u < kMove; ++u) {
    if (uint32_t(page[u]) >= uint32_t(p.n_pages) || uint32_t(to[u]) >= uint32_t(p.n_pages)) page[u] = -1;
    if (page[u] >= 0) x[u] = *reinterpret_cast<const u32x4*>(base + (int64_t(page[u]) * kPage + from[u] % kPage) * row_stride + 8 * piece[u]);
  }
#pragma unroll
  for (int u = 0; u < kMove; ++u)
    if (page[u] >= 0)
      __builtin_nontemporal_store(x[u], reinterpret_cast<u32x4*>(base + (int64_t(to[u]) * kPage + row[u] % kPage) * row_stride + 8 * piece[u]));
}

// ---- host: the plan ----
// Workgroups that a launch is shared out to, about, and tiles of a job at least.
constexpr int kFewGroups = 2048, kManyGroups = 512;
constexpr int kFewLeast = 4, kManyLeast = 6;
// Many rows' lists of up to this many tiles stay whole: one of 8 tiles split in two takes 18.6 us with the join, whole 12.5 (8 x 128
// rows of heads of 64).  Longer ones in pieces of 4, 6 and 8 tiles at least: 24.9, 24.6 and 26.7 (a step of tokens and chunks, up to
// 46 tiles of heads of 96).
constexpr int kManyWhole = 8;
// Few rows: pieces of four tiles, one a wave, as long as that is one round of the CUs; then longer ones, up to 16, in as few whole rounds
// as hold them (8 sequences of up to 2000, 8 K/V heads of 128: by 272 workgroups 18.9 us, by 256 14.0); and from eight rounds on as
// many as make 2048 (64 sequences of up to 16000 positions: 425 us, with 1024 486, with 4096 447).
constexpr int kFewRound = 256, kFewEnough = 16;
// Without weights a sequence of up to this many tiles stays whole, as the join takes another launch: 512 positions of 8 sequences,
// 4 K/V heads of 64: 6.7 us in place of 8.8, heads of 128 9.9 and 10.0; 1024: 9.7 and 8.9, 15.1 and 10.9.
constexpr int kFewWhole = 16;

// Few rows only, and not more workgroups than CUs: paged_whole, of up to 512 positions always, up to 1024 where the pieces would share
// CUs or where there are no weights and heads are small.  In us, this and by pieces: 8 sequences of up to 512, 4 K/V heads of 64, weights
// 6.9 and 9.4; 32 of up to 1000, 8 heads of 64 9.6 and 15.4, with weights 11.1 and 16.4; heads of 128 16.0 and 25.8; but 8 of up to 1000, 4
// heads of 64, with weights 10.2 and 9.1; 64 of up to 500, 8 heads (512 workgroups) 12.9 and 8.3.
constexpr int kWholeGroups = 256, kWholeShort = 512, kWholeSplit = 64;

struct Pieces {
  int64_t each, whole;
  // of a list of `tiles`: one until it has half as much again as the others' pieces
  int of(int64_t tiles) const { return 2 * tiles <= 3 * each || tiles <= whole ? 1 : int(cdiv(tiles, each)); }
};
Pieces many_pieces(int64_t tiles, int n_kv) { return {std::max<int64_t>(kManyLeast, cdiv(tiles * n_kv, kManyGroups)), kManyWhole}; }
Pieces few_pieces(const std::vector<int64_t>& lists, int64_t tiles, int n_kv, bool weighted) {
  const int64_t whole = weighted ? 0 : kFewWhole;
  for (int64_t groups = kFewRound; groups <= kFewGroups && int64_t(lists.size()) * n_kv <= kFewGroups; groups += kFewRound)
    for (Pieces x{std::max<int64_t>(kFewLeast, cdiv(tiles * n_kv, groups)), whole}; x.each <= kFewEnough; ++x.each) {
      int64_t n = 0;
      for (const int64_t t : lists) n += x.of(t);
      if (n * n_kv <= groups) return x;
    }
  return {std::max<int64_t>(kFewEnough, cdiv(tiles * n_kv, kFewGroups)), whole};
}

struct Writer {
  int32_t* words;   // or null: counting
  int64_t at = MSD_PLAN_HEADER;
  int64_t list(int64_t n, int64_t each) {
    const int64_t from = at;
    at += (n * each + 3) / 4 * 4;
    return from;
  }
};

int64_t plan(int n_seqs, const int32_t* seqs, const int32_t* tables, int table_width, int H, int KV, int longest, int32_t* words, int64_t room) {
  if (n_seqs < 0 || n_seqs > 65535 || H <= 0 || KV <= 0 || H % KV || H > 4096 || table_width < 0 || longest < 0 ||
      table_width > (INT32_MAX / kPage))
    return MSD_E_CONFIG;
  if (n_seqs && (!seqs || (table_width && !tables))) return MSD_E_ARG;
  const int64_t g = H / KV;
  int most = 0;   // (lengths up to kLongest: the next tile's first position is a number too)
  int64_t q_end = 0, q_count = 0;
  std::vector<int> few, many;   // sequences
  std::vector<int64_t> few_lists;
  int64_t few_tiles = 0, few_rows = 0, many_tiles = 0, row_tiles = 0, appends = 0, scores = 0;
  auto seen = [&](const int32_t* s, int64_t row) { return s[2] - s[1] + 1 + row / g; };   // positions that the row sees
  for (int b = 0; b < n_seqs; ++b) {
    const int32_t* s = seqs + 3 * b;
    const int64_t rows = s[1] * g;
    if (s[0] < 0 || s[1] < 0 || s[2] < s[1] || s[2] > std::min<int64_t>(int64_t(table_width) * kPage, kLongest) || (longest && s[2] > longest) ||
        s[0] > INT32_MAX - s[1] || rows >= (1 << 30) - 256)
      return MSD_E_CONFIG;
    most = std::max(most, s[2]);
    if (s[1]) q_end = std::max<int64_t>(q_end, int64_t(s[0]) + s[1]);
    q_count += s[1];
    if (rows <= kFewRows) {
      few.push_back(b);
      if (rows) {
        few_lists.push_back(cdiv(s[2], kFewKeys));
        few_tiles += few_lists.back();
      }
      few_rows = std::max(few_rows, rows);
      scores += rows * cdiv(longest ? longest : s[2], kFewKeys);
    } else {
      many.push_back(b);
      for (int64_t r = 0; r < rows; r += kManyRows, ++row_tiles) many_tiles += cdiv(seen(s, std::min(r + kManyRows, rows) - 1), kKeys);
    }
    if (longest) appends += s[1] ? cdiv(s[1], kPage) + 1 : 0;
    else if (s[1]) appends += cdiv(s[2], kPage) - (s[2] - s[1]) / kPage;
  }
  if (longest > std::min<int64_t>(int64_t(table_width) * kPage, kLongest)) return MSD_E_CONFIG;
  const Pieces fp[2] = {few_pieces(few_lists, few_tiles, KV, false), few_pieces(few_lists, few_tiles, KV, true)}, mp = many_pieces(many_tiles, KV);
  int64_t n_few[2] = {}, n_many = 0, few_active = 0;
  bool few_parts[2] = {}, many_parts = false;
  for (int b : few) {
    if (!seqs[3 * b + 1]) continue;
    ++few_active;
    for (int c = 0; c < 2; ++c) {
      const int n = fp[c].of(cdiv(seqs[3 * b + 2], kFewKeys));
      n_few[c] += n;
      few_parts[c] |= n > 1;
    }
  }
  for (int b : many)
    for (int64_t r = 0, rows = seqs[3 * b + 1] * g; r < rows; r += kManyRows) {
      const int n = mp.of(cdiv(seen(seqs + 3 * b, std::min(r + kManyRows, rows) - 1), kKeys));
      n_many += n;
      many_parts |= n > 1;
    }
  if (longest) {   // as many as any lengths up to it give: a piece more than whole ones for each list, none below the least
    const int64_t tiles = cdiv(longest, kFewKeys), most_many = cdiv(cdiv(longest, kKeys), kManyLeast);
    for (int c = 0; c < 2; ++c) {
      const int64_t most_few = tiles <= fp[c].whole ? 1 : cdiv(tiles, kFewLeast);
      n_few[c] = few_active ? std::min(few_active * most_few, few_active + cdiv(kFewGroups, KV)) : 0;
      few_parts[c] = few_active && most_few > 1;
    }
    n_many = row_tiles ? std::min(row_tiles * most_many, row_tiles + cdiv(kManyGroups, KV)) : 0;
    many_parts = row_tiles && most_many > 1;
  }
  const int width = int(cdiv(table_width, 4) * 4);
  Writer w{words};
  const int64_t at_seqs = w.list(n_seqs, 4), at_many = w.list(n_many, 8), at_tiles = w.list(row_tiles, 8), at_manys = w.list(many.size(), 8),
                at_appends = w.list(appends, 4), at_few[2] = {w.list(n_few[0], 8), w.list(n_few[1], 8)},
                at_fews[2] = {w.list(few.size(), 8), w.list(few.size(), 8)}, at_tables = w.list(n_seqs, width);
  // (a launch counts its threads in 32 bits)
  if (w.at >= (int64_t(1) << 28) || scores >= (int64_t(1) << 30) || appends >= (1 << 24) ||
      (n_few[1] + int64_t(few.size()) + n_many + 4 * row_tiles) * KV >= (1 << 24))
    return MSD_E_CONFIG;
  if (!words) return w.at;
  if (room < w.at) return MSD_E_ARG;
  memset(words, 0, size_t(at_tables) * 4);
  // empty jobs, of a sequence that there is not
  for (int c = 0; c < 2; ++c)
    for (int64_t i = 0; i < n_few[c]; ++i) words[at_few[c] + 8 * i + 3] = -1;
  for (int64_t i = 0; i < n_many; ++i) words[at_many + 8 * i + 3] = -1;
  words[MSD_PLAN_WORDS] = int32_t(w.at);
  words[MSD_PLAN_SEQS] = n_seqs;
  words[MSD_PLAN_HEADS] = H;
  words[MSD_PLAN_KV_HEADS] = KV;
  words[MSD_PLAN_WIDTH] = width;
  words[MSD_PLAN_LONGEST] = longest ? longest : most;
  words[MSD_PLAN_Q_END] = int32_t(q_end);
  words[MSD_PLAN_Q_COUNT] = int32_t(q_count);
  words[MSD_PLAN_RESERVED] = longest != 0;
  for (int c = 0; c < 2; ++c) {
    words[N_FEW + c] = int32_t(n_few[c]);
    words[FEW_PARTS + c] = few_parts[c];
    words[AT_FEW + c] = int32_t(at_few[c]);
    words[AT_FEWS + c] = int32_t(at_fews[c]);
  }
  words[N_MANY] = int32_t(n_many);
  words[N_FEWS] = int32_t(few.size());
  words[N_TILES] = int32_t(row_tiles);
  words[N_MANYS] = int32_t(many.size());
  words[N_APPENDS] = int32_t(appends);
  words[MANY_PARTS] = many_parts;
  words[FEW_ROWS] = int32_t(few_rows);
  words[SCORES] = int32_t(scores);
  words[AT_SEQS] = int32_t(at_seqs);
  words[AT_MANY] = int32_t(at_many);
  words[AT_TILES] = int32_t(at_tiles);
  words[AT_MANYS] = int32_t(at_manys);
  words[AT_APPENDS] = int32_t(at_appends);
  words[AT_TABLES] = int32_t(at_tables);

  // pages: what is behind a sequence's length is 0 on the device
  int pages = 0;
  for (int b = 0; b < n_seqs; ++b) {
    int32_t* row = words + at_tables + int64_t(b) * width;
    const int used = int(cdiv(seqs[3 * b + 2], kPage));
    for (int i = 0; i < used; ++i) {
      const int x = tables[int64_t(b) * table_width + i];
      if (x < 0 || x > INT32_MAX / kPage - 1) return MSD_E_CONFIG;
      row[i] = x;
      pages = std::max(pages, x + 1);
    }
    std::fill(row + used, row + width, 0);
  }
  words[MSD_PLAN_PAGES] = pages;
  std::vector<uint8_t> uses(pages, 0);   // 0, 1, more
  for (int b = 0; b < n_seqs; ++b)
    for (int i = 0; i < int(cdiv(seqs[3 * b + 2], kPage)); ++i) {
      uint8_t& x = uses[words[at_tables + int64_t(b) * width + i]];
      x = std::min(x + 1, 2);
    }
  bool shared = false;
  Append* append = reinterpret_cast<Append*>(words + at_appends);
  for (int b = 0; b < n_seqs; ++b) {
    const int32_t *s = seqs + 3 * b, *row = words + at_tables + int64_t(b) * width;
    memcpy(words + at_seqs + 4 * b, s, 12);
    for (int at = s[2] - s[1]; at < s[2];) {
      const int end = std::min(s[2], (at / kPage + 1) * kPage);
      *append++ = {s[0] + at - (s[2] - s[1]), end - at, row[at / kPage] * kPage + at % kPage, 0};
      shared |= uses[row[at / kPage]] > 1;
      at = end;
    }
  }
  words[MSD_PLAN_SHARED] = shared;

  // jobs, the longest first
  struct List { int64_t each; int index; };
  std::vector<List> order;
  auto longest_first = [](const List& a, const List& b) { return a.each > b.each; };
  for (int c = 0; c < 2; ++c) {
    Job* job = reinterpret_cast<Job*>(words + at_few[c]);
    Few* f = reinterpret_cast<Few*>(words + at_fews[c]);
    int slot = 0, score = 0;
    order.clear();
    for (size_t i = 0; i < few.size(); ++i) {
      const int32_t* s = seqs + 3 * few[i];
      const int64_t tiles = cdiv(s[2], kFewKeys);
      const int n = s[1] ? fp[c].of(tiles) : 0;
      f[i] = {s[0], s[1], s[2], few[i], slot, n, score, 0};
      slot += n;
      score += int(s[1] * g * cdiv(longest ? longest : s[2], kFewKeys));
      if (n) order.push_back({cdiv(tiles, n), int(i)});
    }
    std::stable_sort(order.begin(), order.end(), longest_first);
    for (const List& o : order) {
      const Few& x = f[o.index];
      const int64_t tiles = cdiv(x.len, kFewKeys);
      for (int z = 0; z < x.parts; ++z)
        *job++ = {x.q0, x.n, x.len, x.seq, 2 * x.scores + (x.parts == 1), int(tiles * z / x.parts), int(tiles * (z + 1) / x.parts), x.slot + z};
    }
  }
  order.clear();
  Job* job = reinterpret_cast<Job*>(words + at_many);
  RowTile* t = reinterpret_cast<RowTile*>(words + at_tiles);
  Job* m = reinterpret_cast<Job*>(words + at_manys);
  int slot = 0, index = 0;
  for (int b : many) {
    const int32_t* s = seqs + 3 * b;
    *m++ = {s[0], s[1], s[2], b, 0, 0, 0, 0};
    const int64_t rows = s[1] * g;
    for (int64_t r = (rows - 1) / kManyRows * kManyRows; r >= 0; r -= kManyRows, ++index) {   // the longest of a sequence first
      const int64_t tiles = cdiv(seen(s, std::min(r + kManyRows, rows) - 1), kKeys);
      const int n = mp.of(tiles);
      t[index] = {s[0], s[1], s[2], b, int(r), slot, n, int(tiles)};
      slot += n;
      order.push_back({cdiv(tiles, n), index});
    }
  }
  std::stable_sort(order.begin(), order.end(), longest_first);
  for (const List& o : order) {
    const RowTile& x = t[o.index];
    const int64_t tiles = x.tiles;
    for (int z = 0; z < x.parts; ++z)
      *job++ = {x.q0, x.n, x.len, x.seq, x.parts == 1 ? -x.row0 - 1 : x.row0, int(tiles * z / x.parts), int(tiles * (z + 1) / x.parts), x.slot + z};
  }
  words[MSD_PLAN_MAGIC] = kMagic;
  return w.at;
}

// ---- host: the calls ----
bool bad(const void* p) { return !p || reinterpret_cast<uintptr_t>(p) % 16; }
int32_t launched() { return hipGetLastError() == hipSuccess ? MSD_OK : MSD_E_HIP; }
int64_t up(int64_t x) { return cdiv(x, 256) * 256; }

// strides of rows that come in tiles of up to `rows`, and of `heads` heads
bool fits(int64_t row, int64_t head, int64_t rows, int64_t heads) {
  constexpr int64_t most = int64_t(1) << 30;
  return row >= 0 && head >= 0 && row % 8 == 0 && head % 8 == 0 && row <= most / rows && head <= most / heads && rows * row + heads * head < most;
}

int32_t check(const msd_paged* a) {
  if (!a || bad(a->plan) || !a->plan_host || reinterpret_cast<uintptr_t>(a->plan_host) % 4) return MSD_E_ARG;
  const int32_t* h = a->plan_host;
  if (h[MSD_PLAN_MAGIC] != kMagic) return MSD_E_ARG;
  if (a->d_head <= 0 || a->d_head > 128 || a->d_head % 8 || !(a->scale >= 0x1p-60f) || !(a->scale <= 0x1p60f) || a->q_rows < 0 ||
      a->q_rows > INT32_MAX || a->positions < 0 || a->positions > INT32_MAX || a->positions % kPage)
    return MSD_E_CONFIG;
  const int64_t g = h[MSD_PLAN_HEADS] / h[MSD_PLAN_KV_HEADS];
  if (a->q_rows * h[MSD_PLAN_HEADS] > INT32_MAX || h[MSD_PLAN_Q_END] > a->q_rows || h[MSD_PLAN_PAGES] > a->positions / kPage)
    return MSD_E_CONFIG;
  if (!fits(a->q_stride[0], a->q_stride[1], 128, g)) return MSD_E_CONFIG;
  for (const int64_t* s : {a->k_stride, a->v_stride})
    if (s[0] < 0 || s[0] % 8 || s[0] > (int64_t(1) << 40) || !fits(s[1], 0, kPage, 1)) return MSD_E_CONFIG;
  return MSD_OK;
}

// Where a workspace's parts begin, in bytes
struct Space {
  int64_t few_part, few_lse, many_part, many_lse, lse, scores, end;
};
Space space(const msd_paged& a, bool weighted) {
  const int32_t* h = a.plan_host;
  const int64_t few = int64_t(h[N_FEW + weighted]) * h[MSD_PLAN_KV_HEADS] * kFewRows, many = int64_t(h[N_MANY]) * h[MSD_PLAN_KV_HEADS] * kManyRows;
  Space s{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += up(bytes);
    return from;
  };
  s.few_part = take(h[FEW_PARTS + weighted] ? 4 * few * a.d_head : 0);
  s.few_lse = take(h[FEW_PARTS + weighted] || weighted ? 4 * few : 0);
  s.many_part = take(h[MANY_PARTS] ? 4 * many * a.d_head : 0);
  s.many_lse = take(h[MANY_PARTS] ? 4 * many : 0);
  s.lse = take(weighted && h[N_MANYS] ? 4 * a.q_rows * h[MSD_PLAN_HEADS] : 0);
  s.scores = take(weighted ? 4 * int64_t(h[SCORES]) * kFewKeys * h[MSD_PLAN_KV_HEADS] : 0);
  s.end = at;
  return s;
}

}  // namespace msp

using namespace msp;

extern "C" int64_t msd_paged_plan(int32_t n_seqs, const int32_t* seqs, const int32_t* tables, int32_t table_width, int32_t n_heads,
                                  int32_t n_kv_heads, int32_t longest, int32_t* words, int64_t room) {
  try {
    return plan(n_seqs, seqs, tables, table_width, n_heads, n_kv_heads, longest, words, room);
  } catch (...) {   // (no memory for its lists)
    return MSD_E_CONFIG;
  }
}

extern "C" int32_t msd_paged_append(const msd_paged* a, const void* k_new, const int64_t* k_new_stride, const void* v_new,
                                    const int64_t* v_new_stride, void* k, void* v, void* stream) {
  const int32_t rc = check(a);
  if (rc != MSD_OK) return rc;
  if (!k_new_stride || !v_new_stride) return MSD_E_ARG;
  const int32_t* h = a->plan_host;
  const int64_t KV = h[MSD_PLAN_KV_HEADS];
  if (!fits(k_new_stride[0], k_new_stride[1], 128, KV) || !fits(v_new_stride[0], v_new_stride[1], 128, KV)) return MSD_E_CONFIG;
  if (h[MSD_PLAN_SHARED]) return MSD_E_CONFIG;
  if (!h[N_APPENDS]) return MSD_OK;
  if (bad(k_new) || bad(v_new) || bad(k) || bad(v)) return MSD_E_ARG;
  AppendArgs p{static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), k_new_stride[0], k_new_stride[1], v_new_stride[0],
               v_new_stride[1], static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), a->k_stride[0], a->k_stride[1], a->v_stride[0],
               a->v_stride[1], reinterpret_cast<const Append*>(a->plan + h[AT_APPENDS]), int(KV), a->d_head / 8, a->q_rows, a->positions};
  hipLaunchKernelGGL(paged_append, dim3(h[N_APPENDS]), dim3(256), 0, static_cast<hipStream_t>(stream), p);
  return launched();
}

extern "C" int64_t msd_paged_attn_workspace_bytes(const msd_paged* a, int32_t weighted) {
  const int32_t rc = check(a);
  return rc != MSD_OK ? rc : space(*a, weighted != 0).end;
}

extern "C" int32_t msd_paged_attn(const msd_paged* a, const void* q, const void* k, const void* v, void* out, const float* weights,
                                  int32_t weights_width, float* weights_out, void* workspace, void* stream) {
  const int32_t rc = check(a);
  if (rc != MSD_OK) return rc;
  const int32_t* h = a->plan_host;
  const bool weighted = weights_out != nullptr;
  if (weights_width < 0) return MSD_E_CONFIG;
  if (weighted && weights_width && (!weights || reinterpret_cast<uintptr_t>(weights) % 4)) return MSD_E_ARG;
  if (reinterpret_cast<uintptr_t>(weights_out) % 4) return MSD_E_ARG;
  const int64_t KV = h[MSD_PLAN_KV_HEADS], longest = h[MSD_PLAN_LONGEST];
  const int64_t key_blocks = cdiv(longest, 128), weight_blocks = weighted ? cdiv(longest, kWeightKeys) : 0;
  const int n_tiles = h[MANY_PARTS] ? h[N_TILES] : 0, n_fews = h[FEW_PARTS + weighted] || weighted ? h[N_FEWS] : 0;
  // one row of few a workgroup as long as there are few of them (16 parts of 64 rows: 4.0 us, with four rows 5.6; 2048 rows: 6.7 and 5.0)
  const int join_rows = int64_t(n_fews) * KV * h[FEW_ROWS] <= 1024 ? 1 : kJoinRows, few_joins = h[FEW_PARTS + weighted] ? int(cdiv(h[FEW_ROWS], join_rows)) : 0;
  const int64_t finish = int64_t(n_tiles) * KV * (kManyRows / kJoinRows) + int64_t(n_fews) * KV * (few_joins + weight_blocks);
  // (a launch counts its threads in 32 bits)
  constexpr int64_t threads = int64_t(1) << 32;
  if (finish >= threads / kFinish || (weighted && key_blocks * KV * h[N_MANYS] >= threads / (64 * kWaves * kHalves))) return MSD_E_CONFIG;
  if (h[MSD_PLAN_Q_COUNT] && (bad(q) || bad(k) || bad(v) || bad(out))) return MSD_E_ARG;
  const Space at = space(*a, weighted);
  if (at.end && bad(workspace)) return MSD_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto floats = [&](int64_t x) { return reinterpret_cast<float*>(ws + x); };
  Args p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_row = a->q_stride[0];
  p.q_head = a->q_stride[1];
  p.k = {static_cast<const uint16_t*>(k), a->k_stride[0], a->k_stride[1]};
  p.v = {static_cast<const uint16_t*>(v), a->v_stride[0], a->v_stride[1]};
  p.D = a->d_head;
  p.H = h[MSD_PLAN_HEADS];
  p.KV = int(KV);
  p.g = p.H / p.KV;
  magic(uint32_t(p.g), p.g_magic, p.g_shift);
  p.c = a->scale * kLog2e;
  p.q_rows = a->q_rows;
  p.n_seqs = h[MSD_PLAN_SEQS];
  p.width = h[MSD_PLAN_WIDTH];
  p.longest = int(longest);
  p.n_pages = int(a->positions / kPage);
  p.tables = a->plan + h[AT_TABLES];
  p.few = reinterpret_cast<const Job*>(a->plan + h[AT_FEW + weighted]);
  p.many = reinterpret_cast<const Job*>(a->plan + h[AT_MANY]);
  p.n_few = h[N_FEW + weighted];
  p.n_many = h[N_MANY];
  p.out = static_cast<uint16_t*>(out);
  p.few_part = h[FEW_PARTS + weighted] ? floats(at.few_part) : nullptr;
  p.few_lse = floats(at.few_lse);
  p.many_part = h[MANY_PARTS] ? floats(at.many_part) : nullptr;
  p.many_lse = floats(at.many_lse);
  p.lse = weighted ? floats(at.lse) : nullptr;
  p.scores = weighted ? floats(at.scores) : nullptr;
  p.score_words = int64_t(h[SCORES]) * kFewKeys * KV;
  p.weights = weights;
  p.weights_width = weights_width;
  p.weights_out = weights_out;
  const int64_t groups = h[N_FEWS] * KV;
  bool whole = !h[N_MANYS] && groups && groups <= kWholeGroups && longest <= kWholeWaves * kWholeTiles * kFewKeys;
  if (whole)
    with_head(a->d_head, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      whole = h[FEW_ROWS] <= whole_rows<DP>() && (longest <= kWholeShort || groups >= kWholeSplit || (DP <= 64 && !weighted));
      if (!whole) return;
      const Few* fews = reinterpret_cast<const Few*>(a->plan + h[AT_FEWS + weighted]);
      if (weighted) hipLaunchKernelGGL((paged_whole<DP, true>), dim3(unsigned(groups)), dim3(64 * kWholeWaves), 0, s, p, fews);
      else hipLaunchKernelGGL((paged_whole<DP, false>), dim3(unsigned(groups)), dim3(64 * kWholeWaves), 0, s, p, fews);
    });
  if (whole) return launched();
  const Job* manys = reinterpret_cast<const Job*>(a->plan + h[AT_MANYS]);
  with_head(a->d_head, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    const unsigned few = unsigned(h[N_FEW + weighted] * KV), many = unsigned(h[N_MANY] * KV);
    if (few && many) hipLaunchKernelGGL((paged_both<DP>), dim3(few + many), dim3(64 * kWaves), 0, s, p);
    else if (few) hipLaunchKernelGGL((paged_few<DP>), dim3(few), dim3(64 * kWaves), 0, s, p);
    else if (many) hipLaunchKernelGGL((paged_many<DP>), dim3(many), dim3(64 * kWaves), 0, s, p);
  });
  if (finish)
    hipLaunchKernelGGL(paged_finish, dim3(unsigned(finish)), dim3(kFinish), 0, s, p, reinterpret_cast<const RowTile*>(a->plan + h[AT_TILES]),
                       n_tiles, reinterpret_cast<const Few*>(a->plan + h[AT_FEWS + weighted]), n_fews, few_joins, join_rows);
  if (weighted && h[N_MANYS] && key_blocks)
    with_head(a->d_head, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      hipLaunchKernelGGL((paged_weights<DP>), dim3(unsigned(key_blocks * KV * h[N_MANYS])), dim3(64 * kWaves * kHalves), 0, s, p, manys, h[N_MANYS]);
    });
  return launched();
}

extern "C" int32_t msd_paged_evict(const msd_paged* a, int32_t n_layers, int64_t k_layer, int64_t v_layer, void* k, void* v,
                                   const float* weights, int32_t weights_width, int32_t keep, int32_t recent, const int32_t* to,
                                   int32_t to_width, float* weights_out, int32_t* kept, void* stream) {
  const int32_t rc = check(a);
  if (rc != MSD_OK) return rc;
  const int32_t* h = a->plan_host;
  const int64_t heads = int64_t(n_layers) * h[MSD_PLAN_KV_HEADS];
  if (n_layers < 0 || keep < 0 || heads >= 65536 || heads * h[MSD_PLAN_SEQS] * std::max(keep, 1) >= int64_t(1) << 40 || weights_width < 0 ||
      recent < 0 || recent > keep || to_width < 0 || keep > int64_t(to_width) * kPage || k_layer % 8 || v_layer % 8 || k_layer < 0 || v_layer < 0 ||
      k_layer > (int64_t(1) << 44) || v_layer > (int64_t(1) << 44))
    return MSD_E_CONFIG;
  if (!heads || !h[MSD_PLAN_SEQS] || !keep) return MSD_OK;
  if (bad(k) || bad(v) || (weights_width && (!weights || reinterpret_cast<uintptr_t>(weights) % 4)) || !to || reinterpret_cast<uintptr_t>(to) % 4 ||
      !weights_out || reinterpret_cast<uintptr_t>(weights_out) % 4 || !kept || reinterpret_cast<uintptr_t>(kept) % 4)
    return MSD_E_ARG;
  EvictArgs p{};
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  p.k_layer = k_layer;
  p.k_head = a->k_stride[0];
  p.k_row = a->k_stride[1];
  p.v_layer = v_layer;
  p.v_head = a->v_stride[0];
  p.v_row = a->v_stride[1];
  p.weights = weights;
  p.weights_width = weights_width;
  p.keep = keep;
  p.recent = recent;
  p.seqs = reinterpret_cast<const SeqOf*>(a->plan + h[AT_SEQS]);
  p.tables = a->plan + h[AT_TABLES];
  p.to = to;
  p.width = h[MSD_PLAN_WIDTH];
  p.to_width = to_width;
  p.n_pages = int(a->positions / kPage);
  p.longest = h[MSD_PLAN_LONGEST];
  p.n_seqs = h[MSD_PLAN_SEQS];
  p.KV = h[MSD_PLAN_KV_HEADS];
  p.pieces = a->d_head / 8;
  p.weights_out = weights_out;
  p.kept = kept;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 rows(n_layers * p.KV, p.n_seqs);
  if (p.longest <= kShort && int64_t(rows.x) * rows.y >= kFills) {
    hipLaunchKernelGGL(paged_evict_short, rows, dim3(256), 0, s, p);
    return launched();
  }
  const int64_t blocks = cdiv(int64_t(keep) * p.pieces, 256 * kMove);
  if (blocks * p.n_seqs * 256 >= int64_t(1) << 32) return MSD_E_CONFIG;
  if (p.longest <= kShort) hipLaunchKernelGGL((paged_select<256, kShort / 256>), rows, dim3(256), 0, s, p);
  else if (p.longest <= 8192) hipLaunchKernelGGL((paged_select<1024, 8>), rows, dim3(1024), 0, s, p);
  else if (p.longest <= 32768) hipLaunchKernelGGL((paged_select<1024, 32>), rows, dim3(1024), 0, s, p);
  else hipLaunchKernelGGL((paged_select<1024, 0>), rows, dim3(1024), 0, s, p);
  hipLaunchKernelGGL(paged_move, dim3(unsigned(blocks * p.n_seqs), n_layers * p.KV, 2), dim3(256), 0, s, p, int(blocks));
  return launched();
}
