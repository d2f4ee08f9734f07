// What the attention kernels (attn.hip, paged.hip) share: matrix products of 32 x 32 tiles, LDS tiles and how they are
// fetched and read.  The reasons for the layouts stand at the head of attn.hip.
#ifndef MSD_ATTN_TILES_H
#define MSD_ATTN_TILES_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

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
constexpr int kWaves = 4;        // of a workgroup, 32 rows (or keys) each
constexpr int kKeys = 64;        // keys of an LDS tile
constexpr uint32_t kOutside = 0x80000000u;   // a buffer offset past every descriptor: the load gives zeros

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

// 64 lanes' 16 bytes at byte offsets `off` from `base` (wave-uniform) straight to the 1 KB of LDS at byte address `to`
// (lane after lane); kOutside gives zeros.  In assembly, because the compiler would wait for it before
// every LDS read that follows; dma_wait() is the wait, and what the workgroup's other waves fetched needs its barrier too.
// m0, the LDS base, is set in the same statement; the load may take it one wait state after the scalar write, which nothing
// puts between the two inside a statement but the s_nop.
__device__ __forceinline__ void dma(const uint16_t* base, uint32_t off, uint32_t to) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, 0x7fffffff, 0x00020000);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(r) : "m0");
#endif
}
// 64 lanes' 4 bytes to the 256 bytes of LDS at `to`
__device__ __forceinline__ void dma4(const float* base, uint32_t off, uint32_t to) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, 0x7fffffff, 0x00020000);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(r) : "m0");
#endif
}
// Until at most N of this wave's loads are outstanding (they return in order).  The compiler counts it, so that its own
// loads before the last N need no further wait.
template <int N = 0>
__device__ __forceinline__ void dma_wait() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
#endif
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) const uint8_t lds_u8;
  return uint32_t(__builtin_amdgcn_readfirstlane(int(reinterpret_cast<uintptr_t>((lds_u8*)p))));
#else
  return 0;
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

// A tile of R rows on its way to LDS: wave w fetches its instructions w, w + kWaves, ..
template <int DP, int R>
struct Tile {
  static constexpr int P = pitch<DP>(), C = P / 16, NW = kWaves, N = R * P / 1024 / NW;
  static_assert(64 * NW % C == 0, "an instruction's rows are a fixed number apart");
  int row;            // of the first instruction
  uint32_t off[N];
  __device__ __forceinline__ void init(int64_t row_stride, int D, int lane, int wv) {
    row = (64 * wv + lane) / C;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int r = row + 64 * NW / C * u, c = (64 * wv + lane) % C ^ swizzle<P>(r);
      off[u] = 8 * c < D ? uint32_t(r) * uint32_t(row_stride) * 2 + 16 * c : kOutside;
    }
  }
  // rows from `base` on, `left` of which exist: the others are zeros
  __device__ __forceinline__ void load(uint8_t* tile, const uint16_t* base, int left, int wv) const {
    const uint32_t to = lds_address(tile) + 1024 * wv;
#pragma unroll
    for (int u = 0; u < N; ++u) dma(base, row + 64 * NW / C * u < left ? off[u] : kOutside, to + 1024 * NW * u);
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

// LDS reads and matrix products keep their order across; other arithmetic may move
__device__ __forceinline__ void order_reads() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_sched_barrier(0x406);
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

// r / g for r < 2^30 (see magic())
__device__ __forceinline__ int div_by(int r, uint32_t magic, int shift) { return int(__umulhi(2 * uint32_t(r), magic) >> shift); }

// ---- host ----
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// m = ceil(2^(31 + s) / g) with 2^s <= g < 2^(s + 1): g m - 2^(31 + s) is below g < 2^(s + 1), so that floor(r m / 2^(31 +
// s)) is r / g for r < 2^30
inline void magic(uint32_t g, uint32_t& m, int& s) {
  s = 31 - __builtin_clz(g);
  m = uint32_t(((uint64_t(1) << (31 + s)) + g - 1) / g);
}

// f(integral_constant) for the padded head size
template <class F>
void with_head(int D, F f) {
  if (D <= 32) f(std::integral_constant<int, 32>());
  else if (D <= 64) f(std::integral_constant<int, 64>());
  else if (D <= 96) f(std::integral_constant<int, 96>());
  else f(std::integral_constant<int, 128>());
}

}  // namespace msa

#endif  // MSD_ATTN_TILES_H
