// The element-wise and row-wise operators of a training layer (gfx950): rotary positions, RMSNorm with the residual's
// addition, SwiGLU, and the 8-bit checkpoints that the last two can keep for their backward.
//
// Reference: model.py:94-98 (rms_norm), :110-117 (apply_rope), :157-160 (residuals and SwiGLU).
//
// All are bound by memory: each value is read once and written once per pass, in groups of eight values a lane (16 bytes
// of bf16), at any element alignment (the hardware takes unaligned 16-byte accesses; a row's last, partial group goes value
// by value), and everything between is f32.  The rate to compare with is a large copy's, 5.2 TB/s read and written; small calls
// are bound by the launch (3 to 4 us a kernel).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mslayers.h"
#include "internal.h"

namespace msl {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct bf16 { uint16_t x; };

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// Eight values of a row, n of them (n >= 8: all) in memory; the others read as 0
__device__ __forceinline__ void load8(const bf16* p, int n, float (&v)[8]) {
  if (n >= 8) {
    u32x4 x;
    __builtin_memcpy(&x, p, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(x[i] << 16);
      v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? __uint_as_float(uint32_t(p[i].x) << 16) : 0.0f;
  }
}
__device__ __forceinline__ void load8(const float* p, int n, float (&v)[8]) {
  if (n >= 8) {
    __builtin_memcpy(v, p, 32);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
  }
}
__device__ __forceinline__ void store8(bf16* p, int n, const float (&v)[8]) {
  const u32x4 x = {pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
  if (n >= 8) {
    __builtin_memcpy(p, &x, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i].x = uint16_t(x[i >> 1] >> (16 * (i & 1)));
  }
}
__device__ __forceinline__ void store8(float* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = v[i];
  }
}
// to the type and back: what a stored value reads as
__device__ __forceinline__ float rounded(float x, bf16) { return __uint_as_float(pack2(0.0f, x) & 0xffff0000u); }
__device__ __forceinline__ float rounded(float x, float) { return x; }

// lanes of 16 consecutive ones, by the rotations of a DPP row: every lane gets the result
template <int R>
__device__ __forceinline__ uint32_t ror16(uint32_t x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x120 + R, 0xf, 0xf, true));
#else
  return x;
#endif
}
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, ror16<8>(x));
  x = max(x, ror16<4>(x));
  x = max(x, ror16<2>(x));
  return max(x, ror16<1>(x));
}
__device__ __forceinline__ float sum64(float x) {
  x += __uint_as_float(ror16<8>(__float_as_uint(x)));
  x += __uint_as_float(ror16<4>(__float_as_uint(x)));
  x += __uint_as_float(ror16<2>(__float_as_uint(x)));
  x += __uint_as_float(ror16<1>(__float_as_uint(x)));
#if defined(__HIP_DEVICE_COMPILE__)
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
#endif
  return x;
}

// ---- 8-bit checkpoints ----
constexpr int kBlock = 128;   // values that share a scale: 16 lanes of 8
constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100

struct Checkpoint {
  int8_t* q;
  float* scale;
  int64_t pitch;   // values of a padded row
};

__host__ __device__ inline int64_t padded(int64_t d) { return (d + kBlock - 1) / kBlock * kBlock; }

__host__ __device__ inline int64_t checkpoint_bytes(int64_t rows, int64_t d) {
  return (rows * padded(d) + rows * (padded(d) / kBlock) * 4 + 255) / 256 * 256;
}

Checkpoint checkpoint(void* p, int64_t rows, int64_t d) {
  int8_t* q = static_cast<int8_t*>(p);
  return {q, reinterpret_cast<float*>(q + rows * padded(d)), padded(d)};
}

// Half of bf16's bytes: what a training step holds between forward and backward.  Blocks of 128 values of a row, so that a large
// value costs its neighbours' precision only; the scale and the quotients are f32.
// Keeps eight values of a row (group `col` / 8 of it).  All 16 lanes of a block call together; lanes past the row hold
// zeros.  The magnitudes are compared as integers, so a NaN is the largest and makes the block's scale one.
__device__ __forceinline__ void keep8(const Checkpoint& c, int64_t row, int col, const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const float m = __uint_as_float(max16(top));
  const bool small = m < kTiny;
  const float by = small ? 0.0f : 127.0f / m;
  uint32_t w[2] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t(int(rintf(v[i] * by))) & 0xff) << (8 * (i & 3));
  if (col < c.pitch) {
    *reinterpret_cast<uint2*>(c.q + row * c.pitch + col) = make_uint2(w[0], w[1]);
    if (col % kBlock == 0) c.scale[(row * c.pitch + col) / kBlock] = small ? 0.0f : m < INFINITY ? m / 127.0f : NAN;
  }
}
// (col < pitch)
__device__ __forceinline__ void kept8(const Checkpoint& c, int64_t row, int col, float (&v)[8]) {
  const uint2 w = *reinterpret_cast<const uint2*>(c.q + row * c.pitch + col);
  const float by = c.scale[(row * c.pitch + col) / kBlock];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = float(int8_t((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * by;
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// r / n for 0 <= r < 2^31 (a shift where n is a power of two)
struct Div {
  uint32_t n, mul;
  int shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t r) const { return mul ? __umulhi(r, mul) >> shift : r >> shift; }
};
// ceil(2^(32 + s) / n) with 2^s < n < 2^(s + 1): the error n m - 2^(32 + s) is below n <= 2^(s + 1), exact for r < 2^31
Div divider(uint32_t n) {
  Div d{n, 0, 31 - __builtin_clz(n)};
  if (n & (n - 1)) d.mul = uint32_t(((uint64_t(1) << (32 + d.shift)) + n - 1) / n);
  return d;
}

int32_t launched() { return hipGetLastError() == hipSuccess ? MSD_OK : MSD_E_HIP; }
bool odd(const void* p, int type) { return !p || reinterpret_cast<uintptr_t>(p) % (type == MSD_F32 ? 4 : 2); }

// f(value) for the type's element
template <class F>
void with_type(int type, F f) {
  if (type == MSD_F32) f(float());
  else f(bf16());
}

// ---- RMSNorm ----
// A row is held by TPR lanes, V groups of eight values each: group tid + TPR u.  One wave a row up to 1024 values (no
// barrier), 256 lanes up to 4096, 1024 up to 16384: as few lanes as hold the row with 16 values of each operand in
// their registers.  With four times the lanes and one group each: 9.9 and 12.7 us forward and backward in place of 8.7 and
// 9.6 (4096 rows of 1024, bf16, residual), 145 and 167 us in place of 101 and 110 (16383 rows of 4096, 8-bit checkpoint).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* lds, int tid) {
  x = sum64(x);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int wave = tid / 64, first = wave / W * W;
    __syncthreads();
    if (tid % 64 == 0) lds[wave] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) x += lds[first + i];
  }
  return x;
}

__device__ __forceinline__ void load_scale(const void* scale, int type, int col, int n, float (&v)[8]) {
  if (type == MSD_F32) load8(static_cast<const float*>(scale) + col, n, v);
  else load8(static_cast<const bf16*>(scale) + col, n, v);
}

struct RmsArgs {
  const void *x, *residual, *scale, *dy, *dsum;
  int64_t x_stride, residual_stride, dy_stride, dsum_stride, rows;
  int scale_type, d;
  float eps;
  void *y, *sum, *dx, *dscale;
  float *rstd, *part;
  Checkpoint c;
};

// y = s rstd scale, rstd = 1 / sqrt(mean(s^2) + eps).  101 us for 16383 x 4096 (x and residual read, y, the sum and the 8-bit
// checkpoint written: 605 MB, 6.0 TB/s, part of it out of the last-level cache); 8.7 us for 4096 x 1024; 3.5 us for 8 rows.
template <class T, int TPR, int V>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_fwd(RmsArgs p) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  __shared__ float lds[NT / 64];
  const int tid = threadIdx.x, t = tid % TPR;
  const int64_t row = int64_t(blockIdx.x) * (NT / TPR) + tid / TPR;
  if (row >= p.rows) return;   // (whole waves; with several waves a row, one row a workgroup)
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
  float s[V][8], w[V][8];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int col = 8 * (t + TPR * u), n = p.d - col;
    load8(x + col, n, s[u]);
    load_scale(p.scale, p.scale_type, col, n, w[u]);
    if (res) {
      float r[8];
      load8(res + col, n, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[u][i] = rounded(s[u][i] + r[i], T());
    }
  }
  float sq = 0;
#pragma unroll
  for (int u = 0; u < V; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(s[u][i], s[u][i], sq);
  sq = row_sum<TPR>(sq, lds, tid);
  const float rstd = 1.0f / sqrtf(sq / float(p.d) + p.eps);
  if (p.rstd && t == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int col = 8 * (t + TPR * u), n = p.d - col;
    if (p.sum) store8(static_cast<T*>(p.sum) + row * p.d + col, n, s[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[u][i] *= rstd;
    if (p.c.q) keep8(p.c, row, col, s[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[u][i] *= w[u][i];
    store8(static_cast<T*>(p.y) + row * p.d + col, n, s[u]);
  }
}

// With n = s rstd: dx = rstd (dy scale - n mean(dy scale n)) + dsum, dscale = sum over the rows of dy n.
// A workgroup of 1024 lanes takes rows 1024 / TPR at a time and keeps dscale's sums over its rows in registers; at the end
// they are added over its row groups through LDS, in a fixed tree, and go to part[workgroup].  At most 512 parts (256: the
// same time; 1024: 116 + 7.3 us in place of 110 + 4.9 with the sum of the parts).  110 us for 16383 x 4096 from the 8-bit
// checkpoint (473 MB, 4.3 TB/s): the row's sum stands between its loads and its stores; loading the next row ahead costs
// the registers of half the waves (117 us), and workgroups of 512 lanes, whose rows wait for fewer others, gain nothing
// (112).  9.6 us for 4096 x 1024.
template <class T, int TPR, int V>
__global__ __launch_bounds__(1024) void rms_bwd(RmsArgs p) {
  constexpr int G = 1024 / TPR;   // row groups
  __shared__ float lds[16];
  extern __shared__ float sums[];   // G / 2 rows of 8 TPR V
  const int tid = threadIdx.x, t = tid % TPR, g = tid / TPR;
  float w[V][8], acc[V][8] = {};
#pragma unroll
  for (int u = 0; u < V; ++u) load_scale(p.scale, p.scale_type, 8 * (t + TPR * u), p.d - 8 * (t + TPR * u), w[u]);
  for (int64_t row0 = int64_t(blockIdx.x) * G; row0 < p.rows; row0 += int64_t(gridDim.x) * G) {
    const bool ok = row0 + g < p.rows;   // (a group without a row works on the last one again and keeps nothing)
    const int64_t row = ok ? row0 + g : p.rows - 1;
    const float rstd = p.rstd[row];
    float n[V][8], dn[V][8];
    float dot = 0;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int col = 8 * (t + TPR * u), left = p.d - col;
      if (p.c.q) {
        if (left > 0) kept8(p.c, row, col, n[u]);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) n[u][i] = 0;
      } else {
        load8(static_cast<const T*>(p.x) + row * p.x_stride + col, left, n[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) n[u][i] *= rstd;
      }
      load8(static_cast<const T*>(p.dy) + row * p.dy_stride + col, left, dn[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (ok) acc[u][i] = fmaf(dn[u][i], n[u][i], acc[u][i]);
        dn[u][i] *= w[u][i];
        dot = fmaf(dn[u][i], n[u][i], dot);
      }
    }
    dot = row_sum<TPR>(dot, lds, tid) / float(p.d);
    if (!ok) continue;   // (the barriers are behind: a group is whole waves)
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int col = 8 * (t + TPR * u), left = p.d - col;
      float ds[8] = {};
      if (p.dsum) load8(static_cast<const T*>(p.dsum) + row * p.dsum_stride + col, left, ds);
#pragma unroll
      for (int i = 0; i < 8; ++i) ds[i] = fmaf(rstd, fmaf(-dot, n[u][i], dn[u][i]), ds[i]);
      store8(static_cast<T*>(p.dx) + row * p.d + col, left, ds);
    }
  }
  if (!p.part) return;
  for (int half = G / 2; half > 0; half /= 2) {
    __syncthreads();
    if (g >= half && g < 2 * half)
#pragma unroll
      for (int u = 0; u < V; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[(g - half) * 8 * TPR * V + (8 * u + i) * TPR + t] = acc[u][i];
    __syncthreads();
    if (g < half)
#pragma unroll
      for (int u = 0; u < V; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[u][i] += sums[g * 8 * TPR * V + (8 * u + i) * TPR + t];
  }
  if (g == 0)
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int col = 8 * (t + TPR * u);
      store8(p.part + int64_t(blockIdx.x) * p.d + col, p.d - col, acc[u]);
    }
}

// dscale from the workgroups' sums: 16 columns x 16 lanes a workgroup, each lane every 16th part, then the 16 in order.
// 3.0 us for 1024 columns, 4.9 us for 512 parts of 4096.
__global__ __launch_bounds__(256) void rms_dscale(RmsArgs p, int parts) {
  __shared__ float lds[16][17];
  const int c = threadIdx.x % 16, k = threadIdx.x / 16, col = blockIdx.x * 16 + c;
  float a = 0;
  if (col < p.d) {
#pragma unroll 8
    for (int i = k; i < parts; i += 16) a += p.part[int64_t(i) * p.d + col];
  }
  lds[k][c] = a;
  __syncthreads();
  if (k || col >= p.d) return;
  a = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) a += lds[i][c];
  if (p.scale_type == MSD_F32) static_cast<float*>(p.dscale)[col] = a;
  else static_cast<bf16*>(p.dscale)[col].x = uint16_t(pack2(a, 0.0f));
}

int row_lanes(int d) { return d <= 1024 ? 64 : d <= 4096 ? 256 : 1024; }

int rms_parts(int64_t rows, int d) { return int(std::min<int64_t>(cdiv(rows, 1024 / row_lanes(d)), 512)); }

template <class F>
void with_row(int d, F f) {
  using std::integral_constant;
  const int lanes = row_lanes(d);
  const bool two = d > 8 * lanes;
  if (lanes == 64) two ? f(integral_constant<int, 64>(), integral_constant<int, 2>()) : f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (lanes == 256) two ? f(integral_constant<int, 256>(), integral_constant<int, 2>()) : f(integral_constant<int, 256>(), integral_constant<int, 1>());
  else two ? f(integral_constant<int, 1024>(), integral_constant<int, 2>()) : f(integral_constant<int, 1024>(), integral_constant<int, 1>());
}

int32_t rms_check(int64_t rows, int d, int type, int scale_type) {
  if (rows < 0 || rows >= (int64_t(1) << 31) || d < 1 || d > 16384 || (type != MSD_BF16 && type != MSD_F32) ||
      (scale_type != MSD_BF16 && scale_type != MSD_F32))
    return MSD_E_CONFIG;
  // a launch has fewer than 2^32 threads
  return cdiv(rows * row_lanes(d), 256) >= (int64_t(1) << 24) ? MSD_E_CONFIG : MSD_OK;
}

// ---- SwiGLU ----
struct GluArgs {
  const void *gate, *up, *dy;
  int64_t gate_stride, up_stride, dy_stride, rows;
  int d;
  void *y, *dgate, *dup;
  Checkpoint cg, cu;
  Div groups;   // groups of eight values in a row; with a checkpoint whole blocks of 16 groups
};

// A lane's group: row and column.  Workgroup b takes groups 256 U b .. of the rows one behind the other.
struct Place {
  int64_t row;
  int col;
};
__device__ __forceinline__ Place place(const Div& groups, int64_t first, int i) {
  const int64_t row0 = first / groups.n;   // (uniform)
  const uint32_t at = uint32_t(first - row0 * groups.n) + i, r = groups(at);
  return {row0 + r, int(8 * (at - r * groups.n))};
}

// Groups of a lane: the forward takes one (two: 176 us in place of 165 for 16384 x 8192, 5.2 in place of 4.2 for 509 x 2816; the
// same with checkpoints), the backward one (two: 254 us in place of 243, 6.2 in place of 5.1), but two from a checkpoint, whose
// loads are of half the size (one: 243 us in place of 229).
constexpr int backward_groups(bool kept) { return kept ? 2 : 1; }

// y = g sigmoid(g) u.  16384 x 8192 in bf16: 165 us (805 MB, 4.9 TB/s), with the 8-bit checkpoint 206 to 258 us from card to
// card (1.08 GB, 5.2 to 4.2 TB/s).
template <class T, bool KEEP>
__global__ __launch_bounds__(256) void swiglu_fwd(GluArgs p) {
  constexpr int U = 1;
  float g[U][8], u[U][8];
  Place at[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    at[k] = place(p.groups, int64_t(blockIdx.x) * 256 * U, threadIdx.x + 256 * k);
    const int n = at[k].row < p.rows ? p.d - at[k].col : 0;
    load8(static_cast<const T*>(p.gate) + at[k].row * p.gate_stride + at[k].col, n, g[k]);
    load8(static_cast<const T*>(p.up) + at[k].row * p.up_stride + at[k].col, n, u[k]);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    if (at[k].row >= p.rows) continue;   // (whole blocks of 16 lanes: a row is whole blocks)
    if constexpr (KEEP) {
      keep8(p.cg, at[k].row, at[k].col, g[k]);
      keep8(p.cu, at[k].row, at[k].col, u[k]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) g[k][i] = g[k][i] / (1.0f + expf(-g[k][i])) * u[k][i];
    store8(static_cast<T*>(p.y) + at[k].row * p.d + at[k].col, p.d - at[k].col, g[k]);
  }
}

// With sig = sigmoid(g): du = dy g sig, dg = dy u sig (1 + g (1 - sig)).  16384 x 8192 in bf16: 243 us (1.34 GB, 5.5 TB/s), from
// the checkpoint 210 to 249 us (1.08 GB).
template <class T, bool KEPT>
__global__ __launch_bounds__(256) void swiglu_bwd(GluArgs p) {
  constexpr int U = backward_groups(KEPT);
  float g[U][8], u[U][8], dy[U][8];
  Place at[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    at[k] = place(p.groups, int64_t(blockIdx.x) * 256 * U, threadIdx.x + 256 * k);
    const int n = at[k].row < p.rows ? p.d - at[k].col : 0;
    if constexpr (KEPT) {
      if (n > 0) {
        kept8(p.cg, at[k].row, at[k].col, g[k]);
        kept8(p.cu, at[k].row, at[k].col, u[k]);
      }
    } else {
      load8(static_cast<const T*>(p.gate) + at[k].row * p.gate_stride + at[k].col, n, g[k]);
      load8(static_cast<const T*>(p.up) + at[k].row * p.up_stride + at[k].col, n, u[k]);
    }
    load8(static_cast<const T*>(p.dy) + at[k].row * p.dy_stride + at[k].col, n, dy[k]);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    if (at[k].row >= p.rows) continue;
    const int n = p.d - at[k].col;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float sig = 1.0f / (1.0f + expf(-g[k][i]));
      const float du = dy[k][i] * g[k][i] * sig;
      g[k][i] = dy[k][i] * u[k][i] * sig * fmaf(g[k][i], 1.0f - sig, 1.0f);
      u[k][i] = du;
    }
    store8(static_cast<T*>(p.dgate) + at[k].row * p.d + at[k].col, n, g[k]);
    store8(static_cast<T*>(p.dup) + at[k].row * p.d + at[k].col, n, u[k]);
  }
}

int32_t glu_check(int64_t rows, int d, int type) {
  if (rows < 0 || d < 1 || d >= (1 << 24) || rows >= (int64_t(1) << 40) / d || (type != MSD_BF16 && type != MSD_F32)) return MSD_E_CONFIG;
  // a launch has fewer than 2^32 threads
  return cdiv(rows * (padded(d) / 8), 256) >= (int64_t(1) << 24) ? MSD_E_CONFIG : MSD_OK;
}

unsigned glu_setup(GluArgs& p, int64_t rows, int d, const void* checkpoint_, int lane_groups) {
  p.rows = rows;
  p.d = d;
  p.groups = divider(uint32_t(checkpoint_ ? padded(d) / 8 : cdiv(d, 8)));
  if (checkpoint_) {
    uint8_t* c = static_cast<uint8_t*>(const_cast<void*>(checkpoint_));
    p.cg = checkpoint(c, rows, d);
    p.cu = checkpoint(c + checkpoint_bytes(rows, d), rows, d);
  }
  return unsigned(cdiv(rows * p.groups.n, 256 * lane_groups));
}

// ---- rotary positions ----
// (a, c) -> (a cos - c sin, a sin + c cos) amplitude; the gradient is the same turn backwards.  The angle p turns[i] is formed
// in f64 and reduced to less than a turn before it is rounded, so that far positions keep their precision.
// A workgroup takes kTokens tokens: their cosines and sines once, to LDS, for all heads (the f64 product and sincospif
// once a token and pair, not once a head); then units of work, a unit being W values of a head's copied part, W interleaved
// values, or W first and W second values of pairs.  A lane keeps one unit of the token (its head and place) over the
// tokens, kDeep of them in flight.  32767 tokens of 32 + 8 heads of 128 in bf16: 135 us (671 MB, 5.0 TB/s); f32 274 us; 4096 tokens
// of 16 + 4 heads of 64: 7.0 us.  With 4 or 16 tokens a workgroup 142 us (and 9.0 us for the small call, which then has too
// few workgroups); with 1, 2 or 8 tokens in flight within 5 % of 4 either way, by layout.
constexpr int kTokens = 8, kDeep = 4;

struct RopeArgs {
  const void *q, *k, *positions;
  const double* turns;
  void *q_out, *k_out;
  int64_t q_stride[3], k_stride[3], pos_stride[2], start, rows;
  int tokens, H, KV, D, rot, position_bytes, interleaved;
  float amplitude, sign;
  Div by_head_units;
  int token_units, groups;   // units of a token; tokens that the 256 lanes work on at a time
  int rot_units;             // units of a head that turn
};

template <int W>
__device__ __forceinline__ void turn8(float (&a)[8], float (&c)[8], const float2* w) {   // pairs (a[j], c[j])
#pragma unroll
  for (int j = 0; j < W; ++j) {
    const float x = a[j], y = c[j];
    a[j] = x * w[j].x - y * w[j].y;
    c[j] = x * w[j].y + y * w[j].x;
  }
}

template <class T, int W>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs p) {
  extern __shared__ float2 turn[];   // (cos, sin) of kTokens tokens, rot / 2 pairs each
  __shared__ int64_t q_at[kTokens], k_at[kTokens];
  const int half = p.rot / 2;
  const int64_t row0 = int64_t(blockIdx.x) * kTokens;
  const int n = int(min(int64_t(kTokens), p.rows - row0));
  for (int i = threadIdx.x; i < n * half; i += 256) {
    const int t = i / half, j = i - t * half;
    const int64_t row = row0 + t, b = row / p.tokens, tok = row - b * p.tokens;
    int64_t pos = p.start + tok;
    if (p.position_bytes) {
      const int64_t at = b * p.pos_stride[0] + tok * p.pos_stride[1];
      pos = p.position_bytes == 8 ? static_cast<const int64_t*>(p.positions)[at] : int64_t(static_cast<const int32_t*>(p.positions)[at]);
    }
    if (j == 0) {
      q_at[t] = b * p.q_stride[0] + tok * p.q_stride[1];
      k_at[t] = b * p.k_stride[0] + tok * p.k_stride[1];
    }
    const double a = double(pos) * p.turns[j];
    float s, c;
    sincospif(2.0f * float(a - floor(a)), &s, &c);
    turn[i] = make_float2(c * p.amplitude, s * p.amplitude * p.sign);
  }
  __syncthreads();
  const int units = int(p.by_head_units.n), group = p.groups > 1 ? int(threadIdx.x) / p.token_units : 0;
  if (group >= p.groups) return;
  for (int i = p.groups > 1 ? int(threadIdx.x) - group * p.token_units : int(threadIdx.x); i < p.token_units; i += 256) {
    int h = p.by_head_units(i);
    const int u = i - h * units;
    const bool isk = h >= p.H, copied = u >= p.rot_units;
    if (isk) h -= p.H;
    // where the unit's values lie in the head, where its second ones (or, of eight interleaved values, the second four)
    const int at = copied ? p.rot + (u - p.rot_units) * W : p.interleaved ? u * (W == 8 ? 8 : 2) : u * W;
    const int pair = p.interleaved ? u * (W == 8 ? 4 : 1) : u * W;
    const T* from = (isk ? static_cast<const T*>(p.k) + h * p.k_stride[2] : static_cast<const T*>(p.q) + h * p.q_stride[2]) + at;
    const int heads = isk ? p.KV : p.H;
    T* to = static_cast<T*>(isk ? p.k_out : p.q_out) + (row0 * heads + h) * p.D + at;
    const int64_t* row_at = isk ? k_at : q_at;
    const int64_t step = int64_t(heads) * p.D;
    for (int t0 = group; t0 < n; t0 += kDeep * p.groups) {
      float a[kDeep][8], c[kDeep][8];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const int t = t0 + d * p.groups;
        if (t >= n) break;
        const T* x = from + row_at[t];
        if constexpr (W == 8) {
          load8(x, 8, a[d]);
          if (!copied && !p.interleaved) load8(x + half, 8, c[d]);
        } else {
          load8(x, 1, a[d]);
          if (!copied) load8(x + (p.interleaved ? 1 : half), 1, c[d]);
        }
      }
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const int t = t0 + d * p.groups;
        if (t >= n) break;
        T* y = to + t * step;
        const float2* w = turn + t * half + pair;
        if (copied) {
          if constexpr (W == 8) store8(y, 8, a[d]);
          else store8(y, 1, a[d]);
        } else if constexpr (W == 8) {
          if (p.interleaved) {
            float e[8] = {a[d][0], a[d][2], a[d][4], a[d][6]}, f[8] = {a[d][1], a[d][3], a[d][5], a[d][7]};
            turn8<4>(e, f, w);
            const float r[8] = {e[0], f[0], e[1], f[1], e[2], f[2], e[3], f[3]};
            store8(y, 8, r);
          } else {
            turn8<8>(a[d], c[d], w);
            store8(y, 8, a[d]);
            store8(y + half, 8, c[d]);
          }
        } else {
          turn8<1>(a[d], c[d], w);
          store8(y, 1, a[d]);
          store8(y + (p.interleaved ? 1 : half), 1, c[d]);
        }
      }
    }
  }
}

}  // namespace msl

using namespace msl;

extern "C" int64_t msd_checkpoint_bytes(int64_t rows, int32_t d) {
  if (rows < 0 || d < 1 || d >= (1 << 24) || rows >= (int64_t(1) << 40) / d) return MSD_E_CONFIG;
  return checkpoint_bytes(rows, d);
}

extern "C" int32_t msd_rms_forward(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                   const void* scale, int32_t scale_type, int64_t rows, int32_t d, int32_t type, float eps,
                                   void* y, void* sum, float* rstd, void* checkpoint_, void* stream) {
  const int32_t rc = rms_check(rows, d, type, scale_type);
  if (rc != MSD_OK) return rc;
  if (!(eps >= 0) || x_stride < 0 || residual_stride < 0) return MSD_E_CONFIG;
  if (!rows) return MSD_OK;
  if (odd(x, type) || odd(scale, scale_type) || odd(y, type) || (residual && odd(residual, type)) ||
      (residual != nullptr) != (sum != nullptr) || (sum && odd(sum, type)) || reinterpret_cast<uintptr_t>(rstd) % 4 ||
      reinterpret_cast<uintptr_t>(checkpoint_) % 16)
    return MSD_E_ARG;
  RmsArgs p{};
  p.x = x;
  p.x_stride = x_stride;
  p.residual = residual;
  p.residual_stride = residual_stride;
  p.scale = scale;
  p.scale_type = scale_type;
  p.rows = rows;
  p.d = d;
  p.eps = eps;
  p.y = y;
  p.sum = sum;
  p.rstd = rstd;
  if (checkpoint_) p.c = checkpoint(checkpoint_, rows, d);
  with_type(type, [&](auto t) {
    with_row(d, [&](auto lanes, auto v) {
      constexpr int TPR = decltype(lanes)::value, NT = std::max(TPR, 256);
      hipLaunchKernelGGL((rms_fwd<decltype(t), TPR, decltype(v)::value>), dim3(unsigned(cdiv(rows, NT / TPR))), dim3(NT), 0,
                         static_cast<hipStream_t>(stream), p);
    });
  });
  return launched();
}

extern "C" int64_t msd_rms_workspace_bytes(int64_t rows, int32_t d) {
  const int32_t rc = rms_check(rows, d, MSD_BF16, MSD_BF16);
  return rc != MSD_OK ? rc : int64_t(4) * rms_parts(rows, d) * d;
}

extern "C" int32_t msd_rms_backward(const void* s, int64_t s_stride, const float* rstd, const void* checkpoint_,
                                    const void* scale, int32_t scale_type, const void* dy, int64_t dy_stride,
                                    const void* dsum, int64_t dsum_stride, int64_t rows, int32_t d, int32_t type, void* dx,
                                    void* dscale, void* workspace, void* stream) {
  const int32_t rc = rms_check(rows, d, type, scale_type);
  if (rc != MSD_OK) return rc;
  if (s_stride < 0 || dy_stride < 0 || dsum_stride < 0) return MSD_E_CONFIG;
  if ((dscale && odd(dscale, scale_type)) || odd(scale, scale_type)) return MSD_E_ARG;
  if (rows && ((!checkpoint_ && odd(s, type)) || odd(rstd, MSD_F32) || odd(dy, type) || (dsum && odd(dsum, type)) ||
               odd(dx, type) || reinterpret_cast<uintptr_t>(checkpoint_) % 16 || (dscale && odd(workspace, MSD_F32))))
    return MSD_E_ARG;
  RmsArgs p{};
  p.x = s;
  p.x_stride = s_stride;
  p.rstd = const_cast<float*>(rstd);
  if (checkpoint_) p.c = checkpoint(const_cast<void*>(checkpoint_), rows, d);
  p.scale = scale;
  p.scale_type = scale_type;
  p.dy = dy;
  p.dy_stride = dy_stride;
  p.dsum = dsum;
  p.dsum_stride = dsum_stride;
  p.rows = rows;
  p.d = d;
  p.dx = dx;
  p.dscale = dscale;
  p.part = dscale ? static_cast<float*>(workspace) : nullptr;
  const int parts = rms_parts(rows, d);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows)
    with_type(type, [&](auto t) {
      with_row(d, [&](auto lanes, auto v) {
        constexpr int TPR = decltype(lanes)::value, V = decltype(v)::value;
        constexpr size_t lds = size_t(1024 / TPR / 2) * 8 * TPR * V * 4;   // at most 32 KB
        hipLaunchKernelGGL((rms_bwd<decltype(t), TPR, V>), dim3(parts), dim3(1024), lds, st, p);
      });
    });
  if (dscale) hipLaunchKernelGGL(rms_dscale, dim3(unsigned(cdiv(d, 16))), dim3(256), 0, st, p, rows ? parts : 0);
  return launched();
}

extern "C" int32_t msd_swiglu_forward(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, int64_t rows,
                                      int32_t d, int32_t type, void* y, void* checkpoint_, void* stream) {
  const int32_t rc = glu_check(rows, d, type);
  if (rc != MSD_OK) return rc;
  if (gate_stride < 0 || up_stride < 0) return MSD_E_CONFIG;
  if (!rows) return MSD_OK;
  if (odd(gate, type) || odd(up, type) || odd(y, type) || reinterpret_cast<uintptr_t>(checkpoint_) % 16) return MSD_E_ARG;
  GluArgs p{};
  const unsigned blocks = glu_setup(p, rows, d, checkpoint_, 1);
  p.gate = gate;
  p.gate_stride = gate_stride;
  p.up = up;
  p.up_stride = up_stride;
  p.y = y;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(type, [&](auto t) {
    if (checkpoint_) hipLaunchKernelGGL((swiglu_fwd<decltype(t), true>), dim3(blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((swiglu_fwd<decltype(t), false>), dim3(blocks), dim3(256), 0, s, p);
  });
  return launched();
}

extern "C" int32_t msd_swiglu_backward(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride,
                                       const void* checkpoint_, const void* dy, int64_t dy_stride, int64_t rows, int32_t d,
                                       int32_t type, void* dgate, void* dup, void* stream) {
  const int32_t rc = glu_check(rows, d, type);
  if (rc != MSD_OK) return rc;
  if (gate_stride < 0 || up_stride < 0 || dy_stride < 0) return MSD_E_CONFIG;
  if (!rows) return MSD_OK;
  if ((!checkpoint_ && (odd(gate, type) || odd(up, type))) || odd(dy, type) || odd(dgate, type) || odd(dup, type) ||
      reinterpret_cast<uintptr_t>(checkpoint_) % 16)
    return MSD_E_ARG;
  GluArgs p{};
  const unsigned blocks = glu_setup(p, rows, d, checkpoint_, backward_groups(checkpoint_ != nullptr));
  p.gate = gate;
  p.gate_stride = gate_stride;
  p.up = up;
  p.up_stride = up_stride;
  p.dy = dy;
  p.dy_stride = dy_stride;
  p.dgate = dgate;
  p.dup = dup;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(type, [&](auto t) {
    if (checkpoint_) hipLaunchKernelGGL((swiglu_bwd<decltype(t), true>), dim3(blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((swiglu_bwd<decltype(t), false>), dim3(blocks), dim3(256), 0, s, p);
  });
  return launched();
}

extern "C" int32_t msd_rope_apply(const msd_rope* r, const void* q, const void* k, const void* positions, const double* turns,
                                  void* q_out, void* k_out, void* stream) {
  if (!r) return MSD_E_ARG;
  const int64_t rows = int64_t(r->batch) * r->tokens, heads = int64_t(r->n_heads) + r->n_kv_heads;
  if (r->batch < 0 || r->tokens < 0 || r->n_heads < 0 || r->n_kv_heads < 0 || heads > 4096 || r->d_head < 1 ||
      r->d_head > 4096 || r->d_rot < 2 || r->d_rot % 2 || r->d_rot > r->d_head || (r->type != MSD_BF16 && r->type != MSD_F32) ||
      (r->sign != 1 && r->sign != -1) || (r->position_bytes != 0 && r->position_bytes != 4 && r->position_bytes != 8) ||
      rows >= (int64_t(1) << 40) / (std::max<int64_t>(heads, 1) * r->d_head) || cdiv(rows, kTokens) >= (int64_t(1) << 24))
    return MSD_E_CONFIG;
  for (int i = 0; i < 3; ++i)
    if (r->q_stride[i] < 0 || r->k_stride[i] < 0) return MSD_E_CONFIG;
  if (!rows || !heads) return MSD_OK;
  if ((r->n_heads && (odd(q, r->type) || odd(q_out, r->type))) || (r->n_kv_heads && (odd(k, r->type) || odd(k_out, r->type))) ||
      !turns || reinterpret_cast<uintptr_t>(turns) % 8 ||
      (r->position_bytes && (!positions || reinterpret_cast<uintptr_t>(positions) % r->position_bytes)))
    return MSD_E_ARG;
  RopeArgs p{};
  p.q = q;
  p.k = k;
  p.positions = positions;
  p.turns = turns;
  p.q_out = q_out;
  p.k_out = k_out;
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = r->q_stride[i];
    p.k_stride[i] = r->k_stride[i];
  }
  p.pos_stride[0] = r->position_stride[0];
  p.pos_stride[1] = r->position_stride[1];
  p.start = r->start;
  p.rows = rows;
  p.tokens = r->tokens;
  p.H = r->n_heads;
  p.KV = r->n_kv_heads;
  p.D = r->d_head;
  p.rot = r->d_rot;
  p.position_bytes = r->position_bytes;
  p.interleaved = r->interleaved != 0;
  p.amplitude = r->amplitude;
  p.sign = float(r->sign);
  // eight values at a time where the turning and the copied part are whole groups of them (one at a time is there for
  // other sizes: 302 us in place of 135 at 32767 tokens of 40 heads of 128)
  const int half = r->d_rot / 2;
  const bool wide = (r->d_head - r->d_rot) % 8 == 0 && (r->interleaved ? r->d_rot : half) % 8 == 0;
  const int w = wide ? 8 : 1;
  p.rot_units = r->interleaved && wide ? r->d_rot / 8 : half / w;
  const int units = p.rot_units + (r->d_head - r->d_rot) / w;
  p.by_head_units = divider(uint32_t(units));
  p.token_units = int(units * heads);
  p.groups = std::max(256 / p.token_units, 1);
  const size_t lds = size_t(kTokens) * half * 8;   // d_rot 4096: 128 KB
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t err = hipSuccess;
  with_type(r->type, [&](auto t) {
    auto go = [&](auto kernel) {
      if (lds > 64000) err = msdc::ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), lds);
      if (err == hipSuccess)
        hipLaunchKernelGGL(kernel, dim3(unsigned(cdiv(rows, kTokens))), dim3(256), lds, s, p);
    };
    if (wide) go(rope_kernel<decltype(t), 8>);
    else go(rope_kernel<decltype(t), 1>);
  });
  return err != hipSuccess ? MSD_E_HIP : launched();
}
