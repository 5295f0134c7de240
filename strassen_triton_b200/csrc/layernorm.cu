// Layer norm over the last dimension of a matrix of rows, forward and backward.
//
//   y  = xhat * w + b,  xhat = (x - mu) * rstd,  rstd = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  g = dy * w
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// All statistics and sums are fp32; the variance is taken around the mean (a second look at the row),
// not as a difference of squares. Results are rounded once, to the type they are stored in.
//
// Both passes are bound by memory: the forward reads x and writes y, the backward reads x and dy and
// writes dx, each element once. A row lives in the registers of one warp (rows of up to 1024 elements) or
// of one block (up to 16384), NV vectors of VEC elements per thread, so mean, variance and result come
// from one reading; the next row's vectors are requested before the current row is reduced. Threads keep
// their columns from row to row: the parameter gradients add up in fp32 registers over all rows a block
// takes, then in one row of partial sums per block, then over the blocks in their order by a second
// kernel. VEC is 16 bytes where rows and pointers allow it, else 4 bytes, else one element. Longer rows
// take the looping kernels, which read a row again (from L1 / L2) instead of keeping it.
//
// Measured: 16381 x 4096 fp16 with fp32 parameters 48 us forward (5.6 TB/s) and 76 + 4 us backward (5.3 TB/s);
// 8192 x 768 bf16, resident in L2, 6.6 us and 16 us together, where latency counts: a warp has one to five rows.

#include <cuda_runtime.h>

#include "common.h"
#include "ptx_sm100.cuh"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

constexpr int kThreads = 256;

// s / d with the rounding of a division (1 / d alone is rounded already, and a row of one value would differ from its
// mean): the quotient's remainder, formed exactly by the fused operation, corrects it.
__device__ __forceinline__ float mean_of(float s, float inv_d, float d) {
  const float q = s * inv_d;
  return fmaf(fmaf(-q, d, s), inv_d, q);
}

struct NormFwd {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* mean;
  float* rstd;
  int64_t rows, d, ldx, ldy;
  int param_dtype;
  float eps;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_fwd_any_kernel(const NormFwd p) {
  __shared__ float slots[32];
  const float inv_d = 1.f / static_cast<float>(p.d);
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.ldx;
    T* y = static_cast<T*>(p.y) + r * p.ldy;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < p.d; c += kThreads) s += to_f(x[c]);
    const float mu = mean_of(row::block_sum(s, slots), inv_d, static_cast<float>(p.d));
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < p.d; c += kThreads) {
      const float t = to_f(x[c]) - mu;
      q = fmaf(t, t, q);
    }
    const float rs = rsqrtf(row::block_sum(q, slots) * inv_d + p.eps);
    for (int64_t c = threadIdx.x; c < p.d; c += kThreads) {
      float v = (to_f(x[c]) - mu) * rs;
      if (p.w) v *= row::ld_any(p.w, p.param_dtype, c);
      if (p.b) v += row::ld_any(p.b, p.param_dtype, c);
      y[c] = from_f<T>(v);
    }
    if (threadIdx.x == 0 && p.mean) {
      p.mean[r] = mu;
      p.rstd[r] = rs;
    }
  }
}

struct NormBwd {
  const void* x;
  const void* dy;
  const void* w;
  const float* mean;
  const float* rstd;
  void* dx;         // may be null
  float* part_w;    // slices x d partial sums of dw and db (null when not wanted)
  float* part_b;
  int64_t rows, d, ldx, lddy, lddx;
  int slices;
  int param_dtype;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_dx_any_kernel(const NormBwd p) {
  __shared__ float slots[32];
  const float inv_d = 1.f / static_cast<float>(p.d);
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + r * p.lddy;
    T* dx = static_cast<T*>(p.dx) + r * p.lddx;
    const float mu = p.mean[r], rs = p.rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < p.d; c += kThreads) {
      const float g = to_f(dy[c]) * (p.w ? row::ld_any(p.w, p.param_dtype, c) : 1.f);
      s1 += g;
      s2 = fmaf(g, (to_f(x[c]) - mu) * rs, s2);
    }
    const float m1 = row::block_sum(s1, slots) * inv_d;
    const float m2 = row::block_sum(s2, slots) * inv_d;
    for (int64_t c = threadIdx.x; c < p.d; c += kThreads) {
      const float g = to_f(dy[c]) * (p.w ? row::ld_any(p.w, p.param_dtype, c) : 1.f);
      dx[c] = from_f<T>(rs * (g - m1 - (to_f(x[c]) - mu) * rs * m2));
    }
  }
}

// Partial sums of dw and db: 32 columns per block, every slice of the grid's second dimension takes
// rows slice, slice + slices, ...
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_params_any_kernel(const NormBwd p) {
  __shared__ float sw[8][33], sb[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float aw = 0.f, ab = 0.f;
  if (c < p.d) {
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + ty; r < p.rows; r += static_cast<int64_t>(p.slices) * 8) {
      const float g = to_f(static_cast<const T*>(p.dy)[r * p.lddy + c]);
      const float xh = (to_f(static_cast<const T*>(p.x)[r * p.ldx + c]) - p.mean[r]) * p.rstd[r];
      aw = fmaf(g, xh, aw);
      ab += g;
    }
  }
  sw[ty][tx] = aw;
  sb[ty][tx] = ab;
  __syncthreads();
  if (ty == 0 && c < p.d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) aw += sw[k][tx], ab += sb[k][tx];
    if (p.part_w) p.part_w[blockIdx.y * p.d + c] = aw;
    if (p.part_b) p.part_b[blockIdx.y * p.d + c] = ab;
  }
}

// out[c] = sum of the slices: 32 columns per block, every 32nd slice a thread, then over those in order.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) norm_params_sum_kernel(const float* part_w, const float* part_b, void* dw,
                                                                      void* db, int64_t d, int slices, int param_dtype) {
  __shared__ float s[32][33];
  const float* part = blockIdx.y == 0 ? part_w : part_b;
  void* out = blockIdx.y == 0 ? dw : db;
  if (!out) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float a = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int k = ty; k < slices; k += 32) a += part[static_cast<int64_t>(k) * d + c];
  }
  s[ty][tx] = a;
  __syncthreads();
  if (ty == 0 && c < d) {
#pragma unroll
    for (int k = 1; k < 32; ++k) a += s[k][tx];
    row::st_any(out, param_dtype, c, a);
  }
}

// ---- rows kept in registers --------------------------------------------------------------------

using row::add_;
using row::fma_;
using row::hsum;
using row::mul_;
using row::Pack;
using row::Unit;

// VEC parameters of type W from column c on; `fill` where there are none.
template <typename W, int VEC>
__device__ __forceinline__ void ld_params(const void* p, int c, float fill, Pack<W, VEC>& out) {
  if (p) {
    constexpr int N = VEC * sizeof(W) > 16 ? 16 / sizeof(W) : VEC;   // elements of one access
#pragma unroll
    for (int k = 0; k < VEC; k += N)
      *reinterpret_cast<Pack<W, N>*>(out.e + k) = row::ld_const<Pack<W, N>>(static_cast<const W*>(p) + c + k);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) out.e[k] = from_f<W>(fill);
  }
}

// Two sums over a warp, left in lane 0 (x) and lane 16 (y): the halves of the warp take one each.
__device__ __forceinline__ float warp_sums(float2 v) {
  const bool upper = (threadIdx.x & 16) != 0;
  float a = upper ? v.y : v.x;
  a += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}
// Sums over the threads that share a row: a warp (TH = 32), or a block of TH threads, through `slots` and
// one barrier. `slots` alternates between two halves, so the next call may start while slow threads
// still read this one's. The block's warps are added in their order.
template <int TH, bool RING = false>
__device__ __forceinline__ float row_sum(float v, float* slots, int& flip, bool* ok = nullptr) {
  v = row::warp_sum(v);
  if constexpr (TH == 32) return v;
  float* s = slots + flip * 32;
  flip ^= 1;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  if constexpr (RING)
    *ok = __syncthreads_and(*ok);
  else
    __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < TH / 128; ++w) {
    const float4 q = reinterpret_cast<const float4*>(s)[w];
    v += (q.x + q.y) + (q.z + q.w);
  }
  return v;
}
template <int TH, bool RING = false>
__device__ __forceinline__ float2 row_sums(float2 v, float* slots, int& flip, bool* ok = nullptr) {
  const float a = warp_sums(v);
  if constexpr (TH == 32) return make_float2(__shfl_sync(0xffffffffu, a, 0), __shfl_sync(0xffffffffu, a, 16));
  float* s = slots + flip * 32;
  flip ^= 1;
  if ((threadIdx.x & 15) == 0) s[(threadIdx.x & 16) + (threadIdx.x >> 5)] = a;    // x in 0 .. 15, y in 16 .. 31
  if constexpr (RING)
    *ok = __syncthreads_and(*ok);
  else
    __syncthreads();
  float2 t = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < TH / 128; ++w) {
    const float4 q = reinterpret_cast<const float4*>(s)[w], u = reinterpret_cast<const float4*>(s + 16)[w];
    t.x += (q.x + q.y) + (q.z + q.w);
    t.y += (u.x + u.y) + (u.z + u.w);
  }
  return t;
}

constexpr int kWarpRows = 4;      // warps, and rows at a time, of a block in the warp-per-row form
constexpr int kMaxBlock = 512;    // threads of a block in the block-per-row forms: 128, 256 or 512

// Resident blocks per SM the register budget of the backward kernels is set for.
// The forward ring kernel has no sums to keep and runs half as many blocks more.
template <int TH>
constexpr int kFwdResident = TH == 512 ? 1 : 768 / TH;
template <int VEC, int NV, int TH>
constexpr int kResident = TH == 32 ? (NV * VEC <= 8 ? 6 : (NV * VEC <= 16 ? 4 : 3)) : kMaxBlock / TH;

template <typename T, typename W, int VEC, int NV, int TH>
__global__ void __launch_bounds__(TH == 32 ? 32 * kWarpRows : TH) norm_fwd_kernel(const NormFwd p) {
  using P = Pack<T, VEC>;
  using U = Unit<VEC>;
  using F = typename U::type;
  constexpr bool kKeep = NV * VEC <= 16;      // parameters stay in registers from row to row
  __shared__ __align__(16) float slots[64];
  int flip = 0;
  constexpr bool WARP = TH == 32;
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  constexpr int width = TH;
  const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? kWarpRows : 1);
  const int d = static_cast<int>(p.d);
  const float inv_d = 1.f / static_cast<float>(d);
  P next[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) next[i].e[e] = from_f<T>(0.f);   // columns from d on stay zero
  auto fetch = [&](int64_t r) {
    const T* x = static_cast<const T*>(p.x) + r * p.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) next[i] = row::ld_const<P>(x + c);
    }
  };
  if (first < p.rows) fetch(first);
  Pack<W, VEC> kw[kKeep ? NV : 1], kb[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) {
        ld_params<W, VEC>(p.w, c, 1.f, kw[i]);
        ld_params<W, VEC>(p.b, c, 0.f, kb[i]);
      }
    }
  }
  for (int64_t r = first; r < p.rows; r += step) {
    F x[NV][U::count];
    F s = U::all(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < U::count; ++k) {
        x[i][k] = row::unit_of<T, VEC>(next[i], k);
        s = add_(s, x[i][k]);
      }
    if (r + step < p.rows) fetch(r + step);
    const float mu = mean_of(row_sum<TH>(hsum(s), slots, flip), inv_d, static_cast<float>(d));
    const F shift = U::all(-mu);
    F q = U::all(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * width + lane) * VEC < d) {
#pragma unroll
        for (int k = 0; k < U::count; ++k) {
          x[i][k] = add_(x[i][k], shift);
          q = fma_(x[i][k], x[i][k], q);
        }
      }
    }
    const float rs = rsqrtf(row_sum<TH>(hsum(q), slots, flip) * inv_d + p.eps);
    const F scale = U::all(rs);
    T* y = static_cast<T*>(p.y) + r * p.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) {
        Pack<W, VEC> w, b;
        if constexpr (kKeep) {
          w = kw[i], b = kb[i];
        } else {
          ld_params<W, VEC>(p.w, c, 1.f, w);
          ld_params<W, VEC>(p.b, c, 0.f, b);
        }
        P out;
#pragma unroll
        for (int k = 0; k < U::count; ++k)
          row::set_unit<T, VEC>(out, k, fma_(mul_(x[i][k], scale), row::unit_of<W, VEC>(w, k), row::unit_of<W, VEC>(b, k)));
        row::st(y + c, out);
      }
    }
    if (lane == 0 && p.mean) {
      p.mean[r] = mu;
      p.rstd[r] = rs;
    }
  }
}

// Backward: block b leaves its sums of dw and db in row b of part_w and part_b. A row's vectors stay packed in
// their own type and are converted twice (for the sums, for dx): in fp32 they and the column sums would not
// fit the registers. The next row is requested early except where 32 elements a thread leave no room.
template <typename T, typename W, int VEC, int NV, int TH>
__global__ void __launch_bounds__(TH == 32 ? 32 * kWarpRows : TH, kResident<VEC, NV, TH>)
norm_bwd_kernel(const NormBwd p) {
  using P = Pack<T, VEC>;
  using U = Unit<VEC>;
  using F = typename U::type;
  constexpr bool kEarly = NV * VEC <= 24;
  constexpr bool kKeep = NV * VEC <= 16;
  __shared__ __align__(16) float slots[64];
  int flip = 0;
  constexpr bool WARP = TH == 32;
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  constexpr int width = TH;
  const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? kWarpRows : 1);
  const int d = static_cast<int>(p.d);
  const float inv_d = 1.f / static_cast<float>(d);
  F aw[NV][U::count], ab[NV][U::count];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < U::count; ++k) aw[i][k] = ab[i][k] = U::all(0.f);
  P xc[NV], gc[NV], xn[kEarly ? NV : 1], gn[kEarly ? NV : 1];
  float mu = 0.f, rs = 0.f, mun = 0.f, rsn = 0.f;
  auto fetch = [&](int64_t r, P* xd, P* gd, float& m, float& s) {
    const T* x = static_cast<const T*>(p.x) + r * p.ldx;
    const T* g = static_cast<const T*>(p.dy) + r * p.lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) {
        xd[i] = row::ld_const<P>(x + c);
        gd[i] = row::ld_const<P>(g + c);
      }
    }
    m = p.mean[r];
    s = p.rstd[r];
  };
  if (kEarly && first < p.rows) fetch(first, xn, gn, mun, rsn);
  Pack<W, VEC> kw[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) ld_params<W, VEC>(p.w, c, 1.f, kw[i]);
    }
  }
  for (int64_t r = first; r < p.rows; r += step) {
    if constexpr (kEarly) {
#pragma unroll
      for (int i = 0; i < NV; ++i) xc[i] = xn[i], gc[i] = gn[i];
      mu = mun, rs = rsn;
      if (r + step < p.rows) fetch(r + step, xn, gn, mun, rsn);
    } else {
      fetch(r, xc, gc, mu, rs);
    }
    const F shift = U::all(-mu), scale = U::all(rs);
    F s1 = U::all(0.f), s2 = U::all(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) {
        Pack<W, VEC> w;
        if constexpr (kKeep)
          w = kw[i];
        else
          ld_params<W, VEC>(p.w, c, 1.f, w);
#pragma unroll
        for (int k = 0; k < U::count; ++k) {
          const F dy = row::unit_of<T, VEC>(gc[i], k);
          const F xh = mul_(add_(row::unit_of<T, VEC>(xc[i], k), shift), scale);
          aw[i][k] = fma_(dy, xh, aw[i][k]);
          ab[i][k] = add_(ab[i][k], dy);
          const F g = mul_(dy, row::unit_of<W, VEC>(w, k));
          s1 = add_(s1, g);
          s2 = fma_(g, xh, s2);
        }
      }
    }
    if (p.dx) {
      const float2 m = row_sums<TH>(make_float2(hsum(s1), hsum(s2)), slots, flip);
      // dx = rs g - rs m1 - xhat rs m2
      const F m1 = U::all(-m.x * inv_d * rs), m2 = U::all(-m.y * inv_d * rs);
      T* dx = static_cast<T*>(p.dx) + r * p.lddx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * width + lane) * VEC;
        if (c < d) {
          Pack<W, VEC> w;
          if constexpr (kKeep)
            w = kw[i];
          else
            ld_params<W, VEC>(p.w, c, 1.f, w);
          P out;
#pragma unroll
          for (int k = 0; k < U::count; ++k) {
            const F xh = mul_(add_(row::unit_of<T, VEC>(xc[i], k), shift), scale);
            const F g = mul_(row::unit_of<T, VEC>(gc[i], k), row::unit_of<W, VEC>(w, k));
            row::set_unit<T, VEC>(out, k, fma_(g, scale, fma_(xh, m2, m1)));
          }
          row::st(dx + c, out);
        }
      }
    }
  }
  if (!p.part_w && !p.part_b) return;
  if constexpr (WARP) {
    // the block's warps hold the same columns: their sums are added in the order of the warps
    constexpr int kCols = NV * 32 * VEC;
    __shared__ __align__(16) float sw[kCols], sb[kCols];
    for (int k = 0; k < kWarpRows; ++k) {
      if ((threadIdx.x >> 5) == k) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < U::count; ++j) {
            F* tw = reinterpret_cast<F*>(sw + (i * 32 + lane) * VEC) + j;
            F* tb = reinterpret_cast<F*>(sb + (i * 32 + lane) * VEC) + j;
            *tw = k == 0 ? aw[i][j] : add_(*tw, aw[i][j]);
            *tb = k == 0 ? ab[i][j] : add_(*tb, ab[i][j]);
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < d; c += 32 * kWarpRows) {
      if (p.part_w) p.part_w[static_cast<int64_t>(blockIdx.x) * d + c] = sw[c];
      if (p.part_b) p.part_b[static_cast<int64_t>(blockIdx.x) * d + c] = sb[c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * width + lane) * VEC;
      if (c < d) {
        // (an even column of an even d, or single values: rows of partial sums keep pairs aligned)
        F* tw = p.part_w ? reinterpret_cast<F*>(p.part_w + static_cast<int64_t>(blockIdx.x) * d + c) : nullptr;
        F* tb = p.part_b ? reinterpret_cast<F*>(p.part_b + static_cast<int64_t>(blockIdx.x) * d + c) : nullptr;
#pragma unroll
        for (int k = 0; k < U::count; ++k) {
          if (tw) tw[k] = aw[i][k];
          if (tb) tb[k] = ab[i][k];
        }
      }
    }
  }
}

// ---- rows of a block fed through shared memory -------------------------------------------------
// The block-per-row forms read a row, meet at a barrier, and only then finish it: with one row in
// flight per block HBM waits for the barriers (d = 4096, 16-bit, backward: 112 us, here 97; 76 with 16 elements
// a thread instead of 8 and cheaper trees of sums, 109 with 32 on 128 threads).
// Here one thread keeps `stages` rows on their way into shared memory with bulk copies, whatever the
// other threads wait for. A stage is free again after the barrier of its row's sums, which every thread
// reaches after reading it. Waits are bounded: a block that gives up lets its copies land, reports and
// leaves without finishing its rows.

constexpr uint32_t kWhoNorm = 12;
constexpr uint64_t kNormDrainNs = 20ull * 1000 * 1000;

struct RowRing {
  uint32_t data, bars;       // shared-memory addresses: stages, one mbarrier per stage
  uint32_t stage_bytes;
  int stages;
};

struct RingState {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) stage = 0, phase ^= 1u;
  }
};

__device__ __forceinline__ RowRing make_ring(uint8_t* smem, int stages, uint32_t stage_bytes) {
  RowRing ring{ptx::smem_u32(smem) + 128, ptx::smem_u32(smem), stage_bytes, stages};
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) ptx::mbar_init(ring.bars + 8 * s, 1);
    ptx::fence_mbar_init();
  }
  __syncthreads();
  return ring;
}

__device__ __forceinline__ void give_up(const RowRing& ring, const RingState& at, int outstanding, uint32_t* status) {
  if (threadIdx.x != 0) return;
  RingState k = at;
  const uint64_t deadline = ptx::global_timer_ns() + kNormDrainNs;
  for (int i = 0; i < outstanding; ++i, k.next(ring.stages))
    if (!ptx::mbar_wait_until(ring.bars + 8 * k.stage, k.phase, deadline)) break;
  atomicExch(&status[0], 1u);
  atomicExch(&status[1], kWhoNorm);
}

template <typename T, typename W, int VEC, int NV, int TH>
__global__ void __launch_bounds__(TH, kFwdResident<TH>)
norm_fwd_ring_kernel(const NormFwd p, int stages, uint32_t* status) {
  using P = Pack<T, VEC>;
  using U = Unit<VEC>;
  using F = typename U::type;
  constexpr bool kKeep = NV * VEC <= 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float slots[64];
  __shared__ uint32_t abort_word;
  int flip = 0;
  const int d = static_cast<int>(p.d);
  const uint32_t row_bytes = static_cast<uint32_t>(d * sizeof(T));
  const float inv_d = 1.f / static_cast<float>(d);
  if (threadIdx.x == 0) abort_word = 0;
  const RowRing ring = make_ring(smem, stages, row_bytes);
  const int64_t step = gridDim.x;
  auto request = [&](int64_t r, int stage) {
    ptx::mbar_expect_tx(ring.bars + 8 * stage, row_bytes);
    ptx::bulk_load(ring.data + stage * ring.stage_bytes, static_cast<const T*>(p.x) + r * p.ldx, row_bytes, ring.bars + 8 * stage);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < stages && blockIdx.x + s * step < p.rows; ++s) request(blockIdx.x + s * step, s);
  Pack<W, VEC> kw[kKeep ? NV : 1], kb[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
      if (c < d) {
        ld_params<W, VEC>(p.w, c, 1.f, kw[i]);
        ld_params<W, VEC>(p.b, c, 0.f, kb[i]);
      }
    }
  }
  RingState at;
  for (int64_t r = blockIdx.x; r < p.rows; r += step) {
    bool ok = ptx::mbar_wait(ring.bars + 8 * at.stage, at.phase, &abort_word, kWhoNorm);
    const uint8_t* rowp = smem + 128 + at.stage * ring.stage_bytes;
    F x[NV][U::count];
    F s = U::all(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
      if (c < d) {
        const P v = row::ld<P>(rowp + c * sizeof(T));
#pragma unroll
        for (int k = 0; k < U::count; ++k) {
          x[i][k] = row::unit_of<T, VEC>(v, k);
          s = add_(s, x[i][k]);
        }
      }
    }
    const float mu = mean_of(row_sum<TH, true>(hsum(s), slots, flip, &ok), inv_d, static_cast<float>(d));
    if (!ok) {
      const int64_t left = (p.rows - r + step - 1) / step;
      give_up(ring, at, static_cast<int>(left < stages ? left : stages), status);
      return;
    }
    if (threadIdx.x == 0 && r + stages * step < p.rows) request(r + stages * step, at.stage);
    at.next(stages);
    const F shift = U::all(-mu);
    F q = U::all(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (static_cast<int>(i * TH + threadIdx.x) * VEC < d) {
#pragma unroll
        for (int k = 0; k < U::count; ++k) {
          x[i][k] = add_(x[i][k], shift);
          q = fma_(x[i][k], x[i][k], q);
        }
      }
    }
    const float rs = rsqrtf(row_sum<TH, true>(hsum(q), slots, flip, &ok) * inv_d + p.eps);
    const F scale = U::all(rs);
    T* y = static_cast<T*>(p.y) + r * p.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
      if (c < d) {
        Pack<W, VEC> w, b;
        if constexpr (kKeep) {
          w = kw[i], b = kb[i];
        } else {
          ld_params<W, VEC>(p.w, c, 1.f, w);
          ld_params<W, VEC>(p.b, c, 0.f, b);
        }
        P out;
#pragma unroll
        for (int k = 0; k < U::count; ++k)
          row::set_unit<T, VEC>(out, k, fma_(mul_(x[i][k], scale), row::unit_of<W, VEC>(w, k), row::unit_of<W, VEC>(b, k)));
        row::st(y + c, out);
      }
    }
    if (threadIdx.x == 0 && p.mean) {
      p.mean[r] = mu;
      p.rstd[r] = rs;
    }
  }
}

template <typename T, typename W, int VEC, int NV, int TH>
__global__ void __launch_bounds__(TH, kMaxBlock / TH)
norm_bwd_ring_kernel(const NormBwd p, int stages, uint32_t* status) {
  using P = Pack<T, VEC>;
  using U = Unit<VEC>;
  using F = typename U::type;
  constexpr bool kKeep = NV * VEC <= 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float slots[64];
  __shared__ uint32_t abort_word;
  int flip = 0;
  const int d = static_cast<int>(p.d);
  const uint32_t row_bytes = static_cast<uint32_t>(d * sizeof(T));
  const float inv_d = 1.f / static_cast<float>(d);
  if (threadIdx.x == 0) abort_word = 0;
  const RowRing ring = make_ring(smem, stages, 2 * row_bytes);
  const int64_t step = gridDim.x;
  auto request = [&](int64_t r, int stage) {
    const uint32_t bar = ring.bars + 8 * stage, dst = ring.data + stage * ring.stage_bytes;
    ptx::mbar_expect_tx(bar, 2 * row_bytes);
    ptx::bulk_load(dst, static_cast<const T*>(p.x) + r * p.ldx, row_bytes, bar);
    ptx::bulk_load(dst + row_bytes, static_cast<const T*>(p.dy) + r * p.lddy, row_bytes, bar);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < stages && blockIdx.x + s * step < p.rows; ++s) request(blockIdx.x + s * step, s);
  F aw[NV][U::count], ab[NV][U::count];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < U::count; ++k) aw[i][k] = ab[i][k] = U::all(0.f);
  Pack<W, VEC> kw[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
      if (c < d) ld_params<W, VEC>(p.w, c, 1.f, kw[i]);
    }
  }
  RingState at;
  float mun = 0.f, rsn = 0.f;
  if (blockIdx.x < p.rows) mun = p.mean[blockIdx.x], rsn = p.rstd[blockIdx.x];
  for (int64_t r = blockIdx.x; r < p.rows; r += step) {
    const float mu = mun, rs = rsn;
    if (r + step < p.rows) mun = p.mean[r + step], rsn = p.rstd[r + step];
    bool ok = ptx::mbar_wait(ring.bars + 8 * at.stage, at.phase, &abort_word, kWhoNorm);
    const uint8_t* rowp = smem + 128 + at.stage * ring.stage_bytes;
    const F shift = U::all(-mu), scale = U::all(rs);
    F s1 = U::all(0.f), s2 = U::all(0.f);
    P xc[NV], gc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
      if (c < d) {
        xc[i] = row::ld<P>(rowp + c * sizeof(T));
        gc[i] = row::ld<P>(rowp + row_bytes + c * sizeof(T));
        Pack<W, VEC> w;
        if constexpr (kKeep)
          w = kw[i];
        else
          ld_params<W, VEC>(p.w, c, 1.f, w);
#pragma unroll
        for (int k = 0; k < U::count; ++k) {
          const F dy = row::unit_of<T, VEC>(gc[i], k);
          const F xh = mul_(add_(row::unit_of<T, VEC>(xc[i], k), shift), scale);
          aw[i][k] = fma_(dy, xh, aw[i][k]);
          ab[i][k] = add_(ab[i][k], dy);
          const F g = mul_(dy, row::unit_of<W, VEC>(w, k));
          s1 = add_(s1, g);
          s2 = fma_(g, xh, s2);
        }
      }
    }
    const float2 m = row_sums<TH, true>(make_float2(hsum(s1), hsum(s2)), slots, flip, &ok);
    if (!ok) {
      const int64_t left = (p.rows - r + step - 1) / step;
      give_up(ring, at, static_cast<int>(left < stages ? left : stages), status);
      return;
    }
    if (threadIdx.x == 0 && r + stages * step < p.rows) request(r + stages * step, at.stage);
    at.next(stages);
    if (p.dx) {
      const F m1 = U::all(-m.x * inv_d * rs), m2 = U::all(-m.y * inv_d * rs);
      T* dx = static_cast<T*>(p.dx) + r * p.lddx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
        if (c < d) {
          Pack<W, VEC> w;
          if constexpr (kKeep)
            w = kw[i];
          else
            ld_params<W, VEC>(p.w, c, 1.f, w);
          P out;
#pragma unroll
          for (int k = 0; k < U::count; ++k) {
            const F xh = mul_(add_(row::unit_of<T, VEC>(xc[i], k), shift), scale);
            const F g = mul_(row::unit_of<T, VEC>(gc[i], k), row::unit_of<W, VEC>(w, k));
            row::set_unit<T, VEC>(out, k, fma_(g, scale, fma_(xh, m2, m1)));
          }
          row::st(dx + c, out);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = static_cast<int>(i * TH + threadIdx.x) * VEC;
    if (c < d) {
      F* tw = p.part_w ? reinterpret_cast<F*>(p.part_w + static_cast<int64_t>(blockIdx.x) * d + c) : nullptr;
      F* tb = p.part_b ? reinterpret_cast<F*>(p.part_b + static_cast<int64_t>(blockIdx.x) * d + c) : nullptr;
#pragma unroll
      for (int k = 0; k < U::count; ++k) {
        if (tw) tw[k] = aw[i][k];
        if (tb) tb[k] = ab[i][k];
      }
    }
  }
}

// Rows on their way per block: what fits 200 KB of an SM's shared memory shared by `per_sm` blocks, at
// most 8; fewer than two are not worth it (the register forms then keep one row ahead themselves).
constexpr int kRingBudget = 200 * 1024;
int ring_stages(uint32_t stage_bytes, int per_sm) {
  const int n = static_cast<int>(kRingBudget / per_sm / stage_bytes);
  return n > 8 ? 8 : n;
}

template <class K>
int allow_smem(K kernel, size_t bytes, int per_sm) {
  // What a launch gets unasked is 48 KB less the kernel's static shared memory (a few hundred bytes). The limit
  // belongs to the kernel on a device, which rows of many lengths share: it is set to the most any of them asks for,
  // so that a call never lowers it between another thread's setting and its launch.
  if (bytes <= 47 * 1024) return B200S_OK;
  B200S_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 + kRingBudget / per_sm));
  return B200S_OK;
}

// Which kernel a row length takes: elements per vector, vectors per thread, threads on a row (32: a warp;
// 0: the looping kernels).
struct RowForm {
  int vec, nv, threads;
};
RowForm row_form(int64_t d, size_t es, bool al16, bool al4) {
  const int wide = static_cast<int>(16 / es);
  const int vec = al16 && d % wide == 0 ? wide : (es == 2 && al4 && d % 2 == 0 ? 2 : 1);
  const int64_t n = (d + vec - 1) / vec;     // vectors of a row
  // a warp holds up to 1024 elements in 16-byte or 4-byte vectors, 512 in single elements
  const int warp_max = vec == wide ? 1024 / 32 / wide : (vec == 2 ? 16 : 16);
  if (n <= 32 * warp_max) {
    int nv = static_cast<int>((n + 31) / 32);
    if (vec == wide && es == 2) return {vec, nv, 32};                           // 1 .. 4
    if (vec == wide) return {vec, nv <= 1 ? 1 : (nv <= 2 ? 2 : (nv <= 4 ? 4 : (nv <= 6 ? 6 : 8))), 32};
    return {vec, nv <= 1 ? 1 : (nv <= 4 ? 4 : (nv <= 8 ? 8 : 16)), 32};
  }
  // a block with 16 elements a thread, of as few threads as hold the row; 32 elements when 512 threads do not.
  // The work per row that does not depend on its length (two trees of sums, a barrier) favours many
  // elements a thread, registers favour few: see the measurements at the ring kernels.
  for (int t : {128, 256, 512})
    if (n * vec <= 16 * t) return {vec, 16 / vec, t};
  if (vec > 1 && n * vec <= 32 * kMaxBlock) return {vec, 32 / vec, kMaxBlock};
  return {0, 0, 0};
}

// go(Form) for a form: its template arguments.
template <typename T, typename W, int VEC, int NV, int TH>
struct Form {
  using type = T;
  using param = W;
  static constexpr int vec = VEC, nv = NV, threads = TH;
  static constexpr bool warp = TH == 32;
};
template <typename T, typename PT, typename F>
int by_form_of(const RowForm& f, F&& go) {
  constexpr int W = static_cast<int>(16 / sizeof(T));
#define B200S_FORM(V, N, TH) \
  if (f.vec == (V) && f.nv == (N) && f.threads == (TH)) return go(Form<T, PT, V, N, TH>{});
  if constexpr (sizeof(T) == 2) {
    B200S_FORM(W, 1, 32) B200S_FORM(W, 2, 32) B200S_FORM(W, 3, 32) B200S_FORM(W, 4, 32)
    B200S_FORM(2, 1, 32) B200S_FORM(2, 4, 32) B200S_FORM(2, 8, 32) B200S_FORM(2, 16, 32)
    B200S_FORM(2, 8, 128) B200S_FORM(2, 8, 256) B200S_FORM(2, 8, 512) B200S_FORM(2, 16, 512)
  } else {
    B200S_FORM(W, 1, 32) B200S_FORM(W, 2, 32) B200S_FORM(W, 4, 32) B200S_FORM(W, 6, 32) B200S_FORM(W, 8, 32)
  }
  B200S_FORM(W, 16 / W, 128) B200S_FORM(W, 16 / W, 256) B200S_FORM(W, 16 / W, 512) B200S_FORM(W, 32 / W, 512)
  B200S_FORM(1, 1, 32) B200S_FORM(1, 4, 32) B200S_FORM(1, 8, 32) B200S_FORM(1, 16, 32)
  B200S_FORM(1, 16, 128) B200S_FORM(1, 16, 256) B200S_FORM(1, 16, 512)
#undef B200S_FORM
  return B200S_ERR_BAD_SHAPE;   // row_form names no other
}

template <typename T, typename F>
int by_form(const RowForm& f, int param_dtype, F&& go) {
  if constexpr (sizeof(T) == 2)
    if (param_dtype != B200S_FP32) return by_form_of<T, T>(f, go);
  return by_form_of<T, float>(f, go);
}

// Blocks of a form that are resident together on an SM, by the launch bounds of the kernels.
int blocks_per_sm(const RowForm& f) {
  if (f.threads == 32) return f.nv * f.vec <= 8 ? 6 : (f.nv * f.vec <= 16 ? 4 : 3);
  return kMaxBlock / f.threads;
}

// Blocks, and rows of partial sums, of the backward pass.
int bwd_blocks(const RowForm& f, int64_t rows) {
  const int64_t units = f.threads == 32 ? (rows + kWarpRows - 1) / kWarpRows : rows;
  const int64_t cap = 148 * static_cast<int64_t>(blocks_per_sm(f));
  return static_cast<int>(units < 1 ? 1 : (units < cap ? units : cap));
}

bool aligned_rows(const void* p, int64_t ld, int64_t rows, size_t es, uintptr_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && (rows <= 1 || (ld * static_cast<int64_t>(es)) % static_cast<int64_t>(to) == 0);
}

bool known_dtype(int d) { return d == B200S_BF16 || d == B200S_FP16 || d == B200S_FP32; }

int check_rows(int64_t rows, int64_t d, int dtype, int param_dtype) {
  if (rows < 0 || d <= 0 || d > INT32_MAX) return B200S_ERR_BAD_SHAPE;
  if (!known_dtype(dtype) || !known_dtype(param_dtype)) return B200S_ERR_BAD_DTYPE;
  if (param_dtype != dtype && param_dtype != B200S_FP32) return B200S_ERR_BAD_DTYPE;
  return B200S_OK;
}

bool misaligned(const void* p, size_t es) { return reinterpret_cast<uintptr_t>(p) % es != 0; }

template <typename F>
int by_dtype(int dtype, F&& f) {
  if (dtype == B200S_BF16) return f(__nv_bfloat16{});
  if (dtype == B200S_FP16) return f(__half{});
  return f(float{});
}

// Slices the rows are dealt to for the parameter gradients: the partial sums of a launch.
int param_slices(int64_t rows) {
  const int64_t want = (rows + 63) / 64;
  return static_cast<int>(want < 1 ? 1 : (want > 128 ? 128 : want));
}

int64_t row_grid(int64_t rows) { return rows < 148 * 16 ? rows : 148 * 16; }

}  // namespace

}  // namespace b200s

using namespace b200s;

extern "C" {

int b200s_layer_norm(int64_t rows, int64_t d, int dtype, int param_dtype, float eps, const void* x, int64_t ldx,
                     const void* weight, const void* bias, void* y, int64_t ldy, float* mean, float* rstd,
                     void* stream) {
  int rc = check_rows(rows, d, dtype, param_dtype);
  if (rc) return rc;
  if (!(eps >= 0.f)) return B200S_ERR_BAD_SHAPE;
  if (rows == 0) return B200S_OK;
  if (!x || !y || (!mean != !rstd)) return B200S_ERR_NULL_POINTER;
  if ((rows > 1 && ldx < 0) || (rows > 1 && ldy < d)) return B200S_ERR_BAD_STRIDE;
  const size_t es = dtype_size(dtype), ps = dtype_size(param_dtype);
  if (misaligned(x, es) || misaligned(y, es) || misaligned(weight, ps) || misaligned(bias, ps)) return B200S_ERR_BAD_ALIGNMENT;
  if (misaligned(mean, 4) || misaligned(rstd, 4)) return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const NormFwd p{x, weight, bias, y, mean, rstd, rows, d, ldx, ldy, param_dtype, eps};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto fits = [&](uintptr_t to) {
    const uintptr_t pto = to < 16 ? to * ps / es : 16;      // as many parameters as elements, 16 bytes at a time at most
    return aligned_rows(x, ldx, rows, es, to) && aligned_rows(y, ldy, rows, es, to) && !misaligned(weight, pto) && !misaligned(bias, pto);
  };
  const RowForm form = row_form(d, es, fits(16), fits(4));
  return by_dtype(dtype, [&](auto t) -> int {
    if (form.threads) {
      return by_form<decltype(t)>(form, param_dtype, [&](auto f) -> int {
        using F = decltype(f);
        if constexpr (!F::warp && F::vec * sizeof(typename F::type) == 16) {
          constexpr int per_sm = kFwdResident<F::threads>;
          const uint32_t bytes = static_cast<uint32_t>(d * es);
          const int stages = ring_stages(bytes, per_sm);
          if (stages >= 2 && rows > 148 * per_sm) {
            auto kernel = norm_fwd_ring_kernel<typename F::type, typename F::param, F::vec, F::nv, F::threads>;
            int rc2 = allow_smem(kernel, 128 + static_cast<size_t>(stages) * bytes, per_sm);
            if (rc2) return rc2;
            kernel<<<148 * per_sm, form.threads, 128 + static_cast<size_t>(stages) * bytes, s>>>(p, stages, device_status_words());
            B200S_CUDA_OK(cudaGetLastError());
            count_launch();
            return B200S_OK;
          }
        }
        const int64_t units = F::warp ? (rows + kWarpRows - 1) / kWarpRows : rows;
        const int64_t cap = 148 * static_cast<int64_t>(F::warp ? 16 : (form.threads <= 128 ? 8 : (form.threads <= 256 ? 4 : 2)));
        norm_fwd_kernel<typename F::type, typename F::param, F::vec, F::nv, F::threads>
            <<<static_cast<unsigned>(units < cap ? units : cap), F::warp ? 32 * kWarpRows : form.threads, 0, s>>>(p);
        B200S_CUDA_OK(cudaGetLastError());
        count_launch();
        return B200S_OK;
      });
    }
    norm_fwd_any_kernel<decltype(t)><<<static_cast<unsigned>(row_grid(rows)), kThreads, 0, s>>>(p);
    B200S_CUDA_OK(cudaGetLastError());
    count_launch();
    return B200S_OK;
  });
}

int b200s_layer_norm_backward_workspace(int64_t rows, int64_t d, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  if (rows < 0 || d <= 0 || d > INT32_MAX) return B200S_ERR_BAD_SHAPE;
  // room for the partial sums of whichever kernel the operands' type and alignment lead to
  int64_t slices = param_slices(rows);
  for (size_t es : {size_t{2}, size_t{4}})
    for (int al = 0; al < 3; ++al) {
      const RowForm f = row_form(d, es, al == 2, al >= 1);
      if (f.threads && bwd_blocks(f, rows) > slices) slices = bwd_blocks(f, rows);
    }
  *bytes_out = static_cast<size_t>(slices) * static_cast<size_t>(d) * 2 * sizeof(float);
  return B200S_OK;
}

int b200s_layer_norm_backward(int64_t rows, int64_t d, int dtype, int param_dtype, const void* x, int64_t ldx,
                              const void* dy, int64_t lddy, const void* weight, const float* mean, const float* rstd,
                              void* dx, int64_t lddx, void* dweight, void* dbias, void* workspace,
                              size_t workspace_bytes, void* stream) {
  int rc = check_rows(rows, d, dtype, param_dtype);
  if (rc) return rc;
  if (rows > 0 && (!x || !dy || !mean || !rstd)) return B200S_ERR_NULL_POINTER;
  if (rows > 1 && (ldx < 0 || lddy < 0 || (dx && lddx < d))) return B200S_ERR_BAD_STRIDE;
  const size_t es = dtype_size(dtype), ps = dtype_size(param_dtype);
  if (misaligned(x, es) || misaligned(dy, es) || misaligned(dx, es) || misaligned(weight, ps) || misaligned(dweight, ps) ||
      misaligned(dbias, ps) || misaligned(mean, 4) || misaligned(rstd, 4))
    return B200S_ERR_BAD_ALIGNMENT;
  size_t need = 0;
  b200s_layer_norm_backward_workspace(rows, d, &need);
  if (dweight || dbias) {
    if (!workspace) return B200S_ERR_NULL_POINTER;
    if (workspace_bytes < need) return B200S_ERR_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return B200S_ERR_BAD_ALIGNMENT;
  }
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto fits = [&](uintptr_t to) {
    const uintptr_t pto = to < 16 ? to * ps / es : 16;
    return aligned_rows(x, ldx, rows, es, to) && aligned_rows(dy, lddy, rows, es, to) && aligned_rows(dx, lddx, rows, es, to) &&
           !misaligned(weight, pto);
  };
  const RowForm form = rows > 0 ? row_form(d, es, fits(16), fits(4)) : RowForm{0, 0, 0};
  const int slices = form.threads ? bwd_blocks(form, rows) : param_slices(rows);
  float* part = static_cast<float*>(workspace);
  const NormBwd p{x,    dy,  weight, mean, rstd, dx,   dweight ? part : nullptr, dbias ? part + static_cast<int64_t>(slices) * d : nullptr,
                  rows, d,   ldx,    lddy, lddx, slices, param_dtype};
  return by_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned cols = static_cast<unsigned>((d + 31) / 32);
    if (form.threads) {
      int rc2 = by_form<T>(form, param_dtype, [&](auto f) -> int {
        using F = decltype(f);
        if constexpr (!F::warp && F::vec * sizeof(T) == 16) {
          const uint32_t bytes = static_cast<uint32_t>(2 * d * es);
          const int stages = ring_stages(bytes, blocks_per_sm(form));
          if (stages >= 2 && rows > slices) {
            auto kernel = norm_bwd_ring_kernel<T, typename F::param, F::vec, F::nv, F::threads>;
            int rc3 = allow_smem(kernel, 128 + static_cast<size_t>(stages) * bytes, blocks_per_sm(form));
            if (rc3) return rc3;
            kernel<<<slices, form.threads, 128 + static_cast<size_t>(stages) * bytes, s>>>(p, stages, device_status_words());
            B200S_CUDA_OK(cudaGetLastError());
            count_launch();
            return B200S_OK;
          }
        }
        norm_bwd_kernel<T, typename F::param, F::vec, F::nv, F::threads><<<slices, F::warp ? 32 * kWarpRows : form.threads, 0, s>>>(p);
        B200S_CUDA_OK(cudaGetLastError());
        count_launch();
        return B200S_OK;
      });
      if (rc2 || (!dweight && !dbias)) return rc2;
      norm_params_sum_kernel<<<dim3(cols, 2), kSumThreads, 0, s>>>(p.part_w, p.part_b, dweight, dbias, d, slices, param_dtype);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
      return B200S_OK;
    }
    if (dx && rows > 0) {
      norm_dx_any_kernel<T><<<static_cast<unsigned>(row_grid(rows)), kThreads, 0, s>>>(p);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
    }
    if (dweight || dbias) {
      norm_params_any_kernel<T><<<dim3(cols, slices), kThreads, 0, s>>>(p);
      norm_params_sum_kernel<<<dim3(cols, 2), kSumThreads, 0, s>>>(p.part_w, p.part_b, dweight, dbias, d, slices, param_dtype);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch(2);
    }
    return B200S_OK;
  });
}

}  // extern "C"
