// Shared pieces of the row-wise kernels (layer norm, token log probabilities, epilogue passes, gradient
// norms): conversions to and from fp32, vectors of VEC elements, sums over a warp or a block.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200s.h"

namespace b200s {
namespace row {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Element i of a parameter vector whose type is known at run time only.
__device__ __forceinline__ float ld_any(const void* p, int dtype, int64_t i) {
  if (dtype == B200S_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == B200S_FP16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void st_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == B200S_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == B200S_FP16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<float*>(p)[i] = v;
}

// VEC elements moved by one access (VEC * sizeof(T) = 2, 4 or 16 bytes, aligned to that).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T e[VEC];
};

// ---- pairs of fp32 values ------------------------------------------------------------------------
// sm_100 adds, multiplies and fuses two fp32 values per instruction (each lane rounded as the scalar
// form rounds). The single-float overloads let one body serve vectors of one element.
__device__ __forceinline__ uint64_t f2_bits(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 bits_f2(uint64_t b) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(b));
  return v;
}
__device__ __forceinline__ float2 fma_(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return bits_f2(r);
}
__device__ __forceinline__ float2 add_(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return bits_f2(r);
}
__device__ __forceinline__ float2 mul_(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return bits_f2(r);
}
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float add_(float a, float b) { return a + b; }
__device__ __forceinline__ float mul_(float a, float b) { return a * b; }
__device__ __forceinline__ float hsum(float2 a) { return a.x + a.y; }
__device__ __forceinline__ float hsum(float a) { return a; }

// The arithmetic unit of vectors of VEC elements: a pair, or one value.
template <int VEC>
struct Unit {
  using type = float2;
  static constexpr int n = 2, count = VEC / 2;
  static __device__ __forceinline__ float2 all(float v) { return make_float2(v, v); }
};
template <>
struct Unit<1> {
  using type = float;
  static constexpr int n = 1, count = 1;
  static __device__ __forceinline__ float all(float v) { return v; }
};

// Two neighbouring elements <-> a pair.
__device__ __forceinline__ float2 load2(const __nv_bfloat16* e) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(e);
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 load2(const __half* e) { return __half22float2(*reinterpret_cast<const __half2*>(e)); }
__device__ __forceinline__ float2 load2(const float* e) { return *reinterpret_cast<const float2*>(e); }
__device__ __forceinline__ void store2(__nv_bfloat16* e, float2 v) { *reinterpret_cast<__nv_bfloat162*>(e) = __float22bfloat162_rn(v); }
__device__ __forceinline__ void store2(__half* e, float2 v) { *reinterpret_cast<__half2*>(e) = __float22half2_rn(v); }
__device__ __forceinline__ void store2(float* e, float2 v) { *reinterpret_cast<float2*>(e) = v; }

// Unit k of a vector.
template <typename T, int VEC>
__device__ __forceinline__ typename Unit<VEC>::type unit_of(const Pack<T, VEC>& v, int k) {
  if constexpr (VEC == 1)
    return to_f(v.e[0]);
  else
    return load2(v.e + 2 * k);
}
template <typename T, int VEC>
__device__ __forceinline__ void set_unit(Pack<T, VEC>& v, int k, typename Unit<VEC>::type u) {
  if constexpr (VEC == 1)
    v.e[0] = from_f<T>(u);
  else
    store2(v.e + 2 * k, u);
}

// One access of a whole vector. (Copying a Pack member by member leaves the width of the access to the
// compiler, which does not always find it.) ld_const is for data nobody writes during the launch.
template <int BYTES>
struct Raw;
template <>
struct Raw<16> {
  using type = uint4;
};
template <>
struct Raw<8> {
  using type = uint2;
};
template <>
struct Raw<4> {
  using type = uint32_t;
};
template <>
struct Raw<2> {
  using type = unsigned short;
};
template <typename P>
__device__ __forceinline__ P ld(const void* p) {
  using R = typename Raw<sizeof(P)>::type;
  const R q = *static_cast<const R*>(p);
  return *reinterpret_cast<const P*>(&q);
}
template <typename P>
__device__ __forceinline__ P ld_const(const void* p) {
  using R = typename Raw<sizeof(P)>::type;
  const R q = __ldg(static_cast<const R*>(p));
  return *reinterpret_cast<const P*>(&q);
}
template <typename P>
__device__ __forceinline__ void st(void* p, const P& v) {
  using R = typename Raw<sizeof(P)>::type;
  *static_cast<R*>(p) = *reinterpret_cast<const R*>(&v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block, given to every thread. `slots` holds one float per warp; two barriers, so that
// consecutive calls may share it.
__device__ __forceinline__ float block_sum(float v, float* slots) {
  const int warps = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < warps; ++w) t += slots[w];
  __syncthreads();
  return t;
}

}  // namespace row
}  // namespace b200s
