// Activations of the linear layer's epilogue and their derivatives, in fp32.
//
//   relu2(z) = max(z, 0)^2            silu(z) = z sigmoid(z)
//   gelu(z) = z Phi(z), Phi the normal distribution function
//   gelu_tanh(z) = z sigmoid(2 c (z + 0.044715 z^3)), c = sqrt(2 / pi): (1 + tanh a) / 2 = sigmoid(2a)
#pragma once

#include <cuda_runtime.h>

#include "../../include/b200s.h"
#include "rowwise_device.cuh"

namespace b200s {
namespace epi {

constexpr float kTanhC = 0.7978845608028654f;    // sqrt(2 / pi)
constexpr float kTanhA = 0.044715f;
constexpr float kPdf0 = 0.3989422804014327f;     // 1 / sqrt(2 pi)

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if constexpr (ACT == B200S_ACT_RELU) return z < 0.f ? 0.f : z;       // NaN stays NaN
  if constexpr (ACT == B200S_ACT_RELU2) return z < 0.f ? 0.f : z * z;
  if constexpr (ACT == B200S_ACT_SILU) return z * (1.f / (1.f + __expf(-z)));
  if constexpr (ACT == B200S_ACT_GELU) return z * normcdff(z);
  if constexpr (ACT == B200S_ACT_GELU_TANH) return z * (1.f / (1.f + __expf(-2.f * kTanhC * fmaf(kTanhA * z, z * z, z))));
  return z;
}

template <int ACT>
__device__ __forceinline__ float dact(float z) {
  if constexpr (ACT == B200S_ACT_RELU) return z > 0.f ? 1.f : (z == z ? 0.f : z);
  if constexpr (ACT == B200S_ACT_RELU2) return z > 0.f ? 2.f * z : (z == z ? 0.f : z);
  if constexpr (ACT == B200S_ACT_SILU) {
    const float t = fminf(fmaxf(z, -80.f), 80.f);                      // beyond, the limits 0 and 1 hold to the last bit
    const float s = 1.f / (1.f + __expf(-t));
    return (z == z) ? s * fmaf(t, 1.f - s, 1.f) : z;
  }
  if constexpr (ACT == B200S_ACT_GELU) {
    const float t = fminf(fmaxf(z, -20.f), 20.f);
    return (z == z) ? fmaf(t * kPdf0, __expf(-0.5f * t * t), normcdff(t)) : z;
  }
  if constexpr (ACT == B200S_ACT_GELU_TANH) {
    const float t = fminf(fmaxf(z, -20.f), 20.f);
    const float s = 1.f / (1.f + __expf(-2.f * kTanhC * fmaf(kTanhA * t, t * t, t)));
    return (z == z) ? fmaf(t * s * (1.f - s), 2.f * kTanhC * fmaf(3.f * kTanhA * t, t, 1.f), s) : z;
  }
  return 1.f;
}

// ---- the same for 16-bit results: two fast exponentials or reciprocals per value --------------------
// Phi(-a) = e^(-a^2 / 2) P(1 / (1 + 0.35 a)) for a >= 0, P of degree 5: a least-squares fit of
// 0.5 e^(a^2 / 2) erfc(a / sqrt 2), reweighted until its relative error is level (Lawson): 5.5e-6 = 2^-17.5
// for a up to 9, where 16-bit results need 2^-12.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kHalfLog2e = 0.7213475204444817f;
__device__ __forceinline__ float upper_tail(float a, float e) {      // e = e^(-a^2 / 2)
  const float t = rcp(fmaf(0.35f, a, 1.f));
  float p = fmaf(-0.10458728923f, t, 0.29827082271f);
  p = fmaf(p, t, -0.00994253091f);
  p = fmaf(p, t, 0.18356833940f);
  p = fmaf(p, t, 0.13218160375f);
  p = fmaf(p, t, 0.00050789281f);
  return p * e;
}
__device__ __forceinline__ float fast_sigmoid(float z) { return rcp(1.f + ex2(-2.f * kHalfLog2e * z)); }

template <int ACT>
__device__ __forceinline__ float act_fast(float z) {
  if constexpr (ACT == B200S_ACT_SILU) return z * fast_sigmoid(z);
  if constexpr (ACT == B200S_ACT_GELU) {
    const float a = fminf(fabsf(z), 30.f);
    const float q = upper_tail(a, ex2(-kHalfLog2e * a * a));
    return fmaf(-a, q, z < 0.f ? 0.f : z);          // z - z Phi(-z), or z Phi(z)
  }
  if constexpr (ACT == B200S_ACT_GELU_TANH) return z * fast_sigmoid(2.f * kTanhC * fmaf(kTanhA * z, z * z, z));
  return act<ACT>(z);
}
// Two values at a time, with the packed fp32 instructions (the same arithmetic as act_fast).
__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
template <int ACT>
__device__ __forceinline__ float2 act_fast2(float2 z) {
  using row::add_;
  using row::fma_;
  using row::mul_;
  if constexpr (ACT == B200S_ACT_SILU || ACT == B200S_ACT_GELU_TANH) {
    float2 u;
    if constexpr (ACT == B200S_ACT_SILU)
      u = mul_(z, pair(-2.f * kHalfLog2e));
    else
      u = mul_(mul_(z, pair(-4.f * kHalfLog2e * kTanhC)), fma_(mul_(z, z), pair(kTanhA), pair(1.f)));
    const float2 d = add_(make_float2(ex2(u.x), ex2(u.y)), pair(1.f));
    return mul_(z, make_float2(rcp(d.x), rcp(d.y)));
  } else if constexpr (ACT == B200S_ACT_GELU) {
    const float2 a = make_float2(fminf(fabsf(z.x), 30.f), fminf(fabsf(z.y), 30.f));
    const float2 h = mul_(mul_(a, a), pair(-kHalfLog2e));
    const float2 d = fma_(a, pair(0.35f), pair(1.f));
    const float2 t = make_float2(rcp(d.x), rcp(d.y));
    float2 q = fma_(t, pair(0.10458728923f), pair(-0.29827082271f));      // -P(t)
    q = fma_(q, t, pair(0.00994253091f));
    q = fma_(q, t, pair(-0.18356833940f));
    q = fma_(q, t, pair(-0.13218160375f));
    q = fma_(q, t, pair(-0.00050789281f));
    q = mul_(q, make_float2(ex2(h.x), ex2(h.y)));
    return fma_(a, q, make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y));
  } else {
    return make_float2(act<ACT>(z.x), act<ACT>(z.y));
  }
}

template <int ACT>
__device__ __forceinline__ float dact_fast(float z) {
  if constexpr (ACT == B200S_ACT_SILU) {
    const float t = fminf(fmaxf(z, -80.f), 80.f);
    const float s = fast_sigmoid(t);
    return (z == z) ? s * fmaf(t, 1.f - s, 1.f) : z;
  }
  if constexpr (ACT == B200S_ACT_GELU) {
    const float a = fminf(fabsf(z), 30.f);
    const float e = ex2(-kHalfLog2e * a * a);
    const float q = upper_tail(a, e);
    const float w = fmaf(-a * kPdf0, e, q);         // Phi(-a) - a phi(a)
    return (z == z) ? (z < 0.f ? w : 1.f - w) : z;
  }
  if constexpr (ACT == B200S_ACT_GELU_TANH) {
    const float t = fminf(fmaxf(z, -20.f), 20.f);
    const float s = fast_sigmoid(2.f * kTanhC * fmaf(kTanhA * t, t * t, t));
    return (z == z) ? fmaf(t * s * (1.f - s), 2.f * kTanhC * fmaf(3.f * kTanhA * t, t, 1.f), s) : z;
  }
  return dact<ACT>(z);
}

template <int ACT>
__device__ __forceinline__ float2 dact_fast2(float2 z) {
  using row::fma_;
  using row::mul_;
  if constexpr (ACT == B200S_ACT_GELU) {
    const float2 a = make_float2(fminf(fabsf(z.x), 30.f), fminf(fabsf(z.y), 30.f));
    const float2 h = mul_(mul_(a, a), pair(-kHalfLog2e));
    const float2 d = fma_(a, pair(0.35f), pair(1.f));
    const float2 t = make_float2(rcp(d.x), rcp(d.y));
    float2 q = fma_(t, pair(-0.10458728923f), pair(0.29827082271f));
    q = fma_(q, t, pair(-0.00994253091f));
    q = fma_(q, t, pair(0.18356833940f));
    q = fma_(q, t, pair(0.13218160375f));
    q = fma_(q, t, pair(0.00050789281f));
    // Phi(-a) - a phi(a)
    const float2 w = mul_(fma_(a, pair(-kPdf0), q), make_float2(ex2(h.x), ex2(h.y)));
    const float2 r = make_float2(z.x < 0.f ? w.x : 1.f - w.x, z.y < 0.f ? w.y : 1.f - w.y);
    return make_float2(z.x == z.x ? r.x : z.x, z.y == z.y ? r.y : z.y);
  } else {
    return make_float2(dact_fast<ACT>(z.x), dact_fast<ACT>(z.y));
  }
}

// f(std::integral_constant<int, ACT>) for the activation known at run time.
template <int N>
struct Act {
  static constexpr int value = N;
};
template <typename F>
__host__ int by_activation(int a, F&& f) {
  switch (a) {
    case B200S_ACT_NONE: return f(Act<B200S_ACT_NONE>{});
    case B200S_ACT_RELU: return f(Act<B200S_ACT_RELU>{});
    case B200S_ACT_RELU2: return f(Act<B200S_ACT_RELU2>{});
    case B200S_ACT_SILU: return f(Act<B200S_ACT_SILU>{});
    case B200S_ACT_GELU: return f(Act<B200S_ACT_GELU>{});
    case B200S_ACT_GELU_TANH: return f(Act<B200S_ACT_GELU_TANH>{});
  }
  return B200S_ERR_BAD_ALGO;
}

}  // namespace epi
}  // namespace b200s
