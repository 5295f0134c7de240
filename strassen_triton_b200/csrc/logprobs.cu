// Log probabilities of given tokens, with the entropy of every row's distribution and its k most
// likely alternatives, and the gradient of the first two with respect to the logits.
//
//   m = max x, s = sum e^(x-m), u = sum e^(x-m) (x-m)      one pass, m running
//   lse = m + log s, logprob = x_t - lse, entropy = log s - u / s
//   dx_i = gl (1[i = t] - p_i) - ge p_i (log p_i + entropy),  p_i = e^(x_i - lse)
//
// The running maximum, both sums and everything derived from them are fp32. A forbidden token (-inf)
// has probability zero and takes no part in u. A row without any finite logit has no distribution:
// its logprob and lse are -inf, its entropy and its gradient zero. NaN (or +inf) among the logits
// makes the row's results NaN. A target equal to ignore_index gives logprob 0 and no gradient from
// it; any other target outside [0, vocab) gives NaN and is never used as an address.

#include <cuda_runtime.h>

#include "common.h"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

constexpr int kThreads = 256;
constexpr int kMaxTopK = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }

// Running statistics of a set of logits.
struct Stats {
  float m, s, u;
};
__device__ __forceinline__ Stats empty_stats() { return {kNegInf, 0.f, 0.f}; }

// e^(m - to) of statistics moved to the larger maximum `to`.
__device__ __forceinline__ void rescale(Stats& a, float to) {
  if (a.m == to) return;
  if (a.m == kNegInf) {
    a.m = to;    // nothing finite in the set so far: both sums are zero (or NaN, and stay so)
    return;
  }
  const float d = a.m - to;
  const float f = exp2f(d * kLog2e);
  a.u = f * fmaf(a.s, fmaxf(d, -1000.f), a.u);
  a.s *= f;
  a.m = to;
}
__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  const float to = fmaxf(a.m, b.m);
  rescale(a, to);
  rescale(b, to);
  return {to, a.s + b.s, a.u + b.u};
}
// One more logit, not above a.m unless a.m is -inf (then x is -inf or NaN and contributes 0 or NaN).
__device__ __forceinline__ void add(Stats& a, float x) {
  const float d = a.m == kNegInf ? x : x - a.m;
  const float e = exp2f(d * kLog2e);
  a.s += e;
  a.u = fmaf(e, fmaxf(d, -1000.f), a.u);   // e is 0 long before -1000: a forbidden token adds 0, not 0 * inf
}

__device__ __forceinline__ Stats shfl_xor(const Stats& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)};
}

// Unsigned keys in the order of the values: NaN above everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return nan_f();
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// (key, index) as one word: a larger word is the better alternative, ties go to the lower index.
__device__ __forceinline__ uint64_t cand_word(uint32_t key, uint32_t idx) {
  return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - idx);
}

struct LogprobFwd {
  const void* logits;
  const int64_t* targets;
  float* logprob;
  float* lse;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  int64_t rows, ld, ignore_index;
  int32_t vocab, top_k;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_fwd_kernel(const LogprobFwd p) {
  __shared__ Stats warp_stats[kThreads / 32];
  __shared__ uint64_t best[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.logits) + r * p.ld;
    Stats a = empty_stats();
    for (int c = threadIdx.x; c < p.vocab; c += kThreads) {
      const float v = to_f(x[c]);
      if (v > a.m) rescale(a, v);
      add(a, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = merge(a, shfl_xor(a, o));
    if (lane == 0) warp_stats[warp] = a;
    __syncthreads();
    a = warp_stats[0];
    for (int w = 1; w < kThreads / 32; ++w) a = merge(a, warp_stats[w]);
    const float lse = a.m == kNegInf && a.s == 0.f ? kNegInf : (a.m == kNegInf ? nan_f() : a.m + logf(a.s));
    if (threadIdx.x == 0) {
      const int64_t t = p.targets[r];
      float lp = nan_f();
      if (t == p.ignore_index) {
        lp = 0.f;
      } else if (t >= 0 && t < p.vocab) {
        const float xt = to_f(x[t]);
        lp = lse == kNegInf ? kNegInf : (xt - a.m) - logf(a.s);
      }
      p.logprob[r] = lp;
      if (p.lse) p.lse[r] = lse;
      if (p.entropy) p.entropy[r] = lse == kNegInf ? 0.f : logf(a.s) - a.u / a.s;
    }
    // the k best, one after the other: the largest word below the last one found
    uint64_t last = ~uint64_t{0};
    for (int k = 0; k < p.top_k; ++k) {
      uint64_t mine = 0;
      for (int c = threadIdx.x; c < p.vocab; c += kThreads) {
        const uint64_t w = cand_word(order_key(to_f(x[c])), c);
        if (w < last && w > mine) mine = w;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, mine, o);
        if (other > mine) mine = other;
      }
      if (lane == 0) best[warp] = mine;
      __syncthreads();
      for (int w = 0; w < kThreads / 32; ++w)
        if (best[w] > mine) mine = best[w];
      last = mine;
      if (threadIdx.x == 0) {
        const float v = key_value(static_cast<uint32_t>(mine >> 32));
        p.top_ids[r * p.top_k + k] = 0xffffffffu - static_cast<uint32_t>(mine);
        p.top_logprobs[r * p.top_k + k] = lse == kNegInf ? kNegInf : (v - a.m) - logf(a.s);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

struct LogprobBwd {
  const void* logits;
  const int64_t* targets;
  const float* lse;
  const float* entropy;
  const float* dlogprob;   // may be null
  const float* dentropy;   // may be null
  void* dlogits;
  int64_t rows, ld, ldd, ignore_index;
  int32_t vocab, width;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_bwd_kernel(const LogprobBwd p) {
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.logits) + r * p.ld;
    T* d = static_cast<T*>(p.dlogits) + r * p.ldd;
    const int64_t t = p.targets[r];
    const float lse = p.lse[r];
    const bool ignored = t == p.ignore_index;
    float gl = p.dlogprob && !ignored ? p.dlogprob[r] : 0.f;
    const float ge = p.dentropy ? p.dentropy[r] : 0.f;
    const float h = p.dentropy ? p.entropy[r] : 0.f;
    if (!ignored && (t < 0 || t >= p.vocab)) gl = nan_f();
    // an ignored row stays zero whatever its logits hold
    const bool none = lse == kNegInf || (gl == 0.f && ge == 0.f && (ignored || lse == lse));
    for (int c = threadIdx.x; c < p.width; c += kThreads) {
      float v = 0.f;
      if (!none && c < p.vocab) {
        const float lp = to_f(x[c]) - lse;
        const float pr = exp2f(lp * kLog2e);
        v = gl * ((c == t ? 1.f : 0.f) - pr) - ge * pr * (fmaxf(lp, -1000.f) + h);
      }
      d[c] = from_f<T>(v);
    }
  }
}

int check_logits(int64_t rows, int64_t vocab, int dtype) {
  if (rows < 0 || vocab <= 0 || vocab > INT32_MAX - 65536) return B200S_ERR_BAD_SHAPE;
  if (dtype != B200S_BF16 && dtype != B200S_FP16 && dtype != B200S_FP32) return B200S_ERR_BAD_DTYPE;
  return B200S_OK;
}

bool misaligned(const void* p, size_t es) { return reinterpret_cast<uintptr_t>(p) % es != 0; }

int64_t row_grid(int64_t rows) { return rows < 148 * 64 ? rows : 148 * 64; }

}  // namespace

}  // namespace b200s

using namespace b200s;

extern "C" {

int b200s_token_logprobs(int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld, const int64_t* targets,
                         int64_t ignore_index, float* logprob, float* lse, float* entropy, int top_k, int64_t* top_ids,
                         float* top_logprobs, void* stream) {
  int rc = check_logits(rows, vocab, dtype);
  if (rc) return rc;
  if (top_k < 0 || top_k > kMaxTopK || top_k > vocab) return B200S_ERR_BAD_SHAPE;
  if (rows == 0) return B200S_OK;
  if (!logits || !targets || !logprob) return B200S_ERR_NULL_POINTER;
  if (top_k > 0 && (!top_ids || !top_logprobs)) return B200S_ERR_NULL_POINTER;
  if (rows > 1 && ld < 0) return B200S_ERR_BAD_STRIDE;
  if (misaligned(logits, dtype_size(dtype)) || misaligned(targets, 8) || misaligned(logprob, 4) || misaligned(lse, 4) ||
      misaligned(entropy, 4) || misaligned(top_ids, 8) || misaligned(top_logprobs, 4))
    return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const LogprobFwd p{logits, targets, logprob, lse, entropy, top_ids, top_logprobs, rows, ld, ignore_index,
                     static_cast<int32_t>(vocab), top_k};
  const unsigned grid = static_cast<unsigned>(row_grid(rows));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B200S_BF16)
    logprob_fwd_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p);
  else if (dtype == B200S_FP16)
    logprob_fwd_kernel<__half><<<grid, kThreads, 0, s>>>(p);
  else
    logprob_fwd_kernel<float><<<grid, kThreads, 0, s>>>(p);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}

int b200s_token_logprobs_backward(int64_t rows, int64_t vocab, int64_t width, int dtype, const void* logits, int64_t ld,
                                  const int64_t* targets, int64_t ignore_index, const float* lse, const float* entropy,
                                  const float* dlogprob, const float* dentropy, void* dlogits, int64_t ldd,
                                  void* stream) {
  int rc = check_logits(rows, vocab, dtype);
  if (rc) return rc;
  if (width < vocab || width > INT32_MAX - 65536) return B200S_ERR_BAD_SHAPE;
  if (rows == 0) return B200S_OK;
  if (!logits || !targets || !lse || !dlogits || (dentropy && !entropy)) return B200S_ERR_NULL_POINTER;
  if (rows > 1 && (ld < 0 || ldd < width)) return B200S_ERR_BAD_STRIDE;
  if (misaligned(logits, dtype_size(dtype)) || misaligned(dlogits, dtype_size(dtype)) || misaligned(targets, 8) ||
      misaligned(lse, 4) || misaligned(entropy, 4) || misaligned(dlogprob, 4) || misaligned(dentropy, 4))
    return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const LogprobBwd p{logits, targets, lse, entropy, dlogprob, dentropy, dlogits, rows, ld, ldd, ignore_index,
                     static_cast<int32_t>(vocab), static_cast<int32_t>(width)};
  const unsigned grid = static_cast<unsigned>(row_grid(rows));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B200S_BF16)
    logprob_bwd_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p);
  else if (dtype == B200S_FP16)
    logprob_bwd_kernel<__half><<<grid, kThreads, 0, s>>>(p);
  else
    logprob_bwd_kernel<float><<<grid, kThreads, 0, s>>>(p);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}

}  // extern "C"
