// The global L2 norm of a list of gradient tensors, and clipping them to a bound.
//
//   sumsq = sum over tensors and elements of g^2
//   norm = sqrt(sumsq), c = min(1, max_norm / (norm + 1e-6)), out = g * c
//
// A list is cut into chunks of kChunk elements; chunk j of a launch belongs to block j mod grid, so
// what a block adds up, and in which order, depends on the list alone: results repeat bit for bit.
// The squares of one 16-byte vector are added in fp32 (three roundings at most), everything beyond in
// fp64; a vector whose sum leaves the safe range of fp32 (a gradient above 2^60 or all below 2^-42) is
// squared in fp64. The list travels in the kernel's parameters, so a captured graph keeps its own copy.
//
// Both passes are bound by memory. The clipping pass takes the chunks last to first: the end of the list
// is what the norm's pass left in L2 (a model of 326 MB in bf16: about a third of it). GPT-2-124M's gradients,
// 326 MB of bf16, take 62 us for the norm (5.3 TB/s) and 160 us clipped into fp32 (6.1 TB/s).

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "common.h"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

using row::Pack;

constexpr int kThreads = 256;
constexpr int kSmall = 128, kLarge = 512;   // tensors per launch (the list is a kernel parameter, 4 KB or 15 KB)
constexpr int kChunk = 16384;               // elements

template <int CAP>
struct ListParams {
  const void* src[CAP];
  void* dst[CAP];
  int64_t numel[CAP];
  int32_t chunk0[CAP + 1];   // first chunk of each tensor
  uint8_t dtype[CAP], dst_dtype[CAP];
  int32_t count;
};

template <int CAP>
__device__ __forceinline__ int find_tensor(const ListParams<CAP>& p, int chunk) {
  int lo = 0, hi = p.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.chunk0[mid] <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum_f64(double v, double* slots) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.;
  for (int w = 0; w < kThreads / 32; ++w) t += slots[w];
  __syncthreads();
  return t;
}

// Elements from x on up to the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T* x, int n) {
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const int head = off == 0 ? 0 : static_cast<int>(16 / sizeof(T)) - off;
  return head < n ? head : n;
}

template <typename T>
__device__ __forceinline__ double square(T x) {
  const double v = static_cast<double>(to_f(x));
  return v * v;
}

template <typename T>
__device__ __forceinline__ double vector_sumsq(const uint4& q) {
  constexpr int V = 16 / sizeof(T);
  const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(&q);
  float2 s[V / 2];
#pragma unroll
  for (int k = 0; k < V / 2; ++k) {
    const float2 t = row::load2(v.e + 2 * k);
    s[k] = row::mul_(t, t);
  }
#pragma unroll
  for (int w = V / 4; w > 0; w >>= 1)
#pragma unroll
    for (int k = 0; k < w; ++k) s[k] = row::add_(s[k], s[k + w]);
  const float sum = s[0].x + s[0].y;
  if (sum > 0x1p-84f && sum < 0x1p124f) return static_cast<double>(sum);
  if (((q.x | q.y | q.z | q.w) & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu)) == 0) return 0.;
  double d = 0.;
#pragma unroll
  for (int e = 0; e < V; ++e) d += square(v.e[e]);
  return d;
}

template <typename T>
__device__ __forceinline__ double sumsq_span(const T* x, int n) {
  constexpr int V = 16 / sizeof(T), B = 8;
  const int head = head_of(x, n);
  const int vecs = (n - head) / V;
  const int tail = head + vecs * V;
  double a = 0.;
  if (static_cast<int>(threadIdx.x) < head) a += square(x[threadIdx.x]);
  if (tail + static_cast<int>(threadIdx.x) < n) a += square(x[tail + threadIdx.x]);
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  for (int i = threadIdx.x; i < vecs; i += B * kThreads) {
    uint4 q[B];
#pragma unroll
    for (int b = 0; b < B; ++b) q[b] = i + b * kThreads < vecs ? __ldg(body + i + b * kThreads) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int b = 0; b < B; ++b) a += vector_sumsq<T>(q[b]);
  }
  return a;
}

// parts[b] (+)= the squares of block b's chunks; the parts of blocks that do not exist are cleared.
template <int CAP>
__global__ void __launch_bounds__(kThreads, 5) sumsq_kernel(const __grid_constant__ ListParams<CAP> p, double* parts, int accumulate) {
  __shared__ double slots[kThreads / 32];
  const int chunks = p.chunk0[p.count];
  double a = 0.;
  for (int j = blockIdx.x; j < chunks; j += gridDim.x) {
    const int t = find_tensor(p, j);
    const int64_t at = static_cast<int64_t>(j - p.chunk0[t]) * kChunk;
    const int64_t left = p.numel[t] - at;
    const int n = static_cast<int>(left < kChunk ? left : kChunk);
    if (p.dtype[t] == B200S_BF16)
      a += sumsq_span(static_cast<const __nv_bfloat16*>(p.src[t]) + at, n);
    else if (p.dtype[t] == B200S_FP16)
      a += sumsq_span(static_cast<const __half*>(p.src[t]) + at, n);
    else
      a += sumsq_span(static_cast<const float*>(p.src[t]) + at, n);
  }
  a = block_sum_f64(a, slots);
  if (threadIdx.x == 0) parts[blockIdx.x] = accumulate ? parts[blockIdx.x] + a : a;
  if (blockIdx.x == 0 && !accumulate)
    for (int i = gridDim.x + threadIdx.x; i < B200S_NORM_PARTS; i += kThreads) parts[i] = 0.;
}

__device__ __forceinline__ double total_of(const double* parts, int n, double* slots) {
  double a = 0.;
  for (int i = threadIdx.x; i < n; i += kThreads) a += parts[i];
  return block_sum_f64(a, slots);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* parts, int n_parts, float* norm_out) {
  __shared__ double slots[kThreads / 32];
  const double total = total_of(parts, n_parts, slots);
  if (threadIdx.x == 0) *norm_out = static_cast<float>(sqrt(total));
}

// Vectors of as many elements as fill 16 bytes of the wider type, so that a warp's accesses on both sides
// are gapless (bf16 to fp32 with 16-byte loads and two stores each: 224 us for 326 + 652 MB).
template <typename S, typename D>
__device__ __forceinline__ void scale_span(const S* x, D* y, int n, float c) {
  constexpr int V = sizeof(S) > sizeof(D) ? 16 / sizeof(S) : 16 / sizeof(D);
  constexpr int B = 64 / (V * sizeof(S));     // 64 bytes a thread on their way
  int head;
  if constexpr (sizeof(S) >= sizeof(D))
    head = head_of(x, n);
  else
    head = head_of(y, n);
  if (reinterpret_cast<uintptr_t>(y + head) % (V * sizeof(D)) != 0 || reinterpret_cast<uintptr_t>(x + head) % (V * sizeof(S)) != 0) {
    for (int i = threadIdx.x; i < n; i += kThreads) y[i] = from_f<D>(to_f(x[i]) * c);
    return;
  }
  const int vecs = (n - head) / V;
  const int tail = head + vecs * V;
  if (static_cast<int>(threadIdx.x) < head) y[threadIdx.x] = from_f<D>(to_f(x[threadIdx.x]) * c);
  if (tail + static_cast<int>(threadIdx.x) < n) y[tail + threadIdx.x] = from_f<D>(to_f(x[tail + threadIdx.x]) * c);
  const float2 cc = make_float2(c, c);
  for (int i = threadIdx.x; i < vecs; i += B * kThreads) {
    Pack<S, V> v[B];
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (i + b * kThreads < vecs) v[b] = row::ld<Pack<S, V>>(x + head + (i + b * kThreads) * V);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (i + b * kThreads < vecs) {
        Pack<D, V> o;
#pragma unroll
        for (int k = 0; k < V / 2; ++k) row::store2(o.e + 2 * k, row::mul_(row::load2(v[b].e + 2 * k), cc));
        row::st(y + head + (i + b * kThreads) * V, o);
      }
    }
  }
}
template <typename S>
__device__ __forceinline__ void scale_to(const S* x, void* dst, int dst_dtype, int64_t at, int n, float c) {
  if (dst_dtype == B200S_BF16)
    scale_span(x, static_cast<__nv_bfloat16*>(dst) + at, n, c);
  else if (dst_dtype == B200S_FP16)
    scale_span(x, static_cast<__half*>(dst) + at, n, c);
  else
    scale_span(x, static_cast<float*>(dst) + at, n, c);
}

// Every block forms the same norm from the parts, then scales its chunks. A coefficient of 1 leaves
// tensors that are clipped in place untouched; a NaN norm makes the coefficient, and them, NaN.
// S and D are the types of a list whose tensors all go from one to the other, void for any other list. (With all
// nine pairs in one kernel the spans take 255 registers, or spill: 220 .. 290 us for 326 MB of bf16 to fp32.)
template <int CAP, typename S, typename D>
__global__ void __launch_bounds__(kThreads, 5) clip_kernel(const __grid_constant__ ListParams<CAP> p, const double* parts, int n_parts,
                                                        float max_norm, float* norm_out) {
  __shared__ double slots[kThreads / 32];
  const double norm = sqrt(total_of(parts, n_parts, slots));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = static_cast<float>(norm);
  const double q = static_cast<double>(max_norm) / (norm + 1e-6);
  const float c = q >= 1. ? 1.f : static_cast<float>(q);
  const int chunks = p.chunk0[p.count];
  for (int k = blockIdx.x; k < chunks; k += gridDim.x) {
    const int j = chunks - 1 - k;
    const int t = find_tensor(p, j);
    if (c == 1.f && p.dst[t] == p.src[t]) continue;
    const int64_t at = static_cast<int64_t>(j - p.chunk0[t]) * kChunk;
    const int64_t left = p.numel[t] - at;
    const int n = static_cast<int>(left < kChunk ? left : kChunk);
    if constexpr (!std::is_void_v<S>) {
      scale_span(static_cast<const S*>(p.src[t]) + at, static_cast<D*>(p.dst[t]) + at, n, c);
    } else {
      if (p.dtype[t] == B200S_BF16)
        scale_to(static_cast<const __nv_bfloat16*>(p.src[t]) + at, p.dst[t], p.dst_dtype[t], at, n, c);
      else if (p.dtype[t] == B200S_FP16)
        scale_to(static_cast<const __half*>(p.src[t]) + at, p.dst[t], p.dst_dtype[t], at, n, c);
      else
        scale_to(static_cast<const float*>(p.src[t]) + at, p.dst[t], p.dst_dtype[t], at, n, c);
    }
  }
}

bool known_dtype(int d) { return d == B200S_BF16 || d == B200S_FP16 || d == B200S_FP32; }

int check_list(const b200s_tensor* list, int64_t count, bool with_dst) {
  if (count < 0) return B200S_ERR_BAD_SHAPE;
  if (count > 0 && !list) return B200S_ERR_NULL_POINTER;
  for (int64_t i = 0; i < count; ++i) {
    const b200s_tensor& t = list[i];
    if (t.numel < 0 || t.numel > (int64_t{1} << 42)) return B200S_ERR_BAD_SHAPE;
    if (!known_dtype(t.dtype) || (with_dst && !known_dtype(t.dst_dtype))) return B200S_ERR_BAD_DTYPE;
    if (t.numel == 0) continue;
    if (!t.src || (with_dst && !t.dst)) return B200S_ERR_NULL_POINTER;
    if (with_dst && t.dst == t.src && t.dst_dtype != t.dtype) return B200S_ERR_BAD_DTYPE;
    const uintptr_t sa = reinterpret_cast<uintptr_t>(t.src), da = reinterpret_cast<uintptr_t>(t.dst);
    if (sa % dtype_size(t.dtype) || (with_dst && da % dtype_size(t.dst_dtype))) return B200S_ERR_BAD_ALIGNMENT;
  }
  return B200S_OK;
}

// A tensor that is written may not share bytes with any other tensor of the list (two blocks would
// race on it); two that are only read may.
struct Span {
  uintptr_t lo, hi;
  bool write;
};
int check_overlap(const b200s_tensor* list, int64_t count) {
  Span* spans = static_cast<Span*>(std::malloc(sizeof(Span) * 2 * static_cast<size_t>(count) + 1));
  if (!spans) return B200S_ERR_TOO_LARGE;
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    const b200s_tensor& t = list[i];
    if (t.numel == 0) continue;
    const uintptr_t s = reinterpret_cast<uintptr_t>(t.src), d = reinterpret_cast<uintptr_t>(t.dst);
    spans[n++] = {d, d + static_cast<size_t>(t.numel) * dtype_size(t.dst_dtype), true};
    if (s != d) spans[n++] = {s, s + static_cast<size_t>(t.numel) * dtype_size(t.dtype), false};
  }
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t any_end = 0, write_end = 0;
  int rc = B200S_OK;
  for (int64_t i = 0; i < n && rc == B200S_OK; ++i) {
    if (spans[i].lo < (spans[i].write ? any_end : write_end)) rc = B200S_ERR_OVERLAP;
    if (spans[i].hi > any_end) any_end = spans[i].hi;
    if (spans[i].write && spans[i].hi > write_end) write_end = spans[i].hi;
  }
  std::free(spans);
  return rc;
}

// Takes tensors from list[*next] on until the launch is full; returns the number of chunks.
template <int CAP>
int fill(const b200s_tensor* list, int64_t count, int64_t* next, ListParams<CAP>* p) {
  p->count = 0;
  int64_t chunks = 0;
  while (*next < count && p->count < CAP) {
    const b200s_tensor& t = list[*next];
    const int64_t c = (t.numel + kChunk - 1) / kChunk;
    if (chunks + c > INT32_MAX / 2) break;
    ++*next;
    if (t.numel == 0) continue;
    const int i = p->count++;
    p->src[i] = t.src, p->dst[i] = t.dst, p->numel[i] = t.numel;
    p->dtype[i] = static_cast<uint8_t>(t.dtype), p->dst_dtype[i] = static_cast<uint8_t>(t.dst_dtype);
    p->chunk0[i] = static_cast<int32_t>(chunks);
    chunks += c;
  }
  p->chunk0[p->count] = static_cast<int32_t>(chunks);
  return static_cast<int>(chunks);
}

// launch(params, blocks' worth of chunks, is it the first) for every launch a list takes.
template <int CAP, typename F>
int for_launches(const b200s_tensor* list, int64_t count, F&& launch) {
  ListParams<CAP> p;
  int64_t next = 0;
  bool first = true;
  do {
    const int chunks = fill<CAP>(list, count, &next, &p);
    if (chunks == 0 && !first) break;
    launch(p, chunks < 1 ? 1 : chunks, first);
    B200S_CUDA_OK(cudaGetLastError());
    count_launch();
    first = false;
  } while (next < count);
  return B200S_OK;
}
template <typename F>
int for_launches(const b200s_tensor* list, int64_t count, F&& launch) {
  return count <= kSmall ? for_launches<kSmall>(list, count, launch) : for_launches<kLarge>(list, count, launch);
}

}  // namespace

}  // namespace b200s

using namespace b200s;

extern "C" {

int b200s_grad_sumsq(const b200s_tensor* list, int64_t count, double* parts, void* stream) {
  int rc = check_list(list, count, false);
  if (rc) return rc;
  if (!parts) return B200S_ERR_NULL_POINTER;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return for_launches(list, count, [&](const auto& p, int chunks, bool first) {
    const int grid = chunks < B200S_NORM_PARTS ? chunks : B200S_NORM_PARTS;
    sumsq_kernel<<<grid, kThreads, 0, s>>>(p, parts, first ? 0 : 1);
  });
}

int b200s_grad_norm(const double* parts, int n_parts, float* norm_out, void* stream) {
  if (!parts || !norm_out) return B200S_ERR_NULL_POINTER;
  if (n_parts < 1 || n_parts > B200S_NORM_PARTS) return B200S_ERR_BAD_SHAPE;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  norm_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(parts, n_parts, norm_out);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}

int b200s_grad_clip(const b200s_tensor* list, int64_t count, const double* parts, int n_parts, float max_norm,
                    float* norm_out, void* stream) {
  int rc = check_list(list, count, true);
  if (rc) return rc;
  if (!parts || !norm_out) return B200S_ERR_NULL_POINTER;
  if (n_parts < 1 || n_parts > B200S_NORM_PARTS || !(max_norm >= 0.f)) return B200S_ERR_BAD_SHAPE;
  rc = check_overlap(list, count);
  if (rc) return rc;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return for_launches(list, count, [&](const auto& p, int chunks, bool first) {
    constexpr int CAP = sizeof(p) > 4096 ? kLarge : kSmall;
    const int grid = chunks < 148 * 10 ? chunks : 148 * 10;
    float* norm = first ? norm_out : nullptr;
    bool same = true;
    for (int i = 1; i < p.count; ++i) same = same && p.dtype[i] == p.dtype[0] && p.dst_dtype[i] == p.dst_dtype[0];
    const int pair = same && p.count > 0 ? p.dtype[0] * 3 + p.dst_dtype[0] : -1;
    using B = __nv_bfloat16;
    using H = __half;
    auto go = [&](auto from, auto to) {
      using S = std::remove_pointer_t<decltype(from)>;
      using D = std::remove_pointer_t<decltype(to)>;
      clip_kernel<CAP, S, D><<<grid, kThreads, 0, s>>>(p, parts, n_parts, max_norm, norm);
    };
    B* b = nullptr;
    H* h = nullptr;
    float* f = nullptr;
    void* v = nullptr;
    switch (pair) {
      case B200S_BF16 * 3 + B200S_BF16: go(b, b); break;
      case B200S_BF16 * 3 + B200S_FP16: go(b, h); break;
      case B200S_BF16 * 3 + B200S_FP32: go(b, f); break;
      case B200S_FP16 * 3 + B200S_BF16: go(h, b); break;
      case B200S_FP16 * 3 + B200S_FP16: go(h, h); break;
      case B200S_FP16 * 3 + B200S_FP32: go(h, f); break;
      case B200S_FP32 * 3 + B200S_BF16: go(f, b); break;
      case B200S_FP32 * 3 + B200S_FP16: go(f, h); break;
      case B200S_FP32 * 3 + B200S_FP32: go(f, f); break;
      default: go(v, v);
    }
  });
}

}  // extern "C"
