// The global L2 norm of a list of gradient tensors, and clipping them to a bound.
//
//   sumsq = sum over tensors and elements of g^2
//   norm = sqrt(sumsq), c = min(1, max_norm / (norm + 1e-6)), out = g * c
//
// A list is cut into chunks of kChunk elements; chunk j of a launch belongs to block j mod grid, so
// what a block adds up, and in which order, depends on the list alone: results repeat bit for bit.
// Squares are added in fp64: in fp32 a gradient above 1.8e19 would overflow its square and one below
// 1e-23 lose it. The list travels in the kernel's parameters, so a captured graph keeps its own copy.

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdlib>

#include "common.h"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

constexpr int kThreads = 256;
constexpr int kCapacity = 128;     // tensors per launch (the list is a kernel parameter)
constexpr int kChunk = 16384;      // elements

struct ListParams {
  const void* src[kCapacity];
  void* dst[kCapacity];
  int64_t numel[kCapacity];
  int32_t chunk0[kCapacity + 1];   // first chunk of each tensor
  uint8_t dtype[kCapacity], dst_dtype[kCapacity];
  int32_t count;
};

__device__ __forceinline__ int find_tensor(const ListParams& p, int chunk) {
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

template <typename T>
__device__ __forceinline__ double sumsq_span(const T* x, int64_t n) {
  double a = 0.;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const double v = static_cast<double>(to_f(x[i]));
    a = fma(v, v, a);
  }
  return a;
}

// parts[b] (+)= the squares of block b's chunks; the parts of blocks that do not exist are cleared.
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ ListParams p, double* parts, int accumulate) {
  __shared__ double slots[kThreads / 32];
  const int chunks = p.chunk0[p.count];
  double a = 0.;
  for (int j = blockIdx.x; j < chunks; j += gridDim.x) {
    const int t = find_tensor(p, j);
    const int64_t at = static_cast<int64_t>(j - p.chunk0[t]) * kChunk;
    const int64_t left = p.numel[t] - at;
    const int64_t n = left < kChunk ? left : kChunk;
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

template <typename S, typename D>
__device__ __forceinline__ void scale_span(const S* x, D* y, int64_t n, float c) {
  for (int64_t i = threadIdx.x; i < n; i += kThreads) y[i] = from_f<D>(to_f(x[i]) * c);
}
template <typename S>
__device__ __forceinline__ void scale_to(const S* x, void* dst, int dst_dtype, int64_t at, int64_t n, float c) {
  if (dst_dtype == B200S_BF16)
    scale_span(x, static_cast<__nv_bfloat16*>(dst) + at, n, c);
  else if (dst_dtype == B200S_FP16)
    scale_span(x, static_cast<__half*>(dst) + at, n, c);
  else
    scale_span(x, static_cast<float*>(dst) + at, n, c);
}

// Every block forms the same norm from the parts, then scales its chunks. A coefficient of 1 leaves
// tensors that are clipped in place untouched; a NaN norm makes the coefficient, and them, NaN.
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ ListParams p, const double* parts, int n_parts,
                                                        float max_norm, float* norm_out) {
  __shared__ double slots[kThreads / 32];
  const double norm = sqrt(total_of(parts, n_parts, slots));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = static_cast<float>(norm);
  const double q = static_cast<double>(max_norm) / (norm + 1e-6);
  const float c = q >= 1. ? 1.f : static_cast<float>(q);
  const int chunks = p.chunk0[p.count];
  for (int j = blockIdx.x; j < chunks; j += gridDim.x) {
    const int t = find_tensor(p, j);
    if (c == 1.f && p.dst[t] == p.src[t]) continue;
    const int64_t at = static_cast<int64_t>(j - p.chunk0[t]) * kChunk;
    const int64_t left = p.numel[t] - at;
    const int64_t n = left < kChunk ? left : kChunk;
    if (p.dtype[t] == B200S_BF16)
      scale_to(static_cast<const __nv_bfloat16*>(p.src[t]) + at, p.dst[t], p.dst_dtype[t], at, n, c);
    else if (p.dtype[t] == B200S_FP16)
      scale_to(static_cast<const __half*>(p.src[t]) + at, p.dst[t], p.dst_dtype[t], at, n, c);
    else
      scale_to(static_cast<const float*>(p.src[t]) + at, p.dst[t], p.dst_dtype[t], at, n, c);
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
int fill(const b200s_tensor* list, int64_t count, int64_t* next, ListParams* p) {
  p->count = 0;
  int64_t chunks = 0;
  while (*next < count && p->count < kCapacity) {
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
  ListParams p;
  int64_t next = 0;
  bool first = true;
  do {
    int chunks = fill(list, count, &next, &p);
    if (chunks == 0 && !first) break;
    const int grid = chunks < 1 ? 1 : (chunks < B200S_NORM_PARTS ? chunks : B200S_NORM_PARTS);
    sumsq_kernel<<<grid, kThreads, 0, s>>>(p, parts, first ? 0 : 1);
    B200S_CUDA_OK(cudaGetLastError());
    count_launch();
    first = false;
  } while (next < count);
  return B200S_OK;
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
  ListParams p;
  int64_t next = 0;
  bool first = true;
  do {
    int chunks = fill(list, count, &next, &p);
    if (chunks == 0 && !first) break;
    const int grid = chunks < 1 ? 1 : (chunks < 148 * 8 ? chunks : 148 * 8);
    clip_kernel<<<grid, kThreads, 0, s>>>(p, parts, n_parts, max_norm, first ? norm_out : nullptr);
    B200S_CUDA_OK(cudaGetLastError());
    count_launch();
    first = false;
  } while (next < count);
  return B200S_OK;
}

}  // extern "C"
