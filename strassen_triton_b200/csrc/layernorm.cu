// Layer norm over the last dimension of a matrix of rows, forward and backward.
//
//   y  = xhat * w + b,  xhat = (x - mu) * rstd,  rstd = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  g = dy * w
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// All statistics and sums are fp32; the variance is taken around the mean (a second look at the row),
// not as a difference of squares. Results are rounded once, to the type they are stored in.
//
// Rows of any length: a block walks its row in as many steps as it takes and reads it again for the
// variance and for the result; the later readings come from L1 / L2.

#include <cuda_runtime.h>

#include "common.h"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

constexpr int kThreads = 256;

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
    const float mu = row::block_sum(s, slots) * inv_d;
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

// out[c] = sum of the slices, in their order.
__global__ void __launch_bounds__(kThreads) norm_params_sum_kernel(const float* part_w, const float* part_b, void* dw,
                                                                   void* db, int64_t d, int slices, int param_dtype) {
  __shared__ float s[8][33];
  const float* part = blockIdx.y == 0 ? part_w : part_b;
  void* out = blockIdx.y == 0 ? dw : db;
  if (!out) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float a = 0.f;
  if (c < d)
    for (int k = ty; k < slices; k += 8) a += part[static_cast<int64_t>(k) * d + c];
  s[ty][tx] = a;
  __syncthreads();
  if (ty == 0 && c < d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) a += s[k][tx];
    row::st_any(out, param_dtype, c, a);
  }
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
  return by_dtype(dtype, [&](auto t) -> int {
    norm_fwd_any_kernel<decltype(t)><<<static_cast<unsigned>(row_grid(rows)), kThreads, 0, s>>>(p);
    B200S_CUDA_OK(cudaGetLastError());
    count_launch();
    return B200S_OK;
  });
}

int b200s_layer_norm_backward_workspace(int64_t rows, int64_t d, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  if (rows < 0 || d <= 0 || d > INT32_MAX) return B200S_ERR_BAD_SHAPE;
  *bytes_out = static_cast<size_t>(param_slices(rows)) * static_cast<size_t>(d) * 2 * sizeof(float);
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
  const int slices = param_slices(rows);
  float* part = static_cast<float*>(workspace);
  const NormBwd p{x,    dy,  weight, mean, rstd, dx,   dweight ? part : nullptr, dbias ? part + static_cast<int64_t>(slices) * d : nullptr,
                  rows, d,   ldx,    lddy, lddx, slices, param_dtype};
  return by_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (dx && rows > 0) {
      norm_dx_any_kernel<T><<<static_cast<unsigned>(row_grid(rows)), kThreads, 0, s>>>(p);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
    }
    if (dweight || dbias) {
      const unsigned cols = static_cast<unsigned>((d + 31) / 32);
      norm_params_any_kernel<T><<<dim3(cols, slices), kThreads, 0, s>>>(p);
      norm_params_sum_kernel<<<dim3(cols, 2), kThreads, 0, s>>>(p.part_w, p.part_b, dweight, dbias, d, slices, param_dtype);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch(2);
    }
    return B200S_OK;
  });
}

}  // extern "C"
