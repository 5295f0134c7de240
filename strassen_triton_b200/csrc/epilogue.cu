// A matrix product with bias, activation and residual in its epilogue, and the elementwise part of its
// backward pass:
//
//   z = A . B + bias,  C = act(z) + residual                     (b200s_matmul_epilogue)
//   dz = dy * act'(z),  dbias = sum over rows of dz               (b200s_epilogue_backward)
//
// This file holds the forms that work for every product b200s_matmul takes: the product goes to fp32
// scratch, one pass adds the bias, applies the activation, adds the residual and rounds once. The
// pre-activation z the backward pass needs is stored in the type of C.

#include <cuda_runtime.h>

#include "common.h"
#include "epilogue_device.cuh"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

constexpr int kThreads = 256;

struct EpiloguePass {
  const float* z;          // parts x M x N fp32 partial products
  const void* bias;
  const void* residual;
  void* C;
  void* preact;
  int64_t M, N, ldr, ldc, ldp;
  int parts;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) epilogue_kernel(const EpiloguePass p) {
  const int64_t total = p.M * p.N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = i / p.N, c = i - r * p.N;
    float z = p.z[i];
    for (int k = 1; k < p.parts; ++k) z += p.z[k * total + i];
    if (p.bias) z += to_f(static_cast<const T*>(p.bias)[c]);
    if (p.preact) static_cast<T*>(p.preact)[r * p.ldp + c] = from_f<T>(z);
    float y = epi::act<ACT>(z);
    if (p.residual) y += to_f(static_cast<const T*>(p.residual)[r * p.ldr + c]);
    static_cast<T*>(p.C)[r * p.ldc + c] = from_f<T>(y);
  }
}

struct EpilogueBwd {
  const void* z;
  const void* dy;
  void* dz;
  float* part;       // slices x N partial column sums
  int64_t M, N, ldz, ldy, lddz;
  int slices;
};

// 32 columns per block; a slice takes rows slice * 8 + ty, + slices * 8, ...
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) epilogue_bwd_kernel(const EpilogueBwd p) {
  __shared__ float sb[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float a = 0.f;
  if (c < p.N) {
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + ty; r < p.M; r += static_cast<int64_t>(p.slices) * 8) {
      float g = to_f(static_cast<const T*>(p.dy)[r * p.ldy + c]);
      if constexpr (ACT != B200S_ACT_NONE) g *= epi::dact<ACT>(to_f(static_cast<const T*>(p.z)[r * p.ldz + c]));
      if (p.dz) static_cast<T*>(p.dz)[r * p.lddz + c] = from_f<T>(g);
      a += g;
    }
  }
  if (!p.part) return;
  sb[ty][tx] = a;
  __syncthreads();
  if (ty == 0 && c < p.N) {
#pragma unroll
    for (int k = 1; k < 8; ++k) a += sb[k][tx];
    p.part[blockIdx.y * p.N + c] = a;
  }
}

__global__ void __launch_bounds__(kThreads) column_sum_kernel(const float* part, void* out, int64_t n, int slices, int dtype) {
  __shared__ float s[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float a = 0.f;
  if (c < n)
    for (int k = ty; k < slices; k += 8) a += part[static_cast<int64_t>(k) * n + c];
  s[ty][tx] = a;
  __syncthreads();
  if (ty == 0 && c < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) a += s[k][tx];
    row::st_any(out, dtype, c, a);
  }
}

bool known_dtype(int d) { return d == B200S_BF16 || d == B200S_FP16 || d == B200S_FP32; }

int bwd_slices(int64_t M) {
  const int64_t want = (M + 63) / 64;
  return static_cast<int>(want < 1 ? 1 : (want > 128 ? 128 : want));
}

template <typename F>
int by_dtype(int dtype, F&& f) {
  if (dtype == B200S_BF16) return f(__nv_bfloat16{});
  if (dtype == B200S_FP16) return f(__half{});
  return f(float{});
}

size_t round256(size_t x) { return (x + 255) & ~size_t{255}; }

int check_epilogue(const b200s_problem* p, const b200s_epilogue* e) {
  if (!p || !e) return B200S_ERR_NULL_POINTER;
  if (e->activation < B200S_ACT_NONE || e->activation > B200S_ACT_GELU_TANH) return B200S_ERR_BAD_ALGO;
  if (p->beta != 0 || p->batch != 1) return B200S_ERR_BAD_SHAPE;
  if (!known_dtype(p->out_dtype)) return B200S_ERR_BAD_DTYPE;
  if (p->ldc < p->N) return B200S_ERR_BAD_STRIDE;
  if (p->M > 1 && ((e->residual && e->ld_residual < 0) || (e->preact && e->ld_preact < p->N))) return B200S_ERR_BAD_STRIDE;
  const size_t es = dtype_size(p->out_dtype);
  if (reinterpret_cast<uintptr_t>(e->bias) % es || reinterpret_cast<uintptr_t>(e->residual) % es ||
      reinterpret_cast<uintptr_t>(e->preact) % es)
    return B200S_ERR_BAD_ALIGNMENT;
  return B200S_OK;
}

// The product of a general epilogue: fp32, dense rows of N, in scratch.
b200s_problem scratch_product(const b200s_problem* p) {
  b200s_problem q = *p;
  q.out_dtype = B200S_FP32;
  q.ldc = p->N;
  q.strideC = 0;
  return q;
}

}  // namespace

}  // namespace b200s

using namespace b200s;

extern "C" {

int b200s_matmul_epilogue_workspace(const b200s_problem* p, const b200s_epilogue* e, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  int rc = check_epilogue(p, e);
  if (rc) return rc;
  const b200s_problem q = scratch_product(p);
  size_t need = 0;
  rc = b200s_workspace_bytes(&q, &need);
  if (rc) return rc;
  *bytes_out = round256(static_cast<size_t>(p->M) * static_cast<size_t>(p->N) * 4) + need;
  return B200S_OK;
}

int b200s_matmul_epilogue(const b200s_problem* p, const b200s_epilogue* e, const void* A, const void* B, void* C,
                          void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  int rc = b200s_matmul_epilogue_workspace(p, e, &need);
  if (rc) return rc;
  if (!A || !B || !C) return B200S_ERR_NULL_POINTER;
  if (need > 0 && !workspace) return B200S_ERR_NULL_POINTER;
  if (workspace_bytes < need) return B200S_ERR_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return B200S_ERR_BAD_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(C) % dtype_size(p->out_dtype)) return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const b200s_problem q = scratch_product(p);
  const size_t zb = round256(static_cast<size_t>(p->M) * static_cast<size_t>(p->N) * 4);
  uint8_t* rest = static_cast<uint8_t*>(workspace) + zb;
  rc = b200s_matmul(&q, A, B, workspace, need > zb ? rest : nullptr, need - zb, stream);
  if (rc) return rc;
  const EpiloguePass ep{static_cast<const float*>(workspace), e->bias, e->residual, C, e->preact, p->M, p->N, e->ld_residual, p->ldc, e->ld_preact, 1};
  const int64_t blocks = (p->M * p->N + kThreads - 1) / kThreads;
  const unsigned grid = static_cast<unsigned>(blocks < 148 * 32 ? blocks : 148 * 32);
  return by_dtype(p->out_dtype, [&](auto t) {
    return epi::by_activation(e->activation, [&](auto a) -> int {
      epilogue_kernel<decltype(t), decltype(a)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(ep);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
      return B200S_OK;
    });
  });
}

int b200s_epilogue_backward_workspace(int64_t M, int64_t N, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  if (M < 0 || N <= 0 || N > INT32_MAX) return B200S_ERR_BAD_SHAPE;
  *bytes_out = static_cast<size_t>(bwd_slices(M)) * static_cast<size_t>(N) * sizeof(float);
  return B200S_OK;
}

int b200s_epilogue_backward(int64_t M, int64_t N, int dtype, int activation, const void* preact, int64_t ldz,
                            const void* dy, int64_t ldy, void* dz, int64_t lddz, void* dbias, void* workspace,
                            size_t workspace_bytes, void* stream) {
  size_t need = 0;
  int rc = b200s_epilogue_backward_workspace(M, N, &need);
  if (rc) return rc;
  if (!known_dtype(dtype)) return B200S_ERR_BAD_DTYPE;
  if (activation < B200S_ACT_NONE || activation > B200S_ACT_GELU_TANH) return B200S_ERR_BAD_ALGO;
  if (!dz && !dbias) return B200S_ERR_NULL_POINTER;
  if (M > 0 && (!dy || (activation != B200S_ACT_NONE && !preact))) return B200S_ERR_NULL_POINTER;
  if (M > 1 && (ldy < 0 || (activation != B200S_ACT_NONE && ldz < 0) || (dz && lddz < N))) return B200S_ERR_BAD_STRIDE;
  const size_t es = dtype_size(dtype);
  for (const void* q : {preact, dy, static_cast<const void*>(dz), static_cast<const void*>(dbias)})
    if (reinterpret_cast<uintptr_t>(q) % es) return B200S_ERR_BAD_ALIGNMENT;
  if (dbias) {
    if (!workspace) return B200S_ERR_NULL_POINTER;
    if (workspace_bytes < need) return B200S_ERR_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return B200S_ERR_BAD_ALIGNMENT;
  }
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int slices = bwd_slices(M);
  float* part = dbias ? static_cast<float*>(workspace) : nullptr;
  const EpilogueBwd b{preact, dy, dz, part, M, N, ldz, ldy, lddz, slices};
  const unsigned cols = static_cast<unsigned>((N + 31) / 32);
  rc = by_dtype(dtype, [&](auto t) {
    return epi::by_activation(activation, [&](auto a) -> int {
      epilogue_bwd_kernel<decltype(t), decltype(a)::value><<<dim3(cols, slices), kThreads, 0, s>>>(b);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
      return B200S_OK;
    });
  });
  if (rc || !dbias) return rc;
  column_sum_kernel<<<cols, kThreads, 0, s>>>(part, dbias, N, slices, dtype);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}

}  // extern "C"
