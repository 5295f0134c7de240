// A matrix product with bias, activation and residual in its epilogue, and the elementwise part of its
// backward pass:
//
//   z = A . B + bias,  C = act(z) + residual                     (b200s_matmul_epilogue)
//   dz = dy * act'(z),  dbias = sum over rows of dz               (b200s_epilogue_backward)
//
// A dense product of 16-bit operands and results runs its epilogue inside the product's kernel
// (linear_sm100.cu). For every other product b200s_matmul takes (fp32, Strassen), and where K is cut into
// parts, fp32 products go to scratch and one pass here adds them up, adds the bias, applies the activation,
// adds the residual and rounds once.
//
// Two roundings of the backward pass of 16-bit layers are choices. The pre-activation z it needs is stored in the type
// of C: in fp32 it would double the largest tensor kept between the passes (its rounding adds 6e-4 of the gradients'
// norm in bf16, 6e-5 in fp16). dz goes to the products of dx and dw in 16 bits, as the tensor cores take both operands
// (1.6e-3, 2e-4); dbias is summed before that rounding. Together dx and dw have 1.45 times the error of gradients
// that are rounded at the end only (2.4e-3 against 1.7e-3 in bf16, 3.0e-4 against 2.1e-4 in fp16).

#include <cuda_runtime.h>

#include "common.h"
#include "epilogue_device.cuh"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

using row::from_f;
using row::to_f;

constexpr int kThreads = 256;

using row::Pack;

template <typename T, int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (sizeof(T) == 2)
    return epi::act_fast<ACT>(z);
  else
    return epi::act<ACT>(z);
}
template <typename T, int ACT>
__device__ __forceinline__ float dact_of(float z) {
  if constexpr (sizeof(T) == 2)
    return epi::dact_fast<ACT>(z);
  else
    return epi::dact<ACT>(z);
}

struct EpiloguePass {
  const float* z;          // parts x M x ld fp32 partial products
  const void* bias;
  const void* residual;
  void* C;
  void* preact;
  int64_t M, N, ld, ldr, ldc, ldp;
  int parts;
};

// VEC columns of a row per thread and step: bound by reading the partial products.
template <typename T, int ACT, int VEC>
__global__ void __launch_bounds__(kThreads) epilogue_kernel(const EpiloguePass p) {
  using F = Pack<float, VEC>;
  using P = Pack<T, VEC>;
  const int64_t cols = (p.N + VEC - 1) / VEC, total = p.M * cols, stride = p.M * p.ld;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = i / cols, c = (i - r * cols) * VEC;
    const float* at = p.z + r * p.ld + c;
    F z = row::ld<F>(at);
    for (int k = 1; k < p.parts; ++k) {
      const F q = row::ld<F>(at + k * stride);
#pragma unroll
      for (int e = 0; e < VEC; ++e) z.e[e] += q.e[e];
    }
    P out;
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) z.e[e] += to_f(static_cast<const T*>(p.bias)[c + e]);
    }
    if (p.preact) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) out.e[e] = from_f<T>(z.e[e]);
      row::st(static_cast<T*>(p.preact) + r * p.ldp + c, out);
    }
    P res;
    if (p.residual) res = row::ld<P>(static_cast<const T*>(p.residual) + r * p.ldr + c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float y = act_of<T, ACT>(z.e[e]);
      if (p.residual) y += to_f(res.e[e]);
      out.e[e] = from_f<T>(y);
    }
    row::st(static_cast<T*>(p.C) + r * p.ldc + c, out);
  }
}

// Rows copied to where TMA can address them (a padded leading dimension; the padding is left alone), one or two
// matrices by one launch.
struct PadJob {
  const uint16_t* in;
  uint16_t* out;
  int64_t rows, cols, ld_in, ld_out;
  int blocks;      // of the launch that take this matrix's rows
  int pairs;       // two elements an access
};
struct PadJobs {
  PadJob job[2];
  int count;
};
template <int VEC>
__device__ __forceinline__ void pad_rows(const PadJob& j, int64_t first) {
  using P = Pack<uint16_t, VEC>;
  constexpr int B = 4;
  const int64_t rows = j.rows, cols = j.cols, step = j.blocks;
  for (int64_t r = first; r < rows; r += step) {
    const uint16_t* from = j.in + r * j.ld_in;
    uint16_t* to = j.out + r * j.ld_out;
    for (int64_t c0 = threadIdx.x * VEC; c0 < cols; c0 += B * kThreads * VEC) {
      P v[B];
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (c0 + b * kThreads * VEC < cols) v[b] = row::ld_const<P>(from + c0 + b * kThreads * VEC);
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (c0 + b * kThreads * VEC < cols) row::st(to + c0 + b * kThreads * VEC, v[b]);
    }
  }
}
__global__ void __launch_bounds__(kThreads) pad_rows_kernel(const __grid_constant__ PadJobs p) {
  auto run = [](const PadJob& j, int64_t first) {
    if (j.pairs)
      pad_rows<2>(j, first);
    else
      pad_rows<1>(j, first);
  };
  const int block = static_cast<int>(blockIdx.x);
  if (block < p.job[0].blocks)
    run(p.job[0], block);
  else
    run(p.job[1], block - p.job[0].blocks);
}

struct EpilogueBwd {
  const void* z;
  const void* dy;
  void* dz;
  float* part;       // slices x N partial column sums
  int64_t M, N, ldz, ldy, lddz;
  int slices;
};

// 32 VEC columns per block, 8 rows at a time; a slice takes rows slice * 8 + warp, + slices * 8, ... Columns stay
// with their thread, so the sums of dz add up in registers, unrounded. Reads z and dy, writes dz: 8192 x 2304 bf16
// with GELU takes 25 us (113 MB, 4.5 TB/s; the two special functions and 20 instructions a pair weigh as much).
// (Two rows on their way and four blocks an SM; four rows and three blocks 26, two and six, with spills, 30.)
template <typename T, int ACT, int VEC>
__global__ void __launch_bounds__(kThreads, 4) epilogue_bwd_kernel(const EpilogueBwd p) {
  using P = Pack<T, VEC>;
  constexpr int R = 2;      // rows on their way per thread
  __shared__ float sb[8][32 * VEC + 1];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + tx) * VEC;
  const int64_t step = static_cast<int64_t>(p.slices) * 8;
  float a[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) a[e] = 0.f;
  if (c < p.N) {
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * 8 + ty; r0 < p.M; r0 += R * step) {
      P g[R], z[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int64_t r = r0 + k * step;
        if (r < p.M) {
          g[k] = row::ld<P>(static_cast<const T*>(p.dy) + r * p.ldy + c);
          if constexpr (ACT != B200S_ACT_NONE) z[k] = row::ld<P>(static_cast<const T*>(p.z) + r * p.ldz + c);
        }
      }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int64_t r = r0 + k * step;
        if (r < p.M) {
          P out;
          if constexpr (VEC >= 2 && sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              float2 v = row::load2(g[k].e + e);
              if constexpr (ACT != B200S_ACT_NONE) v = row::mul_(v, epi::dact_fast2<ACT>(row::load2(z[k].e + e)));
              a[e] += v.x;
              a[e + 1] += v.y;
              row::store2(out.e + e, v);
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              float v = to_f(g[k].e[e]);
              if constexpr (ACT != B200S_ACT_NONE) v *= dact_of<T, ACT>(to_f(z[k].e[e]));
              a[e] += v;
              out.e[e] = from_f<T>(v);
            }
          }
          if (p.dz) row::st(static_cast<T*>(p.dz) + r * p.lddz + c, out);
        }
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sb[ty][tx * VEC + e] = a[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += kThreads) {
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 * VEC + i;
    if (col >= p.N) continue;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sb[k][i];
    p.part[blockIdx.y * p.N + col] = s;
  }
}

constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) column_sum_kernel(const float* part, void* out, int64_t n, int slices, int dtype) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  float a = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int k = ty; k < slices; k += 32) a += part[static_cast<int64_t>(k) * n + c];
  }
  s[ty][tx] = a;
  __syncthreads();
  if (ty == 0 && c < n) {
#pragma unroll
    for (int k = 1; k < 32; ++k) a += s[k][tx];
    row::st_any(out, dtype, c, a);
  }
}

bool known_dtype(int d) { return d == B200S_BF16 || d == B200S_FP16 || d == B200S_FP32; }

// Slices of the rows: enough blocks for every SM to hold several, at least 16 rows each.
int bwd_slices(int64_t M, int64_t N) {
  const int64_t cols = (N + 255) / 256;
  int64_t want = (148 * 6 + cols - 1) / cols;
  if (want > (M + 15) / 16) want = (M + 15) / 16;
  return static_cast<int>(want < 1 ? 1 : (want > 256 ? 256 : want));
}

bool aligned(const void* p, int64_t ld, int64_t rows, size_t es, size_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && (rows <= 1 || (static_cast<size_t>(ld) * es) % to == 0);
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

// Does the product run with its epilogue in linear_sm100.cu?
int in_kernel(const b200s_problem* p, bool* yes) {
  int32_t algo = 0, depth = 0;
  int rc = b200s_resolve(p, &algo, &depth);
  if (rc) return rc;
  *yes = depth == 0 && dtype_size(p->in_dtype) == 2 && p->out_dtype == p->in_dtype && p->tile_variant == 0;
  return B200S_OK;
}

int64_t partial_ld(int64_t N) { return (N + 3) / 4 * 4; }

int run_pass(const EpiloguePass& ep, int dtype, int activation, cudaStream_t stream) {
  return by_dtype(dtype, [&](auto t) {
    return epi::by_activation(activation, [&](auto a) -> int {
      using T = decltype(t);
      constexpr int ACT = decltype(a)::value;
      const size_t to = 4 * sizeof(T);
      const bool vec = ep.N % 4 == 0 && aligned(ep.z, ep.ld, ep.M, 4, 16) && aligned(ep.C, ep.ldc, ep.M, sizeof(T), to) &&
                       (!ep.preact || aligned(ep.preact, ep.ldp, ep.M, sizeof(T), to)) &&
                       (!ep.residual || aligned(ep.residual, ep.ldr, ep.M, sizeof(T), to));
      const int64_t blocks = (ep.M * (vec ? ep.N / 4 : ep.N) + kThreads - 1) / kThreads;
      const unsigned grid = static_cast<unsigned>(blocks < 148 * 32 ? blocks : 148 * 32);
      if (vec)
        epilogue_kernel<T, ACT, 4><<<grid, kThreads, 0, stream>>>(ep);
      else
        epilogue_kernel<T, ACT, 1><<<grid, kThreads, 0, stream>>>(ep);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
      return B200S_OK;
    });
  });
}

}  // namespace

}  // namespace b200s

using namespace b200s;

extern "C" {

int b200s_matmul_epilogue_workspace(const b200s_problem* p, const b200s_epilogue* e, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  int rc = check_epilogue(p, e);
  if (rc) return rc;
  bool fused = false;
  rc = in_kernel(p, &fused);
  if (rc) return rc;
  if (fused) {
    const LinearPlan plan = plan_linear(p->M, p->N, p->K, p->a_major, p->b_major);
    *bytes_out = plan.splits > 1 ? static_cast<size_t>(plan.splits) * static_cast<size_t>(p->M) * static_cast<size_t>(partial_ld(p->N)) * 4 : 0;
    return B200S_OK;
  }
  const b200s_problem q = scratch_product(p);
  size_t need = 0;
  rc = b200s_workspace_bytes(&q, &need);
  if (rc) return rc;
  *bytes_out = round256(static_cast<size_t>(p->M) * static_cast<size_t>(p->N) * 4) + need;
  return B200S_OK;
}

int b200s_matmul_epilogue(const b200s_problem* p, const b200s_epilogue* e, const void* A, const void* B, void* C,
                          void* workspace, size_t workspace_bytes, void* stream_v) {
  size_t need = 0;
  int rc = b200s_matmul_epilogue_workspace(p, e, &need);
  if (rc) return rc;
  if (!A || !B || !C) return B200S_ERR_NULL_POINTER;
  if (need > 0 && !workspace) return B200S_ERR_NULL_POINTER;
  if (workspace_bytes < need) return B200S_ERR_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return B200S_ERR_BAD_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(C) % dtype_size(p->out_dtype)) return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  bool fused = false;
  rc = in_kernel(p, &fused);
  if (rc) return rc;
  if (fused) {
    const LinearPlan plan = plan_linear(p->M, p->N, p->K, p->a_major, p->b_major);
    const int64_t ldp = partial_ld(p->N);
    const LinearArgs g{A, B, C, e->bias, e->residual, e->preact, static_cast<float*>(workspace), p->M, p->N, p->K,
                       p->lda, p->ldb, p->ldc, e->ld_residual, e->ld_preact, ldp, p->a_major, p->b_major, p->in_dtype, p->out_dtype, e->activation};
    rc = launch_linear(g, plan, stream);
    if (rc || plan.splits == 1) return rc;
    const EpiloguePass ep{static_cast<const float*>(workspace), e->bias, e->residual, C, e->preact, p->M, p->N, ldp, e->ld_residual, p->ldc, e->ld_preact, plan.splits};
    return run_pass(ep, p->out_dtype, e->activation, stream);
  }
  const b200s_problem q = scratch_product(p);
  const size_t zb = round256(static_cast<size_t>(p->M) * static_cast<size_t>(p->N) * 4);
  uint8_t* rest = static_cast<uint8_t*>(workspace) + zb;
  rc = b200s_matmul(&q, A, B, workspace, need > zb ? rest : nullptr, need - zb, stream_v);
  if (rc) return rc;
  const EpiloguePass ep{static_cast<const float*>(workspace), e->bias, e->residual, C, e->preact, p->M, p->N, p->N, e->ld_residual, p->ldc, e->ld_preact, 1};
  return run_pass(ep, p->out_dtype, e->activation, stream);
}

int b200s_epilogue_backward_workspace(int64_t M, int64_t N, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  if (M < 0 || N <= 0 || N > INT32_MAX) return B200S_ERR_BAD_SHAPE;
  *bytes_out = static_cast<size_t>(bwd_slices(M, N)) * static_cast<size_t>(N) * sizeof(float);
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
  const int slices = bwd_slices(M, N);
  float* part = dbias ? static_cast<float*>(workspace) : nullptr;
  const EpilogueBwd b{preact, dy, dz, part, M, N, ldz, ldy, lddz, slices};
  rc = by_dtype(dtype, [&](auto t) {
    return epi::by_activation(activation, [&](auto act) -> int {
      using T = decltype(t);
      constexpr int ACT = decltype(act)::value;
      constexpr int W = static_cast<int>(16 / sizeof(T));
      auto fits = [&](int vec) {
        const size_t to = vec * sizeof(T);
        return N % vec == 0 && aligned(dy, ldy, M, sizeof(T), to) && (ACT == B200S_ACT_NONE || aligned(preact, ldz, M, sizeof(T), to)) &&
               (!dz || aligned(dz, lddz, M, sizeof(T), to));
      };
      auto grid = [&](int vec) { return dim3(static_cast<unsigned>((N + 32 * vec - 1) / (32 * vec)), static_cast<unsigned>(slices)); };
      if (fits(W))
        epilogue_bwd_kernel<T, ACT, W><<<grid(W), kThreads, 0, s>>>(b);
      else if (fits(2))
        epilogue_bwd_kernel<T, ACT, 2><<<grid(2), kThreads, 0, s>>>(b);
      else
        epilogue_bwd_kernel<T, ACT, 1><<<grid(1), kThreads, 0, s>>>(b);
      B200S_CUDA_OK(cudaGetLastError());
      count_launch();
      return B200S_OK;
    });
  });
  if (rc || !dbias) return rc;
  column_sum_kernel<<<static_cast<unsigned>((N + 31) / 32), kSumThreads, 0, s>>>(part, dbias, N, slices, dtype);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}

// ---- the dense 16-bit linear layer in one call each way ------------------------------------------

static int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }
static size_t rows_bytes(int64_t rows, int64_t cols) { return round256(static_cast<size_t>(rows) * static_cast<size_t>(padded(cols)) * 2); }

static size_t product_scratch(int64_t M, int64_t N, int64_t K, int a_major, int b_major) {
  const LinearPlan plan = plan_linear(M, N, K, a_major, b_major);
  return plan.splits > 1 ? round256(static_cast<size_t>(plan.splits) * static_cast<size_t>(M) * static_cast<size_t>(partial_ld(N)) * 4) : 0;
}

static int check_linear(int64_t M, int64_t N, int64_t K, int dtype, int activation) {
  if (M < 0 || N <= 0 || K <= 0 || M > kMaxLinearExtent || N > kMaxLinearExtent || K > kMaxLinearExtent) return B200S_ERR_BAD_SHAPE;
  if (dtype != B200S_BF16 && dtype != B200S_FP16) return B200S_ERR_BAD_DTYPE;
  if (activation < B200S_ACT_NONE || activation > B200S_ACT_GELU_TANH) return B200S_ERR_BAD_ALGO;
  return B200S_OK;
}

static bool addressable(const void* p, int64_t ld, int64_t rows, int64_t cols) {
  return aligned(p, ld, rows, 2, 16) && (rows <= 1 || ld >= cols);
}

// `p`, or (by a job of *jobs) its rows copied to *scratch, which then moves on. *ld becomes the leading dimension
// to use.
static void operand_rows(const void** p, int64_t* ld, int64_t rows, int64_t cols, uint8_t** scratch, PadJobs* jobs) {
  if (addressable(*p, *ld, rows, cols)) {
    if (rows <= 1) *ld = padded(cols);
    return;
  }
  PadJob& j = jobs->job[jobs->count++];
  j.in = static_cast<const uint16_t*>(*p);
  j.out = reinterpret_cast<uint16_t*>(*scratch);
  j.rows = rows, j.cols = cols, j.ld_in = *ld, j.ld_out = padded(cols);
  j.blocks = static_cast<int>(rows < 148 * 16 ? rows : 148 * 16);
  j.pairs = cols % 2 == 0 && aligned(j.in, *ld, rows, 2, 4);
  *p = j.out;
  *ld = j.ld_out;
  *scratch += rows_bytes(rows, cols);
}
static int run_jobs(const PadJobs& jobs, cudaStream_t stream) {
  if (jobs.count == 0) return B200S_OK;
  pad_rows_kernel<<<static_cast<unsigned>(jobs.job[0].blocks + (jobs.count > 1 ? jobs.job[1].blocks : 0)), kThreads, 0, stream>>>(jobs);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}

static int run_linear(LinearArgs g, uint8_t* scratch, cudaStream_t stream) {
  const LinearPlan plan = plan_linear(g.M, g.N, g.K, g.a_major, g.b_major);
  g.partials = reinterpret_cast<float*>(scratch);
  g.ldp = partial_ld(g.N);
  int rc = launch_linear(g, plan, stream);
  if (rc || plan.splits == 1) return rc;
  const EpiloguePass ep{g.partials, g.bias, g.residual, g.C, g.preact, g.M, g.N, g.ldp, g.ldr, g.ldc, g.ldz, plan.splits};
  return run_pass(ep, g.out_dtype, g.activation, stream);
}

int b200s_linear_act_workspace(int64_t M, int64_t N, int64_t K, int dtype, int copies, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  int rc = check_linear(M, N, K, dtype, B200S_ACT_NONE);
  if (rc) return rc;
  *bytes_out = M == 0 ? 0 : product_scratch(M, N, K, B200S_K_MAJOR, B200S_K_MAJOR) + (copies ? rows_bytes(M, K) + rows_bytes(N, K) : 0);
  return B200S_OK;
}

int b200s_linear_act(int64_t M, int64_t N, int64_t K, int dtype, int activation, const void* x, int64_t ldx,
                     const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr, void* y,
                     int64_t ldy, void* z, int64_t ldz, void* workspace, size_t workspace_bytes, void* stream_v) {
  int rc = check_linear(M, N, K, dtype, activation);
  if (rc) return rc;
  if (M == 0) return B200S_OK;
  if (!x || !weight || !y) return B200S_ERR_NULL_POINTER;
  if ((M > 1 && (ldx < 0 || (residual && ldr < 0) || ldy < N || (z && ldz < N))) || (N > 1 && ldw < 0)) return B200S_ERR_BAD_STRIDE;
  for (const void* q : {x, weight, bias, residual, static_cast<const void*>(y), static_cast<const void*>(z)})
    if (reinterpret_cast<uintptr_t>(q) & 1u) return B200S_ERR_BAD_ALIGNMENT;
  size_t need = 0;
  b200s_linear_act_workspace(M, N, K, dtype, !addressable(x, ldx, M, K) || !addressable(weight, ldw, N, K), &need);
  if (need > 0) {
    if (!workspace) return B200S_ERR_NULL_POINTER;
    if (workspace_bytes < need) return B200S_ERR_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return B200S_ERR_BAD_ALIGNMENT;
  }
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  uint8_t* scratch = static_cast<uint8_t*>(workspace);
  PadJobs jobs = {};
  operand_rows(&x, &ldx, M, K, &scratch, &jobs);
  operand_rows(&weight, &ldw, N, K, &scratch, &jobs);
  if ((rc = run_jobs(jobs, stream)) != 0) return rc;
  const LinearArgs g{x, weight, y, bias, residual, z, nullptr, M, N, K, ldx, ldw, ldy, ldr, ldz, 0, B200S_K_MAJOR, B200S_K_MAJOR, dtype, dtype, activation};
  return run_linear(g, scratch, stream);
}

int b200s_linear_act_backward_workspace(int64_t M, int64_t N, int64_t K, int dtype, int activation, int copies, size_t* bytes_out) {
  if (!bytes_out) return B200S_ERR_NULL_POINTER;
  int rc = check_linear(M, N, K, dtype, activation);
  if (rc) return rc;
  size_t sums = 0;
  b200s_epilogue_backward_workspace(M, N, &sums);
  if (M == 0) {
    *bytes_out = round256(sums);
    return B200S_OK;
  }
  const size_t p1 = product_scratch(M, K, N, B200S_K_MAJOR, B200S_MN_MAJOR), p2 = product_scratch(N, K, M, B200S_MN_MAJOR, B200S_MN_MAJOR);
  *bytes_out = (p1 > p2 ? p1 : p2) + round256(sums) + (copies || activation != B200S_ACT_NONE ? rows_bytes(M, N) : 0) +
               (copies ? rows_bytes(M, K) + rows_bytes(N, K) : 0);
  return B200S_OK;
}

int b200s_linear_act_backward(int64_t M, int64_t N, int64_t K, int dtype, int activation, const void* x, int64_t ldx,
                              const void* weight, int64_t ldw, const void* z, int64_t ldz, const void* dy, int64_t lddy,
                              void* dx, int64_t lddx, void* dweight, int64_t lddw, void* dbias, void* workspace,
                              size_t workspace_bytes, void* stream_v) {
  int rc = check_linear(M, N, K, dtype, activation);
  if (rc) return rc;
  if (!dx && !dweight && !dbias) return B200S_OK;
  if (M > 0 && (!dy || (dweight && !x) || (dx && !weight) || (activation != B200S_ACT_NONE && !z))) return B200S_ERR_NULL_POINTER;
  if ((M > 1 && (lddy < 0 || (dweight && ldx < 0) || (dx && lddx < K) || (activation != B200S_ACT_NONE && ldz < 0))) ||
      (N > 1 && ((dx && ldw < 0) || (dweight && lddw < K))))
    return B200S_ERR_BAD_STRIDE;
  for (const void* q : {x, weight, z, dy, static_cast<const void*>(dx), static_cast<const void*>(dweight), static_cast<const void*>(dbias)})
    if (reinterpret_cast<uintptr_t>(q) & 1u) return B200S_ERR_BAD_ALIGNMENT;
  size_t need = 0;
  const bool copies = M > 0 && (!addressable(dy, lddy, M, N) || (dweight && !addressable(x, ldx, M, K)) || (dx && !addressable(weight, ldw, N, K)));
  b200s_linear_act_backward_workspace(M, N, K, dtype, activation, copies, &need);
  if (!workspace) return B200S_ERR_NULL_POINTER;
  if (workspace_bytes < need) return B200S_ERR_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  uint8_t* scratch = static_cast<uint8_t*>(workspace);
  size_t sums = 0;
  b200s_epilogue_backward_workspace(M, N, &sums);
  void* parts = scratch;
  scratch += round256(sums);
  if (M == 0) {
    if (dweight)
      B200S_CUDA_OK(cudaMemset2DAsync(dweight, static_cast<size_t>(N > 1 ? lddw : K) * 2, 0, static_cast<size_t>(K) * 2, static_cast<size_t>(N), stream));
    if (dbias) B200S_CUDA_OK(cudaMemsetAsync(dbias, 0, static_cast<size_t>(N) * 2, stream));
    return B200S_OK;
  }
  // dz: dy itself where nothing has to be multiplied into it and TMA can read it
  const bool products = dx || dweight;
  const bool own = products && (activation != B200S_ACT_NONE || !addressable(dy, lddy, M, N));
  const void* dz = dy;
  int64_t lddz = M > 1 ? lddy : padded(N);
  if (own) {
    dz = scratch, lddz = padded(N);
    scratch += rows_bytes(M, N);
  }
  if (own || dbias) {
    rc = b200s_epilogue_backward(M, N, dtype, activation, z, ldz, dy, lddy, own ? const_cast<void*>(dz) : nullptr, lddz, dbias, parts, sums, stream_v);
    if (rc) return rc;
  }
  PadJobs jobs = {};
  if (dx) operand_rows(&weight, &ldw, N, K, &scratch, &jobs);
  if (dweight) operand_rows(&x, &ldx, M, K, &scratch, &jobs);
  if ((rc = run_jobs(jobs, stream)) != 0) return rc;
  if (dx) {
    const LinearArgs g{dz, weight, dx, nullptr, nullptr, nullptr, nullptr, M, K, N, lddz, ldw, lddx, 0, 0, 0, B200S_K_MAJOR, B200S_MN_MAJOR, dtype, dtype, B200S_ACT_NONE};
    if ((rc = run_linear(g, scratch, stream)) != 0) return rc;
  }
  if (dweight) {
    const LinearArgs g{dz, x, dweight, nullptr, nullptr, nullptr, nullptr, N, K, M, lddz, ldx, lddw, 0, 0, 0, B200S_MN_MAJOR, B200S_MN_MAJOR, dtype, dtype, B200S_ACT_NONE};
    if ((rc = run_linear(g, scratch, stream)) != 0) return rc;
  }
  return B200S_OK;
}

}  // extern "C"
