// Linear layer with its epilogue for sm_100a: z = A . B + bias, C = act(z) + residual, z stored on request.
// 16-bit operands and results, fp32 accumulation, everything after the product in fp32, one rounding.
//
// Two kernels:
//   linear_kernel   tcgen05 tiles. Warp 0 loads 128-byte-swizzled operand tiles by TMA, one lane of warp 1
//                   issues tcgen05.mma into one of two accumulators in tensor memory, warps 2.. take the
//                   other one through the epilogue: bias, activation, residual, rows of results through
//                   shared memory. Tile shapes 256 x 256 and 256 x 128 (CTA pairs), 128 x 128, 128 x 64; K may be cut into
//                   parts whose fp32 partial products a second pass adds up (plan_linear weighs all this).
//   skinny_kernel   up to 16 rows of A (tokens being generated) against K-major weights: bound by reading the
//                   weights once, with mma.sync fed straight from global memory in registers.
//
// What bounds linear_kernel. Products of many tiles: L2 reads of operand tiles. A 256 x 256 pair reads 64 KB per 64
// of K, and with all SMs loading the steps come 0.39 .. 0.48 us apart, about 12 TB/s, where the tensor cores need
// 0.27 (8192 x 4096 x 8192: 374 us, with GELU and bias 389; the library product 337). With K below about 1000 the
// epilogue's arithmetic adds to it: 8192 x 768 -> 2304 takes 27 us plain, 36 with GELU and bias, 40 with z stored too.
// Products of few tiles: the last round. The gradients of that layer are 96 tiles for 74 pairs, two rounds with 22
// pairs at work in the second (dx, 32 us; with a cold L2 38, tensor pipe at 55 %), and 27 tiles in two parts, 54
// pairs at work, with the pass over the partial products behind them (dw, 33 us together). The library products take
// 23 (plain), 22 and 23.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>

#include "common.h"
#include "epilogue_device.cuh"
#include "ptx_sm100.cuh"
#include "rowwise_device.cuh"

namespace b200s {

namespace {

constexpr int kRowBytes = 128;   // one swizzled row of a tile: 64 elements
constexpr int kBK = 64;          // K elements per stage
// Epilogue warps: four for every 64 columns of a tile, eight at most.
template <int BN>
constexpr int epi_warps = BN >= 128 ? 8 : 4;

// Role codes in the status words when a wait runs out.
enum : uint32_t { kWhoProducer = 13, kWhoMma = 14, kWhoMmaAcc = 15, kWhoEpilogue = 16 };
constexpr uint64_t kDrainNs = 20ull * 1000 * 1000;

struct LinearParams {
  int32_t M, N, K;
  int32_t m_tiles, n_tiles, k_blocks, splits, total_tiles;
  int32_t raster_group;
  int32_t a_mn, b_mn, fmt;
  int32_t bf16_out, act;
  int32_t vec_c, vec_z, vec_r;   // C, Z, the residual: rows of whole, aligned 16-byte vectors
  const void* bias;
  const void* residual;
  void* C;
  void* Z;
  int64_t ldc, ldr, ldz;
  uint32_t* status;
};

struct Tile {
  int split, mt, nt, kb0, kb1;
};

__device__ __forceinline__ Tile decode(const LinearParams& p, int tile) {
  Tile t;
  const int per = p.m_tiles * p.n_tiles;
  t.split = tile / per;
  int r = tile - t.split * per;
  const int band = p.raster_group * p.n_tiles;
  const int g = r / band;
  const int first = g * p.raster_group;
  const int size = min(p.raster_group, p.m_tiles - first);
  r -= g * band;
  t.mt = first + r % size;
  t.nt = r / size;
  t.kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * t.split / p.splits);
  t.kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (t.split + 1) / p.splits);
  return t;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  return bf16 ? ptx::pack_bf16(lo, hi) : ptx::pack_f16(lo, hi);
}
__device__ __forceinline__ float2 unpack2(uint32_t u, bool bf16) {
  return bf16 ? make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&u));
}

template <int ACT>
__device__ __forceinline__ void activate(float2 (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = epi::act_fast2<ACT>(v[j]);
}
__device__ __forceinline__ void activate(float2 (&v)[32], int act) {
  switch (act) {      // the same for the whole launch
    case B200S_ACT_RELU: activate<B200S_ACT_RELU>(v); break;
    case B200S_ACT_RELU2: activate<B200S_ACT_RELU2>(v); break;
    case B200S_ACT_SILU: activate<B200S_ACT_SILU>(v); break;
    case B200S_ACT_GELU: activate<B200S_ACT_GELU>(v); break;
    case B200S_ACT_GELU_TANH: activate<B200S_ACT_GELU_TANH>(v); break;
    default: break;
  }
}

// One warp's block of 32 rows x 128 bytes, written by its lanes (lane = row) into a swizzled 4 KB buffer, goes to
// row0, byte column col0 of a matrix of `rows` rows of `row_bytes` bytes, `ld` bytes apart: 16 bytes a lane where the
// rows are whole aligned vectors, else 2 bytes a lane. (With TMA stores instead, two buffers a warp and a stage
// fewer for the operands, 8192 x 4096 -> 8192 with relu2, bias and residual took 519 us back to back, 488 so.)
__device__ __forceinline__ void store_block(uint8_t* dst, int64_t ld, bool vec, int rows, int64_t row_bytes, int row0, int64_t col0,
                                            uint32_t buf, const uint32_t (&h)[32], int lane) {
  const uint32_t srow = buf + static_cast<uint32_t>(lane) * 128u, sw = static_cast<uint32_t>(lane & 7);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    ptx::st_shared_v4(srow + ((static_cast<uint32_t>(j) ^ sw) << 4), h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
  __syncwarp();
  uint8_t* at = dst + static_cast<int64_t>(row0) * ld + col0;
  const int n = min(32, rows - row0);
  const int64_t left = row_bytes - col0;
  if (vec) {
    const int q = lane >> 3, c = (lane & 7) * 16;
    if (c < left) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + q;
        const uint4 v = ptx::ld_shared_v4(buf + static_cast<uint32_t>(r) * 128u + ((static_cast<uint32_t>(lane & 7) ^ static_cast<uint32_t>(r & 7)) << 4));
        if (r < n) *reinterpret_cast<uint4*>(at + r * ld + c) = v;
      }
    }
  } else {
    for (int r = 0; r < n; ++r) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = lane + 32 * k;
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];"
                     : "=h"(v)
                     : "r"(buf + static_cast<uint32_t>(r) * 128u + ((static_cast<uint32_t>(c >> 3) ^ static_cast<uint32_t>(r & 7)) << 4) + (c & 7) * 2u));
        if (2 * c < left) *reinterpret_cast<uint16_t*>(at + r * ld + 2 * c) = v;
      }
    }
  }
  __syncwarp();
}

template <int CG, int BN, int STAGES, bool PARTIAL>
__global__ void __launch_bounds__(64 + 32 * epi_warps<BN>, 1)
linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const LinearParams p) {
  constexpr int kEpiWarps = epi_warps<BN>;
  constexpr int BN_CTA = BN / CG;
  constexpr int A_BYTES = 128 * kRowBytes;
  constexpr int B_BYTES = BN_CTA * kRowBytes;
  constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  constexpr int CHUNK_BYTES = kBK * kRowBytes;       // an MN-major chunk: 64 k-rows of 64 elements
  constexpr int STAGING = kEpiWarps * 4096;
  constexpr uint32_t TMEM_COLS = 2 * BN;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t staging = base + STAGES * STAGE_BYTES;
  const uint32_t bars = staging + STAGING;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bars + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + STAGES * STAGE_BYTES + STAGING + 8 * (2 * STAGES + 4));
  volatile uint32_t* abort_word = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? ptx::cluster_ctarank() : 0u;
  const int cluster = blockIdx.x / CG, clusters = gridDim.x / CG;

  if (threadIdx.x == 0) {
    *abort_word = 0;
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(tfull_bar(b), 1);
      ptx::mbar_init(tempty_bar(b), kEpiWarps * CG);
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmA);
    ptx::prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    ptx::tmem_alloc<CG>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), TMEM_COLS);
    ptx::tmem_relinquish<CG>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool alive = true;
      for (int tile = cluster; alive && tile < p.total_tiles; tile += clusters) {
        const Tile t = decode(p, tile);
        const int m0 = t.mt * (128 * CG) + static_cast<int>(rank) * 128;
        const int n0 = t.nt * BN + static_cast<int>(rank) * BN_CTA;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!ptx::mbar_wait<CG == 2>(empty_bar(stage), phase ^ 1u, abort_word, kWhoProducer)) {
            alive = false;
            break;
          }
          const uint32_t sA = base + stage * STAGE_BYTES, sB = sA + A_BYTES;
          const int k0 = kb * kBK;
          uint32_t fb = full_bar(stage);
          if constexpr (CG == 2) fb = ptx::mapa_cluster(fb, 0);
          if (rank == 0) ptx::mbar_expect_tx(full_bar(stage), CG * STAGE_BYTES);
          auto load = [&](uint32_t dst, const CUtensorMap* m, int c0, int c1) {
            if constexpr (CG == 2)
              ptx::tma_load_3d_pair(dst, m, fb, c0, c1, 0);
            else
              ptx::tma_load_3d(dst, m, fb, c0, c1, 0);
          };
          if (!p.a_mn) {
            load(sA, &tmA, k0, m0);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) load(sA + j * CHUNK_BYTES, &tmA, m0 + j * 64, k0);
          }
          if (!p.b_mn) {
            load(sB, &tmB, k0, n0);
          } else {
#pragma unroll
            for (int j = 0; j < BN_CTA / 64; ++j) load(sB + j * CHUNK_BYTES, &tmB, n0 + j * 64, k0);
          }
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
      }
      if (!alive && rank == 0) {
        // Copies may still be in flight into this cluster's shared memory: let them land, within a limit.
        // Stages below `stage` were armed in this pass over the ring, the others in the one before.
        const uint64_t deadline = ptx::global_timer_ns() + kDrainNs;
        for (uint32_t s = 0; s < static_cast<uint32_t>(STAGES); ++s)
          if (!ptx::mbar_wait_until(full_bar(static_cast<int>(s)), s < stage ? phase : phase ^ 1u, deadline)) break;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = ptx::make_instr_desc(static_cast<uint32_t>(p.fmt), p.a_mn, p.b_mn, 128 * CG, BN);
      const uint32_t a_lbo = p.a_mn ? CHUNK_BYTES : 16u, b_lbo = p.b_mn ? CHUNK_BYTES : 16u;
      const uint32_t a_adv = p.a_mn ? 2 * 1024u : 32u, b_adv = p.b_mn ? 2 * 1024u : 32u;
      const uint64_t a_desc0 = ptx::make_smem_desc(base, a_lbo, 1024u);
      const uint64_t b_desc0 = ptx::make_smem_desc(base + A_BYTES, b_lbo, 1024u);
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool alive = true;
      for (int tile = cluster; alive && tile < p.total_tiles; tile += clusters, ++it) {
        const Tile t = decode(p, tile);
        const int buf = it & 1;
        if (!ptx::mbar_wait<CG == 2>(tempty_bar(buf), ((it >> 1) & 1u) ^ 1u, abort_word, kWhoMmaAcc)) break;
        ptx::tc_fence_after_sync();
        const uint32_t acc = tmem + static_cast<uint32_t>(buf * BN);
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!ptx::mbar_wait<CG == 2>(full_bar(stage), phase, abort_word, kWhoMma)) {
            alive = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t soff = stage * (STAGE_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            ptx::umma<CG, false>(acc, a_desc0 + (soff + k * (a_adv >> 4)), b_desc0 + (soff + k * (b_adv >> 4)), idesc,
                                 (kb != t.kb0 || k != 0) ? 1u : 0u);
          ptx::umma_commit<CG>(empty_bar(stage));
          if constexpr (CG == 2) ptx::umma_commit<CG>(ptx::mapa_cluster(empty_bar(stage), 1));
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
        if (!alive) break;
        ptx::umma_commit<CG>(tfull_bar(buf));
        if constexpr (CG == 2) ptx::umma_commit<CG>(ptx::mapa_cluster(tfull_bar(buf), 1));
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 2;
    const int lane_group = warp & 3;        // this warp's TMEM lanes [32 * lane_group, +32)
    const int half = ew >> 2;               // and share of the tile's columns
    constexpr int WN = BN / (kEpiWarps / 4);
    const uint32_t b = staging + static_cast<uint32_t>(ew) * 4096u;    // this warp's buffer
    const bool bf16 = p.bf16_out != 0;
    int it = 0;
    for (int tile = cluster; tile < p.total_tiles; tile += clusters, ++it) {
      const Tile t = decode(p, tile);
      const int buf = it & 1;
      const int row0 = t.mt * (128 * CG) + static_cast<int>(rank) * 128 + lane_group * 32;
      const int col_first = t.nt * BN + half * WN;
      constexpr int GROUPS = WN / 64;
      // residual of the first columns: on its way while the product is computed (a row of 64 columns is 8 lanes)
      uint4 res[8];
      auto fetch_residual = [&](int col0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = row0 + 4 * i + (lane >> 3), c = col0 + (lane & 7) * 8;
          res[i] = make_uint4(0, 0, 0, 0);
          if (r < p.M && c < p.N)
            res[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.residual) + static_cast<int64_t>(r) * p.ldr + c);
        }
      };
      const bool vec_res = !PARTIAL && p.residual != nullptr && p.vec_r;
      if (vec_res) fetch_residual(col_first);
      // so is the bias: two columns of it per lane and group, handed round with the sums
      uint32_t bias2[GROUPS];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        bias2[g] = 0;
        const int c = col_first + g * 64 + 2 * lane;
        if (!PARTIAL && p.bias != nullptr) {
          const uint16_t* bp = static_cast<const uint16_t*>(p.bias);
          const uint32_t lo = c < p.N ? __ldg(bp + c) : 0, hi = c + 1 < p.N ? __ldg(bp + c + 1) : 0;
          bias2[g] = lo | hi << 16;
        }
      }
      int ok = 1;
      if (lane == 0) ok = ptx::mbar_wait<CG == 2, 32>(tfull_bar(buf), (it >> 1) & 1u, abort_word, kWhoEpilogue) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(lane_group * 32) << 16) + static_cast<uint32_t>(buf * BN + half * WN);
#pragma unroll 1
      for (int g = 0; g < GROUPS; ++g) {
        const int col0 = col_first + g * 64;
        uint32_t r0[32], r1[32];
        ptx::tmem_ld_32x32(taddr + g * 64, r0);
        ptx::tmem_ld_32x32(taddr + g * 64 + 32, r1);
        ptx::tmem_ld_wait();
        if (g == GROUPS - 1) {
          // the accumulator is in registers: the next tile may have it
          ptx::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2)
              ptx::mbar_arrive_cluster(tempty_bar(buf), 0);
            else
              ptx::mbar_arrive(tempty_bar(buf));
          }
        }
        if (col0 >= p.N || row0 >= p.M) continue;
        if constexpr (PARTIAL) {
          uint8_t* dst = static_cast<uint8_t*>(p.C) + static_cast<int64_t>(t.split) * p.M * p.ldc * 4;
          store_block(dst, p.ldc * 4, true, p.M, p.ldc * 4, row0, static_cast<int64_t>(col0) * 4, b, r0, lane);
          if (col0 + 32 < p.N) store_block(dst, p.ldc * 4, true, p.M, p.ldc * 4, row0, static_cast<int64_t>(col0 + 32) * 4, b, r1, lane);
        } else {
          float2 v[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            v[j] = make_float2(__uint_as_float(r0[2 * j]), __uint_as_float(r0[2 * j + 1]));
            v[16 + j] = make_float2(__uint_as_float(r1[2 * j]), __uint_as_float(r1[2 * j + 1]));
          }
          if (p.bias != nullptr) {
            uint32_t mine = bias2[0];
#pragma unroll
            for (int k = 1; k < GROUPS; ++k) mine = g == k ? bias2[k] : mine;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = row::add_(v[j], unpack2(__shfl_sync(0xffffffffu, mine, j), bf16));
          }
          uint32_t h[32];
          if (p.Z != nullptr) {
#pragma unroll
            for (int j = 0; j < 32; ++j) h[j] = pack2(v[j].x, v[j].y, bf16);
            store_block(static_cast<uint8_t*>(p.Z), p.ldz * 2, p.vec_z != 0, p.M, static_cast<int64_t>(p.N) * 2, row0, static_cast<int64_t>(col0) * 2, b, h, lane);
          }
          activate(v, p.act);
          if (p.residual != nullptr) {
            // rows as they were read -> rows of the lanes, through the buffer the result will use
            if (vec_res) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t r = static_cast<uint32_t>(4 * i + (lane >> 3)), j = static_cast<uint32_t>(lane & 7);
                ptx::st_shared_v4(b + r * 128u + ((j ^ (r & 7u)) << 4), res[i].x, res[i].y, res[i].z, res[i].w);
              }
              if (g + 1 < GROUPS) fetch_residual(col0 + 64);
            } else {
              const int rows = min(32, p.M - row0);
              for (int r = 0; r < rows; ++r) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const int c = lane + 32 * k;
                  uint16_t q = 0;
                  if (col0 + c < p.N) q = static_cast<const uint16_t*>(p.residual)[static_cast<int64_t>(row0 + r) * p.ldr + col0 + c];
                  asm volatile("st.shared.u16 [%0], %1;" ::"r"(b + static_cast<uint32_t>(r) * 128u +
                                                               ((static_cast<uint32_t>(c >> 3) ^ static_cast<uint32_t>(r & 7)) << 4) + (c & 7) * 2u),
                               "h"(q)
                               : "memory");
                }
              }
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint4 q = ptx::ld_shared_v4(b + static_cast<uint32_t>(lane) * 128u + ((static_cast<uint32_t>(j) ^ static_cast<uint32_t>(lane & 7)) << 4));
              const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) v[4 * j + k] = row::add_(v[4 * j + k], unpack2(w[k], bf16));
            }
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) h[j] = pack2(v[j].x, v[j].y, bf16);
          store_block(static_cast<uint8_t*>(p.C), p.ldc * 2, p.vec_c != 0, p.M, static_cast<int64_t>(p.N) * 2, row0, static_cast<int64_t>(col0) * 2, b, h, lane);
        }
      }
    }
  }

  // ------------------------------------------------------------ teardown
  ptx::tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  if (threadIdx.x == 0 && *abort_word != 0) {
    atomicExch(&p.status[0], 1u);
    atomicExch(&p.status[1], *abort_word);
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<CG>(tmem, TMEM_COLS);
  }
}

// ---- few rows of A -------------------------------------------------------------------------------
// y^T = W x^T with mma.sync m16n8k16: 16 rows of W (outputs) are the A operand, up to 8 * MT rows of x the
// columns of B. The order of the terms along K is free as long as both operands agree, so lane (g, t) of a
// warp takes 8 consecutive k of its rows, one 16-byte load, as the fragments of two steps: chunks of 32 k are
// read whole, 64 bytes a row, without shared memory. The block's 8 warps take turns over runs of UN chunks and
// add up their sums, 16 NT x 8 MT each, in shared memory.
constexpr int kSkinnyWarps = 8;

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool BF16>
__device__ __forceinline__ float from_bits(uint16_t u) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
  return __half2float(__ushort_as_half(u));
}
template <bool BF16>
__device__ __forceinline__ uint16_t to_bits(float v) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}

struct SkinnyParams {
  const uint16_t* X;
  const uint16_t* W;
  const uint16_t* bias;       // where there is none: any readable element, with bias_step 0
  const uint16_t* residual;   // the same, with res_step and ldr 0
  uint16_t* C;
  uint16_t* Z;
  int64_t ldx, ldw, ldc, ldr, ldz;
  int32_t M, N, K, act;
  int32_t bias_step, res_step, has_z;
};

// 8 elements from column k of a row, zero from column K on (what lies there is not part of the operand).
// Every load of this kernel is unconditional and its address in range by itself: beyond the row's last vector
// the last one is read and dropped.
__device__ __forceinline__ uint4 row8(const uint16_t* row, int k, int K, bool in) {
  const int last = (K - 1) & ~7;
  uint4 q = __ldg(reinterpret_cast<const uint4*>(row + min(k, last)));
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
  const int left = in ? K - k : 0;       // elements of the vector that belong to the row
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = left >= 2 * j + 2 ? w[j] : (left == 2 * j + 1 ? w[j] & 0xffffu : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int MT, int NT, bool BF16>
__global__ void __launch_bounds__(32 * kSkinnyWarps) skinny_kernel(const SkinnyParams p) {
  constexpr int UN = MT + 2 * NT <= 5 ? 4 : 2;       // chunks on their way per warp, side by side
  __shared__ float part[kSkinnyWarps][16 * NT][8 * MT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16 * NT;
  const uint16_t* w[2 * NT];
  bool inw[2 * NT];
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i) {
    inw[i] = n0 + 8 * i + g < p.N;
    w[i] = p.W + static_cast<int64_t>(min(n0 + 8 * i + g, p.N - 1)) * p.ldw;
  }
  const uint16_t* x[MT];
  bool inx[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    inx[j] = 8 * j + g < p.M;
    x[j] = p.X + static_cast<int64_t>(min(8 * j + g, p.M - 1)) * p.ldx;
  }
  float acc[NT][MT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  const int chunks = (p.K + 31) / 32;
  for (int c = warp * UN; c < chunks; c += kSkinnyWarps * UN) {
    uint4 a[UN][2 * NT], xv[UN][MT];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int k = (c + u) * 32 + t * 8;
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) a[u][i] = row8(w[i], k, p.K, inw[i]);
#pragma unroll
      for (int j = 0; j < MT; ++j) xv[u][j] = row8(x[j], k, p.K, inx[j]);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const uint4 &lo = a[u][2 * i], &hi = a[u][2 * i + 1];
          mma16816<BF16>(acc[i][j], lo.x, hi.x, lo.y, hi.y, xv[u][j].x, xv[u][j].y);
          mma16816<BF16>(acc[i][j], lo.z, hi.z, lo.w, hi.w, xv[u][j].z, xv[u][j].w);
        }
  }
  // accumulator element (row g or g + 8 of W, row 2t or 2t + 1 of x)
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      part[warp][16 * i + g][8 * j + 2 * t] = acc[i][j][0];
      part[warp][16 * i + g][8 * j + 2 * t + 1] = acc[i][j][1];
      part[warp][16 * i + g + 8][8 * j + 2 * t] = acc[i][j][2];
      part[warp][16 * i + g + 8][8 * j + 2 * t + 1] = acc[i][j][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * NT * 8 * MT; i += 32 * kSkinnyWarps) {
    const int n = i % (16 * NT), m = i / (16 * NT);
    const int row = min(m, p.M - 1), col = min(n0 + n, p.N - 1);
    const float add = from_bits<BF16>(__ldg(p.bias + static_cast<int64_t>(col) * p.bias_step));
    const float res = from_bits<BF16>(__ldg(p.residual + static_cast<int64_t>(row) * p.ldr + static_cast<int64_t>(col) * p.res_step));
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < kSkinnyWarps; ++k) z += part[k][n][m];
    z += p.bias_step ? add : 0.f;
    float y = z;
    switch (p.act) {
      case B200S_ACT_RELU: y = epi::act_fast<B200S_ACT_RELU>(z); break;
      case B200S_ACT_RELU2: y = epi::act_fast<B200S_ACT_RELU2>(z); break;
      case B200S_ACT_SILU: y = epi::act_fast<B200S_ACT_SILU>(z); break;
      case B200S_ACT_GELU: y = epi::act_fast<B200S_ACT_GELU>(z); break;
      case B200S_ACT_GELU_TANH: y = epi::act_fast<B200S_ACT_GELU_TANH>(z); break;
      default: break;
    }
    y += p.res_step ? res : 0.f;
    if (m < p.M && n0 + n < p.N) {
      if (p.has_z) p.Z[static_cast<int64_t>(m) * p.ldz + n0 + n] = to_bits<BF16>(z);
      p.C[static_cast<int64_t>(m) * p.ldc + n0 + n] = to_bits<BF16>(y);
    }
  }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------

template <int CG, int BN, int STAGES, bool PARTIAL>
int launch_tiles(const CUtensorMap* maps, LinearParams p, cudaStream_t stream) {
  constexpr int kEpiWarps = epi_warps<BN>;
  constexpr int SMEM = STAGES * (128 + BN / CG) * kRowBytes + kEpiWarps * 4096 + 8 * (2 * STAGES + 4) + 16 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  auto kernel = linear_kernel<CG, BN, STAGES, PARTIAL>;
  static std::mutex mu;
  static int resident[64] = {0};       // clusters a device holds at once
  int dev = 0;
  B200S_CUDA_OK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return B200S_ERR_NO_DEVICE;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(64 + 32 * kEpiWarps);
  cfg.dynamicSmemBytes = SMEM;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int fit;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (resident[dev] == 0) {
      B200S_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
      int n = sm_count() / CG;
      if (CG == 2) {
        cfg.gridDim = dim3(sm_count() / 2 * 2);
        int q = 0;
        B200S_CUDA_OK(cudaOccupancyMaxActiveClusters(&q, kernel, &cfg));
        if (q < 1) return B200S_ERR_CUDA;
        if (q < n) n = q;
      }
      resident[dev] = n;
    }
    fit = resident[dev];
  }
  const int allowed = product_sm_count() / CG;
  if (allowed < fit) fit = allowed;
  if (fit < 1) return B200S_ERR_NO_DEVICE;
  cfg.gridDim = dim3((p.total_tiles < fit ? p.total_tiles : fit) * CG);
  cfg.stream = stream;
  B200S_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], p));
  count_launch();
  return B200S_OK;
}

template <bool PARTIAL>
int launch_plan(const LinearPlan& plan, const CUtensorMap* maps, const LinearParams& p, cudaStream_t stream) {
  if (plan.cta_group == 2 && plan.tile_n == 256) return launch_tiles<2, 256, 6, PARTIAL>(maps, p, stream);
  if (plan.cta_group == 2) return launch_tiles<2, 128, 7, PARTIAL>(maps, p, stream);
  if (plan.tile_n == 128) return launch_tiles<1, 128, 6, PARTIAL>(maps, p, stream);
  return launch_tiles<1, 64, 8, PARTIAL>(maps, p, stream);
}

template <int MT, int NT>
int launch_skinny_form(const SkinnyParams& p, bool bf16, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((p.N + 16 * NT - 1) / (16 * NT));
  if (bf16)
    skinny_kernel<MT, NT, true><<<grid, 32 * kSkinnyWarps, 0, stream>>>(p);
  else
    skinny_kernel<MT, NT, false><<<grid, 32 * kSkinnyWarps, 0, stream>>>(p);
  B200S_CUDA_OK(cudaGetLastError());
  count_launch();
  return B200S_OK;
}
// 32 outputs a block where that still leaves most SMs a block (1 x 8192 x 8192: 27 us against 33 with 16).
template <int MT>
int launch_skinny(const SkinnyParams& p, bool bf16, cudaStream_t stream) {
  return MT == 1 && p.N >= 32 * 120 ? launch_skinny_form<1, 2>(p, bf16, stream) : launch_skinny_form<MT, 1>(p, bf16, stream);
}

bool vector_rows(const void* p, int64_t ld, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows <= 1 || (ld * 2) % 16 == 0);
}

}  // namespace

LinearPlan plan_linear(int64_t M, int64_t N, int64_t K, int a_major, int b_major) {
  LinearPlan best{LinearPlan::kTiles, 2, 256, 1};
  // Few rows: the weights are read once, as fast as by a copy (16 x 4096 x 4096: 9.4 us; tiles take 11). With 32
  // rows a block's reading of x costs more than the weights (15.4 us against 11.1 with tiles).
  if (M <= 16 && a_major == B200S_K_MAJOR && b_major == B200S_K_MAJOR) {
    best.kind = LinearPlan::kSkinny;
    return best;
  }
  // Estimated clocks of every tile shape and split. Measured, per 64 of K: 540 clocks for one CTA (its TMA
  // loads), 680 for a pair, never less than the tensor cores need (4096 products a clock and SM), and with all
  // SMs loading 45 bytes a clock and SM from L2; 4.0 and 5.4 us for a launch with one such step. A split adds
  // the pass over the partial products (2.3 us and its traffic, slower where rows are not whole vectors).
  const int64_t kb = (K + kBK - 1) / kBK;
  double least = 0;
  const struct { int cg, bn; } shapes[] = {{2, 256}, {2, 128}, {1, 128}, {1, 64}};
  for (const auto& s : shapes) {
    const int64_t tiles = ((M + 128 * s.cg - 1) / (128 * s.cg)) * ((N + s.bn - 1) / s.bn);
    const int64_t units = 148 / s.cg;
    const double mma = s.bn * 2.0, bytes = (128.0 + s.bn / s.cg) * kRowBytes;
    for (int split = 1; split <= 16 && split <= kb; ++split) {
      const int64_t work = tiles * split, waves = (work + units - 1) / units;
      const double busy = static_cast<double>(work < units ? work : units) / static_cast<double>(units);
      double step = s.cg == 2 ? 680 : 540;
      if (step < mma) step = mma;
      if (step < bytes / 45.0 * busy) step = bytes / 45.0 * busy;
      double clocks = (s.cg == 2 ? 10200 : 7600) + static_cast<double>(waves) * static_cast<double>((kb + split - 1) / split) * step;
      if (split > 1) clocks += 4400 + static_cast<double>(M) * static_cast<double>(N) * (4.0 * split + 2) / (N % 4 == 0 ? 2400 : 900);
      if (least == 0 || clocks < least) {
        least = clocks;
        best.cta_group = s.cg, best.tile_n = s.bn, best.splits = split;
      }
    }
  }
  return best;
}

int launch_linear(const LinearArgs& g, const LinearPlan& plan, cudaStream_t stream) {
  if (g.M > kMaxLinearExtent || g.N > kMaxLinearExtent || g.K > kMaxLinearExtent) return B200S_ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(g.A) & 15u) || (reinterpret_cast<uintptr_t>(g.B) & 15u)) return B200S_ERR_BAD_ALIGNMENT;
  if ((g.lda * 2) % 16 || (g.ldb * 2) % 16) return B200S_ERR_BAD_STRIDE;
  const bool bf16_out = g.out_dtype == B200S_BF16;
  if (plan.kind == LinearPlan::kSkinny) {
    SkinnyParams p = {};
    p.X = static_cast<const uint16_t*>(g.A), p.W = static_cast<const uint16_t*>(g.B);
    p.C = static_cast<uint16_t*>(g.C), p.Z = static_cast<uint16_t*>(g.preact), p.has_z = g.preact != nullptr;
    p.bias = g.bias ? static_cast<const uint16_t*>(g.bias) : p.X, p.bias_step = g.bias ? 1 : 0;
    p.residual = g.residual ? static_cast<const uint16_t*>(g.residual) : p.X, p.res_step = g.residual ? 1 : 0;
    p.ldx = g.lda, p.ldw = g.ldb, p.ldc = g.ldc, p.ldr = g.residual ? g.ldr : 0, p.ldz = g.ldz;
    p.M = static_cast<int32_t>(g.M), p.N = static_cast<int32_t>(g.N), p.K = static_cast<int32_t>(g.K), p.act = g.activation;
    return g.M <= 8 ? launch_skinny<1>(p, bf16_out, stream) : launch_skinny<2>(p, bf16_out, stream);
  }
  const bool partial = plan.splits > 1;
  uint32_t* status = device_status_words();
  if (!status) return B200S_ERR_NO_DEVICE;
  CUtensorMap maps[2];
  const int cg = plan.cta_group, bn_cta = plan.tile_n / cg;
  int rc = g.a_major == B200S_K_MAJOR ? encode_operand_map(&maps[0], g.A, g.in_dtype, g.M, g.K, g.lda, 1, 0, 128, false)
                                      : encode_operand_map(&maps[0], g.A, g.in_dtype, g.K, g.M, g.lda, 1, 0, kBK, false);
  if (rc) return rc;
  rc = g.b_major == B200S_K_MAJOR ? encode_operand_map(&maps[1], g.B, g.in_dtype, g.N, g.K, g.ldb, 1, 0, bn_cta, false)
                                  : encode_operand_map(&maps[1], g.B, g.in_dtype, g.K, g.N, g.ldb, 1, 0, kBK, false);
  if (rc) return rc;
  LinearParams p = {};
  const bool whole = g.N % 8 == 0;
  p.vec_c = whole && vector_rows(g.C, g.ldc, g.M);
  p.vec_z = g.preact && whole && vector_rows(g.preact, g.ldz, g.M);
  p.vec_r = g.residual && whole && vector_rows(g.residual, g.ldr, g.M);
  p.M = static_cast<int32_t>(g.M), p.N = static_cast<int32_t>(g.N), p.K = static_cast<int32_t>(g.K);
  p.m_tiles = static_cast<int32_t>((g.M + 128 * cg - 1) / (128 * cg));
  p.n_tiles = static_cast<int32_t>((g.N + plan.tile_n - 1) / plan.tile_n);
  p.k_blocks = static_cast<int32_t>((g.K + kBK - 1) / kBK);
  p.splits = plan.splits;
  const int64_t total = static_cast<int64_t>(p.m_tiles) * p.n_tiles * plan.splits;
  if (total > INT32_MAX) return B200S_ERR_BAD_SHAPE;
  p.total_tiles = static_cast<int32_t>(total);
  p.raster_group = 8;
  p.a_mn = g.a_major == B200S_MN_MAJOR, p.b_mn = g.b_major == B200S_MN_MAJOR;
  p.fmt = g.in_dtype == B200S_BF16 ? 1 : 0;
  p.bf16_out = bf16_out, p.act = g.activation;
  p.bias = g.bias, p.residual = g.residual, p.C = g.C, p.Z = g.preact;
  p.ldc = g.ldc, p.ldr = g.ldr, p.ldz = g.ldz;
  if (partial) p.C = g.partials, p.ldc = g.ldp;       // rows of whole vectors, the last one filled up
  p.status = status;
  return partial ? launch_plan<true>(plan, maps, p, stream) : launch_plan<false>(plan, maps, p, stream);
}

}  // namespace b200s
