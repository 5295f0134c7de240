// Log probabilities of given tokens, with the entropy of every row's distribution and its k most
// likely alternatives, and the gradient of the first two with respect to the logits.
//
//   m = max x, s = sum e^(x-m), u = sum e^(x-m) (x-m)      one pass, m running
//   lse = m + log s, logprob = x_t - lse, entropy = log s - u / s
//   dx_i = gl (1[i = t] - p_i) - ge p_i (log p_i + entropy),  p_i = e^(x_i - m) / s
//
// The running maximum, both sums and everything derived from them are fp32. The backward pass takes m and log s
// apart: their sum lse is good to |lse| 2^-24 only, which every probability formed from it would carry (logits
// around 1e4: 5e-4 of p; from the two parts a few 1e-6 wherever the logits lie). A forbidden token (-inf)
// has probability zero and takes no part in u. A row without any finite logit has no distribution:
// its logprob and lse are -inf, its entropy and its gradient zero. NaN (or +inf) among the logits
// makes the row's results NaN. A target equal to ignore_index gives logprob 0 and no gradient from
// it; any other target outside [0, vocab) gives NaN and is never used as an address.
//
// Bound by reading the logits (and writing their gradient): 8192 x 50304 bf16 takes 150 us forward (5.5 TB/s, with
// the exponential unit at three quarters) and 250 us backward, less than the 255 of its bytes because it takes
// the rows in reverse and finds the last 100 MB in L2. Rows are shared by clusters of up to 8 blocks while rows
// are few: 8 rows or one take 12 us with entropy and 8 alternatives, 5.6 without.

#include <cuda_runtime.h>

#include "common.h"
#include "ptx_sm100.cuh"
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

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cluster_sync() {
  ptx::cluster_arrive();
  ptx::cluster_wait();
}
// Values at the same shared-memory place in CTA `cta` of the cluster.
__device__ __forceinline__ uint64_t ld_cluster_u64(const void* place, int cta) {
  uint64_t v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(ptx::mapa_cluster(ptx::smem_u32(place), cta)) : "memory");
  return v;
}
__device__ __forceinline__ Stats ld_cluster_stats(const Stats* place, int cta) {
  const uint32_t at = ptx::mapa_cluster(ptx::smem_u32(place), cta);
  Stats a;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a.m) : "r"(at) : "memory");
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a.s) : "r"(at + 4) : "memory");
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a.u) : "r"(at + 8) : "memory");
  return a;
}

struct LogprobFwd {
  const void* logits;
  const int64_t* targets;
  float* logprob;
  float* stats;        // of every row lse, or its two parts: maximum and log of the sum; may be null
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  int64_t rows, ld, ignore_index;
  int32_t vocab, top_k;
  int32_t parts;       // CTAs (a cluster) that share a row
  int32_t split_stats;
};

// The elements of a row as a head up to the first 16-byte boundary, a body of 16-byte vectors and a tail.
template <typename T>
struct RowSpan {
  static constexpr int V = 16 / sizeof(T);
  int head, vecs, n;
  __device__ __forceinline__ RowSpan(const T* x, int n_) : n(n_) {
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    head = off == 0 ? 0 : V - off;
    if (head > n) head = n;
    vecs = (n - head) / V;
  }
  __device__ __forceinline__ int tail() const { return head + vecs * V; }
};

using row::Pack;

// Adds a batch of B vectors to the running statistics: one look for a larger maximum per batch.
template <typename T, bool ENT, int B>
__device__ __forceinline__ void add_batch(Stats& a, const Pack<T, 16 / sizeof(T)> (&v)[B], float2& s2, float2& u2) {
  constexpr int V = 16 / sizeof(T);
  float top = kNegInf;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const float2 x = row::load2(v[b].e + 2 * k);
      top = fmaxf(top, fmaxf(x.x, x.y));
    }
  if (top > a.m) {
    // move what is summed so far to the new maximum
    a.s = s2.x + s2.y;
    a.u = ENT ? u2.x + u2.y : 0.f;
    rescale(a, top);
    s2 = make_float2(a.s, 0.f);
    u2 = make_float2(a.u, 0.f);
  }
  const float shift = a.m == kNegInf ? 0.f : -a.m;      // nothing finite yet: only -inf (adds 0) or NaN
  const float2 sh = make_float2(shift, shift), l2 = make_float2(kLog2e, kLog2e);
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const float2 d = row::add_(row::load2(v[b].e + 2 * k), sh);
      const float2 t = row::mul_(d, l2);
      const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
      s2 = row::add_(s2, e);
      // e is 0 long before -1000: a forbidden token adds 0, not 0 * inf
      if constexpr (ENT) u2 = row::fma_(e, make_float2(fmaxf(d.x, -1000.f), fmaxf(d.y, -1000.f)), u2);
    }
}

constexpr int kCandidates = 2048;

// Scratch of the selection of the best alternatives.
struct TopShared {
  uint64_t cand[kCandidates];
  uint64_t best[kMaxTopK];         // of this CTA
  int count;
  int warp_count[kThreads / 32];
};

// f(index, value) for the elements of vectors v0 .. v1 of a row, plus head and tail of a first and a last part, that
// are not below `least` (a NaN is not).
template <typename T, typename F>
__device__ __forceinline__ void for_elements(const T* x, const RowSpan<T>& sp, int v0, int v1, bool first_part, bool last_part,
                                             float least, F&& f) {
  constexpr int V = RowSpan<T>::V, B = 4;
  auto one = [&](int c) {
    const float v = to_f(x[c]);
    if (!(v < least)) f(c, v);
  };
  if (first_part && static_cast<int>(threadIdx.x) < sp.head) one(threadIdx.x);
  if (last_part && sp.tail() + static_cast<int>(threadIdx.x) < sp.n) one(sp.tail() + threadIdx.x);
  auto look = [&](int i, const uint4& q) {
    const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(&q);
    bool any = false;
#pragma unroll
    for (int e = 0; e < V; ++e) any |= !(to_f(v.e[e]) < least);
    if (any) {        // rare: from memory again, in little code
      const int c = sp.head + i * V;
#pragma unroll 1
      for (int e = 0; e < V; ++e) one(c + e);
    }
  };
  const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
  int i = v0 + threadIdx.x;
  for (; i + (B - 1) * kThreads < v1; i += B * kThreads) {
    uint4 q[B];
#pragma unroll
    for (int b = 0; b < B; ++b) q[b] = __ldg(body + i + b * kThreads);
#pragma unroll
    for (int b = 0; b < B; ++b) look(i + b * kThreads, q[b]);
  }
  uint4 q[B];
#pragma unroll
  for (int b = 0; b < B; ++b)
    if (i + b * kThreads < v1) q[b] = __ldg(body + i + b * kThreads);
#pragma unroll
  for (int b = 0; b < B; ++b)
    if (i + b * kThreads < v1) look(i + b * kThreads, q[b]);
}

// The k best of this CTA's part, best first, into out[0 .. k); fewer elements leave zeros. `mine` is the
// largest value this thread saw. The k-th largest of the threads' maxima bounds the k-th best from below (its
// upper 16 bits do, found bit by bit), so one more pass collects the few elements at or above that bound and
// ranks them. When too many share that bound
// (a masked row, few distinct values) only those above it are collected, and the lowest ids of those equal to it
// are found in order; when even those above it are too many, the k best are searched one after the other.
template <typename T>
__device__ __noinline__ void select_best(const T* x, const RowSpan<T>& sp, int v0, int v1, bool first_part, bool last_part, float mine, int k,
                            TopShared& sh, uint64_t* out) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.count = 0;
  for (int i = tid; i < k; i += kThreads) out[i] = 0;
  const uint32_t own = order_key(mine);
  uint32_t bound = 0;
#pragma unroll 1
  for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
    if (__syncthreads_count(own >= (bound | bit)) >= k) bound |= bit;
  const uint32_t forbidden = order_key(kNegInf);
  auto collect = [&](uint32_t at_least) {
    for_elements<T>(x, sp, v0, v1, first_part, last_part, key_value(at_least), [&](int c, float v) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCandidates) sh.cand[at] = cand_word(order_key(v), c);
    });
  };
  int n = kCandidates + 1;
  if (bound > forbidden) {
    collect(bound);
    __syncthreads();
    n = sh.count;
    __syncthreads();
  }
  if (n > kCandidates) {
    if (bound <= forbidden) {
      bound = forbidden;      // fewer than k threads saw an allowed token: those, then forbidden ones
    } else {
      // the exact k-th largest maximum
#pragma unroll 1
      for (uint32_t bit = 1u << 15; bit != 0; bit >>= 1)
        if (__syncthreads_count(own >= (bound | bit)) >= k) bound |= bit;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (bound != 0xffffffffu) collect(bound + 1);     // above a NaN there is nothing
    __syncthreads();
    n = sh.count;
    __syncthreads();
    if (n <= kCandidates) {
      // the lowest ids whose key equals the bound, in order, until there are k candidates
      int have = n;
      const int c0 = first_part ? 0 : sp.head + v0 * RowSpan<T>::V, c1 = last_part ? sp.n : sp.head + v1 * RowSpan<T>::V;
      for (int base = c0; base < c1 && have < k; base += kThreads) {
        const int c = base + tid;
        const bool hit = c < c1 && order_key(to_f(x[c])) == bound;
        const uint32_t mask = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) sh.warp_count[warp] = __popc(mask);
        __syncthreads();
        int before = __popc(mask & ((1u << lane) - 1)), total = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
          const int cnt = sh.warp_count[w];
          if (w < warp) before += cnt;
          total += cnt;
        }
        if (hit && have + before < kCandidates) sh.cand[have + before] = cand_word(bound, c);
        have += total;
        __syncthreads();
      }
      n = have < kCandidates ? have : kCandidates;
    } else {
      uint64_t last = ~uint64_t{0};
      for (int i = 0; i < k; ++i) {
        uint64_t top = 0;
        for_elements<T>(x, sp, v0, v1, first_part, last_part, kNegInf, [&](int c, float v) {
          const uint64_t w = cand_word(order_key(v), c);
          if (w < last && w > top) top = w;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, top, o);
          if (other > top) top = other;
        }
        if (lane == 0) sh.cand[warp] = top;
        __syncthreads();
        for (int w = 0; w < kThreads / 32; ++w)
          if (sh.cand[w] > top) top = sh.cand[w];
        last = top;
        if (tid == 0) out[i] = top;
        __syncthreads();
      }
      return;
    }
  }
  // words are distinct: a candidate's rank is the number of larger ones
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t w = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n && rank < k; ++j) rank += sh.cand[j] > w;
    if (rank < k) out[rank] = w;
  }
  __syncthreads();
}

// (Five resident blocks keep enough loads on their way; the selection stays out of line, or its registers would
// leave room for one.)
template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kThreads, 5) logprob_fwd_kernel(const LogprobFwd p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int B = 32 / V;            // 32 elements a thread on their way
  __shared__ Stats warp_stats[kThreads / 32];
  __shared__ Stats part_stats;
  __shared__ float2 row_result;        // maximum and log of the sum
  extern __shared__ __align__(16) uint8_t top_raw[];
  TopShared& top = *reinterpret_cast<TopShared*>(top_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int parts = p.parts;
  const int part = parts > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const bool first_part = part == 0, last_part = part == parts - 1;
  for (int64_t r = blockIdx.x / parts; r < p.rows; r += gridDim.x / parts) {
    const T* x = static_cast<const T*>(p.logits) + r * p.ld;
    const RowSpan<T> sp(x, p.vocab);
    const int per = (sp.vecs + parts - 1) / parts;
    const int v0 = min(part * per, sp.vecs), v1 = min(v0 + per, sp.vecs);
    Stats a = empty_stats();
    float2 s2 = make_float2(0.f, 0.f), u2 = s2;
    const Pack<T, V>* body = reinterpret_cast<const Pack<T, V>*>(x + sp.head);
    int i = v0 + threadIdx.x;
    for (; i + (B - 1) * kThreads < v1; i += B * kThreads) {
      Pack<T, V> v[B];
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = row::ld_const<Pack<T, V>>(body + i + b * kThreads);
      add_batch<T, ENT, B>(a, v, s2, u2);
    }
    if (v1 - v0 >= 4 * B * kThreads) {
      // what is left of a long part: a few vectors, one by one
      for (; i < v1; i += kThreads) {
        const Pack<T, V> v[1] = {row::ld_const<Pack<T, V>>(body + i)};
        add_batch<T, ENT, 1>(a, v, s2, u2);
      }
    } else if (i < v1) {
      // of a short one, where each wait counts: one more batch, filled up with forbidden tokens
      Pack<T, V> v[B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (i + b * kThreads < v1) {
          v[b] = row::ld_const<Pack<T, V>>(body + i + b * kThreads);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[b].e[e] = from_f<T>(kNegInf);
        }
      }
      add_batch<T, ENT, B>(a, v, s2, u2);
    }
    a.s = s2.x + s2.y;
    a.u = ENT ? u2.x + u2.y : 0.f;
    auto add_one = [&](int c) {
      const float v = to_f(x[c]);
      if (v > a.m) rescale(a, v);
      add(a, v);
    };
    if (first_part && static_cast<int>(threadIdx.x) < sp.head) add_one(threadIdx.x);
    if (last_part && sp.tail() + static_cast<int>(threadIdx.x) < sp.n) add_one(sp.tail() + threadIdx.x);
    const float mine = a.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = merge(a, shfl_xor(a, o));
    if (lane == 0) warp_stats[warp] = a;
    __syncthreads();
    if (warp == 0) {
      a = lane < kThreads / 32 ? warp_stats[lane] : empty_stats();
#pragma unroll
      for (int o = kThreads / 64; o > 0; o >>= 1) a = merge(a, shfl_xor(a, o));
    }
    if constexpr (TOP) select_best<T>(x, sp, v0, v1, first_part, last_part, mine, p.top_k, top, top.best);
    if (parts > 1) {
      // the first CTA of the cluster gathers statistics and candidates of the others from their shared memory
      if (threadIdx.x == 0) part_stats = a;
      cluster_sync();
      if (first_part && warp == 0) {
        a = lane < parts ? ld_cluster_stats(&part_stats, lane) : empty_stats();
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) a = merge(a, shfl_xor(a, o));
      }
      if constexpr (TOP) {
        if (first_part)
          for (int j = threadIdx.x; j < parts * p.top_k; j += kThreads) {
            const int from = j / p.top_k, at = j - from * p.top_k;
            top.cand[j] = ld_cluster_u64(&top.best[at], from);
          }
      }
      cluster_sync();      // the others may go on (or leave) once everything has been read
    }
    if (first_part) {
      if (threadIdx.x == 0) {
        const float logs = logf(a.s);
        const float lse = a.m == kNegInf ? (a.s == 0.f ? kNegInf : nan_f()) : a.m + logs;
        const int64_t t = p.targets[r];
        float lp = nan_f();
        if (t == p.ignore_index) {
          lp = 0.f;
        } else if (t >= 0 && t < p.vocab) {
          lp = lse == kNegInf ? kNegInf : (to_f(x[t]) - a.m) - logs;
        }
        p.logprob[r] = lp;
        if (p.stats) {
          if (p.split_stats)
            reinterpret_cast<float2*>(p.stats)[r] = make_float2(a.m, logs);
          else
            p.stats[r] = lse;
        }
        if (ENT) p.entropy[r] = lse == kNegInf ? 0.f : logs - a.u / a.s;
        // the alternatives' log probabilities are (x - a.m) - logs; -inf in an empty row, NaN in one whose lse is
        row_result = make_float2(a.m == kNegInf ? lse : a.m, logs);
      }
      if constexpr (TOP) {
        __syncthreads();
        const float m = row_result.x, logs = row_result.y;
        auto put = [&](int at, uint64_t w) {
          p.top_ids[r * p.top_k + at] = 0xffffffffu - static_cast<uint32_t>(w);
          p.top_logprobs[r * p.top_k + at] = m == kNegInf ? kNegInf : (key_value(static_cast<uint32_t>(w >> 32)) - m) - logs;
        };
        if (parts == 1) {
          for (int j = threadIdx.x; j < p.top_k; j += kThreads) put(j, top.best[j]);
        } else {
          const int n = parts * p.top_k;
          for (int j = threadIdx.x; j < n; j += kThreads) {
            const uint64_t w = top.cand[j];
            if (w == 0) continue;       // a part with fewer than top_k elements
            int rank = 0;
            for (int q = 0; q < n; ++q) rank += top.cand[q] > w;
            if (rank < p.top_k) put(rank, w);
          }
        }
      }
    }
    __syncthreads();
  }
}

struct LogprobBwd {
  const void* logits;
  const int64_t* targets;
  const float2* stats;     // maximum and log of the sum, or null:
  const float* lse;        // their sum instead
  const float* entropy;
  const float* dlogprob;   // may be null
  const float* dentropy;   // may be null
  void* dlogits;
  int64_t rows, ld, ldd, ignore_index;
  int32_t vocab, width;
};

// One row per block of the grid's first dimension (the last rows first: the forward pass left their logits in
// L2), its vectors dealt to the blocks of the second.
// Few values live through the loop, so that 32 registers do and eight blocks are resident (8192 x 50304 bf16: 251 us,
// with one register more 272; with an entropy's gradient 270 instead of 301): both gradients are taken times 1 / s,
// and the thread that has the target's column writes it once more at the end.
template <typename T, bool ENT>
__global__ void __launch_bounds__(kThreads) logprob_bwd_kernel(const LogprobBwd p) {
  constexpr int V = 16 / sizeof(T);
  using P = Pack<T, V>;
  const int64_t r = p.rows - 1 - blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + r * p.ld;
  T* d = static_cast<T*>(p.dlogits) + r * p.ldd;
  const int64_t t = p.targets[r];
  const float2 st = p.stats ? p.stats[r] : make_float2(p.lse[r], 0.f);
  const float m = st.x, lse = st.x + st.y;
  const bool ignored = t == p.ignore_index;
  float gl = p.dlogprob && !ignored ? p.dlogprob[r] : 0.f;
  float ge = ENT ? p.dentropy[r] : 0.f;
  const float h = ENT ? p.entropy[r] - st.y : 0.f;      // log p_i + entropy = (x_i - m) + h
  const bool outside = p.dlogprob && !ignored && (t < 0 || t >= p.vocab);      // the entropy does not see the target
  if (outside) gl = nan_f();
  // an ignored row stays zero whatever its logits hold
  const bool none = (lse == kNegInf && !outside) || (gl == 0.f && ge == 0.f && (ignored || lse == lse));
  const int limit = none ? 0 : p.vocab;
  const int target = p.dlogprob && t >= 0 && t < limit && !ignored ? static_cast<int>(t) : -1;
  const float gt = gl;
  gl *= expf(-st.y);
  if constexpr (ENT) ge *= expf(-st.y);
  auto value = [&](float x, float own) {
    const float gap = x - m;
    const float e = exp2_approx(gap * kLog2e);
    float v = fmaf(-gl, e, own);
    if constexpr (ENT) v -= ge * e * (fmaxf(gap, -1000.f) + h);
    return v;
  };
  auto one = [&](int c, float own) { d[c] = from_f<T>(c < limit ? value(to_f(x[c]), own) : 0.f); };
  const int first = static_cast<int>(blockIdx.y) * kThreads + static_cast<int>(threadIdx.x);
  const int step = static_cast<int>(gridDim.y) * kThreads;
  const bool paired = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
  if (!paired) {
    for (int c = first; c < p.width; c += step) one(c, c == target ? gt : 0.f);
    return;
  }
  const RowSpan<T> sp(d, p.width);
  if (first < sp.head) one(first, first == target ? gt : 0.f);
  if (sp.tail() + first < p.width) one(sp.tail() + first, sp.tail() + first == target ? gt : 0.f);
  const T at_target = x[target >= 0 ? target : 0];      // before its vector is written: d may be x
  const float2 sh = make_float2(-m, -m), l2 = make_float2(kLog2e, kLog2e), ng = make_float2(-gl, -gl);
  const float2 ne = make_float2(-ge, -ge), hh = make_float2(h, h);
#pragma unroll 4
  for (int i = first; i < sp.vecs; i += step) {
    const int c = sp.head + i * V;
    P out;
    if (c + V <= limit) {
      const P v = row::ld<P>(x + c);
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        const float2 gap = row::add_(row::load2(v.e + 2 * k), sh);
        const float2 q = row::mul_(gap, l2);
        const float2 e = make_float2(exp2_approx(q.x), exp2_approx(q.y));
        float2 g = ng;
        if constexpr (ENT) g = row::fma_(ne, row::add_(make_float2(fmaxf(gap.x, -1000.f), fmaxf(gap.y, -1000.f)), hh), g);
        row::store2(out.e + 2 * k, row::mul_(g, e));
      }
      row::st(d + c, out);
    } else if (c >= limit) {
#pragma unroll
      for (int e = 0; e < V; ++e) out.e[e] = from_f<T>(0.f);
      row::st(d + c, out);
    } else {
      for (int e = 0; e < V; ++e) one(c + e, 0.f);
    }
  }
  const int at = target - sp.head;
  if (at >= 0 && target < sp.tail() && (at / V - first) % step == 0) d[target] = from_f<T>(value(to_f(at_target), p.dlogprob[r]));
}

int check_logits(int64_t rows, int64_t vocab, int dtype) {
  if (rows < 0 || vocab <= 0 || vocab > INT32_MAX - 65536) return B200S_ERR_BAD_SHAPE;
  if (dtype != B200S_BF16 && dtype != B200S_FP16 && dtype != B200S_FP32) return B200S_ERR_BAD_DTYPE;
  return B200S_OK;
}

bool misaligned(const void* p, size_t es) { return reinterpret_cast<uintptr_t>(p) % es != 0; }

// CTAs that share a row: as many (a power of two up to 8) as it takes to give every SM two, as long as each
// keeps 2048 tokens.
int row_parts(int64_t rows, int64_t vocab) {
  int n = 1;
  while (n < 8 && rows * n < 2 * 148 && vocab >= 2 * 2048 * static_cast<int64_t>(n)) n *= 2;
  return n;
}

template <typename T, bool ENT, bool TOP>
int launch_fwd_form(const LogprobFwd& p, cudaStream_t stream) {
  auto kernel = logprob_fwd_kernel<T, ENT, TOP>;
  const int64_t cap = 148 * 64;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.rows < cap ? p.rows : cap) * p.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = TOP ? sizeof(TopShared) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(p.parts);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  B200S_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p));
  count_launch();
  return B200S_OK;
}

template <typename T>
int launch_fwd(const LogprobFwd& p, cudaStream_t stream) {
  if (p.top_k > 0) return p.entropy ? launch_fwd_form<T, true, true>(p, stream) : launch_fwd_form<T, false, true>(p, stream);
  return p.entropy ? launch_fwd_form<T, true, false>(p, stream) : launch_fwd_form<T, false, false>(p, stream);
}

template <typename T>
int launch_bwd(const LogprobBwd& p, cudaStream_t stream) {
  // a block per row, more when rows are few: at least 2048 columns each
  int64_t parts = 1;
  while (p.rows * parts < 4 * 148 && p.width >= 2 * 2048 * parts) parts *= 2;
  for (int64_t r0 = 0; r0 < p.rows; r0 += int64_t{1} << 30) {
    LogprobBwd q = p;
    const int64_t n = p.rows - r0 < (int64_t{1} << 30) ? p.rows - r0 : int64_t{1} << 30;
    q.rows = n;
    q.logits = static_cast<const T*>(p.logits) + r0 * p.ld;
    q.dlogits = static_cast<T*>(p.dlogits) + r0 * p.ldd;
    q.targets = p.targets + r0;
    if (p.stats) q.stats = p.stats + r0;
    if (p.lse) q.lse = p.lse + r0;
    if (p.entropy) q.entropy = p.entropy + r0;
    if (p.dlogprob) q.dlogprob = p.dlogprob + r0;
    if (p.dentropy) q.dentropy = p.dentropy + r0;
    const dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(parts));
    if (p.dentropy)
      logprob_bwd_kernel<T, true><<<grid, kThreads, 0, stream>>>(q);
    else
      logprob_bwd_kernel<T, false><<<grid, kThreads, 0, stream>>>(q);
    B200S_CUDA_OK(cudaGetLastError());
    count_launch();
  }
  return B200S_OK;
}

}  // namespace

}  // namespace b200s

using namespace b200s;

// Both forward entries: lse, or stats (a maximum and a log of the sum per row), or neither.
static int logprobs_forward(int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld, const int64_t* targets,
                            int64_t ignore_index, float* logprob, float* lse, float* stats, float* entropy, int top_k,
                            int64_t* top_ids, float* top_logprobs, void* stream) {
  int rc = check_logits(rows, vocab, dtype);
  if (rc) return rc;
  if (top_k < 0 || top_k > kMaxTopK || top_k > vocab) return B200S_ERR_BAD_SHAPE;
  if (rows == 0) return B200S_OK;
  if (!logits || !targets || !logprob) return B200S_ERR_NULL_POINTER;
  if (top_k > 0 && (!top_ids || !top_logprobs)) return B200S_ERR_NULL_POINTER;
  if (rows > 1 && ld < 0) return B200S_ERR_BAD_STRIDE;
  if (misaligned(logits, dtype_size(dtype)) || misaligned(targets, 8) || misaligned(logprob, 4) || misaligned(lse, 4) ||
      misaligned(stats, 8) || misaligned(entropy, 4) || misaligned(top_ids, 8) || misaligned(top_logprobs, 4))
    return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const LogprobFwd p{logits, targets, logprob, stats ? stats : lse, entropy, top_ids, top_logprobs, rows, ld, ignore_index,
                     static_cast<int32_t>(vocab), top_k, row_parts(rows, vocab), stats ? 1 : 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B200S_BF16) return launch_fwd<__nv_bfloat16>(p, s);
  if (dtype == B200S_FP16) return launch_fwd<__half>(p, s);
  return launch_fwd<float>(p, s);
}

// Both backward entries: one of lse and stats.
static int logprobs_backward(int64_t rows, int64_t vocab, int64_t width, int dtype, const void* logits, int64_t ld,
                             const int64_t* targets, int64_t ignore_index, const float* lse, const float* stats,
                             const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits, int64_t ldd,
                             void* stream) {
  int rc = check_logits(rows, vocab, dtype);
  if (rc) return rc;
  if (width < vocab || width > INT32_MAX - 65536) return B200S_ERR_BAD_SHAPE;
  if (rows == 0) return B200S_OK;
  if (!logits || !targets || (!lse && !stats) || !dlogits || (dentropy && !entropy)) return B200S_ERR_NULL_POINTER;
  if (rows > 1 && (ld < 0 || ldd < width)) return B200S_ERR_BAD_STRIDE;
  if (misaligned(logits, dtype_size(dtype)) || misaligned(dlogits, dtype_size(dtype)) || misaligned(targets, 8) ||
      misaligned(lse, 4) || misaligned(stats, 8) || misaligned(entropy, 4) || misaligned(dlogprob, 4) || misaligned(dentropy, 4))
    return B200S_ERR_BAD_ALIGNMENT;
  if (!device_status_words()) return B200S_ERR_NO_DEVICE;
  const LogprobBwd p{logits, targets, reinterpret_cast<const float2*>(stats), lse, entropy, dlogprob, dentropy, dlogits, rows, ld,
                     ldd, ignore_index, static_cast<int32_t>(vocab), static_cast<int32_t>(width)};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B200S_BF16) return launch_bwd<__nv_bfloat16>(p, s);
  if (dtype == B200S_FP16) return launch_bwd<__half>(p, s);
  return launch_bwd<float>(p, s);
}

extern "C" {

int b200s_token_logprobs(int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld, const int64_t* targets,
                         int64_t ignore_index, float* logprob, float* lse, float* entropy, int top_k, int64_t* top_ids,
                         float* top_logprobs, void* stream) {
  return logprobs_forward(rows, vocab, dtype, logits, ld, targets, ignore_index, logprob, lse, nullptr, entropy, top_k, top_ids,
                          top_logprobs, stream);
}

int b200s_token_logprobs_stats(int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld, const int64_t* targets,
                               int64_t ignore_index, float* logprob, float* stats, float* entropy, int top_k, int64_t* top_ids,
                               float* top_logprobs, void* stream) {
  return logprobs_forward(rows, vocab, dtype, logits, ld, targets, ignore_index, logprob, nullptr, stats, entropy, top_k, top_ids,
                          top_logprobs, stream);
}

int b200s_token_logprobs_backward(int64_t rows, int64_t vocab, int64_t width, int dtype, const void* logits, int64_t ld,
                                  const int64_t* targets, int64_t ignore_index, const float* lse, const float* entropy,
                                  const float* dlogprob, const float* dentropy, void* dlogits, int64_t ldd,
                                  void* stream) {
  return logprobs_backward(rows, vocab, width, dtype, logits, ld, targets, ignore_index, lse, nullptr, entropy, dlogprob, dentropy,
                           dlogits, ldd, stream);
}

int b200s_token_logprobs_backward_stats(int64_t rows, int64_t vocab, int64_t width, int dtype, const void* logits, int64_t ld,
                                        const int64_t* targets, int64_t ignore_index, const float* stats, const float* entropy,
                                        const float* dlogprob, const float* dentropy, void* dlogits, int64_t ldd,
                                        void* stream) {
  return logprobs_backward(rows, vocab, width, dtype, logits, ld, targets, ignore_index, nullptr, stats, entropy, dlogprob, dentropy,
                           dlogits, ldd, stream);
}

}  // extern "C"
