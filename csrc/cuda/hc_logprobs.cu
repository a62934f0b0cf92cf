// Log probabilities of given tokens, entropies and most likely tokens of rows of logits; gradient of the logits.
//
// With m = max x and S = sum exp(x - m):  log p_i = x_i - m - log S,  H = log S - sum exp(x - m) (x - m) / S.
// One pass over a row: every thread keeps a running maximum and, relative to it, the sum of exp(x - m) and of
// exp(x - m) (x - m), which are rescaled when its maximum grows, after 32 logits at a time; the threads' triples are joined at
// the end.  When there are few rows, a row is shared out among the blocks of a cluster, which join through shared memory of
// the cluster.  Differences are taken before they are scaled for exp2, so logits of any size lose nothing.  What lies so far
// below the maximum that its exp is 0 is raised to a value where it still is, two 16-bit logits an instruction: -inf would
// make 0 times infinity of the second sum.
//
// Most likely tokens: value and index form one 64-bit key, so that no two are equal and the order is the one that the
// header states.  Each thread knows its own maximum after the pass; from one per warp follows a bound that at least
// `top` keys reach, and only the few threads whose maximum reaches it look at their logits again.  What they find is
// ranked by counting.
//
// Both passes read and write each logit once.  Arithmetic is done two values an instruction, for one at a time took 267 us forward
// and 300 us back for 8192 x 50257 logits of bf16, and they take 180 and 265 now: the gradient at 6.2 TB/s, bound by memory, the forward
// pass at 4.6, 0.7 of the copy rate, with 68 % of the issue slots in use (an exponential a logit, and the entropy's sum).
#include <cooperative_groups.h>

#include <type_traits>

#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kRowThreads = 512;     // of a block that has a row, or a part of one
constexpr int kStreamThreads = 128;  // of a block that has one row after the other
constexpr int kMostTop = 64;
constexpr int kCandidates = 2048;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kNothing = -200.0f;  // exp of this and of all below it is 0 in fp32

struct LogprobParams {
  const void* x;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_tokens;
  float* top_logprobs;
  float* stats;
  const float* d_logprobs;
  const float* d_entropy;
  void* dx;
  int64_t rows, vocab, stride, dstride, ignore;
  int top;
  int cluster;
};

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// the larger one, or NaN if one is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Softmax {
  float m, s, t;  // maximum, sum of exp(x - m), sum of exp(x - m) (x - m)
};
// A sum of nothing has m = kLowest, s = t = 0.
__device__ __forceinline__ Softmax join(const Softmax& a, const Softmax& b) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - m, kNothing), db = fmaxf(b.m - m, kNothing);
  const float fa = exp2_fast(da * kLog2e), fb = exp2_fast(db * kLog2e);
  Softmax r;
  r.m = m;
  r.s = fmaf(a.s, fa, b.s * fb);
  r.t = fmaf(fmaf(a.s, da, a.t), fa, fmaf(b.s, db, b.t) * fb);
  return r;
}
__device__ __forceinline__ Softmax warp_join(Softmax v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Softmax u;
    u.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    u.t = __shfl_xor_sync(0xffffffffu, v.t, o);
    // the same operand first in both lanes, so that both get the same bits
    v = (threadIdx.x & o) ? join(u, v) : join(v, u);
  }
  return v;
}

// Values in an order of whole numbers; 0 is below all.  -0 and +0 are equal.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, int64_t index) {
  return (uint64_t)ordered(v) << 32 | (0xffffffffu - (uint32_t)index);
}
// the value of a key (a zero without its sign)
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max64(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Where a row begins within an aligned group: groups of eight values (16-bit types: 16 bytes, fp32: 32 bytes)
template <typename T>
__device__ __forceinline__ int place_of(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) & 7u);
}

constexpr int kAtOnce = 4;  // groups of a thread whose loads are under way together

// Eight logits as they lie in memory, 16-bit types: two in a word
template <typename T>
struct Logits {
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    if (std::is_same<T, __half>::value) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t larger_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  // the largest of several groups, NaN apart
  template <int N>
  static __device__ __forceinline__ float largest(const Logits (&q)[N]) {
    uint32_t m = larger(larger(q[0].w[0], q[0].w[1]), larger(q[0].w[2], q[0].w[3]));
#pragma unroll
    for (int i = 1; i < N; ++i) m = larger(m, larger(larger(q[i].w[0], q[i].w[1]), larger(q[i].w[2], q[i].w[3])));
    float a, b;
    unpack2<T>(m, a, b);
    return fmaxf(a, b);
  }
  __device__ __forceinline__ void pairs(Pair (&v)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      unpack2<T>(w[j], a, b);
      v[j] = pair(a, b);
    }
  }
};
template <>
struct Logits<float> {
  float w[8];
  __device__ __forceinline__ void load(const float* p) { load8(p, w); }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = v[j];
  }
  template <int N>
  static __device__ __forceinline__ float largest(const Logits (&q)[N]) {
    float m = q[0].w[0];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, q[i].w[j]);
    return m;
  }
  __device__ __forceinline__ void pairs(Pair (&v)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = pair(w[2 * j], w[2 * j + 1]);
  }
};

// What is taken for all logits below it, two of a 16-bit type: so far below m that its exp is 0, next to m in the type's steps
// a number apart, and finite.  0: there is none, the differences are raised one by one (fp32; m at the type's lowest).
template <typename T>
__device__ __forceinline__ uint32_t lowest_of(float m) {
  const float c = m - fmaxf(300.0f, fabsf(m) * 0.03125f);
  if (std::is_same<T, __half>::value) return c >= -65000.0f ? pack2<__half>(c, c) : 0u;
  if (std::is_same<T, __nv_bfloat16>::value) return c >= -3e38f ? pack2<__nv_bfloat16>(c, c) : 0u;
  return 0u;
}
// x - m, raised to where exp is 0
template <typename T>
__device__ __forceinline__ void differences(Logits<T> q, float m, uint32_t lowest, Pair (&d)[4]) {
  const Pair minus = pair(-m, -m);
  if constexpr (sizeof(T) == 2) {
    if (lowest) {
#pragma unroll
      for (int j = 0; j < 4; ++j) q.w[j] = Logits<T>::larger_nan(q.w[j], lowest);
      q.pairs(d);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = d[j] + minus;
      return;
    }
  }
  q.pairs(d);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    parts(d[j] + minus, a, b);
    d[j] = pair(max_nan(a, kNothing), max_nan(b, kNothing));
  }
}
__device__ __forceinline__ Pair exp2_pair(Pair v) {
  float a, b;
  parts(v, a, b);
  return pair(exp2_fast(a), exp2_fast(b));
}

// The groups g, g + kThreads, ... of a row; what is not the row's, or from `end` on, is -inf.
template <int kThreads, typename T>
__device__ __forceinline__ void load_some(Logits<T> (&q)[kAtOnce], const T* row, int64_t g, int64_t end, int shift, int64_t vocab) {
  const int64_t last = g + (kAtOnce - 1) * kThreads;
  if (g * 8 >= shift && last < end && (last + 1) * 8 - shift <= vocab) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) q[i].load(row + (g + i * kThreads) * 8 - shift);
  } else {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t first = (g + i * kThreads) * 8 - shift;
      float v[8];
      if (g + i * kThreads < end && first >= 0 && first + 8 <= vocab) {
        q[i].load(row + first);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = g + i * kThreads < end && first + j >= 0 && first + j < vocab ? to_float(row[first + j]) : -INFINITY;
        q[i].set(v);
      }
    }
  }
}

struct TopShared {
  uint64_t list[kCandidates];
  uint64_t warp_key[kRowThreads / 32];
  uint64_t bound;
  uint64_t best[kMostTop];  // of this block, largest first; 0 where there are fewer
  uint64_t last[kRowThreads / 32];
  int count;
};

// The `top` largest keys of the groups of a row that this block has, into sh.best.  A thread has the groups begin + its number,
// and every kThreads-th from there, and thread 0 also group 0 where `begin` is 1.  `mine`: its largest logit; `where`: the
// first group of those among which that stood (the next ones of the thread, up to kAtOnce), -1 for a thread without groups.
template <int kThreads, typename T>
__device__ void block_top(const LogprobParams& p, TopShared& sh, const T* row, int shift, int64_t begin, int64_t end, bool first_too, float mine,
                          int64_t where) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t groups = end - begin;
  const auto each_key = [&](int64_t from, int64_t to, auto f) {
    for (int64_t g = from; g < to; g += kThreads) {
      float v[8];
      load_group(row, g * 8 - shift, p.vocab, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = g * 8 - shift + j;
        if (c >= 0 && c < p.vocab) f(key_of(v[j], c));
      }
    }
  };
  const auto every_key = [&](auto f) {
    if (first_too && threadIdx.x == 0) each_key(0, 1, f);
    each_key(begin + threadIdx.x, end, f);
  };
  uint64_t key = 0;  // this thread's largest
  if (where >= 0) each_key(where, where < begin ? where + 1 : min(end, where + kAtOnce * kThreads), [&](uint64_t one) { key = max64(key, one); });
  // every warp's r-th largest; the (top / r)-th largest of those is reached by at least `top` keys
  const int warps = (int)max((int64_t)1, groups < kThreads ? (groups + 31) / 32 : (kThreads / 32));
  const int r = (p.top + warps - 1) / warps;
  uint64_t k = key, best = 0;
  for (int i = 0; i < r && i < 32; ++i) {
    best = warp_max64(k);
    if (k == best) k = 0;
  }
  if (r > 32) best = 0;
  if (lane == 0) sh.warp_key[warp] = best;
  if (threadIdx.x < kMostTop) sh.best[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.count = 0, sh.bound = 0;
  __syncthreads();
  if (threadIdx.x < kThreads / 32) {
    k = sh.warp_key[threadIdx.x];
    int above = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) above += sh.warp_key[w] > k;
    if (k && above == (p.top + r - 1) / r - 1) sh.bound = k;
  }
  __syncthreads();
  const uint64_t bound = sh.bound;
  if (where >= 0 && ordered(mine) >= (uint32_t)(bound >> 32)) {
    every_key([&](uint64_t one) {
      if (one < bound) return;
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCandidates) sh.list[at] = one;
    });
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kCandidates) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t one = sh.list[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += sh.list[j] > one;
      if (above < p.top) sh.best[above] = one;
    }
  } else {
    // far more candidates than asked for (the largest logits all fell to a few threads): one search per token
    uint64_t below = ~0ull;
    for (int i = 0; i < p.top; ++i) {
      uint64_t found = 0;
      every_key([&](uint64_t one) {
        if (one < below) found = max64(found, one);
      });
      found = warp_max64(found);
      if (lane == 0) sh.last[warp] = found;
      __syncthreads();
      found = 0;
      for (int w = 0; w < (kThreads / 32); ++w) found = max64(found, sh.last[w]);
      __syncthreads();
      if (threadIdx.x == 0) sh.best[i] = found;
      below = found;
    }
  }
  __syncthreads();
}

// a row whose token is left out
template <bool kTop>
__device__ __forceinline__ void leave_out(const LogprobParams& p, int64_t r) {
  if (threadIdx.x == 0) {
    p.logprobs[r] = 0.0f;
    p.entropy[r] = 0.0f;
    if (p.stats) p.stats[r * 3] = p.stats[r * 3 + 1] = p.stats[r * 3 + 2] = 0.0f;
  }
  if (kTop && threadIdx.x < p.top) {
    p.top_tokens[r * p.top + threadIdx.x] = -1;
    p.top_logprobs[r * p.top + threadIdx.x] = 0.0f;
  }
}
// a row whose sums are there; `logit`: of its token, for thread 0
template <bool kTop>
__device__ __forceinline__ void store_row(const LogprobParams& p, int64_t r, int64_t token, float logit, const Softmax& all, const uint64_t* best) {
  const bool sound = all.s > 0.0f && all.s < INFINITY;  // no NaN, no +inf, something above -inf
  const float log_s = logf(all.s);
  if (threadIdx.x == 0) {
    const float h = sound ? log_s - all.t / all.s : NAN;
    p.logprobs[r] = sound && token >= 0 && token < p.vocab ? logit - all.m - log_s : NAN;
    p.entropy[r] = h;
    if (p.stats) {
      p.stats[r * 3] = sound ? all.m : NAN;
      p.stats[r * 3 + 1] = log_s;
      p.stats[r * 3 + 2] = h;
    }
  }
  if (kTop && threadIdx.x < p.top) {
    const uint64_t key = best[threadIdx.x];
    const int64_t i = 0xffffffffu - (uint32_t)key;
    p.top_tokens[r * p.top + threadIdx.x] = sound ? i : -1;
    p.top_logprobs[r * p.top + threadIdx.x] = sound ? value_of(key) - all.m - log_s : NAN;
  }
}

// A thread's sums so far, relative to m, which is near its maximum but not more than kSlack below it: it follows only then, for
// in some thread of a warp the maximum grows nearly every time.  The maximum itself is `best`.
constexpr float kSlack = 8.0f;
template <typename T>
struct Running {
  float m, best;
  Pair s, t;
  uint32_t lowest;
  __device__ __forceinline__ void clear() {
    m = best = kLowest;
    s = t = pair(0.0f, 0.0f);
    lowest = 0;
  }
  // N more groups; whether the maximum has grown
  template <int N>
  __device__ __forceinline__ bool add(const Logits<T> (&q)[N]) {
    const float top = Logits<T>::largest(q);
    const bool more = top > best;
    best = fmaxf(best, top);
    if (top > m + kSlack || m == kLowest) {
      const float d = fmaxf(m - best, kNothing), f = exp2_fast(d * kLog2e);
      const Pair d2 = pair(d, d), f2 = pair(f, f);
      t = fma2(s, d2, t) * f2;
      s = s * f2;
      m = best;
      lowest = lowest_of<T>(best);
    }
    const Pair log2e = pair(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      Pair d[4];
      differences(q[i], m, lowest, d);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const Pair e = exp2_pair(d[k] * log2e);
        s = s + e;
        t = fma2(e, d[k], t);
      }
    }
    return more;
  }
  __device__ __forceinline__ Softmax sums() const { return join({m, both(s), both(t)}, {best, 0.0f, 0.0f}); }
};

// joins the threads' sums; in warp 0 every thread gets those of the block
template <int kThreads>
__device__ __forceinline__ Softmax block_join(Softmax a, Softmax* warp_part) {
  a = warp_join(a);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = threadIdx.x < kThreads / 32 ? warp_part[threadIdx.x] : Softmax{kLowest, 0.0f, 0.0f};
    a = warp_join(a);
  }
  return a;
}

// Few rows: a cluster of p.cluster blocks for each, or one block.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kRowThreads) hc_logprob_kernel(const __grid_constant__ LogprobParams p) {
  __shared__ Softmax warp_part[kRowThreads / 32];
  __shared__ Softmax block_part;
  extern __shared__ __align__(16) unsigned char dynamic[];
  TopShared& sh = *reinterpret_cast<TopShared*>(dynamic);  // only there with kTop
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = blockIdx.x % p.cluster;
  const int64_t r = blockIdx.x / p.cluster;
  const int64_t token = p.tokens[r];
  const T* row = static_cast<const T*>(p.x) + r * p.stride;
  const int shift = place_of(row);
  const int64_t groups = (p.vocab + shift + 7) / 8;
  const int64_t begin = groups * part / p.cluster, end = groups * (part + 1) / p.cluster;
  Logits<T> q[kAtOnce];
  int64_t g = begin + threadIdx.x;
  if (g < end) load_some<kRowThreads>(q, row, g, end, shift, p.vocab);  // on its way while the token comes
  if (token == p.ignore) {  // the same for all threads of the cluster
    if (part == 0) leave_out<kTop>(p, r);
    return;
  }
  const float logit = part == 0 && threadIdx.x == 0 && token >= 0 && token < p.vocab ? to_float(row[token]) : 0.0f;
  Running<T> run;
  run.clear();
  int64_t where = g < end ? g : -1;
  for (; g < end;) {
    if (run.add(q) && kTop) where = g;
    g += kAtOnce * kRowThreads;
    if (g < end) load_some<kRowThreads>(q, row, g, end, shift, p.vocab);
  }
  Softmax a = block_join<kRowThreads>(run.sums(), warp_part);
  if (warp == 0 && lane == 0) block_part = a;
  if (kTop) block_top<kRowThreads>(p, sh, row, shift, begin, end, false, run.best, where);
  if (p.cluster > 1) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0) {
      if (warp == 0) {
        Softmax b = {kLowest, 0.0f, 0.0f};
        if (lane < p.cluster) b = *cluster.map_shared_rank(&block_part, lane);
        a = warp_join(b);
      }
      if (kTop) {
        // the blocks' own largest, ranked together
        const int n = p.cluster * p.top;
        for (int i = threadIdx.x; i < n; i += kRowThreads) sh.list[i] = cluster.map_shared_rank(&sh, i / p.top)->best[i % p.top];
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kRowThreads) {
          const uint64_t one = sh.list[i];
          int above = 0;
          for (int j = 0; j < n; ++j) above += sh.list[j] > one;
          if (one && above < p.top) sh.best[above] = one;
        }
      }
      if (warp == 0 && lane == 0) block_part = a;
    }
    cluster.sync();  // nobody leaves before its part has been read
  } else {
    __syncthreads();
  }
  if (part == 0) store_row<kTop>(p, r, token, logit, block_part, sh.best);
}

// Many rows: a block stays and has one row after the other brought into a ring in shared memory, in pieces of 32 logits a thread
// by bulk copies that do not wait for the end of a row.  What a row costs besides its logits, some 300 instructions a thread, is
// kept small by few threads, and the SM filled by eight blocks, or as many as their shared memory lets in: four of fp32 (48 KB each),
// five of 16 bits and three of fp32 with the best tokens' lists (8192 x 50257 logits of bf16: 267 us with a block of 512 threads for
// each row, 280 with two such blocks an SM and rings).
template <typename T>
constexpr int kPieceBytes = kAtOnce * 8 * (int)sizeof(T) * kStreamThreads;
constexpr int kRing = 3;
__device__ unsigned int g_logprob_status;

template <typename T>
struct Stream {  // what one thread knows to ask for the pieces
  int64_t row, token;
  int piece, pieces;
  const T* from;
  int64_t groups;  // whole ones that begin at `from`
};
template <typename T>
__device__ __forceinline__ void whole_groups(const T* row, int64_t vocab, const T*& from, int64_t& groups) {
  const int shift = place_of(row), skipped = shift ? 8 - shift : 0;
  from = row + skipped;
  groups = (vocab - skipped) / 8;
}

template <typename T, bool kTop>
__global__ void __launch_bounds__(kStreamThreads, 8) hc_logprob_stream_kernel(const __grid_constant__ LogprobParams p) {
  constexpr int kGroups = kAtOnce * kStreamThreads;
  __shared__ Softmax warp_part[(kStreamThreads / 32)];
  __shared__ Softmax block_part;
  __shared__ uint64_t full[kRing], empty[kRing];
  extern __shared__ __align__(128) unsigned char dynamic[];
  TopShared& sh = *reinterpret_cast<TopShared*>(dynamic + kRing * kPieceBytes<T>);  // only there with kTop
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], (kStreamThreads / 32));
    }
    fence_mbar_init();
  }
  __syncthreads();
  // Thread 0 asks for the pieces, kRing - 1 ahead of the one that is worked on.
  Stream<T> ask;
  ask.row = blockIdx.x;
  ask.piece = ask.pieces = 0;
  uint32_t asked = 0;
  bool gave_up = false;
  const auto ask_one = [&] {
    while (ask.piece == ask.pieces) {  // the next row that is read
      if (ask.pieces) ask.row += gridDim.x;
      while (ask.row < p.rows && p.tokens[ask.row] == p.ignore) ask.row += gridDim.x;
      if (ask.row >= p.rows) return;
      whole_groups(static_cast<const T*>(p.x) + ask.row * p.stride, p.vocab, ask.from, ask.groups);
      ask.pieces = (int)((ask.groups + kGroups - 1) / kGroups);
      ask.piece = 0;
    }
    const int stage = asked % kRing;
    if (asked >= kRing && !mbar_wait_bounded(&empty[stage], (asked / kRing - 1) & 1, 2000ull * 1000 * 1000)) gave_up = true;
    const int64_t first = (int64_t)ask.piece * kGroups;
    const uint32_t bytes = (uint32_t)min((int64_t)kGroups, ask.groups - first) * 8 * sizeof(T);
    mbar_expect_tx(&full[stage], bytes);
    bulk_load(dynamic + stage * kPieceBytes<T>, ask.from + first * 8, bytes, &full[stage]);
    ++ask.piece;
    ++asked;
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < kRing - 1; ++i) ask_one();
  uint32_t used = 0;
  int64_t token = blockIdx.x < p.rows ? p.tokens[blockIdx.x] : 0;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const int64_t next_token = r + gridDim.x < p.rows ? p.tokens[r + gridDim.x] : 0;
    if (token == p.ignore) {
      leave_out<kTop>(p, r);
      token = next_token;
      continue;
    }
    const T* row = static_cast<const T*>(p.x) + r * p.stride;
    const int shift = place_of(row);
    const float logit = threadIdx.x == 0 && token >= 0 && token < p.vocab ? to_float(row[token]) : 0.0f;
    const T* from;
    int64_t groups;
    whole_groups(row, p.vocab, from, groups);
    const int64_t all = (p.vocab + shift + 7) / 8;
    const int skipped = shift ? 1 : 0;  // the groups that come through the ring are skipped, skipped + 1, ...
    Running<T> run;
    run.clear();
    int64_t where = skipped + threadIdx.x < all ? skipped + threadIdx.x : -1;
    // what lies before the first whole group, and behind the last one
    for (int edge = 0; edge < 2; ++edge) {
      const int64_t g = edge ? all - 1 : 0;
      if (edge ? skipped + groups == all || threadIdx.x != (all - 1 - skipped) % kStreamThreads : !skipped || threadIdx.x) continue;
      float v[8];
      Logits<T> q[1];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = g * 8 + j >= shift && g * 8 + j - shift < p.vocab ? to_float(row[g * 8 + j - shift]) : -INFINITY;
      q[0].set(v);
      if (run.add(q) && kTop) where = g;
    }
    for (int64_t g0 = 0; g0 < groups; g0 += kGroups, ++used) {
      if (threadIdx.x == 0) ask_one();
      const int stage = used % kRing;
      // after a wait that ran out the others are short (a copy may still be on its way); the status says that sums are wrong
      if (!mbar_wait_bounded(&full[stage], (used / kRing) & 1, gave_up ? 1000ull * 1000 : 2000ull * 1000 * 1000)) gave_up = true;
      const T* piece = reinterpret_cast<const T*>(dynamic + stage * kPieceBytes<T>);
      Logits<T> q[kAtOnce];
      const int64_t g = g0 + threadIdx.x;
      if (g0 + kGroups <= groups) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) q[i].load(piece + (threadIdx.x + i * kStreamThreads) * 8);
        if (run.add(q) && kTop) where = skipped + g;
      } else {
#pragma unroll 1
        for (int i = 0; i < kAtOnce; ++i) {
          if (g + i * kStreamThreads >= groups) break;
          Logits<T> one[1];
          one[0].load(piece + (threadIdx.x + i * kStreamThreads) * 8);
          if (run.add(one) && kTop) where = skipped + g + i * kStreamThreads;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
    if (__any_sync(0xffffffffu, gave_up) && lane == 0) atomicMax(&g_logprob_status, 3u);
    const Softmax a = block_join<kStreamThreads>(run.sums(), warp_part);
    if (threadIdx.x == 0) block_part = a;
    if (kTop) block_top<kStreamThreads>(p, sh, row, shift, skipped, all, skipped, run.best, where);
    __syncthreads();
    store_row<kTop>(p, r, token, logit, block_part, sh.best);
    token = next_token;
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kStreamThreads) hc_logprob_backward_kernel(const __grid_constant__ LogprobParams p) {
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const int64_t token = p.tokens[r];
    const T* row = static_cast<const T*>(p.x) + r * p.stride;
    T* out = static_cast<T*>(p.dx) + r * p.dstride;
    const bool skip = token == p.ignore;
    const int shift = place_of(row);
    const bool same = place_of(out) == shift;
    const int64_t groups = (p.vocab + shift + 7) / 8;
    const bool lost = !skip && (token < 0 || token >= p.vocab);
    const float m = skip ? 0.0f : lost ? NAN : p.stats[r * 3], log_s = p.stats[r * 3 + 1], h = p.stats[r * 3 + 2];
    const float a = !skip && p.d_logprobs ? p.d_logprobs[r] : 0.0f, b = !skip && p.d_entropy ? p.d_entropy[r] : 0.0f;
    // p = exp2((x - m) log2e - log2e log S); dx = p (c1 (x - m) + c0), and a more at the token
    const Pair log2e = pair(kLog2e, kLog2e), less = pair(-log_s * kLog2e, -log_s * kLog2e);
    const float c0 = -fmaf(b, h - log_s, a);
    const Pair first_term = pair(c0, c0), slope = pair(-b, -b);
    const uint32_t lowest = lowest_of<T>(m);
    const int64_t token_group = skip || lost ? -1 : (token + shift) / 8, token_place = (token + shift) % 8;
    for (int64_t g = (int64_t)blockIdx.y * kAtOnce * kStreamThreads + threadIdx.x; g < groups; g += (int64_t)gridDim.y * kAtOnce * kStreamThreads) {
      Logits<T> q[kAtOnce];
      if (!skip) load_some<kStreamThreads>(q, row, g, groups, shift, p.vocab);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int64_t group = g + i * kStreamThreads, first = group * 8 - shift;
        if (group >= groups) break;
        float v[8];
        if (skip) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        } else {
          Pair d[4];
          differences(q[i], m, lowest, d);
#pragma unroll
          for (int j = 0; j < 4; ++j) parts(exp2_pair(fma2(d[j], log2e, less)) * fma2(d[j], slope, first_term), v[2 * j], v[2 * j + 1]);
          if (group == token_group) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += j == token_place ? a : 0.0f;
          }
        }
        if (same) {
          store_group(out, first, p.vocab, v);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (first + j >= 0 && first + j < p.vocab) out[first + j] = from_float<T>(v[j]);
        }
      }
    }
  }
}

}  // namespace dev

namespace {

bool logits_ok(const void* x, int type, size_t rows, size_t vocab, size_t stride) {
  if (!element_type_ok(type) || vocab == 0 || vocab > 0x7fffffffu || stride < vocab || rows > 0x7fffffffu || stride > (1ull << 40))
    return false;
  return rows == 0 || (x && reinterpret_cast<uintptr_t>(x) % element_bytes(type) == 0 && rows <= (1ull << 60) / stride);
}

// Blocks per row: as many as have an SM each, up to the eight of a portable cluster, while each has at least one group of
// eight logits for every other thread (37 rows of 50257: 7.8 us in clusters of four; 12.9 in clusters of eight, which leave SMs two blocks).
int cluster_of(size_t rows, size_t vocab) {
  const size_t sms = device_info().sms;
  int c = 1;
  while (c < 8 && rows * c * 2 <= sms && vocab / (size_t)(c * 2) >= dev::kRowThreads * 8 / 2) c *= 2;
  return c;
}

template <typename T, bool kTop>
cudaError_t run_logprobs(dev::LogprobParams p, cudaStream_t stream) {
  const int64_t sms = device_info().sms;
  // A block for a row has its own start and end, which the ring does without; the ring wants some pieces a row and a row for
  // each of its blocks.
  if (p.rows >= 8 * sms && p.vocab >= 2 * dev::kPieceBytes<T> / (int64_t)sizeof(T)) {
    const int smem = dev::kRing * dev::kPieceBytes<T> + (kTop ? (int)sizeof(dev::TopShared) : 0);
    static unsigned long long allowed = 0;
    const cudaError_t e = allow_smem(dev::hc_logprob_stream_kernel<T, kTop>, smem, &allowed);
    if (e != cudaSuccess) return e;
    dev::hc_logprob_stream_kernel<T, kTop><<<(unsigned)(8 * sms), dev::kStreamThreads, smem, stream>>>(p);
    return cudaGetLastError();
  }
  p.cluster = cluster_of(p.rows, p.vocab);
  if (p.rows > 0x7fffffff / p.cluster) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(p.rows * p.cluster));
  cfg.blockDim = dim3(dev::kRowThreads);
  cfg.dynamicSmemBytes = kTop ? sizeof(dev::TopShared) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  memset(&attr, 0, sizeof(attr));
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, dev::hc_logprob_kernel<T, kTop>, p);
}

template <typename F>
cudaError_t by_type(int type, F f) {
  return type == kF32 ? f(float()) : type == kBf16 ? f(__nv_bfloat16()) : f(__half());
}

}  // namespace

int logprob_status(int clear) { return take_status(dev::g_logprob_status, clear); }

}  // namespace hc

extern "C" {

int hc_token_logprobs(const void* logits, int type, size_t rows, size_t vocab, size_t stride, const int64_t* tokens,
                      int64_t ignore, int top, float* logprobs, float* entropy, int64_t* top_tokens, float* top_logprobs,
                      float* stats, hc_stream_t stream) {
  if (!hc::logits_ok(logits, type, rows, vocab, stride)) return hc::kErrArgument;
  if (top < 0 || top > hc::dev::kMostTop || (size_t)top > vocab) return hc::kErrArgument;
  if (rows == 0) return hc::kOk;
  if (!tokens || !logprobs || !entropy || (top && (!top_tokens || !top_logprobs))) return hc::kErrArgument;
  if (!hc::lies_at(tokens, 8) || !hc::lies_at(logprobs, 4) || !hc::lies_at(entropy, 4) || !hc::lies_at(top_tokens, 8) || !hc::lies_at(top_logprobs, 4) ||
      !hc::lies_at(stats, 4))
    return hc::kErrArgument;
  hc::dev::LogprobParams p = {logits, tokens, logprobs, entropy, top_tokens, top_logprobs, stats, nullptr, nullptr, nullptr,
                              (int64_t)rows, (int64_t)vocab, (int64_t)stride, 0, ignore, top, 1};
  const cudaError_t e = hc::by_type(type, [&](auto t) {
    return top ? hc::run_logprobs<decltype(t), true>(p, stream) : hc::run_logprobs<decltype(t), false>(p, stream);
  });
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

int hc_token_logprobs_backward(const void* logits, int type, size_t rows, size_t vocab, size_t stride,
                               const int64_t* tokens, int64_t ignore, const float* stats, const float* dlogprobs,
                               const float* dentropy, void* dlogits, size_t dstride, hc_stream_t stream) {
  if (!hc::logits_ok(logits, type, rows, vocab, stride) || !hc::logits_ok(dlogits, type, rows, vocab, dstride)) return hc::kErrArgument;
  if (rows == 0) return hc::kOk;
  if (!tokens || !stats) return hc::kErrArgument;
  if (!hc::lies_at(tokens, 8) || !hc::lies_at(stats, 4) || !hc::lies_at(dlogprobs, 4) || !hc::lies_at(dentropy, 4)) return hc::kErrArgument;
  hc::dev::LogprobParams p = {logits, tokens, nullptr, nullptr, nullptr, nullptr, const_cast<float*>(stats), dlogprobs, dentropy, dlogits,
                              (int64_t)rows, (int64_t)vocab, (int64_t)stride, (int64_t)dstride, ignore, 0, 1};
  const size_t chunk = 8 * hc::dev::kAtOnce * hc::dev::kStreamThreads, parts = (vocab + 7 + chunk - 1) / chunk;
  const unsigned y = (unsigned)(rows >= 2048 ? 1 : parts < 1 ? 1 : parts > 64 ? 64 : parts);
  const dim3 grid((unsigned)(rows < 0x7fffffff ? rows : 0x7fffffff), y);
  const cudaError_t e = hc::by_type(type, [&](auto t) {
    hc::dev::hc_logprob_backward_kernel<decltype(t)><<<grid, hc::dev::kStreamThreads, 0, stream>>>(p);
    return cudaGetLastError();
  });
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

}  // extern "C"
