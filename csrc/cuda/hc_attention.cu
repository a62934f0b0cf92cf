// Causal attention with a sliding window and first tokens that stay visible, and its backward pass, on tcgen05 tensor cores.
//
//   query i stands at position p = i + Tk - Tq and sees key j if j <= p and (p - j < window or j < sinks)
//   S = scale Q K^T,  P = softmax of S over what is seen,  O = P V                (a query that sees nothing: 0)
//   delta_i = dO_i . O_i,  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Tiles of 128 queries by 128 keys; tiles that nobody sees are left out, only tiles at an edge of what is seen are masked.  One thread brings
// operands in by TMA, one issues the matrix instructions, eight warps have a row of a tile a thread: scores, probabilities and their
// gradients go from tensor memory to registers and back and never anywhere else.  The second product of each pair reads its first operand, in 16 bits, from where the
// scores lay.  Heads and batch are dimensions of the tensor maps, so a view into a projection's result is read where it lies; several query heads to a key's head read the
// same keys, and dK and dV of such a head are summed in one CTA.  Every sum has a fixed order.
//
// Forward: two tiles of queries share their keys, so that the tensor cores work on one while the other's exponentials are taken, which bound it up to heads of
// 64 (16 a cycle and SM).  The reference that exponentials are taken relative to follows a row's largest score when that is more than 2^8 above it; only then is O
// taken times a factor.  Few queries (with all heads of a key's head at most 128 rows, a new token of each text for one) are one tile, and the keys are shared
// out to several CTAs, whose results a second kernel joins: bound by reading keys and values.
// Backward: dK and dV in a kernel whose CTA has a tile of keys and goes through the queries, dQ in one whose CTA has a tile of queries.  That forms the scores twice (7 products instead of 5), and
// needs no atomic additions, whose order would change the result, and no array of partial dQ.
//
// In fp16, which has no numbers below 2^-24, P is held times a power of two, and dS times one that 2 max|dO_i| max|V_j| (norms of rows, which bound it) gives.
#include <math.h>

#include <type_traits>

#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_tensor.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kTile = 128;  // queries, keys
constexpr int kAttnWarps = 8;  // with a row a thread
constexpr int kAttnThreads = 64 + 32 * kAttnWarps;
constexpr uint64_t kAttnLimitNs = 2000ull * 1000 * 1000;
constexpr float kSlack = 8.0f;  // powers of two that a score may be above its row's reference

__device__ unsigned int g_attention_status;

template <int kD>
struct AttnShape {
  static constexpr int kBoxes = kD / 64;          // of 64 values, 128 bytes
  static constexpr int kBytes = kTile * kD * 2;   // of a tile
  static constexpr int kForwardStages = kD == 128 ? 4 : 8;  // tiles of keys or values
  static constexpr int kForwardSmem = (2 + kForwardStages) * kBytes + 1024;
  static constexpr int kQStages = kD == 128 ? 2 : 4, kDoStages = kD == 128 ? 2 : 4;
  static constexpr int kKvSmem = (2 + kQStages + kDoStages) * kBytes + kQStages * 1024 + 1024;
  static constexpr int kKStages = kD == 128 ? 3 : 5, kVStages = kD == 128 ? 2 : 4;
  static constexpr int kQSmem = (2 + kKStages + kVStages) * kBytes + 1024;
};

struct AttnParams {
  CUtensorMap q, k, v, dout;
  void* o;
  float* less;      // [batch heads][rows]: minus the logarithm (base 2) of a query's sum of exponentials, for the backward pass
  float* part_o;    // [split][query of all][head size], of the CTAs that share the keys out
  float* part_less;
  const float* delta;  // as `less`
  void *dq, *dk, *dv;
  const unsigned int* most;  // bits of max|dO_i|, max|V_j| (fp16)
  int64_t less_ld;
  int batch, heads, kv_heads, group, tq, tk, d, off, window, sinks;
  int packed;   // rows of the one tile that holds the queries of all heads of a key's head, or 0
  int blocks;   // of queries, or of keys
  int splits;
  float scale, scale2;  // scale2: times log2(e)
};

struct AttnBarriers {
  uint64_t full[8], empty[8], more_full[4], more_empty[4];
  uint64_t first, s_full[2], p_ready[2], done[2], s_read, dp_full[2], ds_ready[2], drained;
  uint32_t tmem, gave_up;
};

// A wait that ends: with the barrier, after the limit, or because another role has given up.
__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity, AttnBarriers& sh) {
  long long t0 = 0;
#pragma unroll 1
  for (uint32_t it = 0; !mbar_try_wait(bar, parity); ++it) {
    if ((it & 63u) == 0u) {
      const long long now = clock64();
      if (it == 0u) t0 = now;
      if (*reinterpret_cast<volatile uint32_t*>(&sh.gave_up)) return false;
      if (now - t0 > (long long)kAttnLimitNs * 2 || it >= (1u << 26)) {
        *reinterpret_cast<volatile uint32_t*>(&sh.gave_up) = 1;
        atomicMax(&g_attention_status, 3u);
        return false;
      }
    }
  }
  return true;
}
__device__ __forceinline__ bool attn_wait_all(uint64_t* bar, uint32_t parity, AttnBarriers& sh) { return __all_sync(0xffffffffu, attn_wait(bar, parity, sh)); }

// A place in a ring of N stages
template <int N>
struct Ring {
  int s = 0, count = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    ++count;
    if (++s == N) {
      s = 0;
      phase ^= 1;
    }
  }
};
// what a ring's last loads bring is there before the CTA leaves
template <int N>
__device__ __forceinline__ void ring_end(uint64_t* full, const Ring<N>& r) {
  for (int back = 0; back < N && back < r.count; ++back) {
    const int i = r.count - 1 - back;
    mbar_wait_bounded(&full[i % N], (i / N) & 1, kAttnLimitNs);
  }
}

__device__ __forceinline__ void load_4d(void* dst, const CUtensorMap* map, int x, int t, int h, int b, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)), "l"(map), "r"(x),
               "r"(t), "r"(h), "r"(b), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void load_floats(void* dst, const float* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// a tile: 128 rows from t on
template <int kD>
__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, int t, int h, int b, uint64_t* bar) {
#pragma unroll
  for (int i = 0; i < AttnShape<kD>::kBoxes; ++i) load_4d(dst + i * kTile * 128, map, i * 64, t, h, b, bar);
}

__device__ __forceinline__ void attn_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void attn_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// the first operand in tensor memory: rows in lanes, two values of the sum in a column
__device__ __forceinline__ void attn_mma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// Descriptors of a tile, 128-byte swizzle.  Along: the sum runs along its rows of 128 bytes (eight rows are 1024 bytes).  Across: the sum runs
// over its rows, 64 values across it are a box.
__device__ __forceinline__ uint64_t along(const unsigned char* tile) {
  return (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 / 16) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ uint64_t across(const unsigned char* tile) {
  return (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4) | (uint64_t)(kTile * 128 / 16) << 16 | (uint64_t)(1024 / 16) << 32 | 1ull << 46 | 2ull << 61;
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t operand_format() {
  return sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
}
template <typename T>
__device__ __forceinline__ uint32_t attn_idesc(int n, bool b_across) {
  return 1u << 4 | operand_format<T>() << 7 | operand_format<T>() << 10 | (b_across ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(kTile / 16) << 24;
}
// d = a b^T over the head's values: both tiles along the sum
template <typename T, int kD>
__device__ __forceinline__ void scores(uint32_t d, const unsigned char* a, const unsigned char* b) {
  const uint64_t da = along(a), db = along(b);
  const uint32_t idesc = attn_idesc<T>(kTile, false);
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) {
    const uint32_t at = (i / 4) * (kTile * 128 / 16) + (i % 4) * 2;
    attn_mma(d, da + at, db + at, idesc, i > 0);
  }
}
// d (+)= p b, p in tensor memory; its second 64 columns of the sum begin `second` columns behind the first
template <typename T, int kD>
__device__ __forceinline__ void weighted(uint32_t d, uint32_t p, int second, const unsigned char* b, bool add) {
  const uint64_t db = across(b);
  const uint32_t idesc = attn_idesc<T>(kD, true);
#pragma unroll
  for (int i = 0; i < 8; ++i) attn_mma_from_tmem(d, p + (i / 4) * second + (i % 4) * 8, db + i * 128, idesc, add || i > 0);
}

// ---- what is seen ------------------------------------------------------------------------------------------------------------
// the tiles of keys that positions p0 to p1 see: those of the first tokens, then a stretch
struct KeyTiles {
  int sinks, low, count;
  __device__ __forceinline__ int at(int e) const { return e < sinks ? e : low + e - sinks; }
};
__device__ __forceinline__ KeyTiles key_tiles(const AttnParams& p, int p0, int p1) {
  KeyTiles t = {0, 0, 0};
  if (p1 < 0) return t;
  const int lowest = p0 - p.window + 1;
  t.low = lowest > 0 ? lowest / kTile : 0;
  t.sinks = min((min(p.sinks, p1 + 1) + kTile - 1) / kTile, t.low);
  t.count = t.sinks + p1 / kTile - t.low + 1;
  return t;
}
__device__ __forceinline__ bool any_seen(const AttnParams& p, int p0, int p1, int k0) { return k0 <= p1 && (k0 + kTile - 1 > p0 - p.window || k0 < p.sinks); }
__device__ __forceinline__ bool all_seen(const AttnParams& p, int p0, int p1, int k0) { return k0 + kTile - 1 <= p0 && (p1 - k0 < p.window || k0 + kTile <= p.sinks); }

// barriers and tensor memory; by all threads
__device__ __forceinline__ void attn_begin(AttnBarriers& sh, int ready_warps) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.more_full[i], 1);
      mbar_init(&sh.more_empty[i], 1);
    }
    mbar_init(&sh.first, 1);
    mbar_init(&sh.s_read, kAttnWarps);
    mbar_init(&sh.drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_ready[i], ready_warps);
      mbar_init(&sh.done[i], 1);
      mbar_init(&sh.dp_full[i], 1);
      mbar_init(&sh.ds_ready[i], kAttnWarps);
    }
    sh.gave_up = 0;
    fence_mbar_init();
  }
  if (threadIdx.x >> 5 == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void attn_end(uint32_t tmem) {
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x >> 5 == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}
__device__ __forceinline__ unsigned char* attn_tiles(unsigned char* raw) {
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
}
// a warp has written to tensor memory, or read from it, what the barrier stands for
__device__ __forceinline__ void warp_arrives(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// A row's values, `factor` times what tensor memory has, from `to` on.  `there`, the same for all of a warp: tensor memory has them; `none`: zeros.
template <typename O, int kD>
__device__ __forceinline__ void store_row(uint32_t from, O* to, int d, float factor, bool in, bool there, bool none) {
#pragma unroll
  for (int c = 0; c < kD; c += 32) {
    float v[32];
    if (there) {
      __syncwarp();
      tc_load32(from + c, v);
      tc_load_wait(v);
    }
    if (!in) continue;
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (c + j >= d) continue;
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = there && !none ? v[j + k] * factor : 0.0f;
      store8(to + c + j, w);
    }
  }
}

// ---- forward -----------------------------------------------------------------------------------------------------------------
// Tensor memory: scores of the two tiles of queries at 0 and 128 (the probabilities in their first 64 columns), O at 256 and 384.
template <typename T, int kD>
__global__ void __launch_bounds__(kAttnThreads, 1) hc_attention_kernel(const __grid_constant__ AttnParams p) {
  using S = AttnShape<kD>;
  constexpr int kStages = S::kForwardStages;
  constexpr float kBias = operand_format<T>() ? 0.0f : 6.0f;  // probabilities are held times 2^6 in fp16: at most 2^14
  extern __shared__ unsigned char raw[];
  __shared__ AttnBarriers sh;
  unsigned char* tiles = attn_tiles(raw);
  unsigned char* ring = tiles + 2 * S::kBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the blocks of queries that see most come first
  const int heads = p.packed ? p.kv_heads : p.heads;
  int64_t at = blockIdx.x;
  const int split = (int)(at % p.splits);
  at /= p.splits;
  const int head = (int)(at % heads);
  at /= heads;
  const int b = (int)(at % p.batch), block = p.blocks - 1 - (int)(at / p.batch);
  const int kv_head = p.packed ? head : head / p.group;
  // positions of the two tiles' queries
  const int first = block * 2 * kTile;
  int p0[2], p1[2];
  for (int q = 0; q < 2; ++q) {
    const int i0 = first + q * kTile, i1 = min(i0 + kTile, p.tq) - 1;
    const bool there = i0 <= i1 && (q == 0 || !p.packed);
    p0[q] = p.off + i0;
    p1[q] = there ? p.off + (p.packed ? p.tq - 1 : i1) : -1;
  }
  const KeyTiles list = key_tiles(p, p0[0], max(p1[0], p1[1]));
  const int e0 = (int)((int64_t)list.count * split / p.splits), e1 = (int)((int64_t)list.count * (split + 1) / p.splits);
  attn_begin(sh, kAttnWarps / 2);
  const uint32_t tmem = sh.tmem;
  if (warp == 0) {
    if (lane == 0) {
      Ring<kStages> r;
      bool ok = true;
      const bool second = !p.packed && first + kTile < p.tq;
      if (e0 < e1) {
        if (p.packed) {
          mbar_expect_tx(&sh.first, p.packed * 128 * S::kBoxes);
          for (int i = 0; i < S::kBoxes; ++i) load_4d(tiles + i * kTile * 128, &p.q, i * 64, 0, head * p.group, b, &sh.first);
        } else {
          mbar_expect_tx(&sh.first, second ? 2 * S::kBytes : S::kBytes);
          load_tile<kD>(tiles, &p.q, first, head, b, &sh.first);
          if (second) load_tile<kD>(tiles + S::kBytes, &p.q, first + kTile, head, b, &sh.first);
        }
      }
      for (int e = e0; ok && e < e1; ++e) {
        for (int kv = 0; kv < 2; ++kv) {
          if (!attn_wait(&sh.empty[r.s], r.phase ^ 1, sh)) {
            ok = false;
            break;
          }
          mbar_expect_tx(&sh.full[r.s], S::kBytes);
          load_tile<kD>(ring + r.s * S::kBytes, kv ? &p.v : &p.k, list.at(e) * kTile, kv_head, b, &sh.full[r.s]);
          r.next();
        }
      }
      ring_end(sh.full, r);
      if (e0 < e1) mbar_wait_bounded(&sh.first, 0, kAttnLimitNs);
    }
  } else if (warp == 1) {
    if (lane == 0 && e0 < e1) {
      Ring<kStages> r;  // of what is waited for next
      int scored[2] = {0, 0}, summed[2] = {0, 0};
      const auto score = [&](int q, int e, const unsigned char* k) {
        if (!any_seen(p, p0[q], p1[q], list.at(e) * kTile)) return true;
        if (scored[q] && !attn_wait(&sh.done[q], (scored[q] - 1) & 1, sh)) return false;  // the probabilities that lie there have been read
        tc_fence_after();
        scores<T, kD>(tmem + q * kTile, tiles + q * S::kBytes, k);
        attn_commit(&sh.s_full[q]);
        ++scored[q];
        return true;
      };
      const auto sum = [&](int q, int e, const unsigned char* v) {
        if (!any_seen(p, p0[q], p1[q], list.at(e) * kTile)) return true;
        if (!attn_wait(&sh.p_ready[q], summed[q] & 1, sh)) return false;
        tc_fence_after();
        weighted<T, kD>(tmem + 256 + q * kTile, tmem + q * kTile, 32, v, summed[q] > 0);
        attn_commit(&sh.done[q]);
        ++summed[q];
        return true;
      };
      bool ok = attn_wait(&sh.first, 0, sh) && attn_wait(&sh.full[r.s], r.phase, sh);
      if (ok) {
        tc_fence_after();
        const unsigned char* k = ring + r.s * S::kBytes;
        ok = score(0, e0, k) && score(1, e0, k);
        attn_commit(&sh.empty[r.s]);
        r.next();
      }
      for (int e = e0; ok && e < e1; ++e) {
        if (!attn_wait(&sh.full[r.s], r.phase, sh)) break;
        tc_fence_after();
        const int v_stage = r.s;
        const unsigned char* v = ring + v_stage * S::kBytes;
        r.next();
        if (!sum(0, e, v)) break;
        const bool more = e + 1 < e1;
        const unsigned char* k = ring + r.s * S::kBytes;
        if (more) {
          if (!attn_wait(&sh.full[r.s], r.phase, sh)) break;
          tc_fence_after();
          if (!score(0, e + 1, k)) break;
        }
        if (!sum(1, e, v)) break;
        attn_commit(&sh.empty[v_stage]);
        if (more) {
          if (!score(1, e + 1, k)) break;
          attn_commit(&sh.empty[r.s]);
          r.next();
        }
      }
      attn_commit(&sh.drained);  // matrix instructions in flight are done before the CTA leaves
      mbar_wait_bounded(&sh.drained, 0, kAttnLimitNs);
    }
  } else {
    const int quarter = warp & 3, q = (warp - 2) >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lanes + q * kTile, o_at = lanes + 256 + q * kTile;
    const int i = p.packed ? row % p.tq : first + q * kTile + row;
    const bool in = p.packed ? q == 0 && row < p.packed : i < p.tq;
    const bool some = __any_sync(0xffffffffu, in);
    const int h = p.packed ? head * p.group + row / p.tq : head, position = p.off + i;
    const float slack = kSlack / p.scale2;
    float most = -INFINITY, sum = 0.0f, ref = 0.0f;
    int taken = 0;
    bool ok = true;
    for (int e = e0; e < e1; ++e) {
      const int k0 = list.at(e) * kTile;
      if (!any_seen(p, p0[q], p1[q], k0)) continue;
      if (!attn_wait_all(&sh.s_full[q], taken & 1, sh)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (some) {
        float v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc_load32(s_at + c * 32, v[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tc_load_wait(v[c]);
        if (!all_seen(p, p0[q], p1[q], k0)) {
          const int high = position - k0, low = position - p.window + 1 - k0, sinks = p.sinks - k0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const int n = c * 32 + j;
              if (n > high || (n < low && n >= sinks)) v[c][j] = -INFINITY;
            }
        }
        float tops[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tops[c] = fmaxf(v[c][0], v[c][1]);
#pragma unroll
          for (int j = 2; j < 32; j += 2) tops[c] = fmaxf(tops[c], fmaxf(v[c][j], v[c][j + 1]));
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const bool grows = top > most + slack;
        float factor = 1.0f;
        if (grows) {
          factor = power2((most - top) * p.scale2);
          most = top;
          ref = top * p.scale2 - kBias;
          sum *= factor;
        }
        if (taken && __any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int c = 0; c < kD; c += 32) {
            float o[32];
            __syncwarp();
            tc_load32(o_at + c, o);
            tc_load_wait(o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= factor;
            tc_store32(o_at + c, o);
          }
        }
        const Pair scale = pair(p.scale2, p.scale2), less = pair(-ref, -ref);
        Pair total = pair(0.0f, 0.0f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t words[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float x, y;
            parts(fma2(pair(v[c][j], v[c][j + 1]), scale, less), x, y);
            x = power2(x);
            y = power2(y);
            total = total + pair(x, y);
            words[j / 2] = pack2<T>(x, y);
          }
          tc_store16(s_at + c * 16, words);
        }
        sum += both(total);
        tc_store_wait();
      }
      ++taken;
      warp_arrives(&sh.p_ready[q]);
    }
    if (ok && taken && !attn_wait_all(&sh.done[q], (taken - 1) & 1, sh)) ok = false;
    if (ok && some) {
      tc_fence_after();
      const bool none = sum == 0.0f;  // (a NaN is not)
      const float factor = none ? 0.0f : 1.0f / sum;
      const int64_t head_at = (int64_t)b * p.heads + h;
      if (p.part_o) {
        const int64_t all = (int64_t)p.batch * p.heads * p.tq, query = head_at * p.tq + i;
        store_row<float, kD>(o_at, p.part_o + (split * all + query) * p.d, p.d, factor, in, taken > 0, none);
        if (in) p.part_less[split * all + query] = none ? INFINITY : -(ref + log2f(sum));
      } else {
        store_row<T, kD>(o_at, static_cast<T*>(p.o) + (((int64_t)b * p.tq + i) * p.heads + h) * p.d, p.d, factor, in, taken > 0, none);
        if (in && p.less) p.less[head_at * p.less_ld + i] = none ? -INFINITY : -(ref + log2f(sum));
      }
    }
  }
  attn_end(tmem);
}

// Joins the results of CTAs that shared the keys out: a warp a query and head.
template <typename T>
__global__ void __launch_bounds__(256) hc_attention_join_kernel(const float* part_o, const float* part_less, int splits, int64_t queries, int tq, int heads, int d, T* o, float* less,
                                                                int64_t less_ld) {
  const int lane = threadIdx.x & 31;
  const int64_t query = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (query >= queries) return;
  // minus a split's logarithm, +inf where it has seen nothing: the least of them is the reference
  float least = INFINITY;
  bool bad = false;
  for (int s = lane; s < splits; s += 32) {
    const float v = part_less[s * queries + query];
    least = fminf(least, v);
    bad = bad || v != v;
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, k));
  bad = __any_sync(0xffffffffu, bad);
  const bool none = least == INFINITY && !bad;
  float sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; !none && s < splits; ++s) {
    const float theirs = part_less[s * queries + query];
    const float weight = theirs == INFINITY ? 0.0f : exp2f(least - theirs);
    sum += weight;
    if (lane * 4 < d && theirs != INFINITY) {
      const float4 w = *reinterpret_cast<const float4*>(part_o + (s * queries + query) * d + lane * 4);
      v[0] += weight * w.x, v[1] += weight * w.y, v[2] += weight * w.z, v[3] += weight * w.w;
    }
  }
  const float factor = none ? 0.0f : 1.0f / sum;
  const int64_t head = query / tq, b = head / heads;
  const int i = (int)(query - head * tq);
  if (lane * 4 < d) {
    uint2 w = make_uint2(pack2<T>(v[0] * factor, v[1] * factor), pack2<T>(v[2] * factor, v[3] * factor));
    *reinterpret_cast<uint2*>(o + ((b * tq + i) * heads + head % heads) * d + lane * 4) = w;
  }
  if (less && lane == 0) less[head * less_ld + i] = none ? -INFINITY : bad ? least + __int_as_float(0x7fc00000) : least - log2f(sum);
}

// ---- backward ----------------------------------------------------------------------------------------------------------------
// delta = dO . O of every query and head; eight values a thread, so `kLanes` threads a query
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) hc_attention_delta_kernel(const T* dout, int64_t stride_b, int64_t stride_h, int64_t stride_t, const T* o, int batch, int heads, int tq, int d, float* delta,
                                                                 int64_t ld, unsigned int* most) {
  const int64_t total = (int64_t)batch * heads * tq;
  const int part = threadIdx.x % kLanes;
  unsigned int largest = 0;
  for (int64_t first = blockIdx.x * (256ll / kLanes); first < total; first += gridDim.x * (256ll / kLanes)) {
    const int64_t n = first + threadIdx.x / kLanes;  // as O lies: head after head of a query
    float dot = 0.0f, square = 0.0f;
    int64_t h = 0, b = 0;
    int i = 0;
    if (n < total) {
      h = n % heads;
      const int64_t r = n / heads;
      b = r / tq;
      i = (int)(r - b * tq);
      if (part * 8 < d) {
        float x[8], y[8];
        load8(dout + b * stride_b + h * stride_h + i * stride_t + part * 8, x);
        load8(o + n * d + part * 8, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dot = fmaf(x[j], y[j], dot);
          square = fmaf(x[j], x[j], square);
        }
      }
    }
#pragma unroll
    for (int k = kLanes / 2; k > 0; k >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, k);
      square += __shfl_xor_sync(0xffffffffu, square, k);
    }
    if (n < total && part == 0) delta[(b * heads + h) * ld + i] = dot;
    if (square < INFINITY) largest = max(largest, __float_as_uint(square));
  }
  if (!most) return;
  largest = __reduce_max_sync(0xffffffffu, largest);
  if ((threadIdx.x & 31) == 0 && largest) atomicMax(most, largest);
}
// the largest square of a norm of the rows of V
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) hc_attention_norm_kernel(const T* v, int64_t stride_b, int64_t stride_h, int64_t stride_t, int batch, int heads, int tk, int d, unsigned int* most) {
  const int64_t total = (int64_t)batch * heads * tk;
  const int part = threadIdx.x % kLanes;
  unsigned int largest = 0;
  for (int64_t first = blockIdx.x * (256ll / kLanes); first < total; first += gridDim.x * (256ll / kLanes)) {
    const int64_t n = first + threadIdx.x / kLanes;
    float square = 0.0f;
    if (n < total && part * 8 < d) {
      const int64_t h = n % heads, r = n / heads, b = r / tk;
      float x[8];
      load8(v + b * stride_b + h * stride_h + (r - b * tk) * stride_t + part * 8, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) square = fmaf(x[j], x[j], square);
    }
#pragma unroll
    for (int k = kLanes / 2; k > 0; k >>= 1) square += __shfl_xor_sync(0xffffffffu, square, k);
    if (square < INFINITY) largest = max(largest, __float_as_uint(square));
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  if ((threadIdx.x & 31) == 0 && largest) atomicMax(most, largest);
}
// The power of two that dS is held times in fp16: 2 max|dO_i| max|V_j|, which |dS| does not exceed, comes to below 2^15 (from the squares of both).
__device__ __forceinline__ float ds_power(const unsigned int* most, int sign) {
  const int e = (int)(most[0] >> 23) - 127 + (int)(most[1] >> 23) - 127 + 2;  // the product of the squares is below 2^e
  const int k = most[0] && most[1] ? min(max(13 - (e + 1) / 2, -100), 100) : 0;
  return __int_as_float((127 + sign * k) << 23);
}

// dK and dV of a tile of keys.  Tensor memory: scores (keys in lanes, queries in columns) at 0, dO V^T at 128, dV at 256, dK at 384.  The two halves of the warps have 64
// queries each, whose probabilities lie at the beginning of their own 64 columns.
template <typename T, int kD>
__global__ void __launch_bounds__(kAttnThreads, 1) hc_attention_dkv_kernel(const __grid_constant__ AttnParams p) {
  using S = AttnShape<kD>;
  constexpr int kQ = S::kQStages, kDo = S::kDoStages;
  constexpr float kBias = operand_format<T>() ? 0.0f : 14.0f;  // probabilities are held times 2^14 in fp16
  extern __shared__ unsigned char raw[];
  __shared__ AttnBarriers sh;
  unsigned char *k_tile = attn_tiles(raw), *v_tile = k_tile + S::kBytes, *q_ring = v_tile + S::kBytes, *do_ring = q_ring + kQ * S::kBytes;
  float* sides = reinterpret_cast<float*>(do_ring + kDo * S::kBytes);  // of a stage of queries: less, delta
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t at = blockIdx.x;
  const int head = (int)(at % p.kv_heads);
  at /= p.kv_heads;
  const int b = (int)(at % p.batch), block = (int)(at / p.batch);
  const int k0 = block * kTile, k1 = min(k0 + kTile, p.tk) - 1;
  // the queries that see one of them, in tiles
  const int i_first = max(k0 - p.off, 0), i_last = k0 < p.sinks ? p.tq - 1 : (int)min((int64_t)p.tq - 1, (int64_t)k1 + p.window - 1 - p.off);
  const int t_first = i_first / kTile, tiles = i_first <= i_last ? i_last / kTile - t_first + 1 : 0, count = tiles * p.group;
  attn_begin(sh, kAttnWarps);
  const uint32_t tmem = sh.tmem;
  if (warp == 0) {
    if (lane == 0 && count) {
      Ring<kQ> rq;
      Ring<kDo> rd;
      mbar_expect_tx(&sh.first, 2 * S::kBytes);
      load_tile<kD>(k_tile, &p.k, k0, head, b, &sh.first);
      load_tile<kD>(v_tile, &p.v, k0, head, b, &sh.first);
      for (int e = 0; e < count; ++e) {
        const int h = head * p.group + e / tiles, i0 = (t_first + e % tiles) * kTile;
        const int64_t side = ((int64_t)b * p.heads + h) * p.less_ld + i0;
        if (!attn_wait(&sh.empty[rq.s], rq.phase ^ 1, sh)) break;
        mbar_expect_tx(&sh.full[rq.s], S::kBytes + 1024);
        load_tile<kD>(q_ring + rq.s * S::kBytes, &p.q, i0, h, b, &sh.full[rq.s]);
        load_floats(sides + rq.s * 256, p.less + side, 512, &sh.full[rq.s]);
        load_floats(sides + rq.s * 256 + 128, p.delta + side, 512, &sh.full[rq.s]);
        rq.next();
        if (!attn_wait(&sh.more_empty[rd.s], rd.phase ^ 1, sh)) break;
        mbar_expect_tx(&sh.more_full[rd.s], S::kBytes);
        load_tile<kD>(do_ring + rd.s * S::kBytes, &p.dout, i0, h, b, &sh.more_full[rd.s]);
        rd.next();
      }
      ring_end(sh.full, rq);
      ring_end(sh.more_full, rd);
      mbar_wait_bounded(&sh.first, 0, kAttnLimitNs);
    }
  } else if (warp == 1) {
    if (lane == 0 && count) {
      Ring<kQ> rq;   // of the tile whose scores come next
      Ring<kDo> rd;
      const auto score = [&] {  // of the next tile of queries
        if (!attn_wait(&sh.full[rq.s], rq.phase, sh)) return false;
        tc_fence_after();
        scores<T, kD>(tmem, k_tile, q_ring + rq.s * S::kBytes);
        attn_commit(&sh.s_full[0]);
        return true;
      };
      const auto second = [&] {
        if (!attn_wait(&sh.more_full[rd.s], rd.phase, sh)) return false;
        tc_fence_after();
        scores<T, kD>(tmem + kTile, v_tile, do_ring + rd.s * S::kBytes);
        attn_commit(&sh.dp_full[0]);
        return true;
      };
      if (attn_wait(&sh.first, 0, sh) && score() && second()) {
        for (int e = 0; e < count; ++e) {
          const uint32_t turn = e & 1;
          const int sq = rq.s, sd = rd.s;
          if (!attn_wait(&sh.p_ready[0], turn, sh)) break;
          tc_fence_after();
          weighted<T, kD>(tmem + 256, tmem, 64, do_ring + sd * S::kBytes, e > 0);
          attn_commit(&sh.done[0]);
          attn_commit(&sh.more_empty[sd]);
          rq.next();
          rd.next();
          if (e + 1 < count && (!attn_wait(&sh.done[0], turn, sh) || !score())) break;
          if (!attn_wait(&sh.ds_ready[0], turn, sh)) break;
          tc_fence_after();
          weighted<T, kD>(tmem + 384, tmem + kTile, 64, q_ring + sq * S::kBytes, e > 0);
          attn_commit(&sh.done[1]);
          attn_commit(&sh.empty[sq]);
          if (e + 1 < count && (!attn_wait(&sh.done[1], turn, sh) || !second())) break;
        }
      }
      attn_commit(&sh.drained);
      mbar_wait_bounded(&sh.drained, 0, kAttnLimitNs);
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, j = k0 + quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lanes + half * 64, dp_at = lanes + kTile + half * 64;
    const float power = operand_format<T>() ? 1.0f : ds_power(p.most, 1), back = operand_format<T>() ? 1.0f : ds_power(p.most, -1);
    const float gain = operand_format<T>() ? 1.0f : power * (1.0f / 16384.0f);
    const Pair scale = pair(p.scale2, p.scale2), bias = pair(kBias, kBias);
    Ring<kQ> rq;
    bool ok = true;
    for (int e = 0; e < count; ++e) {
      const uint32_t turn = e & 1;
      const int i0 = (t_first + e % tiles) * kTile;
      const float* less = sides + rq.s * 256 + half * 64;
      if (!attn_wait_all(&sh.full[rq.s], rq.phase, sh) || !attn_wait_all(&sh.s_full[0], turn, sh)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float v[2][32];
      tc_load32(s_at, v[0]);
      tc_load32(s_at + 32, v[1]);
      tc_load_wait(v[0]);
      tc_load_wait(v[1]);
      const int pa = p.off + i0, pb = p.off + min(i0 + kTile, p.tq) - 1;
      const bool whole = all_seen(p, pa, pb, k0) && i0 + kTile <= p.tq;
      // the columns (queries) that see this row's key
      const int low = j - pa - half * 64;
      const int high = min(p.tq - i0, (int)min((int64_t)kTile, j < p.sinks ? (int64_t)kTile : (int64_t)j + p.window - pa)) - half * 64;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t words[16];
#pragma unroll
        for (int n = 0; n < 32; n += 4) {
          const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(less + c * 32 + n);
          Pair l0 = {l.x}, l1 = {l.y};
          if (!operand_format<T>()) {
            l0 = l0 + bias;
            l1 = l1 + bias;
          }
          parts(fma2(pair(v[c][n], v[c][n + 1]), scale, l0), v[c][n], v[c][n + 1]);
          parts(fma2(pair(v[c][n + 2], v[c][n + 3]), scale, l1), v[c][n + 2], v[c][n + 3]);
        }
#pragma unroll
        for (int n = 0; n < 32; ++n) v[c][n] = power2(v[c][n]);
        if (!whole) {
#pragma unroll
          for (int n = 0; n < 32; ++n)
            if (c * 32 + n < low || c * 32 + n >= high) v[c][n] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < 32; n += 2) words[n / 2] = pack2<T>(v[c][n], v[c][n + 1]);
        tc_store16(s_at + c * 16, words);
      }
      tc_store_wait();
      warp_arrives(&sh.p_ready[0]);
      if (!attn_wait_all(&sh.dp_full[0], turn, sh)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float g[32];
        __syncwarp();
        tc_load32(dp_at + c * 32, g);
        tc_load_wait(g);
        uint32_t words[16];
#pragma unroll
        for (int n = 0; n < 32; n += 4) {
          const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(less + 128 + c * 32 + n);
          const Pair minus = pair(-1.0f, -1.0f);
          Pair a = fma2(Pair{l.x}, minus, pair(g[n], g[n + 1])), w = fma2(Pair{l.y}, minus, pair(g[n + 2], g[n + 3]));
          Pair pa2 = pair(v[c][n], v[c][n + 1]), pb2 = pair(v[c][n + 2], v[c][n + 3]);
          if (!operand_format<T>()) {
            pa2 = pa2 * pair(gain, gain);
            pb2 = pb2 * pair(gain, gain);
          }
          parts(a * pa2, g[n], g[n + 1]);
          parts(w * pb2, g[n + 2], g[n + 3]);
        }
        if (!whole) {  // also where a query that does not see the key, or is none, has no number
#pragma unroll
          for (int n = 0; n < 32; ++n)
            if (c * 32 + n < low || c * 32 + n >= high) g[n] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < 32; n += 2) words[n / 2] = pack2<T>(g[n], g[n + 1]);
        tc_store16(dp_at + c * 16, words);
      }
      tc_store_wait();
      warp_arrives(&sh.ds_ready[0]);
      rq.next();
    }
    if (ok && count) ok = attn_wait_all(&sh.done[0], (count - 1) & 1, sh) && attn_wait_all(&sh.done[1], (count - 1) & 1, sh);
    if (ok) {
      tc_fence_after();
      // the first half of the warps stores dV, the second dK
      T* to = static_cast<T*>(half ? p.dk : p.dv) + (((int64_t)b * p.tk + j) * p.kv_heads + head) * p.d;
      const float factor = half ? p.scale * back : operand_format<T>() ? 1.0f : 1.0f / 16384.0f;
      store_row<T, kD>(lanes + 256 + half * kTile, to, p.d, factor, j < p.tk, count > 0, false);
    }
  }
  attn_end(tmem);
}

// dQ of a tile of queries.  Tensor memory: scores (queries in lanes) at 0, dO V^T at 128 and 256 in turn, dQ at 384.
template <typename T, int kD>
__global__ void __launch_bounds__(kAttnThreads, 1) hc_attention_dq_kernel(const __grid_constant__ AttnParams p) {
  using S = AttnShape<kD>;
  constexpr int kK = S::kKStages, kV = S::kVStages;
  extern __shared__ unsigned char raw[];
  __shared__ AttnBarriers sh;
  unsigned char *q_tile = attn_tiles(raw), *do_tile = q_tile + S::kBytes, *k_ring = do_tile + S::kBytes, *v_ring = k_ring + kK * S::kBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t at = blockIdx.x;
  const int head = (int)(at % p.heads);
  at /= p.heads;
  const int b = (int)(at % p.batch), block = p.blocks - 1 - (int)(at / p.batch);
  const int i0 = block * kTile, p0 = p.off + i0, p1 = p.off + min(i0 + kTile, p.tq) - 1;
  const KeyTiles list = key_tiles(p, p0, p1);
  const int count = list.count;
  attn_begin(sh, kAttnWarps);
  const uint32_t tmem = sh.tmem;
  if (warp == 0) {
    if (lane == 0 && count) {
      Ring<kK> rk;
      Ring<kV> rv;
      mbar_expect_tx(&sh.first, 2 * S::kBytes);
      load_tile<kD>(q_tile, &p.q, i0, head, b, &sh.first);
      load_tile<kD>(do_tile, &p.dout, i0, head, b, &sh.first);
      for (int e = 0; e < count; ++e) {
        const int k0 = list.at(e) * kTile;
        if (!attn_wait(&sh.empty[rk.s], rk.phase ^ 1, sh)) break;
        mbar_expect_tx(&sh.full[rk.s], S::kBytes);
        load_tile<kD>(k_ring + rk.s * S::kBytes, &p.k, k0, head / p.group, b, &sh.full[rk.s]);
        rk.next();
        if (!attn_wait(&sh.more_empty[rv.s], rv.phase ^ 1, sh)) break;
        mbar_expect_tx(&sh.more_full[rv.s], S::kBytes);
        load_tile<kD>(v_ring + rv.s * S::kBytes, &p.v, k0, head / p.group, b, &sh.more_full[rv.s]);
        rv.next();
      }
      ring_end(sh.full, rk);
      ring_end(sh.more_full, rv);
      mbar_wait_bounded(&sh.first, 0, kAttnLimitNs);
    }
  } else if (warp == 1) {
    if (lane == 0 && count) {
      Ring<kK> rk, used;  // of the tile whose scores come next; of the one whose dS comes next
      Ring<kV> rv;
      const auto score = [&](int e) {
        if (!attn_wait(&sh.full[rk.s], rk.phase, sh)) return false;
        if (e && !attn_wait(&sh.s_read, (e - 1) & 1, sh)) return false;
        tc_fence_after();
        scores<T, kD>(tmem, q_tile, k_ring + rk.s * S::kBytes);
        attn_commit(&sh.s_full[0]);
        rk.next();
        if (!attn_wait(&sh.more_full[rv.s], rv.phase, sh)) return false;
        if (e >= 2 && !attn_wait(&sh.done[e & 1], (e / 2 - 1) & 1, sh)) return false;
        tc_fence_after();
        scores<T, kD>(tmem + (1 + (e & 1)) * kTile, do_tile, v_ring + rv.s * S::kBytes);
        attn_commit(&sh.dp_full[e & 1]);
        attn_commit(&sh.more_empty[rv.s]);
        rv.next();
        return true;
      };
      if (attn_wait(&sh.first, 0, sh) && score(0)) {
        for (int e = 0; e < count; ++e) {
          if (e + 1 < count && !score(e + 1)) break;
          if (!attn_wait(&sh.ds_ready[e & 1], (e / 2) & 1, sh)) break;
          tc_fence_after();
          weighted<T, kD>(tmem + 384, tmem + (1 + (e & 1)) * kTile, 64, k_ring + used.s * S::kBytes, e > 0);
          attn_commit(&sh.done[e & 1]);
          attn_commit(&sh.empty[used.s]);
          used.next();
        }
      }
      attn_commit(&sh.drained);
      mbar_wait_bounded(&sh.drained, 0, kAttnLimitNs);
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, i = i0 + quarter * 32 + lane, position = p.off + i;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lanes + half * 64;
    const float power = operand_format<T>() ? 1.0f : ds_power(p.most, 1), back = operand_format<T>() ? 1.0f : ds_power(p.most, -1);
    const bool in = i < p.tq;
    const int64_t side = ((int64_t)b * p.heads + head) * p.less_ld + i;
    const float less = in ? p.less[side] : -INFINITY, delta = in ? p.delta[side] : 0.0f;
    const Pair scale = pair(p.scale2, p.scale2), less2 = pair(less, less), delta2 = pair(-delta, -delta), gain = pair(power, power);
    bool ok = true;
    for (int e = 0; e < count; ++e) {
      const int k0 = list.at(e) * kTile;
      if (!attn_wait_all(&sh.s_full[0], e & 1, sh)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float v[2][32];
      tc_load32(s_at, v[0]);
      tc_load32(s_at + 32, v[1]);
      tc_load_wait(v[0]);
      tc_load_wait(v[1]);
      warp_arrives(&sh.s_read);
      const bool whole = all_seen(p, p0, p1, k0);
      const int high = position - k0 - half * 64, low = position - p.window + 1 - k0 - half * 64, sinks = p.sinks - k0 - half * 64;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int n = 0; n < 32; n += 2) {
          float x, y;
          parts(fma2(pair(v[c][n], v[c][n + 1]), scale, less2), x, y);
          v[c][n] = power2(x);
          v[c][n + 1] = power2(y);
        }
      }
      if (!attn_wait_all(&sh.dp_full[e & 1], (e / 2) & 1, sh)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t dp_at = lanes + (1 + (e & 1)) * kTile + half * 64;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float g[32];
        __syncwarp();
        tc_load32(dp_at + c * 32, g);
        tc_load_wait(g);
        uint32_t words[16];
#pragma unroll
        for (int n = 0; n < 32; n += 2) {
          Pair a = (pair(g[n], g[n + 1]) + delta2) * pair(v[c][n], v[c][n + 1]);
          if (!operand_format<T>()) a = a * gain;
          parts(a, g[n], g[n + 1]);
        }
        if (!whole) {
#pragma unroll
          for (int n = 0; n < 32; ++n) {
            const int m = c * 32 + n;
            if (m > high || (m < low && m >= sinks)) g[n] = 0.0f;
          }
        }
#pragma unroll
        for (int n = 0; n < 32; n += 2) words[n / 2] = pack2<T>(g[n], g[n + 1]);
        tc_store16(dp_at + c * 16, words);
      }
      tc_store_wait();
      warp_arrives(&sh.ds_ready[e & 1]);
    }
    if (ok && count) ok = attn_wait_all(&sh.done[(count - 1) & 1], ((count - 1) / 2) & 1, sh);
    if (ok && !half) {
      tc_fence_after();
      T* to = static_cast<T*>(p.dq) + (((int64_t)b * p.tq + i) * p.heads + head) * p.d;
      store_row<T, kD>(lanes + 384, to, p.d, p.scale * back, in, count > 0, false);
    }
  }
  attn_end(tmem);
}

}  // namespace dev

namespace {

constexpr size_t kMostLength = (size_t)1 << 24, kMostHeads = (size_t)1 << 15;
constexpr int kNoWindow = 1 << 28;

struct Sizes {
  size_t batch, heads, kv_heads, queries, keys, d;
};
bool sizes_ok(const Sizes& s) {
  return s.d >= 8 && s.d <= 128 && s.d % 8 == 0 && s.queries < kMostLength && s.keys < kMostLength && s.kv_heads > 0 && s.heads < kMostHeads && s.heads >= s.kv_heads &&
         s.heads % s.kv_heads == 0 && s.batch < ((size_t)1 << 24) && s.batch * s.heads < ((size_t)1 << 24) && s.batch * s.heads * ((s.queries + 127) / 128 + (s.keys + 127) / 128) < ((size_t)1 << 30);
}
size_t up(size_t v, size_t unit) { return (v + unit - 1) / unit * unit; }

// rows of a head of `length` positions: boxes of 64 values of `rows` positions of `heads` heads
bool make_head_map(CUtensorMap* map, int type, const hc_heads& t, size_t d, size_t length, size_t heads, size_t batch, int rows, int box_heads) {
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)length, (cuuint64_t)heads, (cuuint64_t)batch};
  // the distance of the only one of its kind is of no account
  cuuint64_t strides[3] = {(cuuint64_t)(length > 1 ? t.position : d) * 2, (cuuint64_t)(heads > 1 ? t.head : d) * 2, (cuuint64_t)(batch > 1 ? t.batch : d) * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)rows, (cuuint32_t)box_heads, 1};
  cuuint32_t step[4] = {1, 1, 1, 1};
  return encode_tiled(map, type == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(t.data), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}
bool heads_ok(const hc_heads& t, size_t d, size_t length, size_t heads, size_t batch) {
  const auto ok = [&](size_t stride, size_t n) { return n <= 1 || (stride >= d && stride % 8 == 0 && stride < ((size_t)1 << 38)); };
  return t.data && (reinterpret_cast<uintptr_t>(t.data) & 15u) == 0 && ok(t.position, length) && ok(t.head, heads) && ok(t.batch, batch);
}

int64_t attn_sms() { return device_info().sms > 0 ? device_info().sms : 1; }

// Into how many CTAs the keys of a tile of queries are shared out, where there are fewer of those than SMs: a CTA costs some three tiles besides its own, joining a part one.
struct Plan {
  int packed, blocks, splits;
};
Plan plan_of(const Sizes& s, size_t window, size_t sinks) {
  Plan p;
  const size_t group = s.heads / s.kv_heads;
  p.packed = s.queries * group <= 128 ? (int)(s.queries * group) : 0;
  p.blocks = p.packed ? 1 : (int)((s.queries + 255) / 256);
  const int64_t ctas = (int64_t)s.batch * (p.packed ? s.kv_heads : s.heads) * p.blocks, sms = attn_sms();
  const size_t seen = window ? (window + sinks + s.queries < s.keys ? window + sinks + s.queries : s.keys) : s.keys;
  const int64_t tiles = (int64_t)(seen + 127) / 128;
  p.splits = 1;
  int64_t least = (ctas + sms - 1) / sms * (tiles + 3);
  for (int n = 2; n <= 64 && n <= tiles && ctas < sms * 2; ++n) {
    const int64_t cost = (ctas * n + sms - 1) / sms * ((tiles + n - 1) / n + 3) + 1 + n / 16;
    if (cost < least) {
      least = cost;
      p.splits = n;
    }
  }
  return p;
}

size_t stats_ld(size_t queries) { return up(queries, 128); }

void fill_attention(dev::AttnParams* p, const Sizes& s, size_t window, size_t sinks, float scale) {
  memset(p, 0, sizeof(*p));
  p->batch = (int)s.batch, p->heads = (int)s.heads, p->kv_heads = (int)s.kv_heads, p->group = (int)(s.heads / s.kv_heads);
  p->tq = (int)s.queries, p->tk = (int)s.keys, p->d = (int)s.d, p->off = (int)s.keys - (int)s.queries;
  p->window = window && window < (size_t)kNoWindow ? (int)window : kNoWindow;
  p->sinks = (int)(sinks < s.keys ? sinks : s.keys);
  p->scale = scale;
  p->scale2 = scale * 1.4426950408889634f;
  p->less_ld = (int64_t)stats_ld(s.queries);
}

template <typename T, int kD>
cudaError_t run_forward(const dev::AttnParams& p, const Plan& plan, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  constexpr int smem = dev::AttnShape<kD>::kForwardSmem;
  cudaError_t e = allow_smem(dev::hc_attention_kernel<T, kD>, smem, &allowed);
  if (e != cudaSuccess) return e;
  const int64_t ctas = (int64_t)p.batch * (p.packed ? p.kv_heads : p.heads) * p.blocks * p.splits;
  dev::hc_attention_kernel<T, kD><<<(unsigned)ctas, dev::kAttnThreads, smem, stream>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || plan.splits == 1) return e;
  const int64_t queries = (int64_t)p.batch * p.heads * p.tq;
  dev::hc_attention_join_kernel<T><<<(unsigned)((queries + 7) / 8), 256, 0, stream>>>(p.part_o, p.part_less, p.splits, queries, p.tq, p.heads, p.d, static_cast<T*>(p.o), p.less, p.less_ld);
  return cudaGetLastError();
}

template <typename T, int kD>
cudaError_t run_backward(dev::AttnParams& p, const hc_heads& dout, const hc_heads& v, const void* o, float* delta, unsigned int* most, cudaStream_t stream) {
  static unsigned long long allowed_kv = 0, allowed_q = 0;
  using S = dev::AttnShape<kD>;
  cudaError_t e = allow_smem(dev::hc_attention_dkv_kernel<T, kD>, S::kKvSmem, &allowed_kv);
  if (e == cudaSuccess) e = allow_smem(dev::hc_attention_dq_kernel<T, kD>, S::kQSmem, &allowed_q);
  if (e != cudaSuccess) return e;
  constexpr int kLanes = kD / 8;
  const int64_t most_blocks = attn_sms() * 8;
  const auto blocks_for = [&](int64_t rows) { return (unsigned)((rows + 256 / kLanes - 1) / (256 / kLanes) < most_blocks ? (rows + 256 / kLanes - 1) / (256 / kLanes) : most_blocks); };
  dev::hc_attention_delta_kernel<T, kLanes><<<blocks_for((int64_t)p.batch * p.heads * p.tq), 256, 0, stream>>>(
      static_cast<const T*>(dout.data), (int64_t)dout.batch, (int64_t)dout.head, (int64_t)dout.position, static_cast<const T*>(o), p.batch, p.heads, p.tq, p.d, delta, p.less_ld, most);
  if (most)
    dev::hc_attention_norm_kernel<T, kLanes><<<blocks_for((int64_t)p.batch * p.kv_heads * p.tk), 256, 0, stream>>>(
        static_cast<const T*>(v.data), (int64_t)v.batch, (int64_t)v.head, (int64_t)v.position, p.batch, p.kv_heads, p.tk, p.d, most + 1);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (p.dk) {
    p.blocks = (p.tk + dev::kTile - 1) / dev::kTile;
    dev::hc_attention_dkv_kernel<T, kD><<<(unsigned)((int64_t)p.batch * p.kv_heads * p.blocks), dev::kAttnThreads, S::kKvSmem, stream>>>(p);
  }
  if (p.dq) {
    p.blocks = (p.tq + dev::kTile - 1) / dev::kTile;
    dev::hc_attention_dq_kernel<T, kD><<<(unsigned)((int64_t)p.batch * p.heads * p.blocks), dev::kAttnThreads, S::kQSmem, stream>>>(p);
  }
  return cudaGetLastError();
}

size_t forward_bytes(const Sizes& s, size_t window, size_t sinks) {
  const Plan plan = plan_of(s, window, sinks);
  const size_t rows = s.batch * s.heads * s.queries;
  return plan.splits > 1 ? up(rows * plan.splits * s.d * sizeof(float), 256) + up(rows * plan.splits * sizeof(float), 256) : 0;
}
size_t backward_bytes(const Sizes& s) { return up(s.batch * s.heads * stats_ld(s.queries) * sizeof(float), 256) + 256; }

}  // namespace

int attention_status(int clear) { return take_status(dev::g_attention_status, clear); }

}  // namespace hc

extern "C" {

size_t hc_attention_stats(size_t batch, size_t heads, size_t queries) { return batch * heads * hc::stats_ld(queries); }

size_t hc_attention_bytes(size_t batch, size_t heads, size_t kv_heads, size_t queries, size_t keys, size_t head_size, size_t window, size_t sinks) {
  const hc::Sizes s = {batch, heads, kv_heads, queries, keys, head_size};
  return hc::sizes_ok(s) && batch && queries && keys ? hc::forward_bytes(s, window, sinks) : 0;
}

int hc_attention(hc_heads q, hc_heads k, hc_heads v, int type, void* out, float* stats, size_t batch, size_t heads, size_t kv_heads, size_t queries, size_t keys, size_t head_size,
                 size_t window, size_t sinks, float scale, void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  const Sizes s = {batch, heads, kv_heads, queries, keys, head_size};
  if ((type != kBf16 && type != kF16) || !sizes_ok(s) || !(scale > 0.0f) || !(scale < INFINITY) || !lies_at(out, 16) || !lies_at(stats, 16)) return kErrArgument;
  if (batch == 0 || queries == 0) return kOk;
  if (!out) return kErrArgument;
  if (keys == 0) {
    // nobody sees anything; the backward pass of such a call reads no statistics
    return cudaMemsetAsync(out, 0, batch * queries * heads * head_size * 2, stream) == cudaSuccess ? kOk : kErrCuda;
  }
  if (!heads_ok(q, head_size, queries, heads, batch) || !heads_ok(k, head_size, keys, kv_heads, batch) || !heads_ok(v, head_size, keys, kv_heads, batch)) return kErrArgument;
  const Plan plan = plan_of(s, window, sinks);
  const size_t need = forward_bytes(s, window, sinks), rows = batch * heads * queries;
  if (need && (!scratch || !lies_at(scratch, 256) || scratch_bytes < need)) return kErrArgument;
  dev::AttnParams p;
  fill_attention(&p, s, window, sinks, scale);
  p.packed = plan.packed;
  p.blocks = plan.blocks;
  p.splits = plan.splits;
  p.o = out;
  p.less = stats;
  if (plan.splits > 1) {
    p.part_o = static_cast<float*>(scratch);
    p.part_less = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + up(rows * plan.splits * head_size * sizeof(float), 256));
  }
  if (!make_head_map(&p.q, type, q, head_size, queries, heads, batch, plan.packed ? (int)queries : dev::kTile, plan.packed ? p.group : 1) ||
      !make_head_map(&p.k, type, k, head_size, keys, kv_heads, batch, dev::kTile, 1) || !make_head_map(&p.v, type, v, head_size, keys, kv_heads, batch, dev::kTile, 1))
    return kErrArgument;
  cudaError_t e;
  if (type == kBf16) e = head_size <= 64 ? run_forward<__nv_bfloat16, 64>(p, plan, stream) : run_forward<__nv_bfloat16, 128>(p, plan, stream);
  else e = head_size <= 64 ? run_forward<__half, 64>(p, plan, stream) : run_forward<__half, 128>(p, plan, stream);
  return e == cudaSuccess ? kOk : kErrCuda;
}

size_t hc_attention_backward_bytes(size_t batch, size_t heads, size_t kv_heads, size_t queries, size_t keys, size_t head_size) {
  const hc::Sizes s = {batch, heads, kv_heads, queries, keys, head_size};
  return hc::sizes_ok(s) && batch && queries && keys ? hc::backward_bytes(s) : 0;
}

int hc_attention_backward(hc_heads dout, const void* out, hc_heads q, hc_heads k, hc_heads v, int type, const float* stats, void* dq, void* dk, void* dv, size_t batch, size_t heads,
                          size_t kv_heads, size_t queries, size_t keys, size_t head_size, size_t window, size_t sinks, float scale, void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  const Sizes s = {batch, heads, kv_heads, queries, keys, head_size};
  if ((type != kBf16 && type != kF16) || !sizes_ok(s) || !(scale > 0.0f) || !(scale < INFINITY) || (!dk != !dv)) return kErrArgument;
  if (!lies_at(out, 16) || !lies_at(stats, 16) || !lies_at(dq, 16) || !lies_at(dk, 16) || !lies_at(dv, 16)) return kErrArgument;
  if (batch == 0 || (!dq && !dk)) return kOk;
  if (queries == 0 || keys == 0) {
    cudaError_t e = cudaSuccess;
    if (dq && queries) e = cudaMemsetAsync(dq, 0, batch * queries * heads * head_size * 2, stream);
    if (e == cudaSuccess && dk && keys) e = cudaMemsetAsync(dk, 0, batch * keys * kv_heads * head_size * 2, stream);
    if (e == cudaSuccess && dv && keys) e = cudaMemsetAsync(dv, 0, batch * keys * kv_heads * head_size * 2, stream);
    return e == cudaSuccess ? kOk : kErrCuda;
  }
  if (!out || !stats || !heads_ok(dout, head_size, queries, heads, batch) || !heads_ok(q, head_size, queries, heads, batch) || !heads_ok(k, head_size, keys, kv_heads, batch) ||
      !heads_ok(v, head_size, keys, kv_heads, batch))
    return kErrArgument;
  const size_t need = backward_bytes(s);
  if (!scratch || !lies_at(scratch, 256) || scratch_bytes < need) return kErrArgument;
  dev::AttnParams p;
  fill_attention(&p, s, window, sinks, scale);
  float* delta = static_cast<float*>(scratch);
  unsigned int* most = type == kF16 ? reinterpret_cast<unsigned int*>(static_cast<unsigned char*>(scratch) + need - 256) : nullptr;
  if (most && cudaMemsetAsync(most, 0, 8, stream) != cudaSuccess) return kErrCuda;
  p.less = const_cast<float*>(stats);
  p.delta = delta;
  p.most = most;
  p.dq = dq, p.dk = dk, p.dv = dv;
  if (!make_head_map(&p.q, type, q, head_size, queries, heads, batch, dev::kTile, 1) || !make_head_map(&p.dout, type, dout, head_size, queries, heads, batch, dev::kTile, 1) ||
      !make_head_map(&p.k, type, k, head_size, keys, kv_heads, batch, dev::kTile, 1) || !make_head_map(&p.v, type, v, head_size, keys, kv_heads, batch, dev::kTile, 1))
    return kErrArgument;
  cudaError_t e;
  if (type == kBf16) e = head_size <= 64 ? run_backward<__nv_bfloat16, 64>(p, dout, v, out, delta, most, stream) : run_backward<__nv_bfloat16, 128>(p, dout, v, out, delta, most, stream);
  else e = head_size <= 64 ? run_backward<__half, 64>(p, dout, v, out, delta, most, stream) : run_backward<__half, 128>(p, dout, v, out, delta, most, stream);
  return e == cudaSuccess ? kOk : kErrCuda;
}

}  // extern "C"
