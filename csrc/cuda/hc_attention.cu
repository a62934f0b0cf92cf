// Causal attention with a sliding window and first tokens that stay visible, and its backward pass, on tcgen05 tensor cores.
//
//   query i stands at position p = i + Tk - Tq and sees key j if j <= p and (p - j < window or j < sinks)
//   S = scale Q K^T,  P = softmax of S over what is seen,  O = P V                (a query that sees nothing: 0)
//   delta_i = dO_i . O_i,  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Tiles of 128 rows, steps of 64 of the other side; steps that nobody sees are left out, only steps at an edge of what is seen are masked.  One thread brings
// operands in by TMA, two warps issue the matrix instructions, eight or sixteen have a row of a tile a thread: scores, probabilities and their
// gradients go from tensor memory to registers and back and never anywhere else.  The second product of each pair reads its first operand, in 16 bits, from where the
// scores lay.  Heads and batch are dimensions of the tensor maps, so a view into a projection's result is read where it lies; several query heads to a key's head read the
// same keys, and dK and dV of such a head are summed in one CTA.  Every sum has a fixed order.
//
// Forward: two tiles of queries share their keys, so that the tensor cores work on one while the other's exponentials are taken, which bound it up to heads of
// 64 (16 a cycle and SM).  The reference that exponentials are taken relative to follows a row's largest score when that is more than 2^8 above it; only then is O
// taken times a factor.  Few queries (with all heads of a key's head at most 128 rows; up to 8 have a kernel of their own) are one tile, and the keys are shared
// out to the CTAs of a cluster, which join their results over its shared memory: bound by reading keys and values.
// Backward: dK and dV in a kernel whose CTA has a tile of keys and goes through the queries, dQ in one whose CTA has a tile of queries.  That forms the scores twice (8 products instead of 5, P K below among them), and
// needs no atomic additions, whose order would change the result, and no array of partial dQ.
//
// In fp16, which has no numbers below 2^-24, P is held times 2^6 in the forward pass (its reference may be 2^8 below a row's largest), times 2^14 for few rows and in the keys' pass, and as it is in the
// queries' pass, where P K needs no more than a few bits; dS times a power that 2 max|dO_i| max|V_j| (norms of rows, which bound it) gives, over the queries and keys of a sequence's key head: what else
// is in the batch has no part in it.
#include <math.h>

#include <type_traits>

#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_tensor.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kTile = 128;  // rows of a tile, one a thread
constexpr int kStep = 64;   // columns that are worked on at a time
constexpr int kMostSplits = 8;  // CTAs of a cluster
constexpr uint64_t kAttnLimitNs = 2000ull * 1000 * 1000;
constexpr float kSlack = 8.0f;  // powers of two that a score may be above its row's reference

__device__ unsigned int g_attention_status;

template <int kD>
struct AttnShape {
  static constexpr int kBoxes = kD / 64;          // of 64 values, 128 bytes
  static constexpr int kBytes = kTile * kD * 2;   // of a tile
  static constexpr int kStepBytes = kStep * kD * 2;
  // Heads of up to 64 values: two CTAs an SM, with half of the tensor memory each.
  static constexpr int kResident = kD == 128 ? 1 : 2;
  static constexpr int kColumns = 512 / kResident;
  // Registers a thread that share_registers counts on, or 0 where it is not used; a kernel that was built with fewer is not launched.
  static constexpr int kForwardRegisters = kResident == 2 ? 80 : 0, kBackwardRegisters = kResident == 2 ? 80 : 96;
  static constexpr int kSlots = kD == 128 ? 2 : 1;  // forward: steps of scores of a tile
  static constexpr int kForwardStages = kD == 128 ? 10 : 8;  // steps, half of them of keys and half of values
  static constexpr int kForwardSmem = 2 * kBytes + kForwardStages * kStepBytes + 1024;
  static constexpr int kForwardThreads = 32 * (4 + 8);
  static constexpr int kGroups = kD == 128 ? 2 : 1;  // backward: of eight warps, which take the steps in turn
  static constexpr int kStages = 4;                  // backward: a step of both streams, and what belongs to its queries
  static constexpr int kBackwardSmem = 2 * kBytes + kStages * (2 * kStepBytes + 512) + 1024;
  static constexpr int kBackwardThreads = 32 * (4 + 8 * kGroups);
};

struct AttnParams {
  CUtensorMap q, k, v, dout;                          // in steps of 64 positions (forward, q: tiles)
  CUtensorMap q_tile, k_tile, v_tile, dout_tile;  // in tiles of 128 (backward)
  void* o;       // the result (backward: read)
  float* less;      // [batch heads][rows]: minus the logarithm (base 2) of a query's sum of exponentials, for the backward pass
  float* delta;  // as `less`
  void *dq, *dk, *dv;
  const unsigned int* most;  // [batch][key heads]: bits of the squares of max|dO_i|, max|V_j| (fp16)
  int64_t less_ld;
  int batch, heads, kv_heads, group, tq, tk, d, off, window, sinks;
  int packed;   // rows of the one tile that holds the queries of all heads of a key's head, or 0
  int blocks;   // of queries, or of keys
  int splits;   // CTAs of a cluster that share the keys (forward) or the heads (dK and dV) of a tile
  float scale, scale2;  // scale2: times log2(e)
};

struct AttnBarriers {
  uint64_t full[16], empty[16], first, drained, met, dots;
  uint64_t s_full[4], p_ready[4], done[4], dp_full[2], ds_ready[2], ds_done[2];
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

// A place in a ring of N stages, or of the first of them
template <int N>
struct Ring {
  int s = 0, count = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages = N) {
    ++count;
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
};
// what a ring's last loads bring is there before the CTA leaves
template <int N>
__device__ __forceinline__ void ring_end(uint64_t* full, const Ring<N>& r, int stages = N) {
  for (int back = 0; back < stages && back < r.count; ++back) {
    const int i = r.count - 1 - back;
    mbar_wait_bounded(&full[i % stages], (i / stages) & 1, kAttnLimitNs);
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
// kRows rows from t on
template <int kD, int kRows>
__device__ __forceinline__ void load_rows(unsigned char* dst, const CUtensorMap* map, int t, int h, int b, uint64_t* bar) {
#pragma unroll
  for (int i = 0; i < AttnShape<kD>::kBoxes; ++i) load_4d(dst + i * kRows * 128, map, i * 64, t, h, b, bar);
}

// The matrix instructions' warp runs as a whole, so that the compiler keeps descriptors and addresses in uniform registers, which these instructions take them from, and one
// lane of it issues.  With one lane in all of its code an instruction cost 130 to 290 cycles, several times what the tensor cores take for it.
__device__ __forceinline__ bool elected() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ void attn_commit(bool leader, uint64_t* bar) {
  if (leader) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void attn_mma(bool leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if (leader)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// the first operand in tensor memory: rows in lanes, two values of the sum in a column
__device__ __forceinline__ void attn_mma_from_tmem(bool leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  if (leader)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// Descriptors of a tile or a step, 128-byte swizzle.  Along: the sum runs along its rows of 128 bytes (eight rows are 1024 bytes).  Across: the sum runs
// over its rows, 64 values across it are a box.
__device__ __forceinline__ uint64_t along(const unsigned char* tile) {
  return (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 / 16) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ uint64_t across(const unsigned char* step) {
  return (uint64_t)((smem_u32(step) & 0x3ffff) >> 4) | (uint64_t)(kStep * 128 / 16) << 16 | (uint64_t)(1024 / 16) << 32 | 1ull << 46 | 2ull << 61;
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t operand_format() {
  return sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
}
template <typename T>
__device__ __forceinline__ uint32_t attn_idesc(int n, bool b_across) {
  return 1u << 4 | operand_format<T>() << 7 | operand_format<T>() << 10 | (b_across ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(kTile / 16) << 24;
}
// d = a b^T over the head's values, of a tile and a step (their descriptors along the sum)
template <typename T, int kD>
__device__ __forceinline__ void scores(bool leader, uint32_t d, uint64_t a, uint64_t b) {
  const uint32_t idesc = attn_idesc<T>(kStep, false);
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) attn_mma(leader, d, a + (i / 4) * (kTile * 128 / 16) + (i % 4) * 2, b + (i / 4) * (kStep * 128 / 16) + (i % 4) * 2, idesc, i > 0);
}
// d (+)= p b, p in tensor memory, its second 32 values of the sum `second` columns behind the first, b a step (its descriptor across the sum)
template <typename T, int kD>
__device__ __forceinline__ void weighted(bool leader, uint32_t d, uint32_t p, int second, uint64_t b, bool add) {
  const uint32_t idesc = attn_idesc<T>(kD, true);
#pragma unroll
  for (int i = 0; i < kStep / 16; ++i) attn_mma_from_tmem(leader, d, p + i / 2 * second + i % 2 * 8, b + i * 128, idesc, add || i > 0);
}

// Registers that the warps with roles, the first four, leave to those with rows.  Together they are no more than the CTA was launched with, or the others would wait for ever.
constexpr int kRoleRegisters = 48;
template <int kRegisters, int kThreads, int kLaunched>
__device__ __forceinline__ void share_registers(bool role) {
  static_assert(128 * kRoleRegisters + (kThreads - 128) * kRegisters <= kThreads * kLaunched, "what the CTA has");
  if (role) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegisters));
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}

// ---- clusters -----------------------------------------------------------------------------------------------------------------
// All threads of all CTAs of a cluster come to both of these, in any case; `all`: the cluster's size.  The instructions want whole warps, which rows and columns shared out by thread may have split.
__device__ __forceinline__ void cluster_meet(int all) {
  __syncwarp();
  if (all > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 peer_load4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float peer_load(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// ---- what is seen ------------------------------------------------------------------------------------------------------------
// the steps of keys that positions p0 to p1 see: those of the first tokens, then a stretch
struct KeySteps {
  int sinks, low, count;
  __device__ __forceinline__ int at(int e) const { return (e < sinks ? e : low + e - sinks) * kStep; }
};
__device__ __forceinline__ KeySteps key_steps(const AttnParams& p, int p0, int p1) {
  KeySteps t = {0, 0, 0};
  if (p1 < 0) return t;
  const int lowest = p0 - p.window + 1;
  t.low = lowest > 0 ? lowest / kStep : 0;
  t.sinks = min((min(p.sinks, p1 + 1) + kStep - 1) / kStep, t.low);
  t.count = t.sinks + p1 / kStep - t.low + 1;
  return t;
}
// Which of a list's steps positions p0 to p1, some of those that it was made for, see something of: those below `first`, and from `from` up to below `to`.
struct StepsSeen {
  int first, from, to;
  __device__ __forceinline__ bool has(int e) const { return e < first || (e >= from && e < to); }
};
__device__ __forceinline__ StepsSeen steps_seen(const AttnParams& p, const KeySteps& list, int p0, int p1) {
  if (p1 < 0) return {0, 0, 0};
  const int shift = list.sinks - list.low, lowest = p0 - p.window + 1;
  StepsSeen s;
  s.to = p1 / kStep + shift + 1;
  s.from = (lowest > 0 ? lowest / kStep : 0) + shift;
  s.first = min(max(list.sinks, (p.sinks + kStep - 1) / kStep + shift), s.to);
  return s;
}
// of `keys` keys from k0 on
__device__ __forceinline__ bool all_seen(const AttnParams& p, int p0, int p1, int k0, int keys) { return k0 + keys - 1 <= p0 && (p1 - k0 < p.window || k0 + keys <= p.sinks); }

// of the 32 columns from `at` on those from `low` up to below `high`, and those below `sinks`, as bits
__device__ __forceinline__ uint32_t ones_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen_bits(int low, int high, int sinks, int at) { return ones_below(high - at) & (~ones_below(low - at) | ones_below(sinks - at)); }

// barriers and tensor memory; by all threads.  `rows`: warps that work on a step, `released`: roles that have to be done with a stage.
// `loads`: by thread 0 as soon as the barriers are there, so that the first copies are on their way meanwhile.
template <int kColumns, typename F>
__device__ __forceinline__ void attn_begin(AttnBarriers& sh, int warps, int rows, int released, F loads) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 16; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], released);
    }
    mbar_init(&sh.first, 1);
    mbar_init(&sh.drained, 2);
    mbar_init(&sh.met, warps);
    mbar_init(&sh.dots, warps);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_ready[i], rows);
      mbar_init(&sh.done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.dp_full[i], 1);
      mbar_init(&sh.ds_ready[i], rows);
      mbar_init(&sh.ds_done[i], 1);
    }
    sh.gave_up = 0;
    fence_mbar_init();
    loads();
  }
  if (threadIdx.x >> 5 == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
template <int kColumns>
__device__ __forceinline__ void attn_end(uint32_t tmem) {
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x >> 5 == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kColumns));
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

// kCount of a row's values, `factor` times what tensor memory has, from `to` on; `d`: how many the row has from there.  `there`, the same for all of a warp: tensor memory has them; `none`: zeros.
template <typename O, int kCount>
__device__ __forceinline__ void store_row(uint32_t from, O* to, int d, float factor, bool in, bool there, bool none) {
#pragma unroll 1
  for (int c = 0; c < kCount; c += 32) {
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
// the largest of three, which is one instruction
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two tiles of queries, with four warps and a warp that issues their matrix instructions each.  Tensor memory: one or two steps of scores of each tile (the probabilities in their first 32
// columns), then O of both.  With two steps the next one's scores are formed while a step is worked on; heads of up to 64 values have one, and two CTAs on an SM.
template <typename T, int kD>
__global__ void __launch_bounds__(AttnShape<kD>::kForwardThreads, AttnShape<kD>::kResident) hc_attention_kernel(const __grid_constant__ AttnParams p) {
  using S = AttnShape<kD>;
  constexpr int kStages = S::kForwardStages, kSlots = S::kSlots, kO = 2 * kSlots * kStep;
  constexpr float kBias = operand_format<T>() ? 0.0f : 6.0f;  // probabilities are held times 2^6 in fp16: at most 2^14
  extern __shared__ unsigned char raw[];
  __shared__ AttnBarriers sh;
  unsigned char* tiles = attn_tiles(raw);
  unsigned char* ring = tiles + 2 * S::kBytes;
  // what the CTAs of a cluster join lies where the operands were
  constexpr int kRow = kD + 4;  // floats from row to row, so that neighbours' pieces do not meet in a bank
  static_assert(2 * kTile * (kRow + 1) * 4 <= S::kForwardSmem - 1024, "room for the parts");
  float *joined = reinterpret_cast<float*>(tiles), *part_less = joined + 2 * kTile * kRow;
  const bool shared = p.packed || p.splits > 1;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
    p0[q] = p.packed ? p.off : p.off + i0;
    p1[q] = p.packed ? p.off + p.tq - 1 : i0 <= i1 ? p.off + i1 : -1;
  }
  const KeySteps list = key_steps(p, p0[0], max(p1[0], p1[1]));
  const int e0 = (int)((int64_t)list.count * split / p.splits), e1 = (int)((int64_t)list.count * (split + 1) / p.splits);
  // One tile of queries is worked on twice, with every second step of the keys each.
  attn_begin<S::kColumns>(sh, 8, 4, p.packed ? 1 : 2, [&] {
    if (e0 >= e1) return;
    const bool second = !p.packed && first + kTile < p.tq;
    if (p.packed) {
      mbar_expect_tx(&sh.first, p.packed * 128 * S::kBoxes);
      for (int i = 0; i < S::kBoxes; ++i) load_4d(tiles + i * kTile * 128, &p.q, i * 64, 0, head * p.group, b, &sh.first);
    } else {
      mbar_expect_tx(&sh.first, second ? 2 * S::kBytes : S::kBytes);
      load_rows<kD, kTile>(tiles, &p.q, first, head, b, &sh.first);
      if (second) load_rows<kD, kTile>(tiles + S::kBytes, &p.q, first + kTile, head, b, &sh.first);
    }
  });
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  if constexpr (S::kResident == 2) share_registers<96, S::kForwardThreads, S::kForwardRegisters>(warp < 4);
  constexpr int kRing = kStages / 2;  // of keys; behind it that of values
  unsigned char* v_ring = ring + kRing * S::kStepBytes;
  // Groups that take the steps in turn need an even number of stages, so that a stage is always of the same group: one that does not wait for each of a barrier's phases cannot tell them apart.
  const int stages = p.packed ? kRing / 2 * 2 : kRing;
  if (warp == 0) {
    if (lane == 0 && e0 < e1) {
      Ring<kRing> rk, rv;
      for (int e = e0; e < e1; ++e) {
        const int k0 = list.at(e);
        if (!attn_wait(&sh.empty[rk.s], rk.phase ^ 1, sh)) break;
        mbar_expect_tx(&sh.full[rk.s], S::kStepBytes);
        load_rows<kD, kStep>(ring + rk.s * S::kStepBytes, &p.k, k0, kv_head, b, &sh.full[rk.s]);
        rk.next(stages);
        if (!attn_wait(&sh.empty[8 + rv.s], rv.phase ^ 1, sh)) break;
        mbar_expect_tx(&sh.full[8 + rv.s], S::kStepBytes);
        load_rows<kD, kStep>(v_ring + rv.s * S::kStepBytes, &p.v, k0, kv_head, b, &sh.full[8 + rv.s]);
        rv.next(stages);
      }
      ring_end(sh.full, rk, stages);
      ring_end(sh.full + 8, rv, stages);
      mbar_wait_bounded(&sh.first, 0, kAttnLimitNs);
    }
  } else if (warp <= 2) {
    if (e0 < e1) {
      const int q = warp - 1, by = p.packed ? 2 : 1;
      const bool leader = elected();
      const StepsSeen seen = p.packed ? StepsSeen{e1, 0, 0} : steps_seen(p, list, p0[q], p1[q]);
      const uint64_t q_at = along(tiles + (p.packed ? 0 : q * S::kBytes)), k_at = along(ring), v_at = across(v_ring);
      constexpr int kUnits = S::kStepBytes / 16;
      int scored = 0, summed = 0;
      Ring<kRing> rk, rv;
      const int start = p.packed ? e0 + ((e0 ^ q) & 1) : e0;  // its first step
      if (start != e0) {
        rk.next(stages);
        rv.next(stages);
      }
      const auto score = [&](int e) {
        if (!attn_wait_all(&sh.full[rk.s], rk.phase, sh)) return false;
        if (seen.has(e)) {
          const int n = scored++, slot = q * kSlots + n % kSlots;
          if (n >= kSlots && !attn_wait_all(&sh.done[slot], (n / kSlots - 1) & 1, sh)) return false;  // the probabilities that lie there have been read
          tc_fence_after();
          scores<T, kD>(leader, tmem + slot * kStep, q_at, k_at + rk.s * kUnits);
          attn_commit(leader, &sh.s_full[slot]);
        }
        attn_commit(leader, &sh.empty[rk.s]);
        rk.next(stages);
        if (by == 2) rk.next(stages);
        return true;
      };
      const auto sum = [&](int e) {
        if (!attn_wait_all(&sh.full[8 + rv.s], rv.phase, sh)) return false;
        if (seen.has(e)) {
          const int n = summed++, slot = q * kSlots + n % kSlots;
          if (!attn_wait_all(&sh.p_ready[slot], (n / kSlots) & 1, sh)) return false;
          tc_fence_after();
          weighted<T, kD>(leader, tmem + kO + q * kD, tmem + slot * kStep, 16, v_at + rv.s * kUnits, n > 0);
          attn_commit(leader, &sh.done[slot]);
        }
        attn_commit(leader, &sh.empty[8 + rv.s]);
        rv.next(stages);
        if (by == 2) rv.next(stages);
        return true;
      };
      bool ok = attn_wait_all(&sh.first, 0, sh);
      int ahead = start;  // the next step whose scores are formed
      for (int n = 0; ok && n < kSlots && ahead < e1; ++n, ahead += by) ok = score(ahead);
      for (int e = start; ok && e < e1; e += by, ahead += by) ok = sum(e) && (ahead >= e1 || score(ahead));
      attn_commit(leader, &sh.drained);  // matrix instructions in flight are done before the CTA leaves
      if (lane == 0) mbar_wait_bounded(&sh.drained, 0, kAttnLimitNs);
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, q = (warp - 4) >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), o_at = lanes + kO + q * kD;
    const int i = p.packed ? row % p.tq : first + q * kTile + row;
    const bool in = p.packed ? row < p.packed : i < p.tq;
    const bool some = __any_sync(0xffffffffu, in);
    const int h = p.packed ? head * p.group + row / p.tq : head, position = p.off + i;
    const float slack = kSlack / p.scale2;
    float most = -INFINITY, sum = 0.0f, ref = 0.0f;
    int taken = 0;
    bool ok = true;
    const StepsSeen seen_steps = p.packed ? StepsSeen{e1, 0, 0} : steps_seen(p, list, p0[q], p1[q]);
    for (int e = p.packed ? e0 + ((e0 ^ q) & 1) : e0; ok && e < e1; e += p.packed ? 2 : 1) {
      if (!seen_steps.has(e)) continue;
      const int k0 = list.at(e), slot = q * kSlots + taken % kSlots;
      const uint32_t s_at = lanes + slot * kStep;
      ok = attn_wait_all(&sh.s_full[slot], (taken / kSlots) & 1, sh);
      if (!ok) break;
      tc_fence_after();
      if (some) {
        // twice, so that the steps that are seen as a whole, most of them, run through no code for the others
        const auto take = [&](auto masked) {
          constexpr bool kMasked = decltype(masked)::value;
          // where the registers do not hold all of a row's scores they are read twice
          constexpr int kHeld = kD == 128 ? 2 : 1;
          float v[kHeld][32];
          const int high = position + 1 - k0, low = position - p.window + 1 - k0, sinks = min(p.sinks - k0, high);
          const auto read = [&](int c, float(&w)[32]) {
            tc_load32(s_at + c * 32, w);
            tc_load_wait(w);
            if (kMasked) {
              const uint32_t seen = seen_bits(low, high, sinks, c * 32);
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = seen >> j & 1 ? w[j] : -INFINITY;
            }
          };
          float top = -INFINITY;
#pragma unroll kHeld
          for (int c = 0; c < 2; ++c) {
            float(&w)[32] = v[c % kHeld];
            read(c, w);
            float tops[2] = {fmaxf(w[0], w[1]), fmaxf(w[16], w[17])};
#pragma unroll
            for (int j = 2; j < 16; j += 2) {
              tops[0] = max3(tops[0], w[j], w[j + 1]);
              tops[1] = max3(tops[1], w[16 + j], w[17 + j]);
            }
            top = max3(top, tops[0], tops[1]);
          }
          const bool grows = top > most + slack;
          if (__any_sync(0xffffffffu, grows)) {
            float factor = 1.0f;
            if (grows) {
              factor = power2((most - top) * p.scale2);
              most = top;
              ref = top * p.scale2 - kBias;
              sum *= factor;
            }
            __syncwarp();  // tensor memory is read by whole warps
            if (taken) {
              // O has everything up to the step before
              ok = attn_wait_all(&sh.done[q * kSlots + (taken - 1) % kSlots], ((taken - 1) / kSlots) & 1, sh);
              if (!ok) return;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < kD; c += 32) {
                float o[32];
                tc_load32(o_at + c, o);
                tc_load_wait(o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] *= factor;
                tc_store32(o_at + c, o);
              }
            }
          }
          const Pair scale = pair(p.scale2, p.scale2), less = pair(-ref, -ref);
          Pair total[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
#pragma unroll kHeld
          for (int c = 0; c < 2; ++c) {
            float(&w)[32] = v[c % kHeld];
            if (kHeld == 1) read(c, w);
            uint32_t words[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float x, y;
              parts(fma2(pair(w[j], w[j + 1]), scale, less), x, y);
              x = power2(x);
              y = power2(y);
              total[j / 2 % 2] = total[j / 2 % 2] + pair(x, y);
              words[j / 2] = pack2<T>(x, y);
            }
            tc_store16(s_at + c * 16, words);
          }
          sum += both(total[0] + total[1]);
          tc_store_wait();
        };
        if (all_seen(p, p0[q], p1[q], k0, kStep)) take(std::false_type());
        else take(std::true_type());
        if (!ok) break;
      }
      ++taken;
      warp_arrives(&sh.p_ready[slot]);
    }
    if (ok && e0 < e1) ok = attn_wait_all(&sh.drained, 0, sh);
    if (ok && some) {
      tc_fence_after();
      const bool none = sum == 0.0f;  // (a NaN is not)
      const float factor = none ? 0.0f : 1.0f / sum;
      const int64_t head_at = (int64_t)b * p.heads + h;
      if (shared) {
        store_row<float, kD>(o_at, joined + (q * kTile + row) * kRow, kD, factor, in, taken > 0, none);
        if (in) part_less[q * kTile + row] = none ? INFINITY : -(ref + log2f(sum));
      } else {
        store_row<T, kD>(o_at, static_cast<T*>(p.o) + (((int64_t)b * p.tq + i) * p.heads + h) * p.d, p.d, factor, in, taken > 0, none);
        if (in && p.less) p.less[head_at * p.less_ld + i] = none ? -INFINITY : -(ref + log2f(sum));
      }
    }
    if (!ok && shared && in) part_less[q * kTile + row] = __int_as_float(0x7fc00000);  // a wait ran out: no numbers
  }
  attn_end<S::kColumns>(tmem);
  if (!shared) return;
  // O = sum of the parts' O times 2^(their logarithm), over the sum of those; four columns of a row a thread, the rows' pieces go round the CTAs
  cluster_meet(p.splits);
  const int halves = p.packed ? 2 : 1, rows = p.packed ? p.packed : min(2 * kTile, p.tq - first), all = p.splits * halves;
  for (int n = threadIdx.x * p.splits + split; n < rows * (kD / 4); n += S::kForwardThreads * p.splits) {
    const int row = n / (kD / 4), c = n % (kD / 4) * 4;
    const auto lies = [&](int k) { return row + (p.packed ? k % 2 * kTile : 0); };  // part k's row in its CTA
    const auto rank = [&](int k) { return p.packed ? k / 2 : k; };
    float least = INFINITY, sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    float theirs[2 * kMostSplits];  // loads are on their way together
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 2 * kMostSplits; ++k) theirs[k] = k < all ? peer_load(peer_address(part_less + lies(k), rank(k))) : INFINITY;
#pragma unroll
    for (int k = 0; k < 2 * kMostSplits; ++k) {
      least = fminf(least, theirs[k]);
      bad = bad || theirs[k] != theirs[k];
    }
    const bool none = least == INFINITY && !bad;
#pragma unroll
    for (int k0 = 0; k0 < 2 * kMostSplits; k0 += 4) {
      if (k0 >= all) break;
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = k0 + k < all ? peer_load4(peer_address(joined + lies(k0 + k) * kRow + c, rank(k0 + k))) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (theirs[k0 + k] == INFINITY) continue;
        const float weight = power2(least - theirs[k0 + k]);
        sum += weight;
        v[0] += weight * x[k].x, v[1] += weight * x[k].y, v[2] += weight * x[k].z, v[3] += weight * x[k].w;
      }
    }
    const float factor = none ? 0.0f : 1.0f / sum;
    const int i = p.packed ? row % p.tq : first + row, h = p.packed ? head * p.group + row / p.tq : head;
    if (c < p.d)
      *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + (((int64_t)b * p.tq + i) * p.heads + h) * p.d + c) =
          make_uint2(pack2<T>(v[0] * factor, v[1] * factor), pack2<T>(v[2] * factor, v[3] * factor));
    if (c == 0 && p.less) p.less[((int64_t)b * p.heads + h) * p.less_ld + i] = none ? -INFINITY : least - log2f(sum);
  }
  cluster_meet(p.splits);  // nobody leaves while its shared memory is read
}

// ---- forward, few rows -------------------------------------------------------------------------------------------------------
// Up to eight rows (queries times heads of a key's head), a new token for one, where the kernel above mostly waits for its own beginning.  No tensor memory and no mbarriers: a warp loads 16 keys and
// values at a time from global memory as mma.sync's first operand wants them (S^T = K Q^T, O^T = V^T P^T, so that the rows are its eight columns and no operand is empty), and keeps a maximum, a sum
// and O of its own keys, which CTA and cluster join.  Bound by reading keys and values, and by latency where they are few.  bf16, times in a graph: 12 heads of 64, 1024 keys 3.9 us (9.1 with
// the kernel above); 32 heads on 8 of 128, 1024 keys 6.1 us (10.3); 8 x 16 heads on 4 of 128, 4096 keys 16.4 us (21.5); 64 x 12 heads of 64, 1024 keys 38 us, 5.3 TB/s (56); 16 x 16 heads on 4 of 128, 8196
// keys 49 us (52).  32 keys at a time, with heads up to 64: 5.3 us instead of 4.2; the next keys' loads before the work on these: spills, 73 us instead of 51 at 32 x 16 heads on 8, 2048 keys of 128.
struct FewRows {
  const void *q, *k, *v;
  int64_t q_batch, q_head, q_position, k_batch, k_head, k_position, v_batch, v_head, v_position;
  void* o;
  float* less;
  int64_t less_ld;
  int heads, kv_heads, group, tq, d, off, window, sinks, splits, split_bits;  // splits: 2^split_bits
  unsigned heads_of;  // 2^16 / tq, rounded up
  float scale2;
};
constexpr int kFewWarps = 8, kFewRows = 8, kFewKeys = 16;  // keys of a warp at once
// eight rows of eight 16-bit values, a row's neighbours 2t and 2t + 1 in lane 4 row + t, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T, int kD, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == 16 ? 1 : kD == 64 ? 3 : 2) hc_attention_few_kernel(const __grid_constant__ FewRows p) {
  constexpr int kQ = kD / 32, kV = kD / 64;
  constexpr float kBias = operand_format<T>() ? 0.0f : 14.0f;  // probabilities, and with them sums and O, are held times 2^14 in fp16
  __shared__ __align__(16) float values[kFewWarps][kFewRows][kD];
  __shared__ __align__(16) float joined[kFewRows][kD];
  __shared__ float2 sums[kFewWarps][kFewRows], joined_sums[kFewRows];  // maximum, sum of exponentials
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, rows = p.group * p.tq;
  const unsigned at = blockIdx.x >> p.split_bits;
  const int rank = blockIdx.x & (p.splits - 1), b = at / (unsigned)p.kv_heads, head = at - b * p.kv_heads;
  const auto head_of = [&](int row) { return (int)((unsigned)row * p.heads_of >> 16); };  // row / tq
  // the keys that some row sees, counted without the gap between the first tokens and the window
  const int last = p.off + p.tq - 1, from = max(p.off - p.window + 1, 0), sinks = min(p.sinks, from), count = last < 0 ? 0 : sinks + last - from + 1;
  const T *k = static_cast<const T*>(p.k) + b * p.k_batch + head * p.k_head, *v = static_cast<const T*>(p.v) + b * p.v_batch + head * p.v_head;
  const auto key_of = [&](int n) { return n < sinks ? n : n - sinks + from; };
  // eight values of key number n, from 8 c on
  const auto load = [&](const T* at, int64_t position, int n, int c) { return n < count && c * 8 < p.d ? *reinterpret_cast<const uint4*>(at + key_of(n) * position + c * 8) : make_uint4(0, 0, 0, 0); };
  uint4 q[kQ];  // of row g
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const int c = t + 4 * i;
    q[i] = make_uint4(0, 0, 0, 0);
    if (g < rows && c * 8 < p.d) q[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_batch + (head * p.group + head_of(g)) * p.q_head + (g - head_of(g) * p.tq) * p.q_position + c * 8);
  }
  float o[kV][4][4];  // of rows 2t (0, 2) and 2t + 1 (1, 3), values 8 (g + 8 i) + 2 u (0, 1) and the next
#pragma unroll
  for (int i = 0; i < kV; ++i)
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][u][j] = 0.0f;
  float most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  int position[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) position[r] = p.off + 2 * t + r - head_of(2 * t + r) * p.tq;
  for (int first = (rank * kWarps + warp) * kFewKeys; first < count; first += p.splits * kWarps * kFewKeys) {
    uint4 x[2][kQ], y[4][kV];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kQ; ++i) x[h][i] = load(k, p.k_position, first + h * 8 + g, t + 4 * i);
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < kV; ++i) y[h][i] = load(v, p.v_position, first + (h >> 1) * 8 + 2 * t + (h & 1), g + 8 * i);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of keys g (0, 1) and g + 8, rows 2t (0, 2) and 2t + 1
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      mma_16x8x16<T>(s, x[0][i].x, x[1][i].x, x[0][i].y, x[1][i].y, q[i].x, q[i].y);
      mma_16x8x16<T>(s, x[0][i].z, x[1][i].z, x[0][i].w, x[1][i].w, q[i].z, q[i].w);
    }
    float top[2] = {most[0], most[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = first + (j >> 1) * 8 + g, key = key_of(n), at = position[j & 1];
      const bool seen = n < count && key <= at && (at - key < p.window || key < p.sinks);
      s[j] = seen ? s[j] * p.scale2 : -INFINITY;
      top[j & 1] = fmaxf(top[j & 1], s[j]);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int n = 4; n < 32; n <<= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], n));
      const float ref = top[r] == -INFINITY ? 0.0f : top[r], before = power2(most[r] - ref);
      most[r] = top[r];
      s[r] = power2(s[r] - ref + kBias);
      s[2 + r] = power2(s[2 + r] - ref + kBias);
      sum[r] = sum[r] * before + (s[r] + s[2 + r]);
#pragma unroll
      for (int i = 0; i < kV; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          o[i][u][r] *= before;
          o[i][u][2 + r] *= before;
        }
    }
    const uint32_t b0 = transposed(pack2<T>(s[0], s[1])), b1 = transposed(pack2<T>(s[2], s[3]));
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const auto word = [&](int h, int u) { return u == 0 ? y[h][i].x : u == 1 ? y[h][i].y : u == 2 ? y[h][i].z : y[h][i].w; };
#pragma unroll
      for (int u = 0; u < 4; ++u)
        mma_16x8x16<T>(o[i][u], __byte_perm(word(0, u), word(1, u), 0x5410), __byte_perm(word(0, u), word(1, u), 0x7632), __byte_perm(word(2, u), word(3, u), 0x5410),
                       __byte_perm(word(2, u), word(3, u), 0x7632), b0, b1);
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int n = 4; n < 32; n <<= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], n);
  const auto put = [&](int at) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = 2 * t + r;
      if (row >= rows) continue;
      if (g == 0) sums[at][row] = make_float2(most[r], sum[r]);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        float* to = &values[at][row][8 * (g + 8 * i)];
        *reinterpret_cast<float4*>(to) = make_float4(o[i][0][r], o[i][0][2 + r], o[i][1][r], o[i][1][2 + r]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(o[i][2][r], o[i][2][2 + r], o[i][3][r], o[i][3][2 + r]);
      }
    }
  };
  if (kWarps > kFewWarps) {  // the second eight warps' go to the first
    if (warp >= kFewWarps) put(warp - kFewWarps);
    __syncthreads();
    if (warp < kFewWarps) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 2 * t + r;
        if (row >= rows) continue;
        const float2 other = sums[warp][row];
        const float top = fmaxf(most[r], other.x), ref = top == -INFINITY ? 0.0f : top, a = power2(most[r] - ref), c = power2(other.x - ref);
        most[r] = top;
        sum[r] = sum[r] * a + other.y * c;
#pragma unroll
        for (int i = 0; i < kV; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 w = *reinterpret_cast<const float2*>(&values[warp][row][8 * (g + 8 * i) + 2 * u]);
            o[i][u][r] = o[i][u][r] * a + w.x * c;
            o[i][u][2 + r] = o[i][u][2 + r] * a + w.y * c;
          }
      }
      __syncwarp();  // all of it is read
    }
  }
  if (warp < kFewWarps) put(warp);
  __syncthreads();
  // of `all` parts: a row's four values, maximum and sum
  const auto join = [](int all, auto sum_at, auto value_at, float2& total, float4& x) {
    float2 s[kFewWarps];
    float4 y[kFewWarps];
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < kFewWarps; ++n) {
      s[n] = n < all ? sum_at(n) : make_float2(-INFINITY, 0.0f);
      y[n] = n < all ? value_at(n) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      top = fmaxf(top, s[n].x);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    total = make_float2(top, 0.0f);
    x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int n = 0; n < kFewWarps; ++n) {
      const float weight = power2(s[n].x - ref);
      total.y += weight * s[n].y;
      x.x += weight * y[n].x, x.y += weight * y[n].y, x.z += weight * y[n].z, x.w += weight * y[n].w;
    }
  };
  const auto store = [&](int r, int col, float2 total, float4 x) {
    const bool none = total.y == 0.0f;  // (a NaN is not)
    const float factor = none ? 0.0f : 1.0f / total.y;
    const int i = r - head_of(r) * p.tq, h = head * p.group + head_of(r);
    if (col < p.d)
      *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + (((int64_t)b * p.tq + i) * p.heads + h) * p.d + col) = make_uint2(pack2<T>(x.x * factor, x.y * factor), pack2<T>(x.z * factor, x.w * factor));
    if (col == 0 && p.less) p.less[((int64_t)b * p.heads + h) * p.less_ld + i] = none ? -INFINITY : kBias - (total.x + log2f(total.y));
  };
  static_assert(kFewRows * (kD / 4) <= 32 * kFewWarps && kMostSplits <= kFewWarps, "a thread's part");
  const int row = threadIdx.x / (kD / 4), col = threadIdx.x % (kD / 4) * 4;
  float2 total;
  float4 x;
  if (row < rows) {
    join(kFewWarps, [&](int n) { return sums[n][row]; }, [&](int n) { return *reinterpret_cast<const float4*>(&values[n][row][col]); }, total, x);
    if (p.splits == 1) store(row, col, total, x);
  }
  if (p.splits == 1) return;
  if (row < rows) {
    *reinterpret_cast<float4*>(&joined[row][col]) = x;
    if (col == 0) joined_sums[row] = total;
  }
  cluster_meet(p.splits);
  if (row < rows && threadIdx.x % p.splits == rank) {
    join(
        p.splits,
        [&](int n) {
          const uint32_t at = peer_address(&joined_sums[row], n);
          return make_float2(peer_load(at), peer_load(at + 4));
        },
        [&](int n) { return peer_load4(peer_address(&joined[row][col], n)); }, total, x);
    store(row, col, total, x);
  }
  cluster_meet(p.splits);  // nobody leaves while its shared memory is read
}

// ---- backward ----------------------------------------------------------------------------------------------------------------
// fp16: for each sequence's key head the largest square of a norm of dO's rows (the first `blocks[0] * heads[0] * batch` blocks) and of V's.  Eight values a thread, four rows of a thread on their way together; a block has
// 4 * 256 / kLanes rows of a head.
struct RowsOf {
  const void* data[2];
  int64_t stride_b[2], stride_h[2], stride_t[2];
  int heads[2], length[2], blocks[2];
  int64_t first_blocks;
};
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) hc_attention_rows_kernel(const __grid_constant__ RowsOf of, int d, unsigned int* most) {
  constexpr int kAtOnce = 4, kApart = 256 / kLanes;
  const int n = blockIdx.x >= of.first_blocks, block = (int)(blockIdx.x - (n ? of.first_blocks : 0));
  const int head_at = block / of.blocks[n], b = head_at / of.heads[n], h = head_at - b * of.heads[n];
  const int part = threadIdx.x % kLanes, first = (block - head_at * of.blocks[n]) * (kAtOnce * kApart) + threadIdx.x / kLanes;
  const T* from = static_cast<const T*>(of.data[n]) + b * of.stride_b[n] + h * of.stride_h[n] + part * 8;
  uint4 x[kAtOnce];
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k) {
    const int i = first + k * kApart;
    x[k] = part * 8 < d && i < of.length[n] ? *reinterpret_cast<const uint4*>(from + i * of.stride_t[n]) : make_uint4(0, 0, 0, 0);
  }
  launch_dependents();
  unsigned int largest = 0;
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k) {
    float u[8], square = 0.0f;
    unpack2<T>(x[k].x, u[0], u[1]), unpack2<T>(x[k].y, u[2], u[3]), unpack2<T>(x[k].z, u[4], u[5]), unpack2<T>(x[k].w, u[6], u[7]);
#pragma unroll
    for (int j = 0; j < 8; ++j) square = fmaf(u[j], u[j], square);
#pragma unroll
    for (int m = kLanes / 2; m > 0; m >>= 1) square += __shfl_xor_sync(0xffffffffu, square, m);
    if (square < INFINITY) largest = max(largest, __float_as_uint(square));
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  if ((threadIdx.x & 31) == 0 && largest) atomicMax(most + 2 * ((int64_t)b * of.heads[1] + h / (of.heads[n] / of.heads[1])) + n, largest);
}
// The power of two that dS is held times in fp16: 2 max|dO_i| max|V_j|, which |dS| does not exceed, comes to below 2^15 (from the squares of both).
__device__ __forceinline__ float ds_power(const unsigned int* most, int sign) {
  const int e = (int)(most[0] >> 23) - 127 + (int)(most[1] >> 23) - 127 + 2;  // the product of the squares is below 2^e
  const int k = most[0] && most[1] ? min(max(13 - (e + 1) / 2, -100), 100) : 0;
  return __int_as_float((127 + sign * k) << 23);
}

// The backward pass of a tile of 128 keys (kKeys: dV = P^T dO, dK = scale dS^T Q; a stream of queries, 64 at a time) or of 128 queries (dQ = scale dS K; a stream of keys).  The tile
// lies in lanes, the stream in columns.  Eight warps work on a step, four on each half of its columns; with heads of more than 64 values two groups of eight take the steps in turn, with smaller ones
// two CTAs are on an SM, so that exponentials, multiplications and the tensor cores' work overlap.  One warp issues the products that form scores, one those that sum.
// Tensor memory: scores of the groups' steps, then dO V^T (P and dS at the beginning of each half's 32 columns), then the two sums.
//
// The queries' pass takes delta from dO and O itself (from a kernel before it all passes took 154 us instead of 151 at 8 x 12 x 1024 x 64, and one us less of 967 at 16 heads
// on 4, 8192 x 128).  delta from the rounded O, whose probabilities were rounded too, is wrong by some 2^-9 of itself, and all of a row's dS with it: half of the error of dQ and dK (1024 x 1024, 2.8e-3 of dQ's norm, where
// all other roundings come to 2.5e-3).  The rows of dS sum to 0, so the sum of what they are instead is what delta lacks: r = sum_j P (dP - delta).  The queries' pass finds r on
// its way, sums P K beside dS K, and gives dQ = scale (dS K - r P K); delta + r goes to the keys' pass, which comes behind it.  For dQ, r is
// the sum of the rounded dS, so that of what their rounding adds up to the keys' mean has no part either.
template <typename T, int kD, bool kKeys>
__global__ void __launch_bounds__(AttnShape<kD>::kBackwardThreads, AttnShape<kD>::kResident) hc_attention_backward_kernel(const __grid_constant__ AttnParams p) {
  using S = AttnShape<kD>;
  constexpr int kStages = S::kStages, kStageBytes = 2 * S::kStepBytes, kGroups = S::kGroups, kParts = 2 * kGroups;
  constexpr int kDp = kGroups * kStep, kSum1 = 2 * kDp, kSum2 = kSum1 + kD;  // columns of tensor memory
  constexpr bool kF16 = operand_format<T>() == 0;
  extern __shared__ unsigned char raw[];
  __shared__ AttnBarriers sh;
  __shared__ float2 lacking[kParts][kTile];  // sums of a row's dS, and of the rounded
  __shared__ float dots[kParts][kTile];      // parts of delta
  unsigned char *tile1 = attn_tiles(raw), *tile2 = tile1 + S::kBytes, *ring = tile2 + S::kBytes;
  float* sides = reinterpret_cast<float*>(ring + kStages * kStageBytes);  // of a step of queries: less, delta
  // what the CTAs of a cluster join lies where the operands were: dV and dK side by side
  constexpr int kRow = 2 * kD + 4;
  static_assert(kTile * kRow * 4 <= S::kBackwardSmem - 1024, "room for the parts");
  float* joined = reinterpret_cast<float*>(tile1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int heads = kKeys ? p.kv_heads : p.heads;
  int64_t at = blockIdx.x;
  const int rank = kKeys ? (int)(at % p.splits) : 0;  // in a cluster that shares a tile of keys' query heads out
  if (kKeys) at /= p.splits;
  const int head = (int)(at % heads);
  at /= heads;
  const int b = (int)(at % p.batch), block = kKeys ? (int)(at / p.batch) : p.blocks - 1 - (int)(at / p.batch);
  const int t0 = block * kTile;  // the tile's first row
  const int64_t most_at = 2 * ((int64_t)b * p.kv_heads + (kKeys ? head : head / p.group));  // of p.most
  // the stream: queries that see one of the keys, head after head; or the keys that the queries see
  const int q_first = max(t0 - p.off, 0) / kStep,
            q_last = t0 < p.sinks ? p.tq - 1 : (int)min((int64_t)p.tq - 1, (int64_t)min(t0 + kTile, p.tk) - 1 + p.window - 1 - p.off);
  const int q_steps = q_last >= max(t0 - p.off, 0) ? q_last / kStep - q_first + 1 : 0;
  const int p0 = p.off + t0, p1 = p.off + min(t0 + kTile, p.tq) - 1;
  const KeySteps list = kKeys ? KeySteps{0, 0, 0} : key_steps(p, p0, p1);
  const int own_heads = p.group / p.splits, count = kKeys ? q_steps * own_heads : list.count;
  // for delta: 32 values of a row of O each, on their way while the CTA begins
  uint4 y[4];
  float less1 = 0.0f;
  if (!kKeys && warp >= 4) {
    const int row = (warp & 3) * 32 + lane, t = t0 + row, c = ((warp - 4) >> 2) * 32;
    const T* o = static_cast<const T*>(p.o) + (((int64_t)b * p.tq + t) * p.heads + head) * p.d + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = t < p.tq && c + j * 8 < p.d ? *reinterpret_cast<const uint4*>(o + j * 8) : make_uint4(0, 0, 0, 0);
    if (t < p.tq) less1 = p.less[((int64_t)b * p.heads + head) * p.less_ld + t];
  }
  attn_begin<S::kColumns>(sh, 8 * kGroups, 8, 1, [&] {
    if (!count) return;
    mbar_expect_tx(&sh.first, 2 * S::kBytes);
    load_rows<kD, kTile>(tile1, kKeys ? &p.k_tile : &p.q_tile, t0, head, b, &sh.first);
    load_rows<kD, kTile>(tile2, kKeys ? &p.v_tile : &p.dout_tile, t0, head, b, &sh.first);
  });
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  share_registers<(S::kResident == 2 ? 96 : 104), S::kBackwardThreads, S::kBackwardRegisters>(warp < 4);
  if (warp == 0) {
    if (kKeys && lane == 0) grid_dependency_wait();  // behind the queries' pass, whose delta comes in with the queries; the norms were there when it let this kernel begin
    if (lane == 0 && count) {
      Ring<kStages> r;
      int h = kKeys ? head * p.group + rank * own_heads : head / p.group, step = 0;
      for (int e = 0; e < count; ++e) {
        if (!attn_wait(&sh.empty[r.s], r.phase ^ 1, sh)) break;
        const int at0 = kKeys ? (q_first + step) * kStep : list.at(e);
        unsigned char* to = ring + r.s * kStageBytes;
        mbar_expect_tx(&sh.full[r.s], kStageBytes + (kKeys ? 512 : 0));
        load_rows<kD, kStep>(to, kKeys ? &p.q : &p.k, at0, h, b, &sh.full[r.s]);
        load_rows<kD, kStep>(to + S::kStepBytes, kKeys ? &p.dout : &p.v, at0, h, b, &sh.full[r.s]);
        if (kKeys) {
          const int64_t side = ((int64_t)b * p.heads + h) * p.less_ld + at0;
          load_floats(sides + r.s * 128, p.less + side, 256, &sh.full[r.s]);
          load_floats(sides + r.s * 128 + 64, p.delta + side, 256, &sh.full[r.s]);
          if (++step == q_steps) {
            step = 0;
            ++h;
          }
        }
        r.next();
      }
      ring_end(sh.full, r);
      mbar_wait_bounded(&sh.first, 0, kAttnLimitNs);
    }
  } else if (warp <= 2) {
    if (count) {
      // what is waited for the k-th time has parity k & 1
      const bool leader = elected();
      constexpr int kUnits = kStageBytes / 16, kSecond = S::kStepBytes / 16;
      const uint64_t tile1_at = along(tile1), tile2_at = along(tile2), ring_along = along(ring), ring_across = across(ring);
      bool ok = true;
      if (warp == 1) {
        ok = attn_wait_all(&sh.first, 0, sh);
        for (int e = 0; ok && e < count; ++e) {
          const int g = e % kGroups;
          const uint32_t before = (e / kGroups - 1) & 1;
          ok = attn_wait_all(&sh.full[e % kStages], (e / kStages) & 1, sh) && (e < kGroups || attn_wait_all(&sh.done[g], before, sh));
          if (!ok) break;
          tc_fence_after();
          scores<T, kD>(leader, tmem + g * kStep, tile1_at, ring_along + e % kStages * kUnits);
          attn_commit(leader, &sh.s_full[g]);
          ok = e < kGroups || attn_wait_all(&sh.ds_done[g], before, sh);
          if (!ok) break;
          tc_fence_after();
          scores<T, kD>(leader, tmem + kDp + g * kStep, tile2_at, ring_along + e % kStages * kUnits + kSecond);
          attn_commit(leader, &sh.dp_full[g]);
        }
      } else {
        const auto second_sum = [&](int e) {
          const int g = e % kGroups;
          if (!attn_wait_all(&sh.ds_ready[g], (e / kGroups) & 1, sh)) return false;
          tc_fence_after();
          weighted<T, kD>(leader, tmem + kSum2, tmem + kDp + g * kStep, 32, ring_across + e % kStages * kUnits, e > 0);
          attn_commit(leader, &sh.ds_done[g]);
          attn_commit(leader, &sh.empty[e % kStages]);  // all four products of the step are done then
          return true;
        };
        for (int e = 0; ok && e < count; ++e) {
          const int g = e % kGroups;
          ok = attn_wait_all(&sh.full[e % kStages], (e / kStages) & 1, sh) && attn_wait_all(&sh.p_ready[g], (e / kGroups) & 1, sh);
          if (!ok) break;
          tc_fence_after();
          weighted<T, kD>(leader, tmem + kSum1, tmem + g * kStep, 32, ring_across + e % kStages * kUnits + (kKeys ? kSecond : 0), e > 0);
          attn_commit(leader, &sh.done[g]);
          ok = e < kGroups - 1 || second_sum(e - (kGroups - 1));
        }
        for (int e = count - min(kGroups - 1, count); ok && e < count; ++e) ok = second_sum(e);
      }
      attn_commit(leader, &sh.drained);
      if (lane == 0) mbar_wait_bounded(&sh.drained, 0, kAttnLimitNs);
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, part = (warp - 4) >> 2, g = part >> 1, half = part & 1, row = quarter * 32 + lane, t = t0 + row;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lanes + g * kStep + half * 32, dp_at = s_at + kDp;
    constexpr float kBias = kF16 && kKeys ? 14.0f : 0.0f;  // P^T is held times 2^14 in fp16 (what P K is for needs no more than a few bits)
    if (!kKeys) {
      if (kF16) grid_dependency_wait();  // behind the largest norms
      if (p.dk) launch_dependents();  // the keys' pass; without it, what comes next waits for the end
    }
    const float power = kF16 ? ds_power(p.most + most_at, 1) : 1.0f, back = kF16 ? ds_power(p.most + most_at, -1) : 1.0f;
    const Pair gain = pair(power * (kBias ? 1.0f / 16384.0f : 1.0f), power * (kBias ? 1.0f / 16384.0f : 1.0f));
    const Pair scale = pair(p.scale2, p.scale2), minus = pair(-1.0f, -1.0f), bias = pair(kBias, kBias);
    const bool in = t < (kKeys ? p.tk : p.tq);
    const int64_t side = ((int64_t)b * p.heads + head) * p.less_ld + t;
    float delta = 0.0f;
    Pair less = pair(-INFINITY, -INFINITY), delta2 = pair(0.0f, 0.0f), lacks = pair(0.0f, 0.0f), rounded = pair(0.0f, 0.0f);
    if (!kKeys && count) {
      // delta = dO . O, dO's row from the tile
      const int c = part * 32;
      if (in) less = pair(less1, less1);
      attn_wait_all(&sh.first, 0, sh);  // when this or the wait for the other parts runs out, so do those below
      const unsigned char* at = tile2 + c / 64 * (kTile * 128) + row * 128;
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 x = *reinterpret_cast<const uint4*>(at + ((c % 64 / 8 + j) ^ (row & 7)) * 16);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y[j].x, y[j].y, y[j].z, y[j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float u[2], w[2];
          unpack2<T>(xs[k], u[0], u[1]);
          unpack2<T>(ys[k], w[0], w[1]);
          dot = fmaf(u[1], w[1], fmaf(u[0], w[0], dot));
        }
      }
      dots[part][row] = dot;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.dots);
      attn_wait_all(&sh.dots, 0, sh);
#pragma unroll
      for (int k = 0; k < kParts; ++k) delta += dots[k][row];
      delta2 = pair(delta, delta);
    }
    int step = g;
    if (kKeys)
      while (q_steps && step >= q_steps) step -= q_steps;
    bool ok = true;
    for (int e = g; e < count; e += kGroups) {
      const uint32_t turn = (e / kGroups) & 1;
      const float* side_at = sides + e % kStages * 128 + half * 32;
      if ((kKeys && !attn_wait_all(&sh.full[e % kStages], (e / kStages) & 1, sh)) || !attn_wait_all(&sh.s_full[g], turn, sh)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // what this row sees, or is seen by
      const int i0 = (q_first + step) * kStep, pa = p.off + i0, k0 = kKeys ? t0 : list.at(e), position = p.off + t;
      const bool whole = kKeys ? i0 + kStep <= p.tq && all_seen(p, pa, pa + kStep - 1, t0, kTile) : all_seen(p, p0, p1, k0, kStep);
      // twice, so that the steps that are seen as a whole, most of them, run through no code for the others
      const auto take = [&](auto masked) {
        constexpr bool kMasked = decltype(masked)::value;
        float v[32];
        tc_load32(s_at, v);
        uint32_t seen = 0xffffffffu;
        if (kMasked && kKeys) {
          const int high = min(p.tq - i0, (int)min((int64_t)kStep, t < p.sinks ? (int64_t)kStep : (int64_t)t + p.window - pa));
          seen = seen_bits(t - pa, high, 0, half * 32);
        } else if (kMasked) {
          const int high = position - k0 + 1;
          seen = seen_bits(position - p.window + 1 - k0, high, min(p.sinks - k0, high), half * 32);
        }
        tc_load_wait(v);
#pragma unroll
        for (int n = 0; n < 32; n += 4) {
          Pair l0 = less, l1 = less;
          if (kKeys) {
            const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(side_at + n);
            l0 = Pair{l.x};
            l1 = Pair{l.y};
            if (kBias) {
              l0 = l0 + bias;
              l1 = l1 + bias;
            }
          }
          parts(fma2(pair(v[n], v[n + 1]), scale, l0), v[n], v[n + 1]);
          parts(fma2(pair(v[n + 2], v[n + 3]), scale, l1), v[n + 2], v[n + 3]);
        }
#pragma unroll
        for (int n = 0; n < 32; ++n) v[n] = power2(v[n]);
        if (kMasked) {
#pragma unroll
          for (int n = 0; n < 32; ++n) v[n] = seen >> n & 1 ? v[n] : 0.0f;
        }
        uint32_t words[16];
#pragma unroll
        for (int n = 0; n < 32; n += 2) words[n / 2] = pack2<T>(v[n], v[n + 1]);
        tc_store16(s_at, words);
        tc_store_wait();
        warp_arrives(&sh.p_ready[g]);
        if (!attn_wait_all(&sh.dp_full[g], turn, sh)) {
          ok = false;
          return;
        }
        tc_fence_after();
        float d[32];
        tc_load32(dp_at, d);
        tc_load_wait(d);
#pragma unroll
        for (int n = 0; n < 32; n += 4) {
          Pair l0 = delta2, l1 = delta2;
          if (kKeys) {
            const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(side_at + 64 + n);
            l0 = Pair{l.x};
            l1 = Pair{l.y};
          }
          Pair x = fma2(l0, minus, pair(d[n], d[n + 1])) * pair(v[n], v[n + 1]), y = fma2(l1, minus, pair(d[n + 2], d[n + 3])) * pair(v[n + 2], v[n + 3]);
          if (kF16) {
            x = x * gain;
            y = y * gain;
          }
          parts(x, d[n], d[n + 1]);
          parts(y, d[n + 2], d[n + 3]);
        }
        if (kMasked) {  // also where one that is not seen, or a query that is none, has no number
#pragma unroll
          for (int n = 0; n < 32; ++n) d[n] = seen >> n & 1 ? d[n] : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < 32; n += 2) {
          words[n / 2] = pack2<T>(d[n], d[n + 1]);
          if (!kKeys) {
            lacks = lacks + pair(d[n], d[n + 1]);
            unpack2<T>(words[n / 2], d[n], d[n + 1]);
            rounded = rounded + pair(d[n], d[n + 1]);
          }
        }
        tc_store16(dp_at, words);
        tc_store_wait();
        warp_arrives(&sh.ds_ready[g]);
      };
      if (whole) take(std::false_type());
      else take(std::true_type());
      if (!ok) break;
      if (kKeys) {
        step += kGroups;
        while (step >= q_steps) step -= q_steps;
      }
    }
    if (ok && count) ok = attn_wait_all(&sh.drained, 0, sh);
    if (ok && kKeys) {
      tc_fence_after();
      // 64 of the columns of dV and dK each
      const bool second = part * 64 >= kD;
      const int c = part * 64 % kD;
      if (p.splits > 1) {
        store_row<float, 64>(lanes + kSum1 + part * 64, joined + row * kRow + part * 64, 64, 1.0f, true, count > 0, false);
      } else {
        T* to = static_cast<T*>(second ? p.dk : p.dv) + (((int64_t)b * p.tk + t) * p.kv_heads + head) * p.d + c;
        store_row<T, 64>(lanes + kSum1 + part * 64, to, p.d - c, second ? p.scale * back : kF16 ? 1.0f / 16384.0f : 1.0f, in, count > 0, false);
      }
    }
    if (!ok && kKeys && p.splits > 1)  // a wait ran out: no numbers
      for (int c = 0; c < 64; ++c) joined[row * kRow + part * 64 + c] = __int_as_float(0x7fc00000);
    if (ok && !kKeys) {
      lacking[part][row] = make_float2(both(lacks) * back, both(rounded) * back);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.met);
      ok = attn_wait_all(&sh.met, 0, sh);
      float lack = 0.0f, r = 0.0f;
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        lack += lacking[k][row].x;
        r += lacking[k][row].y;
      }
      if (ok && in && part == 0) p.delta[side] = delta + lack;
      __syncwarp();
      tc_fence_after();
      // 32 of the columns each
      static_assert(kParts * 32 == kD, "a part's columns");
      const int c = part * 32;
      float x[32], y[32];
      if (count) {
        tc_load32(lanes + kSum1 + c, x);
        tc_load32(lanes + kSum2 + c, y);
        tc_load_wait(x);
        tc_load_wait(y);
      }
      if (ok && in && p.dq) {
        T* to = static_cast<T*>(p.dq) + (((int64_t)b * p.tq + t) * p.heads + head) * p.d + c;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (c + j >= p.d) continue;
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = count ? p.scale * (y[j + k] * back - r * x[j + k]) : 0.0f;
          store8(to + j, v);
        }
      }
    }
  }
  attn_end<S::kColumns>(tmem);
  if (!kKeys || p.splits == 1) return;
  cluster_meet(p.splits);
  const float back = kF16 ? ds_power(p.most + most_at, -1) : 1.0f;
  for (int n = threadIdx.x * p.splits + rank; n < min(kTile, p.tk - t0) * (kD / 4); n += S::kBackwardThreads * p.splits) {
    const int row = n / (kD / 4), column = n % (kD / 4) * 8;  // of dV and dK side by side
    const bool second = column >= kD;
    const int c = second ? column - kD : column;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // a pair
      const uint32_t from = peer_address(joined + row * kRow + column, k);
      const float4 x = peer_load4(from), y = peer_load4(from + 16);
      v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    const float factor = second ? p.scale * back : kF16 ? 1.0f / 16384.0f : 1.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= factor;
    if (c < p.d) store8(static_cast<T*>(second ? p.dk : p.dv) + (((int64_t)b * p.tk + t0 + row) * p.kv_heads + head) * p.d + c, v);
  }
  cluster_meet(p.splits);
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

// Into how many CTAs (a cluster of up to eight) the keys of a tile of queries are shared out where there are fewer tiles than SMs take: a CTA costs some four steps of 64 keys besides its own,
// joining two more.
struct Plan {
  int packed, blocks, splits;
};
Plan plan_of(const Sizes& s, size_t window, size_t sinks) {
  Plan p;
  const size_t group = s.heads / s.kv_heads;
  p.packed = s.queries * group <= 128 ? (int)(s.queries * group) : 0;
  p.blocks = p.packed ? 1 : (int)((s.queries + 255) / 256);
  const int64_t ctas = (int64_t)s.batch * (p.packed ? s.kv_heads : s.heads) * p.blocks, slots = attn_sms() * (s.d > 64 ? 1 : 2);
  const size_t seen = window && window + sinks + 256 < s.keys ? window + sinks + 256 : s.keys;
  const int64_t steps = (int64_t)(seen + 63) / 64;
  p.splits = 1;
  int64_t least = (ctas + slots - 1) / slots * (steps + 4);
  for (int n = 2; n <= 8 && n <= steps && ctas < slots; n *= 2) {
    const int64_t cost = (ctas * n + slots - 1) / slots * ((steps + n - 1) / n + 4) + 2;
    if (cost < least) {
      least = cost;
      p.splits = n;
    }
  }
  return p;
}
// Whether the query heads that share a tile of keys are shared out to a pair of CTAs: where there are fewer than eight tiles for each place, so that the last ones to end weigh little (16 heads on 4,
// 8192 positions of 128 values: 1038 us for both passes instead of 1091; with clusters of four, which do not fill the GPU, 1260).
int kv_splits(const Sizes& s) {
  const size_t group = s.heads / s.kv_heads, tiles = s.batch * s.kv_heads * ((s.keys + 127) / 128), slots = (size_t)attn_sms() * (s.d > 64 ? 1 : 2);
  return group % 2 == 0 && tiles < slots * 8 ? 2 : 1;
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
cudaError_t run_forward(const dev::AttnParams& p, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  constexpr int smem = dev::AttnShape<kD>::kForwardSmem;
  const cudaError_t e = allow_smem(dev::hc_attention_kernel<T, kD>, smem, &allowed, dev::AttnShape<kD>::kForwardRegisters);
  if (e != cudaSuccess) return e;
  const int64_t ctas = (int64_t)p.batch * (p.packed ? p.kv_heads : p.heads) * p.blocks * p.splits;
  return launch_with(dev::hc_attention_kernel<T, kD>, ctas, p.splits, dev::AttnShape<kD>::kForwardThreads, smem, stream, false, p);
}

// How the keys of few rows are shared out: CTAs of a cluster, and where the largest clusters have more keys than they load at once perhaps sixteen warps a CTA instead of eight, so that their rounds of
// CTAs and, in each, of loads and two more for beginning and joining are fewest.  16 x 16 heads on 4, 8196 keys of 128: 4 CTAs in one round 49 us, 8 in two 53; 12 heads of 64, 32768 keys:
// sixteen warps 25 us, eight 43.  Clusters of sixteen CTAs take 45 us instead of 79 for a single key's head with 65536 keys, but 21 instead of 16 for eight with 8192, as they do not all find room at once.
// No CTAs: the rows are not that few.
struct FewPlan {
  int splits, warps;
};
FewPlan few_plan(const Sizes& s, size_t window, size_t sinks) {
  if (s.heads / s.kv_heads * s.queries > dev::kFewRows) return {0, 0};
  const size_t reach = window && window + sinks + s.queries < s.keys ? window + sinks + s.queries : s.keys;
  const int64_t ctas = (int64_t)(s.batch * s.kv_heads);
  FewPlan p = {1, dev::kFewWarps};
  int64_t least = 0;
  for (int n = 1; n <= dev::kMostSplits; n *= 2)
    for (int w = dev::kFewWarps; w <= (n >= dev::kMostSplits ? 2 : 1) * dev::kFewWarps; w *= 2) {
      const int64_t at_once = (int64_t)n * w * dev::kFewKeys, places = attn_sms() * (w > dev::kFewWarps ? 1 : s.d > 64 ? 2 : 3);
      const int64_t cost = (ctas * n + places - 1) / places * (((int64_t)reach + at_once - 1) / at_once + 2);
      if (least == 0 || cost < least) {
        least = cost;
        p = {n, w};
      }
    }
  return p;
}
template <typename T, int kD>
cudaError_t run_few(const dev::FewRows& p, int warps, int batch, cudaStream_t stream) {
  const auto kernel = warps > dev::kFewWarps ? dev::hc_attention_few_kernel<T, kD, 2 * dev::kFewWarps> : dev::hc_attention_few_kernel<T, kD, dev::kFewWarps>;
  return launch_with(kernel, batch * p.kv_heads * p.splits, p.splits, 32 * warps, 0, stream, false, p);
}

template <typename T, int kD>
cudaError_t run_backward(dev::AttnParams& p, const hc_heads& dout, const hc_heads& v, unsigned int* most, cudaStream_t stream) {
  static unsigned long long allowed_kv = 0, allowed_q = 0;
  constexpr int smem = dev::AttnShape<kD>::kBackwardSmem, registers = dev::AttnShape<kD>::kBackwardRegisters;
  cudaError_t e = allow_smem(dev::hc_attention_backward_kernel<T, kD, true>, smem, &allowed_kv, registers);
  if (e == cudaSuccess) e = allow_smem(dev::hc_attention_backward_kernel<T, kD, false>, smem, &allowed_q, registers);
  if (e != cudaSuccess) return e;
  if (most) {
    constexpr int kLanes = kD / 8, kRows = 4 * 256 / kLanes;  // of a block
    const dev::RowsOf of = {{dout.data, v.data},
                            {(int64_t)dout.batch, (int64_t)v.batch},
                            {(int64_t)dout.head, (int64_t)v.head},
                            {(int64_t)dout.position, (int64_t)v.position},
                            {p.heads, p.kv_heads},
                            {p.tq, p.tk},
                            {(p.tq + kRows - 1) / kRows, (p.tk + kRows - 1) / kRows},
                            (int64_t)p.batch * p.heads * ((p.tq + kRows - 1) / kRows)};
    dev::hc_attention_rows_kernel<T, kLanes><<<(unsigned)(of.first_blocks + (int64_t)p.batch * p.kv_heads * of.blocks[1]), 256, 0, stream>>>(of, p.d, most);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  // dq or not: the keys' pass needs the delta that this one completes
  const int splits = p.splits;
  p.splits = 1;
  p.blocks = (p.tq + dev::kTile - 1) / dev::kTile;
  e = launch_with(dev::hc_attention_backward_kernel<T, kD, false>, (int64_t)p.batch * p.heads * p.blocks, 1, dev::AttnShape<kD>::kBackwardThreads, smem, stream, most != nullptr, p);
  if (e != cudaSuccess || !p.dk) return e;
  p.splits = splits;
  p.blocks = (p.tk + dev::kTile - 1) / dev::kTile;
  // beside the queries' pass: 8 x 12 heads of 64, 1024 positions, bf16, all three kernels 151 us, 155 without
  return launch_with(dev::hc_attention_backward_kernel<T, kD, true>, (int64_t)p.batch * p.kv_heads * p.blocks * splits, splits, dev::AttnShape<kD>::kBackwardThreads, smem, stream, true, p);
}

// delta, and behind it what fp16's powers of two are made of
size_t delta_bytes(const Sizes& s) { return up(s.batch * s.heads * stats_ld(s.queries) * sizeof(float), 256); }
size_t most_bytes(const Sizes& s) { return s.batch * s.kv_heads * 2 * sizeof(unsigned int); }
size_t backward_bytes(const Sizes& s) { return delta_bytes(s) + up(most_bytes(s), 256); }

}  // namespace

int attention_status(int clear) { return take_status(dev::g_attention_status, clear); }

}  // namespace hc

extern "C" {

size_t hc_attention_stats(size_t batch, size_t heads, size_t queries) { return batch * heads * hc::stats_ld(queries); }

int hc_attention(hc_heads q, hc_heads k, hc_heads v, int type, void* out, float* stats, size_t batch, size_t heads, size_t kv_heads, size_t queries, size_t keys, size_t head_size,
                 size_t window, size_t sinks, float scale, hc_stream_t stream) {
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
  if (const FewPlan few = few_plan(s, window, sinks); few.splits) {
    dev::AttnParams all;
    fill_attention(&all, s, window, sinks, scale);
    const int bits = few.splits == 1 ? 0 : few.splits == 2 ? 1 : few.splits == 4 ? 2 : 3;
    const dev::FewRows p = {q.data, k.data, v.data, (int64_t)q.batch, (int64_t)q.head, (int64_t)q.position, (int64_t)k.batch, (int64_t)k.head, (int64_t)k.position, (int64_t)v.batch,
                            (int64_t)v.head, (int64_t)v.position, out, stats, all.less_ld, all.heads, all.kv_heads, all.group, all.tq, all.d, all.off, all.window, all.sinks, few.splits, bits,
                            (unsigned)((65536 + queries - 1) / queries), all.scale2};
    const auto run = type == kBf16 ? head_size <= 64 ? run_few<__nv_bfloat16, 64> : run_few<__nv_bfloat16, 128> : head_size <= 64 ? run_few<__half, 64> : run_few<__half, 128>;
    return run(p, few.warps, all.batch, stream) == cudaSuccess ? kOk : kErrCuda;
  }
  const Plan plan = plan_of(s, window, sinks);
  dev::AttnParams p;
  fill_attention(&p, s, window, sinks, scale);
  p.packed = plan.packed;
  p.blocks = plan.blocks;
  p.splits = plan.splits;
  p.o = out;
  p.less = stats;
  if (!make_head_map(&p.q, type, q, head_size, queries, heads, batch, plan.packed ? (int)queries : dev::kTile, plan.packed ? p.group : 1) ||
      !make_head_map(&p.k, type, k, head_size, keys, kv_heads, batch, dev::kStep, 1) || !make_head_map(&p.v, type, v, head_size, keys, kv_heads, batch, dev::kStep, 1))
    return kErrArgument;
  cudaError_t e;
  if (type == kBf16) e = head_size <= 64 ? run_forward<__nv_bfloat16, 64>(p, stream) : run_forward<__nv_bfloat16, 128>(p, stream);
  else e = head_size <= 64 ? run_forward<__half, 64>(p, stream) : run_forward<__half, 128>(p, stream);
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
  unsigned int* most = type == kF16 ? reinterpret_cast<unsigned int*>(static_cast<unsigned char*>(scratch) + delta_bytes(s)) : nullptr;
  if (most && cudaMemsetAsync(most, 0, most_bytes(s), stream) != cudaSuccess) return kErrCuda;
  p.less = const_cast<float*>(stats);
  p.delta = static_cast<float*>(scratch);
  p.o = const_cast<void*>(out);
  p.most = most;
  p.dq = dq, p.dk = dk, p.dv = dv;
  p.splits = kv_splits(s);
  const auto map = [&](CUtensorMap* m, const hc_heads& t, size_t length, size_t of, int rows) { return make_head_map(m, type, t, head_size, length, of, batch, rows, 1); };
  if (!map(&p.q, q, queries, heads, dev::kStep) || !map(&p.q_tile, q, queries, heads, dev::kTile) || !map(&p.dout, dout, queries, heads, dev::kStep) ||
      !map(&p.dout_tile, dout, queries, heads, dev::kTile) || !map(&p.k, k, keys, kv_heads, dev::kStep) || !map(&p.k_tile, k, keys, kv_heads, dev::kTile) ||
      !map(&p.v, v, keys, kv_heads, dev::kStep) || !map(&p.v_tile, v, keys, kv_heads, dev::kTile))
    return kErrArgument;
  cudaError_t e;
  if (type == kBf16) e = head_size <= 64 ? run_backward<__nv_bfloat16, 64>(p, dout, v, most, stream) : run_backward<__nv_bfloat16, 128>(p, dout, v, most, stream);
  else e = head_size <= 64 ? run_backward<__half, 64>(p, dout, v, most, stream) : run_backward<__half, 128>(p, dout, v, most, stream);
  return e == cudaSuccess ? kOk : kErrCuda;
}

}  // extern "C"
