// out[m, n] = sum over k of a[m, k] b[n, k] on tcgen05 tensor cores, for the operators that are products.
//
// Two SMs work on a tile of 256 x BN together (or one on 128 x 64, for small results): each loads its 128 rows of the first
// operand and one half of the second, and the matrix instruction reads both halves.  An SM loads 64 bytes a cycle at most,
// which is what 256 x 256 takes at full rate (a tile of 128 x 256 on one SM takes 96: 8192 x 4096 x 8192 ran at 1.18 PFLOP/s).
// One CTA per SM goes through tiles: one thread brings operands in by TMA (128-byte swizzle, 64 of the sum at a time, as many
// stages as shared memory holds), one issues the matrix instructions (fp32 accumulators in tensor memory, two of them, so that
// a tile is stored while the next one is computed), eight warps store.  An operand may lie along the sum or across it: boxes
// and descriptors differ, the data is not moved, so the products of a backward pass need no transposed copies.
//
// Results leave through shared memory: a warp puts 32 rows of 32 values there (swizzled, so that no two of its threads meet
// in a bank) and one TMA store takes them; what is added to a result comes in the same way, one piece ahead, and is
// overwritten by the result in place.  Stored from registers, a row a thread, the projection 8192 x 2304 x 768 took 101 us.
#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kBM = 128, kBK = 64;  // rows of a CTA, part of the sum in a stage
constexpr int kStoreWarps = 8;
constexpr int kGemmThreads = 64 + 32 * kStoreWarps;
constexpr int kOperandA = kBM * kBK * 2;
constexpr int kGemmLinearWide = 4;  // kGemmLinear whose sums are formed in parts
constexpr int kGemmGramWide = 5;    // kGemmGram, the same
constexpr uint64_t kGemmLimitNs = 2000ull * 1000 * 1000;

struct GemmParams {
  CUtensorMap map_a, map_b;
  CUtensorMap map_out, map_out2, map_in, map_in2;  // boxes of 32 x 32 values; of those that tma_* names
  CUtensorMap map_mirror;                          // the same of a symmetric result, without swizzle
  int64_t m, n;
  int k_blocks;
  int tiles_m, tiles_n, tiles;  // of one matrix
  int batch;
  int parts;  // of the sum, in the place of a batch
  int a_across, b_across;  // the operand lies across the sum: boxes of 64 values across it
  uint32_t idesc;
  uint64_t desc_a, desc_b;    // without the address
  uint32_t step_a, step_b;    // from one 16 of the sum to the next, in 16 bytes
  GemmSide out, out2, in, in2;
  int out_type, type;
  const void* bias;
  int bias_type, activation;
  float ca, cb, cc;
  const float* scale;
  const unsigned int* most;
  int tma_out, tma_out2, tma_in, tma_in2;              // moved by TMA: rows that begin at 16 bytes
  int wide_boxes;                                      // map_out and map_out2 are of boxes of 32 x 64 values
};

__device__ unsigned int g_train_status;

constexpr int kSlot = 4096;            // 32 x 32 values of 4 bytes, or two of 2 bytes
constexpr int kWarpStage = 2 * kSlot;  // of each storing warp

// kCtas: 2 work on a tile, or 1
template <int BN, int kCtas>
struct GemmShape {
  static constexpr int kB = BN / kCtas;  // rows of the second operand in a CTA
  static constexpr int kStage = kOperandA + kB * kBK * 2;
  static constexpr int kStages = kStage > 24 * 1024 ? 5 : 6;
  static constexpr int kSmem = kStages * kStage + kStoreWarps * kWarpStage + 1024;
  static constexpr int kColumns = 2 * BN;  // of tensor memory
  static constexpr int kRows = kBM * kCtas;
};

struct GemmBarriers {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drained, stage_done, stage_go;
  uint64_t loaded[kStoreWarps][2];
  alignas(16) float bias[kStoreWarps][32];
  uint32_t tmem;
  uint32_t gave_up;
};

// Addresses of the cluster's shared memory: a CTA's own are valid as they are.
__device__ __forceinline__ uint32_t leader_address(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// bytes are counted at a barrier of this CTA or, in a pair, of the first one
template <int kCtas>
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if (kCtas == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives at the barrier, in a pair at both CTAs', when the matrix instructions so far are done
template <int kCtas>
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  if (kCtas == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int kCtas>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if (kCtas == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// 32 columns of this warp's 32 rows: thread i has row i.  The values are there after tc_load_wait.
__device__ __forceinline__ void tc_load32(uint32_t addr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_load_wait(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));  // no use of a value moves in front of the wait
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z, const void* src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z),
               "r"(smem_u32(src))
               : "memory");
}

// A wait that ends: with the barrier, after the limit, or because another role has given up.
__device__ __forceinline__ bool gemm_wait(uint64_t* bar, uint32_t parity, GemmBarriers& sh) {
  long long t0 = 0;
#pragma unroll 1
  for (uint32_t it = 0; !mbar_try_wait(bar, parity); ++it) {
    if ((it & 63u) == 0u) {
      const long long now = clock64();
      if (it == 0u) t0 = now;
      if (*reinterpret_cast<volatile uint32_t*>(&sh.gave_up)) return false;
      if (now - t0 > (long long)kGemmLimitNs * 2 || it >= (1u << 26)) {
        *reinterpret_cast<volatile uint32_t*>(&sh.gave_up) = 1;
        atomicMax(&g_train_status, 3u);
        return false;
      }
    }
  }
  return true;
}

// Tile t of a matrix.  Symmetric results: only tiles that reach the diagonal or below it.  Others: 16 rows of tiles at a
// time, so that the tiles at work share their operands in L2.
template <int BN, int kRows, int MODE>
__device__ __forceinline__ void tile_place(const GemmParams& p, int t, int& mi, int& ni) {
  if (MODE == kGemmGram || MODE == kGemmGramWide || MODE == kGemmPoly) {
    mi = 0;
    for (;;) {
      int count = (mi * kRows + kRows - 1) / BN + 1;
      if (count > p.tiles_n) count = p.tiles_n;
      if (t < count) break;
      t -= count;
      ++mi;
    }
    ni = t;
  } else {
    const int per = 16 * p.tiles_n, group = t / per, r = t - group * per;
    const int rows = min(16, p.tiles_m - group * 16);
    mi = group * 16 + r % rows;
    ni = r / rows;
  }
}

template <int kAct>
__device__ __forceinline__ void activate_all(float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) activate_pair<kAct>(v[j], v[j + 1]);
}

constexpr float kLow = 2048.0f;  // lo is held times this: as precise next to hi as fp16 can be

// 16 bytes of row `lane` of a swizzled piece: rows of 128 bytes (fp32) or 64
__device__ __forceinline__ float4* wide_at(unsigned char* piece, int lane, int i) {
  return reinterpret_cast<float4*>(piece + lane * 128 + ((i ^ (lane & 7)) << 4));
}
__device__ __forceinline__ uint4* half_at(unsigned char* piece, int lane, int i) {
  return reinterpret_cast<uint4*>(piece + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4));
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  unpack2<T>(w.x, v[0], v[1]);
  unpack2<T>(w.y, v[2], v[3]);
  unpack2<T>(w.z, v[4], v[5]);
  unpack2<T>(w.w, v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
__device__ __forceinline__ uint4 pack8_as(const float* v, int type) {
  return type == kBf16 ? pack8<__nv_bfloat16>(v) : pack8<__half>(v);
}

// One piece of a result: 32 rows from `row0`, 32 columns from `col0` of matrix z, in v (thread i has row i).  `slot` has
// what TMA has brought for it, and what TMA is to take away is put there; `bias`: of this thread's column.
template <int MODE>
__device__ __forceinline__ void gemm_finish(const GemmParams& p, int z, int row0, int col0, float (&v)[32], unsigned char* slot, float bias,
                                            float* shared_bias, bool mirror) {
  const int lane = threadIdx.x & 31;
  const int64_t row = row0 + lane;
  const int64_t count = row < p.m ? p.n - col0 : 0;  // columns of this row (may be over 32)
  unsigned char* second = slot + kSlot / 2;
  if (MODE == kGemmLinear) {
    if (p.most) {
      const float power = gradient_power(p.most, -1);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= power;
    }
    if (p.bias) {
      shared_bias[lane] = bias;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 b = *reinterpret_cast<const float4*>(shared_bias + j);
        v[j] += b.x, v[j + 1] += b.y, v[j + 2] += b.z, v[j + 3] += b.w;
      }
    }
    if (p.tma_out2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *half_at(second, lane, i) = pack8_as(v + i * 8, p.type);
    } else if (p.out2.data) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) param_put(p.out2.data, p.type, row * p.out2.ld + col0 + j, v[j]);
    }
    if (p.activation == kActGeluTanh) activate_all<kActGeluTanh>(v);
    else if (p.activation == kActRelu) activate_all<kActRelu>(v);
    else if (p.activation == kActSilu) activate_all<kActSilu>(v);
    if (p.in.data && !p.tma_in) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) v[j] += param_at(p.in.data, p.out_type, row * p.in.ld + col0 + j);
    }
    if (p.out_type == kF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float4* at = wide_at(slot, lane, i);
        if (p.tma_in) {
          const float4 r = *at;
          v[i * 4] += r.x, v[i * 4 + 1] += r.y, v[i * 4 + 2] += r.z, v[i * 4 + 3] += r.w;
        }
        if (p.tma_out) *at = make_float4(v[i * 4], v[i * 4 + 1], v[i * 4 + 2], v[i * 4 + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4* at = half_at(slot, lane, i);
        if (p.tma_in) {
          float r[8];
          if (p.type == kBf16) unpack8<__nv_bfloat16>(*at, r);
          else unpack8<__half>(*at, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i * 8 + j] += r[j];
        }
        if (p.tma_out) *at = pack8_as(v + i * 8, p.type);
      }
    }
    if (!p.tma_out) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) param_put(p.out.data, p.out_type, row * p.out.ld + col0 + j, v[j]);
    }
  } else if (MODE == kGemmUpdate) {
    const bool last = !p.out2.data;
    const float scale = last ? p.scale[z] : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 *at = half_at(slot, lane, i), *at2 = half_at(second, lane, i);
      float hi[8], lo[8];
      unpack8<__half>(*at, hi);
      unpack8<__half>(*at2, lo);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i * 8 + j] = fmaf(p.ca, fmaf(lo[j], 1.0f / kLow, hi[j]), v[i * 8 + j]) * scale;
      if (!last) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hi[j] = to_float(__float2half_rn(v[i * 8 + j]));
          lo[j] = (v[i * 8 + j] - hi[j]) * kLow;
        }
        *at = pack8<__half>(hi);
        *at2 = pack8<__half>(lo);
      } else if (p.tma_out) {
        *at = pack8<__nv_bfloat16>(v + i * 8);
      }
    }
    if (!p.tma_out) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) param_put(p.out.data, kBf16, z * p.out.stride + row * p.out.ld + col0 + j, v[j]);
    }
  } else {
    const float square = MODE == kGemmPoly ? p.scale[z] * p.scale[z] : 0.0f, c1 = p.cb * square, c2 = p.cc * square * square;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4* at = half_at(slot, lane, i);
      if (MODE == kGemmPoly) {
        float q[8];
        unpack8<__half>(*at, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i * 8 + j] = fmaf(c2, v[i * 8 + j], c1 * q[j]);
      }
      *at = pack8<__half>(v + i * 8);
    }
    if (mirror) {  // not swizzled: the threads of a warp write neighbours
      __half* t = reinterpret_cast<__half*>(second) + lane;
#pragma unroll
      for (int j = 0; j < 32; ++j) t[j * 32] = __float2half_rn(v[j]);
    }
  }
}

// brings what is added to the result at (row0, col0) into a slot
template <int MODE>
__device__ __forceinline__ void gemm_fetch(const GemmParams& p, int z, int row0, int col0, unsigned char* slot, uint64_t* bar) {
  const bool whole = MODE == kGemmUpdate || (MODE == kGemmLinear && p.out_type == kF32);
  mbar_expect_tx(bar, whole ? kSlot : kSlot / 2);
  load_box<1>(slot, &p.map_in, col0, row0, z, smem_u32(bar));
  if (MODE == kGemmUpdate) load_box<1>(slot + kSlot / 2, &p.map_in2, col0, row0, z, smem_u32(bar));
}

// Half of a piece of 64 columns, which only TMA stores: 32 rows of 128 bytes in `out`, what the activation is applied to in `z`.
__device__ __forceinline__ void gemm_finish_half(const GemmParams& p, float (&v)[32], int half, unsigned char* out, unsigned char* z, float bias,
                                                 float* shared_bias) {
  const int lane = threadIdx.x & 31;
  if (p.most) {
    const float power = gradient_power(p.most, -1);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= power;
  }
  if (p.bias) {
    __syncwarp();
    shared_bias[lane] = bias;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 b = *reinterpret_cast<const float4*>(shared_bias + j);
      v[j] += b.x, v[j + 1] += b.y, v[j + 2] += b.z, v[j + 3] += b.w;
    }
  }
  if (p.tma_out2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(wide_at(z, lane, half * 4 + i)) = pack8_as(v + i * 8, p.type);
  }
  if (p.activation == kActGeluTanh) activate_all<kActGeluTanh>(v);
  else if (p.activation == kActRelu) activate_all<kActRelu>(v);
  else if (p.activation == kActSilu) activate_all<kActSilu>(v);
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(wide_at(out, lane, half * 4 + i)) = pack8_as(v + i * 8, p.type);
}

// What the three roles carry from tile to tile (and, in a chain of products, from one to the next).
struct Loading {
  int s = 0, issued = 0;
  uint32_t phase = 0;
  bool ok = true;
};
struct Multiplying {
  int s = 0, acc = 0;
  uint32_t phase = 0, acc_phase = 0;
  bool ok = true;
};
struct Storing {
  int acc = 0;
  uint32_t acc_phase = 0, uses = 0;  // uses: pieces so far, which take the two slots in turn
  uint32_t phases = 0;               // of the slots' barriers, a bit each
  int on_their_way = 0;              // pieces that have been asked for and not been waited for
  bool ok = true;
};
// A result in fp32 gets its sum in parts of 1024: the tensor core does not round to nearest when it adds to an accumulator, and
// what that loses over a whole sum (6e-6 of the result over 8192) is ten times what fp32 additions do.  Where all terms are
// positive it loses 6.5e-9 of the result a term (3.4e-3 over 2^19), so 16-bit results get theirs in parts, too, where what
// is lost would come to more than a quarter of half the result's step (2^-14, 2^-11): 5.3e-5 and 4.3e-4 at the lengths below.
// Of tiles of 256 x 256 a thread then has 128 sums, and keeps 216 bytes outside of its 168 registers.
constexpr int kChunk = 16;  // stages
constexpr int64_t kLongF16 = 8192, kLongBf16 = 65536;

template <int BN, int kCtas, int MODE>
__device__ __forceinline__ void load_tiles(const GemmParams& p, GemmBarriers& sh, unsigned char* stages, Loading& st, int unit, int units, int rank) {
  using S = GemmShape<BN, kCtas>;
  const int total = p.tiles * p.batch;
  for (int t = unit; st.ok && t < total; t += units) {
    const int z = t / p.tiles;
    int mi, ni;
    tile_place<BN, S::kRows, MODE>(p, t - z * p.tiles, mi, ni);
    const int row = mi * S::kRows + rank * kBM, col = ni * BN + rank * S::kB;
    const int zz = p.parts > 1 ? 0 : z, k0 = p.parts > 1 ? z * p.k_blocks : 0;
    for (int kb = 0; kb < p.k_blocks; ++kb) {
      const int k = (k0 + kb) * kBK;
      if (!gemm_wait(&sh.empty[st.s], st.phase ^ 1, sh)) {
        st.ok = false;
        break;
      }
      unsigned char* a = stages + st.s * S::kStage;
      unsigned char* b = a + kOperandA;
      const uint32_t bar = kCtas == 2 ? leader_address(&sh.full[st.s]) : smem_u32(&sh.full[st.s]);
      if (rank == 0) mbar_expect_tx(&sh.full[st.s], S::kStage * kCtas);
      if (p.a_across) {
        for (int i = 0; i < kBM / 64; ++i) load_box<kCtas>(a + i * 8192, &p.map_a, row + i * 64, k, zz, bar);
      } else {
        load_box<kCtas>(a, &p.map_a, k, row, zz, bar);
      }
      if (p.b_across) {
        for (int i = 0; i < S::kB / 64; ++i) load_box<kCtas>(b + i * 8192, &p.map_b, col + i * 64, k, zz, bar);
      } else {
        load_box<kCtas>(b, &p.map_b, k, col, zz, bar);
      }
      ++st.issued;
      if (++st.s == S::kStages) {
        st.s = 0;
        st.phase ^= 1;
      }
    }
  }
}
// Copies in flight land before the CTA leaves.  Those of a pair are counted at its first CTA; the second one leaves behind it,
// and after a wait that ran out, when they may differ in what they have issued, a millisecond later.
template <int BN, int kCtas>
__device__ __forceinline__ void load_end(GemmBarriers& sh, const Loading& st, int rank) {
  using S = GemmShape<BN, kCtas>;
  if (rank == 0) {
    for (int back = 0; back < S::kStages && back < st.issued; ++back) {
      const int i = st.issued - 1 - back;
      mbar_wait_bounded(&sh.full[i % S::kStages], (i / S::kStages) & 1, kGemmLimitNs);
    }
  } else if (!st.ok) {
    const long long t0 = clock64();
    for (int i = 0; i < (1 << 22) && clock64() - t0 < 2000000; ++i) {
    }
  }
}

template <int BN, int kCtas, int MODE>
__device__ __forceinline__ void multiply_tiles(const GemmParams& p, GemmBarriers& sh, unsigned char* stages, Multiplying& st, uint32_t tmem, int unit, int units) {
  using S = GemmShape<BN, kCtas>;
  const int total = p.tiles * p.batch;
  for (int t = unit; st.ok && t < total; t += units) {
    for (int begin = 0; begin < p.k_blocks; begin += kChunk) {
      const int end = MODE == kGemmLinearWide || MODE == kGemmGramWide ? min(begin + kChunk, p.k_blocks) : p.k_blocks;
      if (!gemm_wait(&sh.acc_empty[st.acc], st.acc_phase ^ 1, sh)) {
        st.ok = false;
        return;
      }
      tc_fence_after();
      const uint32_t d = tmem + st.acc * BN;
      for (int kb = begin; kb < end; ++kb) {
        if (!gemm_wait(&sh.full[st.s], st.phase, sh)) {
          st.ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = smem_u32(stages + st.s * S::kStage);
        const uint64_t da = p.desc_a | (uint64_t)((a & 0x3ffff) >> 4), db = p.desc_b | (uint64_t)(((a + kOperandA) & 0x3ffff) >> 4);
#pragma unroll
        for (int i = 0; i < kBK / 16; ++i) tc_mma<kCtas>(d, da + i * p.step_a, db + i * p.step_b, p.idesc, kb > begin || i > 0);
        tc_commit<kCtas>(&sh.empty[st.s]);
        if (++st.s == S::kStages) {
          st.s = 0;
          st.phase ^= 1;
        }
      }
      tc_commit<kCtas>(&sh.acc_full[st.acc]);
      if (++st.acc == 2) {
        st.acc = 0;
        st.acc_phase ^= 1;
      }
      if (!st.ok || end == p.k_blocks) break;
    }
  }
}

// the accumulator has been read
template <int kCtas>
__device__ __forceinline__ void release_accumulator(GemmBarriers& sh, Storing& st, int rank) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if (rank == 0) mbar_arrive(&sh.acc_empty[st.acc]);
    else
      asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_address(&sh.acc_empty[st.acc])) : "memory");
  }
  if (++st.acc == 2) {
    st.acc = 0;
    st.acc_phase ^= 1;
  }
}

template <int BN, int kCtas, int MODE>
__device__ __forceinline__ void store_tiles(const GemmParams& p, GemmBarriers& sh, unsigned char* mine, Storing& st, uint32_t tmem, int unit, int units, int rank) {
  using S = GemmShape<BN, kCtas>;
  constexpr bool kWide = MODE == kGemmLinearWide || MODE == kGemmGramWide, kLinear = MODE == kGemmLinear || MODE == kGemmLinearWide;
  constexpr bool kSymmetric = MODE == kGemmGram || MODE == kGemmGramWide || MODE == kGemmPoly;
  constexpr int kMode = MODE == kGemmLinearWide ? kGemmLinear : MODE == kGemmGramWide ? kGemmGram : MODE;
  constexpr int kPieces = kWide ? (BN / 32 + 1) / 2 : 1;  // of a warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3;      // the rows of tensor memory that this warp can reach
  const int half = (warp - 2) >> 2;  // every second piece of 32 columns
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  uint64_t* loaded = sh.loaded[warp - 2];
  float* shared_bias = sh.bias[warp - 2];
  const bool fetches = MODE == kGemmPoly || MODE == kGemmUpdate || (kLinear && p.tma_in);
  const int total = p.tiles * p.batch;
  for (int t = unit; t < total; t += units) {
    const int z = t / p.tiles;
    int mi, ni;
    tile_place<BN, S::kRows, MODE>(p, t - z * p.tiles, mi, ni);
    const int row0 = mi * S::kRows + rank * kBM + quarter * 32, col0 = ni * BN;
    // pieces of these rows that hold something (of a symmetric result: at the diagonal of blocks of 32, or below it)
    int pieces = row0 < p.m ? (int)min((int64_t)(BN / 32), (p.n - col0 + 31) / 32) : 0;
    if (kSymmetric && pieces) pieces = min(pieces, row0 / 32 - col0 / 32 + 1);
    float bias = 0.0f;
    if (half < pieces && !(MODE == kGemmLinear && BN >= 128 && p.wide_boxes)) {
      if (fetches && lane == 0) {
        tma_wait_group_read<0>();
        gemm_fetch<kMode>(p, z, row0, col0 + half * 32, mine + (st.uses & 1) * kSlot, &loaded[st.uses & 1]);
        ++st.on_their_way;
      }
      if (kLinear && p.bias && col0 + half * 32 + lane < p.n) bias = param_at(p.bias, p.bias_type, col0 + half * 32 + lane);
    }
    float sums[kPieces][32];
    if (kWide) {
#pragma unroll
      for (int q = 0; q < kPieces; ++q)
#pragma unroll
        for (int j = 0; j < 32; ++j) sums[q][j] = 0.0f;
      for (int begin = 0; begin < p.k_blocks; begin += kChunk) {
        if (!__all_sync(0xffffffffu, gemm_wait(&sh.acc_full[st.acc], st.acc_phase, sh))) {
          st.ok = false;
          return;
        }
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
          if (half + 2 * q >= pieces) break;
          float v[32];
          __syncwarp();
          tc_load32(lanes + st.acc * BN + (half + 2 * q) * 32, v);
          tc_load_wait(v);
#pragma unroll
          for (int j = 0; j < 32; ++j) sums[q][j] += v[j];
        }
        release_accumulator<kCtas>(sh, st, rank);
      }
    } else {
      if (!__all_sync(0xffffffffu, gemm_wait(&sh.acc_full[st.acc], st.acc_phase, sh))) {
        st.ok = false;
        return;
      }
      tc_fence_after();
    }
    const auto piece = [&](int c, float (&v)[32]) {  // false: a wait ran out
      const int col = col0 + c * 32;
      unsigned char* slot = mine + (st.uses & 1) * kSlot;
      float next_bias = 0.0f;
      if (c + 2 < pieces) {
        if (fetches && lane == 0) {
          tma_wait_group_read<0>();
          gemm_fetch<kMode>(p, z, row0, col + 64, mine + ((st.uses + 1) & 1) * kSlot, &loaded[(st.uses + 1) & 1]);
          ++st.on_their_way;
        }
        if (kLinear && p.bias && col + 64 + lane < p.n) next_bias = param_at(p.bias, p.bias_type, col + 64 + lane);
      }
      if (!fetches && lane == 0) tma_wait_group_read<1>();
      __syncwarp();
      if (!kWide) {
        tc_load32(lanes + st.acc * BN + c * 32, v);
        tc_load_wait(v);
      }
      if (fetches) {
        const uint32_t slot_number = st.uses & 1;
        if (!__all_sync(0xffffffffu, gemm_wait(&loaded[slot_number], st.phases >> slot_number & 1, sh))) return false;
        st.phases ^= 1u << slot_number;
        --st.on_their_way;
      }
      const bool mirror = kSymmetric && col / 32 < row0 / 32;
      gemm_finish<kMode>(p, z, row0, col, v, slot, bias, shared_bias, mirror);
      bias = next_bias;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        if (p.tma_out) tma_store_3d(&p.map_out, col, row0, z, slot);
        if (p.tma_out2) tma_store_3d(&p.map_out2, col, row0, z, slot + kSlot / 2);
        if (mirror) tma_store_3d(&p.map_mirror, row0, col, z, slot + kSlot / 2);
        tma_commit_group();
      }
      ++st.uses;
      return true;
    };
    if (kWide) {
#pragma unroll 1
      for (int q = 0; half + 2 * q < pieces; ++q) {  // not unrolled: what is done to a piece is long
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          v[j] = sums[0][j];
#pragma unroll
          for (int k = 1; k < kPieces; ++k) v[j] = q == k ? sums[k][j] : v[j];
        }
        if (!piece(half + 2 * q, v)) {
          st.ok = false;
          return;
        }
      }
    } else if (MODE == kGemmLinear && BN >= 128 && p.wide_boxes) {
      // Half as many pieces and rows of boxes: what a piece costs besides its values (waits, the fence, the store's issue, some
      // 1300 of 2200 cycles) is what bounds short sums (8192 x 64 -> 2304: 16.5 us instead of 23.3, 8192 x 768 -> 2304: 29 and 32).
#pragma unroll 1
      for (int c = half * 2; c < pieces; c += 4) {
        const int col = col0 + c * 32;
        float bias2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (p.bias && col + h * 32 + lane < p.n) bias2[h] = param_at(p.bias, p.bias_type, col + h * 32 + lane);
        unsigned char* slot = p.tma_out2 ? mine : mine + (st.uses & 1) * kSlot;
        if (lane == 0) {
          if (p.tma_out2) tma_wait_group_read<0>();
          else tma_wait_group_read<1>();
        }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tc_load32(lanes + st.acc * BN + (c + h) * 32, sums[0]);
          tc_load_wait(sums[0]);
          gemm_finish_half(p, sums[0], h, slot, mine + kSlot, bias2[h], shared_bias);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(&p.map_out, col, row0, z, slot);
          if (p.tma_out2) tma_store_3d(&p.map_out2, col, row0, z, mine + kSlot);
          tma_commit_group();
        }
        ++st.uses;
      }
      release_accumulator<kCtas>(sh, st, rank);
    } else {
#pragma unroll 1
      for (int c = half; c < pieces; c += 2) {
        if (!piece(c, sums[0])) {
          st.ok = false;
          return;
        }
      }
      release_accumulator<kCtas>(sh, st, rank);
    }
  }
}
// what was fetched and not used (after a wait that ran out) lands before the CTA leaves, and all stores have read what they
// take from its shared memory
__device__ __forceinline__ void store_end(GemmBarriers& sh, Storing& st) {
  if ((threadIdx.x & 31) != 0) return;
  uint64_t* loaded = sh.loaded[(threadIdx.x >> 5) - 2];
  for (; st.on_their_way > 0; --st.on_their_way, ++st.uses) {
    mbar_wait_bounded(&loaded[st.uses & 1], st.phases >> (st.uses & 1) & 1, kGemmLimitNs);
    st.phases ^= 1u << (st.uses & 1);
  }
  tma_wait_group_read<0>();
}

// barriers and tensor memory; by all threads
template <int BN, int kCtas>
__device__ __forceinline__ void gemm_begin(GemmBarriers& sh) {
  using S = GemmShape<BN, kCtas>;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sh.acc_full[a], 1);
      mbar_init(&sh.acc_empty[a], kStoreWarps * kCtas);
    }
    mbar_init(&sh.drained, 1);
    mbar_init(&sh.stage_done, kStoreWarps);
    mbar_init(&sh.stage_go, 1);
    for (int w = 0; w < kStoreWarps; ++w) {
      mbar_init(&sh.loaded[w][0], 1);
      mbar_init(&sh.loaded[w][1], 1);
    }
    sh.gave_up = 0;
    fence_mbar_init();
  }
  if (threadIdx.x >> 5 == 1) {
    if (kCtas == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(S::kColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(S::kColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (kCtas == 2) cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
}
template <int BN, int kCtas>
__device__ __forceinline__ void gemm_end(uint32_t tmem) {
  using S = GemmShape<BN, kCtas>;
  __syncthreads();
  if (kCtas == 2) cluster_sync();  // nobody leaves while the other one's memory is read or its barriers are used
  if (threadIdx.x >> 5 == 1) {
    __syncwarp();
    tc_fence_after();
    if (kCtas == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kColumns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kColumns));
  }
}
__device__ __forceinline__ unsigned char* gemm_stages(unsigned char* raw) {
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
}

template <int BN, int kCtas, int MODE>
__global__ void __launch_bounds__(kGemmThreads, 1) hc_gemm_kernel(const __grid_constant__ GemmParams p) {
  using S = GemmShape<BN, kCtas>;
  extern __shared__ unsigned char raw[];
  __shared__ GemmBarriers sh;
  unsigned char* stages = gemm_stages(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kCtas == 2 ? (int)(blockIdx.x & 1) : 0;  // in the pair; the first one issues the matrix instructions
  const int unit = blockIdx.x / kCtas, units = gridDim.x / kCtas;
  if (threadIdx.x == 0) {
    tma_prefetch_map(&p.map_a);
    tma_prefetch_map(&p.map_b);
  }
  gemm_begin<BN, kCtas>(sh);
  const uint32_t tmem = sh.tmem;
  if (warp == 0) {
    if (lane == 0) {
      Loading st;
      load_tiles<BN, kCtas, MODE>(p, sh, stages, st, unit, units, rank);
      load_end<BN, kCtas>(sh, st, rank);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      Multiplying st;
      multiply_tiles<BN, kCtas, MODE>(p, sh, stages, st, tmem, unit, units);
      // matrix instructions in flight are done before the CTA leaves, too
      tc_commit<kCtas>(&sh.drained);
      mbar_wait_bounded(&sh.drained, 0, kGemmLimitNs);
    }
  } else {
    Storing st;
    store_tiles<BN, kCtas, MODE>(p, sh, stages + S::kStages * S::kStage + (warp - 2) * kWarpStage, st, tmem, unit, units, rank);
    store_end(sh, st);
  }
  gemm_end<BN, kCtas>(tmem);
}

// ---- all products of a Newton-Schulz iteration in one launch -----------------------------------------------------------
// Each product needs all of the one before it, so the CTAs, which are all on the GPU (a cooperative launch), meet between them:
// a CTA whose stores are complete adds one to a counter and waits, with a limit, until all have.
struct ChainParams {
  GemmParams gram[2], poly, update[2], last;
  int steps;
  unsigned int* arrived;  // 0 at the start
};

// by the loading thread, between product number `stage` and the next
__device__ __forceinline__ bool meet(GemmBarriers& sh, unsigned int* arrived, int stage) {
  if (!gemm_wait(&sh.stage_done, stage & 1, sh)) return false;
  asm volatile("fence.proxy.async;" ::: "memory");
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(arrived) : "memory");
  const unsigned int want = gridDim.x * (unsigned)(stage + 1);
  const long long t0 = clock64();
  for (uint32_t it = 0;; ++it) {
    unsigned int n;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(arrived) : "memory");
    if (n >= want) break;
    if (*reinterpret_cast<volatile uint32_t*>(&sh.gave_up)) return false;
    if (clock64() - t0 > (long long)kGemmLimitNs * 2 || it >= (1u << 28)) {
      *reinterpret_cast<volatile uint32_t*>(&sh.gave_up) = 1;
      atomicMax(&g_train_status, 3u);
      return false;
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");
  mbar_arrive(&sh.stage_go);
  return true;
}

template <int BN, int kCtas, bool kLong>  // kLong: the long side is beyond kLongF16
__global__ void __launch_bounds__(kGemmThreads, 1) hc_gemm_chain_kernel(const __grid_constant__ ChainParams c) {
  using S = GemmShape<BN, kCtas>;
  constexpr int kGram = kLong ? kGemmGramWide : kGemmGram;
  extern __shared__ unsigned char raw[];
  __shared__ GemmBarriers sh;
  unsigned char* stages = gemm_stages(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kCtas == 2 ? (int)(blockIdx.x & 1) : 0;
  const int unit = blockIdx.x / kCtas, units = gridDim.x / kCtas;
  gemm_begin<BN, kCtas>(sh);
  const uint32_t tmem = sh.tmem;
  const int products = 3 * c.steps;
  if (warp == 0) {
    if (lane == 0) {
      Loading st;
      for (int i = 0; i < products && st.ok; ++i) {
        const int step = i / 3;
        if (i % 3 == 0) load_tiles<BN, kCtas, kGram>(c.gram[step & 1], sh, stages, st, unit, units, rank);
        else if (i % 3 == 1) load_tiles<BN, kCtas, kGemmPoly>(c.poly, sh, stages, st, unit, units, rank);
        else load_tiles<BN, kCtas, kGemmUpdate>(step == c.steps - 1 ? c.last : c.update[step & 1], sh, stages, st, unit, units, rank);
        if (st.ok && i + 1 < products) st.ok = meet(sh, c.arrived, i);
      }
      load_end<BN, kCtas>(sh, st, rank);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      Multiplying st;
      for (int i = 0; i < products && st.ok; ++i) {
        const int step = i / 3;
        if (i % 3 == 0) multiply_tiles<BN, kCtas, kGram>(c.gram[step & 1], sh, stages, st, tmem, unit, units);
        else if (i % 3 == 1) multiply_tiles<BN, kCtas, kGemmPoly>(c.poly, sh, stages, st, tmem, unit, units);
        else multiply_tiles<BN, kCtas, kGemmUpdate>(step == c.steps - 1 ? c.last : c.update[step & 1], sh, stages, st, tmem, unit, units);
      }
      tc_commit<kCtas>(&sh.drained);
      mbar_wait_bounded(&sh.drained, 0, kGemmLimitNs);
    }
  } else {
    Storing st;
    unsigned char* mine = stages + S::kStages * S::kStage + (warp - 2) * kWarpStage;
    for (int i = 0; i < products && st.ok; ++i) {
      const int step = i / 3;
      if (i % 3 == 0) store_tiles<BN, kCtas, kGram>(c.gram[step & 1], sh, mine, st, tmem, unit, units, rank);
      else if (i % 3 == 1) store_tiles<BN, kCtas, kGemmPoly>(c.poly, sh, mine, st, tmem, unit, units, rank);
      else store_tiles<BN, kCtas, kGemmUpdate>(step == c.steps - 1 ? c.last : c.update[step & 1], sh, mine, st, tmem, unit, units, rank);
      if (!st.ok || i + 1 == products) break;
      if (lane == 0) {
        tma_wait_group<0>();  // what this warp has stored is there
        asm volatile("fence.proxy.async;" ::: "memory");
        mbar_arrive(&sh.stage_done);
      }
      st.ok = __all_sync(0xffffffffu, gemm_wait(&sh.stage_go, i & 1, sh));
      asm volatile("fence.proxy.async;" ::: "memory");
    }
    store_end(sh, st);
  }
  gemm_end<BN, kCtas>(tmem);
}

}  // namespace dev

bool gemm_operand_ok(const void* data, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(data) & 15u) == 0 && ld % 8 == 0;
}

namespace {

// boxes of 64 x `box_rows` of a batch of row-major matrices of 16-bit values; outside of a matrix zeros are read
bool make_matrix_map(CUtensorMap* map, int type, const void* base, int64_t inner, int64_t rows, int64_t batch, int64_t ld, int64_t stride,
                     int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(batch > 1 ? stride : ld) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  cuuint32_t step[3] = {1, 1, 1};
  return fn(map, type == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box,
            step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Shared memory descriptor without its address: 128-byte swizzle; eight rows of 128 bytes are 1024 bytes, and 64 values
// across the sum a box of 8192.
uint64_t descriptor(bool k_major) {
  const uint64_t leading = k_major ? 1 : 8192 / 16, stride = 1024 / 16;
  return leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}

// A map of boxes of 32 x 32 values (`wide`: 32 x 64 of 16 bits) of something beside the accumulator, if its rows begin at 16 bytes.  TMA stores whole 16
// bytes, also at the end of a row (seen on a B200): what it stores to has rows of whole 16 bytes, or no more behind a row than
// rounds it up to eight values.
bool make_side_map(CUtensorMap* map, const GemmSide& s, int type, const GemmCall& c, bool stored, bool mirror = false, bool wide = false) {
  const size_t bytes = element_bytes(type);
  if (stored && c.n * bytes % 16 && s.ld != (c.n + 7) / 8 * 8) return false;
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn || !s.data || (reinterpret_cast<uintptr_t>(s.data) & 15u) || s.ld * bytes % 16 || (c.batch > 1 && s.stride * bytes % 16)) return false;
  cuuint64_t dims[3] = {(cuuint64_t)c.n, (cuuint64_t)c.m, (cuuint64_t)c.batch};
  cuuint64_t strides[2] = {(cuuint64_t)(s.ld * bytes), (cuuint64_t)((c.batch > 1 ? s.stride : s.ld) * bytes)};
  cuuint32_t box[3] = {wide ? 64u : 32u, 32, 1};
  cuuint32_t step[3] = {1, 1, 1};
  return fn(map, type == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            s.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            mirror ? CU_TENSOR_MAP_SWIZZLE_NONE : type == kF32 || wide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// tiles of one matrix
template <int MODE>
int64_t count_tiles(const GemmCall& c, int rows, int bn) {
  const int64_t tm = (c.m + rows - 1) / rows, tn = (c.n + bn - 1) / bn;
  if (MODE != kGemmGram && MODE != kGemmPoly) return tm * tn;
  int64_t tiles = 0;
  for (int64_t i = 0; i < tm; ++i) {
    const int64_t count = (i * rows + rows - 1) / bn + 1;
    tiles += count < tn ? count : tn;
  }
  return tiles;
}

template <int BN, int kCtas, int MODE>
cudaError_t fill_params(const GemmCall& given, dev::GemmParams* out) {
  GemmCall c = given;
  using S = dev::GemmShape<BN, kCtas>;
  dev::GemmParams& p = *out;
  memset(&p, 0, sizeof(p));
  p.m = c.m;
  p.n = c.n;
  p.k_blocks = (int)((c.k + dev::kBK - 1) / dev::kBK);
  const int64_t operands = c.batch;
  p.parts = c.parts;
  if (c.parts > 1) {
    p.k_blocks = (p.k_blocks + c.parts - 1) / c.parts;  // what a part has behind the end of the sum reads as zeros
    c.batch = c.parts;
  }
  p.tiles_m = (int)((c.m + S::kRows - 1) / S::kRows);
  p.tiles_n = (int)((c.n + BN - 1) / BN);
  p.batch = (int)c.batch;
  const int64_t tiles = count_tiles<MODE>(c, S::kRows, BN);
  if (tiles * c.batch > 1 << 30) return cudaErrorInvalidValue;
  p.tiles = (int)tiles;
  p.a_across = !c.a.k_major;
  p.b_across = !c.b.k_major;
  if (!make_matrix_map(&p.map_a, c.type, c.a.data, c.a.k_major ? c.k : c.m, c.a.k_major ? c.m : c.k, operands, c.a.ld, c.a.stride,
                       c.a.k_major ? dev::kBM : dev::kBK))
    return cudaErrorInvalidValue;
  if (!make_matrix_map(&p.map_b, c.type, c.b.data, c.b.k_major ? c.k : c.n, c.b.k_major ? c.n : c.k, operands, c.b.ld, c.b.stride,
                       c.b.k_major ? S::kB : dev::kBK))
    return cudaErrorInvalidValue;
  p.desc_a = descriptor(c.a.k_major);
  p.desc_b = descriptor(c.b.k_major);
  p.step_a = c.a.k_major ? 2 : 128;
  p.step_b = c.b.k_major ? 2 : 128;
  const uint32_t format = c.type == kBf16 ? 1u : 0u;
  p.idesc = 1u << 4 | format << 7 | format << 10 | (c.a.k_major ? 0u : 1u << 15) | (c.b.k_major ? 0u : 1u << 16) | (uint32_t)(BN / 8) << 17 |
            (uint32_t)(S::kRows / 16) << 24;
  p.out = c.out;
  p.out2 = c.out2;
  p.in = c.in;
  p.in2 = c.in2;
  p.out_type = c.out_type;
  p.type = c.type;
  p.bias = c.bias;
  p.bias_type = c.bias_type;
  p.activation = c.activation;
  p.ca = c.ca;
  p.cb = c.cb;
  p.cc = c.cc;
  p.scale = c.scale;
  p.most = c.most;
  constexpr bool kLinear = MODE == kGemmLinear || MODE == dev::kGemmLinearWide, kUpdate = MODE == kGemmUpdate;
  if (MODE == kGemmLinear && BN >= 128 && c.out_type != kF32 && !c.in.data && make_side_map(&p.map_out, c.out, c.out_type, c, true, false, true))
    p.wide_boxes = !c.out2.data || make_side_map(&p.map_out2, c.out2, c.type, c, true, false, true);
  p.tma_out = p.wide_boxes || make_side_map(&p.map_out, c.out, c.out_type, c, true);
  p.tma_out2 = c.out2.data && (kUpdate || (kLinear && c.out_type != kF32)) && (p.wide_boxes || make_side_map(&p.map_out2, c.out2, c.type, c, true));
  p.tma_in = c.in.data && make_side_map(&p.map_in, c.in, kLinear ? c.out_type : kF16, c, false);
  p.tma_in2 = kUpdate && make_side_map(&p.map_in2, c.in2, kF16, c, false);
  // the iteration's own arrays lie as TMA wants them
  if (!kLinear && ((MODE != kGemmGram && !p.tma_in) || (kUpdate && (!p.tma_in2 || (c.out2.data && (!p.tma_out || !p.tma_out2)))))) return cudaErrorInvalidValue;
  if ((MODE == kGemmGram || MODE == kGemmPoly) && (!p.tma_out || !make_side_map(&p.map_mirror, c.out, kF16, c, true, true))) return cudaErrorInvalidValue;
  return cudaSuccess;
}

// a launch of pairs of CTAs, or of single ones
template <int kCtas, typename K, typename P>
cudaError_t launch_units(K kernel, const P& p, int64_t total, int smem, bool meeting, cudaStream_t stream) {
  const int64_t units = device_info().sms / kCtas;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)((total < units ? total : units) * kCtas));
  cfg.blockDim = dim3(dev::kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  memset(attr, 0, sizeof(attr));
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeCooperative;
  attr[1].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = meeting ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int BN, int kCtas, int MODE>
cudaError_t run_gemm(const GemmCall& c, cudaStream_t stream) {
  using S = dev::GemmShape<BN, kCtas>;
  dev::GemmParams p;
  cudaError_t e = fill_params<BN, kCtas, MODE>(c, &p);
  static unsigned long long allowed = 0;
  if (e == cudaSuccess) e = allow_smem(dev::hc_gemm_kernel<BN, kCtas, MODE>, S::kSmem, &allowed);
  if (e != cudaSuccess) return e;
  return launch_units<kCtas>(dev::hc_gemm_kernel<BN, kCtas, MODE>, p, (int64_t)p.tiles * p.batch, S::kSmem, false, stream);
}

// Cycles that a launch takes: those of the unit (a pair of SMs, or one) with the most tiles.  A stage of a tile costs what the
// matrix instructions take or what loading it takes at 64 bytes a cycle, whichever is more, a tile some 1000 for its start
// and four for each of its columns.  With a single row of tiles no SM finds in L2 what another one has read, and a stage is there
// some 650 cycles after the one before it (64 rows, a sum of 8192: 44 us with 1024 columns, 47 with 8192).
int64_t sm_count() { return device_info().sms > 1 ? device_info().sms : 2; }
struct TileChoice {
  int bn, ctas;
  int64_t cost;
};
template <int MODE>
TileChoice best_tile(const GemmCall& c, int parts, int64_t sms) {
  const int64_t stages = ((c.k + dev::kBK - 1) / dev::kBK + parts - 1) / parts;
  const int shapes[3][3] = {{256, 2, 512}, {128, 2, 384}, {64, 1, 384}};
  TileChoice best = {0, 0, 0};
  for (const auto& s : shapes) {
    const int64_t tiles = count_tiles<MODE>(c, dev::kBM * s[1], s[0]) * c.batch * parts, units = sms / s[1];
    const int stage = MODE == kGemmLinear && c.m <= dev::kBM * s[1] && s[2] < 650 ? 650 : s[2];
    const int64_t cost = (tiles + units - 1) / units * (stages * stage + 1000 + 4 * s[0]);
    if (best.bn == 0 || cost < best.cost) best = {s[0], s[1], cost};
  }
  return best;
}

template <int MODE>
cudaError_t run_gemm_mode(const GemmCall& c, cudaStream_t stream) {
  const TileChoice tile = best_tile<MODE>(c, c.parts > 1 ? c.parts : 1, sm_count());
  if (tile.bn == 256) return run_gemm<256, 2, MODE>(c, stream);
  if (tile.bn == 128) return run_gemm<128, 2, MODE>(c, stream);
  return run_gemm<64, 1, MODE>(c, stream);
}

// A chain's products with the same tiles.  A product ends with its slowest CTA; the next one begins some 2500 cycles later.
TileChoice best_chain_tile(const GemmCall& gram, const GemmCall& poly, const GemmCall& update) {
  const int64_t sms = sm_count();
  const int shapes[3][3] = {{256, 2, 512}, {128, 2, 384}, {64, 1, 384}};
  TileChoice best = {0, 0, 0};
  for (const auto& s : shapes) {
    int64_t cost = 0;
    const GemmCall* calls[3] = {&gram, &poly, &update};
    for (int i = 0; i < 3; ++i) {
      const GemmCall& c = *calls[i];
      const int64_t tiles = (i < 2 ? count_tiles<kGemmGram>(c, dev::kBM * s[1], s[0]) : count_tiles<kGemmUpdate>(c, dev::kBM * s[1], s[0])) * c.batch;
      const int64_t units = sms / s[1], stages = (c.k + dev::kBK - 1) / dev::kBK;
      cost += (tiles + units - 1) / units * (stages * s[2] + 1000 + 4 * s[0]);
    }
    if (best.bn == 0 || cost < best.cost) best = {s[0], s[1], cost};
  }
  return best;
}

template <int BN, int kCtas, bool kLong>
cudaError_t run_chain_of(const GemmChain& c, cudaStream_t stream) {
  using S = dev::GemmShape<BN, kCtas>;
  static_assert(sizeof(dev::ChainParams) <= 32000, "arguments of a kernel");
  dev::ChainParams p;
  cudaError_t e = cudaSuccess;
  for (int i = 0; i < 2; ++i) {
    if (e == cudaSuccess) e = fill_params<BN, kCtas, kGemmGram>(c.gram[i], &p.gram[i]);
    if (e == cudaSuccess) e = fill_params<BN, kCtas, kGemmUpdate>(c.update[i], &p.update[i]);
  }
  if (e == cudaSuccess) e = fill_params<BN, kCtas, kGemmPoly>(c.poly, &p.poly);
  if (e == cudaSuccess) e = fill_params<BN, kCtas, kGemmUpdate>(c.last, &p.last);
  p.steps = c.steps;
  p.arrived = c.arrived;
  static unsigned long long allowed = 0;
  if (e == cudaSuccess) e = allow_smem(dev::hc_gemm_chain_kernel<BN, kCtas, kLong>, S::kSmem, &allowed);
  if (e != cudaSuccess) return e;
  const int64_t total = (int64_t)p.last.tiles * p.last.batch;  // the product with the most tiles
  return launch_units<kCtas>(dev::hc_gemm_chain_kernel<BN, kCtas, kLong>, p, total, S::kSmem, true, stream);
}
// S sums the long side, and its diagonal is all positive; the other sums are as long as the short side, which memory bounds.
template <int BN, int kCtas>
cudaError_t run_chain(const GemmChain& c, cudaStream_t stream) {
  return c.gram[0].k > dev::kLongF16 ? run_chain_of<BN, kCtas, true>(c, stream) : run_chain_of<BN, kCtas, false>(c, stream);
}

}  // namespace

int gemm_parts(int64_t m, int64_t n, int64_t k) {
  GemmCall c;
  memset(&c, 0, sizeof(c));
  c.m = m, c.n = n, c.k = k, c.batch = 1;
  int best = 1;
  if (k < 512) return 1;
  const int64_t sms = sm_count();
  int64_t least = best_tile<kGemmLinear>(c, 1, sms).cost;
  for (int parts = 2; parts <= 16; ++parts) {
    if (k < parts * 256) break;
    // the parts are written and read once more, some 3000 bytes a cycle, by a launch that takes some 5000 cycles besides
    const int64_t cost = best_tile<kGemmLinear>(c, parts, sms).cost + 5000 + m * n * 8 * parts / 3000;
    if (cost < least) {
      least = cost;
      best = parts;
    }
  }
  return best;
}

cudaError_t launch_gemm(const GemmCall& c, cudaStream_t stream) {
  // sums in parts cost 8 % at 8192 x 4096 x 8192 (392 us with a bf16 result, 403 with fp32, 437 with fp32 sums in parts), 6 % at
  // 4096 x 4096 x 16384 in fp16 (432 and 458 us)
  const int64_t length = c.k / (c.parts > 1 ? c.parts : 1);
  const bool wide = length > (c.precise ? dev::kChunk * dev::kBK : c.type == kF16 ? dev::kLongF16 : dev::kLongBf16);
  return wide ? run_gemm_mode<dev::kGemmLinearWide>(c, stream) : run_gemm_mode<kGemmLinear>(c, stream);
}

cudaError_t launch_chain(const GemmChain& c, cudaStream_t stream) {
  const TileChoice tile = best_chain_tile(c.gram[0], c.poly, c.update[0]);
  if (tile.bn == 256) return run_chain<256, 2>(c, stream);
  if (tile.bn == 128) return run_chain<128, 2>(c, stream);
  return run_chain<64, 1>(c, stream);
}

}  // namespace hc

extern "C" int hc_train_status(int clear) {
  if (cudaDeviceSynchronize() != cudaSuccess) return hc::kErrCuda;
  const int all[3] = {hc::take_status(hc::dev::g_train_status, clear), hc::norm_status(clear), hc::logprob_status(clear)};
  return all[0] ? all[0] : all[1] ? all[1] : all[2];
}
