// out[m, n] = sum over k of a[m, k] b[n, k] on tcgen05 tensor cores, for the operators that are products.
//
// One CTA per SM goes through tiles of 128 x BN.  One thread brings the operands' tiles in by TMA (128-byte swizzle, 64
// of the sum at a time, as many stages as shared memory holds), one issues the matrix instructions (fp32 accumulators in
// tensor memory, two of them, so that a tile is stored while the next one is computed), four warps store.  An operand
// may lie along the sum or across it: tile and descriptor differ, the data is not moved, so the products of a backward
// pass need no transposed copies.
#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kBM = 128, kBK = 64;
constexpr int kGemmThreads = 192;
constexpr int kOperandA = kBM * kBK * 2;
constexpr uint64_t kGemmLimitNs = 2000ull * 1000 * 1000;

struct GemmParams {
  CUtensorMap map_a, map_b;
  int64_t m, n;
  int k_blocks;
  int tiles_m, tiles_n, tiles;  // of one matrix
  int batch;
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
  int vector_out, vector_out2, vector_in, vector_in2;  // rows begin at 16 bytes
};

__device__ unsigned int g_train_status;

template <int BN>
struct GemmShape {
  static constexpr int kStage = kOperandA + BN * kBK * 2;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kColumns = 2 * BN;  // of tensor memory
};

struct GemmBarriers {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drained;
  uint32_t tmem;
  uint32_t gave_up;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// 32 columns of this warp's 32 rows: thread i has row i
__device__ __forceinline__ void tc_load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
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
template <int BN, int MODE>
__device__ __forceinline__ void tile_place(const GemmParams& p, int t, int& mi, int& ni) {
  if (MODE == kGemmGram || MODE == kGemmPoly) {
    mi = 0;
    for (;;) {
      int count = (mi * kBM + kBM - 1) / BN + 1;
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

__device__ __forceinline__ float sigmoid(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
__device__ __forceinline__ float activate(float z, int kind) {
  if (kind == kActGeluTanh) return z * sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));  // (1 + tanh u) / 2 = sigmoid(2 u)
  if (kind == kActSilu) return z * sigmoid(z);
  if (kind == kActRelu) return z > 0.0f ? z : z != z ? z : 0.0f;
  return z;
}

// 32 columns of one row
template <typename T>
__device__ __forceinline__ void read32(const T* p, int64_t count, bool vector, float (&v)[32]) {
  if (vector && count >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float w[8];
      load8(p + i * 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i * 8 + j] = w[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = j < count ? to_float(p[j]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void write32(T* p, int64_t count, bool vector, const float (&v)[32]) {
  if (vector && count >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = v[i * 8 + j];
      store8(p + i * 8, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < count) p[j] = from_float<T>(v[j]);
  }
}
__device__ __forceinline__ void write32_as(void* p, int type, int64_t at, int64_t count, bool vector, const float (&v)[32]) {
  if (type == kF32) write32(static_cast<float*>(p) + at, count, vector, v);
  else if (type == kBf16) write32(static_cast<__nv_bfloat16*>(p) + at, count, vector, v);
  else write32(static_cast<__half*>(p) + at, count, vector, v);
}
__device__ __forceinline__ void read32_as(const void* p, int type, int64_t at, int64_t count, bool vector, float (&v)[32]) {
  if (type == kF32) read32(static_cast<const float*>(p) + at, count, vector, v);
  else if (type == kBf16) read32(static_cast<const __nv_bfloat16*>(p) + at, count, vector, v);
  else read32(static_cast<const __half*>(p) + at, count, vector, v);
}

constexpr float kLow = 2048.0f;  // lo is held times this: as precise next to hi as fp16 can be

// row, columns col .. col + 31 of matrix z
template <int MODE>
__device__ __forceinline__ void gemm_finish(const GemmParams& p, int64_t z, int64_t row, int64_t col, float (&v)[32]) {
  const int64_t count = row < p.m ? p.n - col : 0;
  if (count <= 0) return;
  const int64_t at = z * p.out.stride + row * p.out.ld + col;
  if (MODE == kGemmLinear) {
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) v[j] += param_at(p.bias, p.bias_type, col + j);
    }
    if (p.out2.data) write32_as(p.out2.data, p.type, row * p.out2.ld + col, count, p.vector_out2, v);
    if (p.activation != kActNone) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = activate(v[j], p.activation);
    }
    if (p.in.data) {
      float r[32];
      read32_as(p.in.data, p.out_type, row * p.in.ld + col, count, p.vector_in, r);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += r[j];
    }
    write32_as(p.out.data, p.out_type, at, count, p.vector_out, v);
  } else if (MODE == kGemmUpdate) {
    float hi[32], lo[32];
    const int64_t from = z * p.in.stride + row * p.in.ld + col;
    read32(static_cast<const __half*>(p.in.data) + from, count, p.vector_in, hi);
    read32(static_cast<const __half*>(p.in2.data) + from, count, p.vector_in2, lo);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = fmaf(p.ca, fmaf(lo[j], 1.0f / kLow, hi[j]), v[j]);
    if (p.out2.data) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        hi[j] = to_float(__float2half_rn(v[j]));
        lo[j] = (v[j] - hi[j]) * kLow;
      }
      write32(static_cast<__half*>(p.out.data) + at, count, p.vector_out, hi);
      write32(static_cast<__half*>(p.out2.data) + at, count, p.vector_out2, lo);
    } else {
      const float scale = p.scale[z];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= scale;
      write32_as(p.out.data, p.out_type, at, count, p.vector_out, v);
    }
  } else {
    if (col > row) return;  // the mirror image of another tile's
    if (MODE == kGemmPoly) {
      const float square = p.scale[z] * p.scale[z], c1 = p.cb * square, c2 = p.cc * square * square;
      float q[32];
      read32(static_cast<const __half*>(p.in.data) + z * p.in.stride + row * p.in.ld + col, count, p.vector_in, q);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = fmaf(c2, v[j], c1 * q[j]);
    }
    __half* out = static_cast<__half*>(p.out.data);
    const int64_t own = min(count, row - col + 1);
    write32(out + at, own, p.vector_out, v);
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < count && col + j < row) out[z * p.out.stride + (col + j) * p.out.ld + row] = __float2half_rn(v[j]);
  }
}

template <int BN, int MODE>
__global__ void __launch_bounds__(kGemmThreads, 1) hc_gemm_kernel(const __grid_constant__ GemmParams p) {
  using S = GemmShape<BN>;
  extern __shared__ unsigned char raw[];
  __shared__ GemmBarriers sh;
  unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sh.acc_full[a], 1);
      mbar_init(&sh.acc_empty[a], 4);
    }
    mbar_init(&sh.drained, 1);
    sh.gave_up = 0;
    fence_mbar_init();
    tma_prefetch_map(&p.map_a);
    tma_prefetch_map(&p.map_b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(S::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const int total = p.tiles * p.batch;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      int issued = 0;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const int z = t / p.tiles;
        int mi, ni;
        tile_place<BN, MODE>(p, t - z * p.tiles, mi, ni);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!gemm_wait(&sh.empty[s], phase ^ 1, sh)) {
            ok = false;
            break;
          }
          unsigned char* a = stages + s * S::kStage;
          unsigned char* b = a + kOperandA;
          mbar_expect_tx(&sh.full[s], S::kStage);
          if (p.a_across) {
            for (int i = 0; i < kBM / 64; ++i) tma_load_3d(a + i * 8192, &p.map_a, mi * kBM + i * 64, kb * kBK, z, &sh.full[s]);
          } else {
            tma_load_3d(a, &p.map_a, kb * kBK, mi * kBM, z, &sh.full[s]);
          }
          if (p.b_across) {
            for (int i = 0; i < BN / 64; ++i) tma_load_3d(b + i * 8192, &p.map_b, ni * BN + i * 64, kb * kBK, z, &sh.full[s]);
          } else {
            tma_load_3d(b, &p.map_b, kb * kBK, ni * BN, z, &sh.full[s]);
          }
          ++issued;
          if (++s == S::kStages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // copies in flight land before the CTA leaves
      for (int back = 0; back < S::kStages && back < issued; ++back) {
        const int i = issued - 1 - back;
        mbar_wait_bounded(&sh.full[i % S::kStages], (i / S::kStages) & 1, kGemmLimitNs);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int s = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        if (!gemm_wait(&sh.acc_empty[acc], acc_phase ^ 1, sh)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!gemm_wait(&sh.full[s], phase, sh)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(stages + s * S::kStage);
          const uint64_t da = p.desc_a | (uint64_t)((a & 0x3ffff) >> 4), db = p.desc_b | (uint64_t)(((a + kOperandA) & 0x3ffff) >> 4);
#pragma unroll
          for (int i = 0; i < kBK / 16; ++i) tc_mma(d, da + i * p.step_a, db + i * p.step_b, p.idesc, kb > 0 || i > 0);
          tc_commit(&sh.empty[s]);
          if (++s == S::kStages) {
            s = 0;
            phase ^= 1;
          }
        }
        tc_commit(&sh.acc_full[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // so do the matrix instructions
      tc_commit(&sh.drained);
      mbar_wait_bounded(&sh.drained, 0, kGemmLimitNs);
    }
  } else {
    int acc = 0;
    uint32_t acc_phase = 0;
    const int quarter = warp & 3;  // the rows of tensor memory that this warp can reach
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const int z = t / p.tiles;
      int mi, ni;
      tile_place<BN, MODE>(p, t - z * p.tiles, mi, ni);
      const bool ok = gemm_wait(&sh.acc_full[acc], acc_phase, sh);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const int64_t row = (int64_t)mi * kBM + quarter * 32 + lane;
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        float v[32];
        __syncwarp();
        tc_load32(tmem + ((uint32_t)(quarter * 32) << 16) + acc * BN + c, v);
        gemm_finish<MODE>(p, z, row, (int64_t)ni * BN + c, v);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.acc_empty[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kColumns));
  }
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

bool vector_side(const GemmSide& s, size_t bytes) {
  return s.data && (reinterpret_cast<uintptr_t>(s.data) & 15u) == 0 && s.ld * bytes % 16 == 0 && s.stride * bytes % 16 == 0;
}

template <int BN, int MODE>
cudaError_t run_gemm(const GemmCall& c, cudaStream_t stream) {
  using S = dev::GemmShape<BN>;
  dev::GemmParams p;
  memset(&p, 0, sizeof(p));
  p.m = c.m;
  p.n = c.n;
  p.k_blocks = (int)((c.k + dev::kBK - 1) / dev::kBK);
  p.tiles_m = (int)((c.m + dev::kBM - 1) / dev::kBM);
  p.tiles_n = (int)((c.n + BN - 1) / BN);
  p.batch = (int)c.batch;
  int64_t tiles = 0;
  if (MODE == kGemmGram || MODE == kGemmPoly) {
    for (int i = 0; i < p.tiles_m; ++i) {
      const int count = (i * dev::kBM + dev::kBM - 1) / BN + 1;
      tiles += count < p.tiles_n ? count : p.tiles_n;
    }
  } else {
    tiles = (int64_t)p.tiles_m * p.tiles_n;
  }
  if (tiles * c.batch > 0x7fffffff) return cudaErrorInvalidValue;
  p.tiles = (int)tiles;
  p.a_across = !c.a.k_major;
  p.b_across = !c.b.k_major;
  if (!make_matrix_map(&p.map_a, c.type, c.a.data, c.a.k_major ? c.k : c.m, c.a.k_major ? c.m : c.k, c.batch, c.a.ld, c.a.stride,
                       c.a.k_major ? dev::kBM : dev::kBK))
    return cudaErrorInvalidValue;
  if (!make_matrix_map(&p.map_b, c.type, c.b.data, c.b.k_major ? c.k : c.n, c.b.k_major ? c.n : c.k, c.batch, c.b.ld, c.b.stride,
                       c.b.k_major ? BN : dev::kBK))
    return cudaErrorInvalidValue;
  p.desc_a = descriptor(c.a.k_major);
  p.desc_b = descriptor(c.b.k_major);
  p.step_a = c.a.k_major ? 2 : 128;
  p.step_b = c.b.k_major ? 2 : 128;
  const uint32_t format = c.type == kBf16 ? 1u : 0u;
  p.idesc = 1u << 4 | format << 7 | format << 10 | (c.a.k_major ? 0u : 1u << 15) | (c.b.k_major ? 0u : 1u << 16) | (uint32_t)(BN / 8) << 17 |
            (uint32_t)(dev::kBM / 16) << 24;
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
  const size_t wide = MODE == kGemmLinear || (MODE == kGemmUpdate && !c.out2.data) ? element_bytes(c.out_type) : 2;
  p.vector_out = vector_side(c.out, wide);
  p.vector_out2 = vector_side(c.out2, 2);
  p.vector_in = vector_side(c.in, MODE == kGemmLinear ? element_bytes(c.out_type) : 2);
  p.vector_in2 = vector_side(c.in2, 2);
  const cudaError_t e = set_smem(dev::hc_gemm_kernel<BN, MODE>, S::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t total = tiles * c.batch;
  const int sms = device_info().sms;
  dev::hc_gemm_kernel<BN, MODE><<<(int)(total < sms ? total : sms), dev::kGemmThreads, S::kSmem, stream>>>(p);
  return cudaGetLastError();
}

// Width of a tile.  What a tile takes is its columns (the tensor core's time) and a constant for what does not shrink with
// it (128 rows of the first operand are loaded for a tile of any width); the launch takes as long as the SM with the most tiles.
template <int MODE>
cudaError_t run_gemm_mode(const GemmCall& c, cudaStream_t stream) {
  const int64_t sms = device_info().sms > 0 ? device_info().sms : 1;
  const int64_t tm = (c.m + 127) / 128 * c.batch;
  int64_t best = 0;
  int width = 0;
  for (int bn = 256; bn >= 64; bn /= 2) {
    const int64_t tiles = tm * ((c.n + bn - 1) / bn);
    const int64_t cost = (tiles + sms - 1) / sms * (bn + 32);
    if (width == 0 || cost < best) {
      best = cost;
      width = bn;
    }
  }
  if (width == 256) return run_gemm<256, MODE>(c, stream);
  if (width == 128) return run_gemm<128, MODE>(c, stream);
  return run_gemm<64, MODE>(c, stream);
}

}  // namespace

cudaError_t launch_gemm(const GemmCall& c, cudaStream_t stream) {
  if (c.mode == kGemmLinear) return run_gemm_mode<kGemmLinear>(c, stream);
  if (c.mode == kGemmGram) return run_gemm_mode<kGemmGram>(c, stream);
  if (c.mode == kGemmPoly) return run_gemm_mode<kGemmPoly>(c, stream);
  return run_gemm_mode<kGemmUpdate>(c, stream);
}

}  // namespace hc

extern "C" int hc_train_status(int clear) {
  unsigned int status = 0;
  if (cudaMemcpyFromSymbol(&status, hc::dev::g_train_status, sizeof(status)) != cudaSuccess) return hc::kErrCuda;
  if (clear && status) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(hc::dev::g_train_status, &zero, sizeof(zero)) != cudaSuccess) return hc::kErrCuda;
  }
  return (int)status;
}
