// act(x W^T + b) + residual and its backward pass: the products are hc_gemm.cu's, here is what lies around them.
#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

// ---- a few rows -----------------------------------------------------------------------------------------------------
// With up to sixteen rows the weights are read once and everything else is small, so the kernel is made for reading: sixteen
// rows of W are a block's, its warps share the sum in stretches of 64, and each lane feeds mma.sync straight from 16-byte
// loads of W and x, since any order of the sum will do as long as both operands have the same one.  Eight rows of x are the
// n of one instruction.  The tensor core's own sum is taken up into fp32 every 16 stretches of a warp, as in the large
// products.  Bound by reading W: one row of 4096 -> 4096 takes 5.9 us (5.7 TB/s), of 8192 -> 8192 27 us (5.0 TB/s), with fp32
// multiplications in place of mma.sync 8 rows took 39 and 143 us.  Rows of W that begin anywhere cost more loads (12.6 us for
// 5001 -> 2049, 20 MB).
struct FewRowsParams {
  const void *x, *w, *bias, *residual;
  void *out, *z;
  int64_t ldx, ldw, ldr, ldo, ldz;
  int64_t inner, width;
  int rows, out_type, bias_type, activation;
};

__device__ __forceinline__ float act_value(float z, int kind) {
  float other = 0.0f;
  if (kind == kActGeluTanh) activate_pair<kActGeluTanh>(z, other);
  else if (kind == kActRelu) activate_pair<kActRelu>(z, other);
  else if (kind == kActSilu) activate_pair<kActSilu>(z, other);
  return z;
}

// Eight 16-bit elements from p on, which may begin anywhere, with zeros from the `count`th on: the three words between an odd
// element at either end, or the two at the end, shifted into place.
__device__ __forceinline__ uint4 any_group(const uint16_t* p, int64_t count) {
  uint4 w = make_uint4(0, 0, 0, 0);
  if (count >= 8) {
    const bool odd = (reinterpret_cast<uintptr_t>(p) & 2u) != 0;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(p + odd);
    const uint32_t a = q[0], b = q[1], c = q[2], first = p[odd ? 0 : 6], last = p[7];
    w = odd ? make_uint4(first | a << 16, __funnelshift_r(a, b, 16), __funnelshift_r(b, c, 16), c >> 16 | last << 16) : make_uint4(a, b, c, first | last << 16);
  } else {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < count ? p[j] : 0u;
    w = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
  return w;
}
// Eight elements of a lane for a step of 32 along the sum; zeros behind the end.
template <typename T, bool kVector>
__device__ __forceinline__ uint4 few_group(const T* row, int64_t k, int64_t end, int t) {
  if (!kVector) return any_group(reinterpret_cast<const uint16_t*>(row + k + 8 * t), end - k - 8 * t);
  return k + 8 * t < end ? *reinterpret_cast<const uint4*>(row + k + 8 * t) : make_uint4(0, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void few_mma<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void few_mma<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kFewWarps = 16;  // at most, of a block
template <typename T, int N, bool kVector>  // N: eights of rows
__global__ void __launch_bounds__(kFewWarps * 32) hc_few_rows_kernel(const __grid_constant__ FewRowsParams p) {
  __shared__ float parts[kFewWarps][N * 8][17];
  constexpr int kSteps = 4;  // of 32 along the sum, whose loads are under way together
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t stride = warps * 32ll * kSteps;
  const int g = lane >> 2, t = lane & 3;
  const int64_t first = blockIdx.x * 16ll, last = p.width - 1;
  const T* w0 = static_cast<const T*>(p.w) + (first + g < last ? first + g : last) * p.ldw;
  const T* w1 = static_cast<const T*>(p.w) + (first + g + 8 < last ? first + g + 8 : last) * p.ldw;
  const T* x[N];
  int64_t end[N];  // of a row of x; a row that is not there ends before its start
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int row = n * 8 + g;
    x[n] = static_cast<const T*>(p.x) + (row < p.rows ? row : 0) * p.ldx;
    end[n] = row < p.rows ? p.inner : 0;
  }
  float sum[N][4], part[N][4];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[n][j] = part[n][j] = 0.0f;
  int taken = 0;
  for (int64_t k0 = warp * 64ll; k0 < p.inner; k0 += stride) {
    uint4 a[kSteps], b[kSteps], v[kSteps][N];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t k = k0 + (s >> 1) * (warps * 64ll) + (s & 1) * 32;
      a[s] = few_group<T, kVector>(w0, k, p.inner, t);
      b[s] = few_group<T, kVector>(w1, k, p.inner, t);
#pragma unroll
      for (int n = 0; n < N; ++n) v[s][n] = few_group<T, kVector>(x[n], k, end[n], t);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        few_mma<T>(part[n], a[s].x, b[s].x, a[s].y, b[s].y, v[s][n].x, v[s][n].y);
        few_mma<T>(part[n], a[s].z, b[s].z, a[s].w, b[s].w, v[s][n].z, v[s][n].w);
      }
    if (++taken == 32 / kSteps || k0 + stride >= p.inner) {
      taken = 0;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[n][j] += part[n][j];
          part[n][j] = 0.0f;
        }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) parts[warp][n * 8 + 2 * t + (j & 1)][g + (j >> 1) * 8] = sum[n][j];
  __syncthreads();
  for (int i = threadIdx.x; i < N * 128; i += blockDim.x) {
    const int r = i >> 4;
    const int64_t n = first + (i & 15);
    if (r >= p.rows || n >= p.width) continue;
    float z = 0.0f;
    for (int w = 0; w < warps; ++w) z += parts[w][r][i & 15];
    if (p.bias) z += param_at(p.bias, p.bias_type, n);
    if (p.z) static_cast<T*>(p.z)[r * p.ldz + n] = from_float<T>(z);
    z = act_value(z, p.activation);
    if (p.residual) z += param_at(p.residual, p.out_type, r * p.ldr + n);
    param_put(p.out, p.out_type, r * p.ldo + n, z);
  }
}

// ---- rows of the backward pass ----------------------------------------------------------------------------------------
// dz = dy act'(z), rounded for the products, and the sums of its columns.  A thread has eight columns, a block 256 and a
// share of the rows.  Bound by memory.  Of an fp32 dy fp16 does not hold all that the results may be made of: `most` then gives
// the power of two that dz is taken times.
struct RowsBackwardParams {
  const void *dy, *z;
  void* dz;
  float* partial;  // [share][width]
  const unsigned int* most;
  int64_t ldy, ldz, ldd, rows, width;
  int activation, shares;
};

// The largest finite |value| of a matrix, as bits (whose order is that of the values); `most` is 0 before.  Bound by reading, in a pass of
// its own, since no value can be rounded before the largest one is known: 6 us for 8192 x 768, 27 for 8192 x 4096 (5 TB/s).  kVector: without
// gaps, from 16 bytes on.
template <bool kVector>
__global__ void __launch_bounds__(256, 8) hc_largest_kernel(const float* v, int64_t ld, int64_t rows, int64_t width, unsigned int* most) {
  const int64_t first = blockIdx.x * 256ll + threadIdx.x, step = gridDim.x * 256ll, total = rows * width;
  unsigned int m = 0;
  const auto take = [&](float a) {
    const unsigned int bits = __float_as_uint(a) & 0x7fffffffu;
    if (bits < 0x7f800000u) m = max(m, bits);
  };
  const int64_t fours = kVector ? total / 4 : 0;
#pragma unroll 4
  for (int64_t i = first; i < fours; i += step) {
    const float4 a = reinterpret_cast<const float4*>(v)[i];
    take(a.x), take(a.y), take(a.z), take(a.w);
  }
#pragma unroll 2
  for (int64_t i = fours * 4 + first; i < total; i += step) take(kVector ? v[i] : v[i / width * ld + i % width]);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m) atomicMax(most, m);
}

template <typename Y, typename T, bool kVector, int kAct>
__global__ void __launch_bounds__(256, kAct == kActNone ? 3 : 2) hc_rows_backward_kernel(const __grid_constant__ RowsBackwardParams p) {
  __shared__ float sums[8][256];
  constexpr int kAtOnce = 4;  // rows whose loads are under way together
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = blockIdx.x * 256ll + lane * 8, step = p.shares * 8ll;
  Pair total[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) total[j] = pair(0.0f, 0.0f);
  const bool whole = kVector && col + 8 <= p.width;
  for (int64_t r0 = blockIdx.y * 8ll + warp; r0 < p.rows && col < p.width; r0 += step * kAtOnce) {
    float g[kAtOnce][8], a[kAtOnce][8];
    if (whole && r0 + (kAtOnce - 1) * step < p.rows) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        load8(static_cast<const Y*>(p.dy) + (r0 + i * step) * p.ldy + col, g[i]);
        if (kAct != kActNone) load8(static_cast<const T*>(p.z) + (r0 + i * step) * p.ldz + col, a[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int64_t r = r0 + i * step;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = r < p.rows && col + j < p.width;
          g[i][j] = in ? to_float(static_cast<const Y*>(p.dy)[r * p.ldy + col + j]) : 0.0f;
          a[i][j] = kAct != kActNone && in ? to_float(static_cast<const T*>(p.z)[r * p.ldz + col + j]) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t r = r0 + i * step;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Pair v = slope_pair<kAct>(pair(g[i][2 * j], g[i][2 * j + 1]), a[i][2 * j], a[i][2 * j + 1]);
        total[j] = total[j] + v;
        parts(v, g[i][2 * j], g[i][2 * j + 1]);
      }
      if (p.dz && r < p.rows) {
        if (p.most) {
          const float power = gradient_power(p.most, 1);
#pragma unroll
          for (int j = 0; j < 8; ++j) g[i][j] *= power;
        }
        T* dz = static_cast<T*>(p.dz) + r * p.ldd + col;
        if (whole) {
          store8(dz, g[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < p.width) dz[j] = from_float<T>(g[i][j]);
        }
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) parts(total[j], sums[warp][lane * 8 + 2 * j], sums[warp][lane * 8 + 2 * j + 1]);
  __syncthreads();
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
  if (c < p.width) p.partial[blockIdx.y * p.width + c] = s;
}

__global__ void __launch_bounds__(256) hc_rows_finish_kernel(const float* partial, int shares, int64_t width, void* out, int type) {
  __shared__ float sums[8][32];
  const int64_t c = blockIdx.x * 32ll + (threadIdx.x & 31);
  float s = 0.0f;
  if (c < width)
    for (int i = threadIdx.x >> 5; i < shares; i += 8) s += partial[i * width + c];
  sums[threadIdx.x >> 5][threadIdx.x & 31] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || c >= width) return;
  s = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
  param_put(out, type, c, s);
}

// ---- products whose sum is shared out ---------------------------------------------------------------------------------
// A product with few tiles and a long sum gives parts of the sum to different SMs, which leave fp32 matrices; they are added
// here, in the order of the sum, and what follows a product is done to them.
struct JoinParams {
  const float* parts;
  int64_t ld, stride;  // rows of a part begin at 32 bytes
  int count;
  int64_t rows, width;
  const void *bias, *residual;
  void *out, *z;
  const unsigned int* most;
  int64_t ldr, ldo, ldz;
  int type, out_type, bias_type, activation;
};
// the first `count` of eight values, from element i on
__device__ __forceinline__ void join_put(void* base, int type, int64_t i, const float (&v)[8], int64_t count) {
  unsigned char* to = static_cast<unsigned char*>(base) + i * (type == kF32 ? 4 : 2);
  if (count >= 8 && (reinterpret_cast<uintptr_t>(to) & 15u) == 0) {
    if (type == kF32) store8(reinterpret_cast<float*>(to), v);
    else if (type == kBf16) store8(reinterpret_cast<__nv_bfloat16*>(to), v);
    else store8(reinterpret_cast<__half*>(to), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) param_put(base, type, i + j, v[j]);
  }
}
__global__ void __launch_bounds__(256) hc_join_kernel(const __grid_constant__ JoinParams p) {
  const int64_t groups = (p.width + 7) / 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < p.rows * groups; i += gridDim.x * 256ll) {
    const int64_t r = i / groups, c = (i - r * groups) * 8, count = p.width - c;
    const float* part = p.parts + r * p.ld + c;
    float s[8], v[8];
    load8(part, s);
    for (int k = 1; k < p.count; ++k) {
      load8(part + k * p.stride, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
    if (p.most) {
      const float power = gradient_power(p.most, -1);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] *= power;
    }
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < count) s[j] += param_at(p.bias, p.bias_type, c + j);
    }
    if (p.z) join_put(p.z, p.type, r * p.ldz + c, s, count);
    if (p.activation != kActNone) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = act_value(s[j], p.activation);
    }
    if (p.residual) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < count) s[j] += param_at(p.residual, p.out_type, r * p.ldr + c + j);
    }
    join_put(p.out, p.out_type, r * p.ldo + c, s, count);
  }
}

// ---- rows that begin anywhere, as the products read them -----------------------------------------------------------------
// Rows of 16-bit values, copied to rows that begin at 16 bytes, zeros behind their ends.  Bound by memory: a thread brings eight.
__global__ void __launch_bounds__(256) hc_align_rows_kernel(const uint16_t* from, int64_t ld, int64_t rows, int64_t width, uint4* to, int64_t groups) {
  const int64_t used = (width + 7) / 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * used; i += gridDim.x * 256ll) {
    const int64_t r = i / used, c = i - r * used;
    to[r * groups + c] = any_group(from + r * ld + c * 8, width - c * 8);
  }
}

}  // namespace dev

namespace {

constexpr size_t kMostSize = (size_t)1 << 26;  // of each side: a tile's sum then stays far below the limit of a wait
// Up to here the kernel for few rows: 8 us with 16 rows of 4096 -> 4096, 30 to 36 of 8192 -> 8192.  The large products take 16 and 37
// with 17 rows; this kernel with four eights of rows took 16 to 18 and 88 to 108, for every block reads all of x.
constexpr size_t kFewRows = HC_LINEAR_FEW_ROWS;

bool sizes_ok(size_t rows, size_t inner, size_t width) {
  return inner > 0 && width > 0 && inner < kMostSize && width < kMostSize && rows < kMostSize;
}
bool stride_ok(size_t stride, size_t least) { return stride >= least && stride < ((size_t)1 << 32); }
bool product_type(int type) { return type == kBf16 || type == kF16; }

// As many blocks as the SMs hold at a time, two each (with an activation; three without), each with a share of the rows.
int shares_of(size_t rows, size_t width, int activation) {
  const size_t sms = device_info().sms > 0 ? device_info().sms : 1;
  const size_t strips = (width + 255) / 256, most = (rows + 31) / 32;
  size_t shares = sms * (activation == kActNone ? 3 : 2) / strips;
  if (shares > most) shares = most;
  if (shares > 128) shares = 128;
  return (int)(shares ? shares : 1);
}

template <typename T, int N>
void few_rows_of(const dev::FewRowsParams& p, bool vector, cudaStream_t stream) {
  // eight warps a block; sixteen where that leaves SMs without a block and each warp has a step to go
  const unsigned grid = (unsigned)((p.width + 15) / 16);
  const unsigned threads = (int)grid <= device_info().sms && p.inner >= 1024 ? 512 : 256;
  if (vector) dev::hc_few_rows_kernel<T, N, true><<<grid, threads, 0, stream>>>(p);
  else dev::hc_few_rows_kernel<T, N, false><<<grid, threads, 0, stream>>>(p);
}
template <typename T>
void few_rows(const dev::FewRowsParams& p, bool vector, cudaStream_t stream) {
  static_assert(kFewRows <= 16, "two eights of rows");
  if (p.rows <= 8) few_rows_of<T, 1>(p, vector, stream);
  else few_rows_of<T, 2>(p, vector, stream);
}

template <typename Y, typename T, int kAct>
void rows_backward_of(const dev::RowsBackwardParams& p, bool vector, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.width + 255) / 256), (unsigned)p.shares);
  if (vector) dev::hc_rows_backward_kernel<Y, T, true, kAct><<<grid, 256, 0, stream>>>(p);
  else dev::hc_rows_backward_kernel<Y, T, false, kAct><<<grid, 256, 0, stream>>>(p);
}
template <typename Y, typename T>
void rows_backward(const dev::RowsBackwardParams& p, bool vector, cudaStream_t stream) {
  if (p.activation == kActNone) rows_backward_of<Y, T, kActNone>(p, vector, stream);
  else if (p.activation == kActGeluTanh) rows_backward_of<Y, T, kActGeluTanh>(p, vector, stream);
  else if (p.activation == kActRelu) rows_backward_of<Y, T, kActRelu>(p, vector, stream);
  else rows_backward_of<Y, T, kActSilu>(p, vector, stream);
}

size_t rounded(size_t v, size_t unit) { return (v + unit - 1) / unit * unit; }
// scratch memory of a product: the parts of its sum
size_t product_bytes(int parts, size_t m, size_t n) {
  return parts > 1 ? rounded((size_t)parts * m * rounded(n, 8) * sizeof(float), 256) : 0;
}
cudaError_t run_product(GemmCall c, int parts, void* scratch, cudaStream_t stream) {
  c.precise = c.out_type == kF32;
  if (parts <= 1) return launch_gemm(c, stream);
  dev::JoinParams p;
  p.parts = static_cast<const float*>(scratch);
  p.ld = (c.n + 7) / 8 * 8;
  p.stride = c.m * p.ld;
  p.count = parts;
  p.rows = c.m, p.width = c.n;
  p.bias = c.bias, p.residual = c.in.data, p.out = c.out.data, p.z = c.out2.data;
  p.ldr = c.in.ld, p.ldo = c.out.ld, p.ldz = c.out2.ld;
  p.type = c.type, p.out_type = c.out_type, p.bias_type = c.bias_type, p.activation = c.activation;
  p.most = c.most;
  c.most = nullptr;
  c.parts = parts;
  c.out_type = kF32;
  c.out = {scratch, p.ld, p.stride};
  c.out2 = c.in = GemmSide{nullptr, 0, 0};
  c.bias = nullptr;
  c.activation = kActNone;
  const cudaError_t e = launch_gemm(c, stream);
  if (e != cudaSuccess) return e;
  const int64_t blocks = (p.rows * (p.ld / 8) + 255) / 256;
  dev::hc_join_kernel<<<(unsigned)(blocks < 2368 ? blocks : 2368), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

// scratch memory of a backward pass: sums of columns, parts of a product's sum, dz, the largest |dy|
constexpr size_t kMostBytes = 256;
struct BackwardLayout {
  size_t sums, parts, total;
  int dx_parts, dw_parts;
};
BackwardLayout backward_layout(size_t rows, size_t inner, size_t width, int keep_dz) {
  BackwardLayout l;
  l.sums = rounded((size_t)shares_of(rows, width, kActNone) * width * sizeof(float), 256);  // the most there are
  l.dx_parts = gemm_parts((int64_t)rows, (int64_t)inner, (int64_t)width);
  l.dw_parts = gemm_parts((int64_t)width, (int64_t)inner, (int64_t)rows);
  const size_t dx = product_bytes(l.dx_parts, rows, inner), dw = product_bytes(l.dw_parts, width, inner);  // one after the other
  l.parts = dx > dw ? dx : dw;
  l.total = l.sums + l.parts + (keep_dz ? rounded(rows * rounded(width, 8) * 2, 256) + kMostBytes : 0);
  return l;
}

bool aligned_rows(const void* p, size_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 8 == 0; }

}  // namespace
}  // namespace hc

extern "C" {

int hc_align_rows(const void* from, size_t from_stride, size_t rows, size_t width, void* to, size_t to_stride, hc_stream_t stream) {
  using namespace hc;
  if (!stride_ok(from_stride, width) || !stride_ok(to_stride, width) || rows >= kMostSize || width >= kMostSize) return kErrArgument;
  if (rows == 0 || width == 0) return kOk;
  if (!from || !to || (reinterpret_cast<uintptr_t>(from) & 1u) || !gemm_operand_ok(to, (int64_t)to_stride)) return kErrArgument;
  const size_t blocks = (rows * ((width + 7) / 8) + 255) / 256, most = (size_t)(device_info().sms > 0 ? device_info().sms : 1) * 8;
  dev::hc_align_rows_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(
      static_cast<const uint16_t*>(from), (int64_t)from_stride, (int64_t)rows, (int64_t)width, static_cast<uint4*>(to), (int64_t)to_stride / 8);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

size_t hc_linear_bytes(size_t rows, size_t inner, size_t width) {
  return hc::sizes_ok(rows, inner, width) && rows > hc::kFewRows
             ? hc::product_bytes(hc::gemm_parts((int64_t)rows, (int64_t)width, (int64_t)inner), rows, width) : 0;
}

int hc_linear(const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, const void* bias, int bias_type,
              const void* residual, size_t residual_stride, void* out, int out_type, size_t out_stride, void* z, size_t z_stride,
              int activation, size_t rows, size_t inner, size_t width, void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  if (!product_type(type) || (out_type != kF32 && out_type != type) || !element_type_ok(bias_type)) return kErrArgument;
  if (activation < kActNone || activation > kActSilu || !sizes_ok(rows, inner, width)) return kErrArgument;
  if (!stride_ok(x_stride, inner) || !stride_ok(weight_stride, inner) || !stride_ok(out_stride, width)) return kErrArgument;
  if ((residual && !stride_ok(residual_stride, width)) || (z && !stride_ok(z_stride, width))) return kErrArgument;
  if (rows == 0) return kOk;
  if (!x || !weight || !out) return kErrArgument;
  if (!lies_at(x, 2) || !lies_at(weight, 2) || !lies_at(z, 2) || !lies_at(bias, element_bytes(bias_type)) || !lies_at(residual, element_bytes(out_type)) ||
      !lies_at(out, element_bytes(out_type)))
    return kErrArgument;
  if (rows <= kFewRows) {
    const dev::FewRowsParams p = {x, weight, bias, residual, out, z, (int64_t)x_stride, (int64_t)weight_stride, (int64_t)residual_stride,
                                  (int64_t)out_stride, (int64_t)z_stride, (int64_t)inner, (int64_t)width, (int)rows, out_type, bias_type, activation};
    const bool vector = inner % 8 == 0 && aligned_rows(x, x_stride) && aligned_rows(weight, weight_stride);
    if (type == kBf16) few_rows<__nv_bfloat16>(p, vector, stream);
    else few_rows<__half>(p, vector, stream);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
  }
  if (!gemm_operand_ok(x, x_stride) || !gemm_operand_ok(weight, weight_stride)) return kErrArgument;
  const int parts = gemm_parts((int64_t)rows, (int64_t)width, (int64_t)inner);
  const size_t need = product_bytes(parts, rows, width);
  if (need && (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255u) || scratch_bytes < need)) return kErrArgument;
  GemmCall c;
  memset(&c, 0, sizeof(c));
  c.type = type;
  c.m = rows, c.n = width, c.k = inner, c.batch = 1;
  c.a = {x, (int64_t)x_stride, 0, true};
  c.b = {weight, (int64_t)weight_stride, 0, true};
  c.out = {out, (int64_t)out_stride, 0};
  c.out2 = {z, (int64_t)z_stride, 0};
  c.in = {const_cast<void*>(residual), (int64_t)residual_stride, 0};
  c.out_type = out_type;
  c.bias = bias;
  c.bias_type = bias_type;
  c.activation = activation;
  return run_product(c, parts, scratch, stream) == cudaSuccess ? kOk : kErrCuda;
}

size_t hc_linear_backward_bytes(size_t rows, size_t inner, size_t width, int keep_dz) {
  return hc::sizes_ok(rows, inner, width) && rows ? hc::backward_layout(rows, inner, width, keep_dz).total : 0;
}

int hc_linear_backward(const void* dy, int dy_type, size_t dy_stride, const void* z, size_t z_stride, int activation, int keep_dz,
                       const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, void* dx, size_t dx_stride,
                       void* dweight, size_t dweight_stride, void* dbias, int bias_type, size_t rows, size_t inner, size_t width,
                       void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  if (!product_type(type) || (dy_type != kF32 && dy_type != type) || !element_type_ok(bias_type)) return kErrArgument;
  if (activation < kActNone || activation > kActSilu || !sizes_ok(rows, inner, width) || !stride_ok(dy_stride, width)) return kErrArgument;
  if (activation != kActNone && !stride_ok(z_stride, width)) return kErrArgument;
  if ((dx && (!stride_ok(weight_stride, inner) || !stride_ok(dx_stride, inner))) || (dweight && (!stride_ok(x_stride, inner) || !stride_ok(dweight_stride, inner))))
    return kErrArgument;
  if (!lies_at(dy, element_bytes(dy_type)) || !lies_at(z, 2) || !lies_at(dx, 2) || !lies_at(dweight, 2) || !lies_at(dbias, element_bytes(bias_type)))
    return kErrArgument;
  if (!keep_dz && (dx || dweight) && (activation != kActNone || dy_type != type)) return kErrArgument;
  if (rows == 0) {
    cudaError_t e = dweight ? cudaMemset2DAsync(dweight, dweight_stride * 2, 0, inner * 2, width, stream) : cudaSuccess;
    if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, width * element_bytes(bias_type), stream);
    return e == cudaSuccess ? kOk : kErrCuda;
  }
  if (!dx && !dweight && !dbias) return kOk;
  if (!dy || (activation != kActNone && !z)) return kErrArgument;
  if ((dx && (!weight || !gemm_operand_ok(weight, weight_stride))) || (dweight && (!x || !gemm_operand_ok(x, x_stride)))) return kErrArgument;
  const BackwardLayout l = backward_layout(rows, inner, width, keep_dz);
  if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255u) || scratch_bytes < l.total) return kErrArgument;
  unsigned char* at = static_cast<unsigned char*>(scratch);
  const bool products = dx || dweight;
  const void* dz = keep_dz ? at + l.sums + l.parts : dy;
  const size_t dz_stride = keep_dz ? (width + 7) / 8 * 8 : dy_stride;
  if (products && !gemm_operand_ok(dz, dz_stride)) return kErrArgument;
  unsigned int* most = nullptr;
  if (products && type == kF16 && dy_type == kF32) {
    most = reinterpret_cast<unsigned int*>(at + l.total - kMostBytes);
    if (cudaMemsetAsync(most, 0, sizeof(*most), stream) != cudaSuccess) return kErrCuda;
    const size_t blocks = (rows * width + 4095) / 4096, resident = (size_t)(device_info().sms > 0 ? device_info().sms : 1) * 8;
    const unsigned grid = (unsigned)(blocks < resident ? blocks : resident);
    const float* from = static_cast<const float*>(dy);
    if (dy_stride == width && lies_at(dy, 16)) dev::hc_largest_kernel<true><<<grid, 256, 0, stream>>>(from, (int64_t)dy_stride, (int64_t)rows, (int64_t)width, most);
    else dev::hc_largest_kernel<false><<<grid, 256, 0, stream>>>(from, (int64_t)dy_stride, (int64_t)rows, (int64_t)width, most);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  }
  if (dbias || (products && keep_dz)) {
    const dev::RowsBackwardParams p = {dy, z, products && keep_dz ? const_cast<void*>(dz) : nullptr, dbias ? reinterpret_cast<float*>(at) : nullptr, most,
                                       (int64_t)dy_stride, (int64_t)z_stride, (int64_t)dz_stride, (int64_t)rows, (int64_t)width, activation,
                                       shares_of(rows, width, activation)};
    const bool vector = aligned_rows(dy, dy_stride) && (activation == kActNone || aligned_rows(z, z_stride));
    if (type == kBf16) {
      if (dy_type == kF32) rows_backward<float, __nv_bfloat16>(p, vector, stream);
      else rows_backward<__nv_bfloat16, __nv_bfloat16>(p, vector, stream);
    } else {
      if (dy_type == kF32) rows_backward<float, __half>(p, vector, stream);
      else rows_backward<__half, __half>(p, vector, stream);
    }
    if (dbias) dev::hc_rows_finish_kernel<<<(unsigned)((width + 31) / 32), 256, 0, stream>>>(p.partial, p.shares, (int64_t)width, dbias, bias_type);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  }
  GemmCall c;
  memset(&c, 0, sizeof(c));
  c.type = c.out_type = type;
  c.batch = 1;
  c.most = most;
  if (dx) {
    c.m = rows, c.n = inner, c.k = width;
    c.a = {dz, (int64_t)dz_stride, 0, true};
    c.b = {weight, (int64_t)weight_stride, 0, false};
    c.out = {dx, (int64_t)dx_stride, 0};
    if (run_product(c, l.dx_parts, at + l.sums, stream) != cudaSuccess) return kErrCuda;
  }
  if (dweight) {
    c.m = width, c.n = inner, c.k = rows;
    c.a = {dz, (int64_t)dz_stride, 0, false};
    c.b = {x, (int64_t)x_stride, 0, false};
    c.out = {dweight, (int64_t)dweight_stride, 0};
    if (run_product(c, l.dw_parts, at + l.sums, stream) != cudaSuccess) return kErrCuda;
  }
  return kOk;
}

}  // extern "C"
