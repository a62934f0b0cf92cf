// Newton-Schulz iteration of a batch of matrices: X = G / (|G| + eps), then X = a X + (b S + c S S) X with S = X X^T, or
// X = a X + X (b S + c S S) with S = X^T X where that is the smaller one.  Three products a step, of which the first two give
// symmetric matrices and compute one half, all of them in one launch (hc_gemm.cu).
//
// Operands are fp16: 11 bits, and no entry of X, S or the polynomial leaves its range once |X| <= 1.  What is rounded off
// X in directions that G hardly has would grow by `a` in every step (485 times in five); products with X carry none of it
// there, only the term a X does, so that term takes X from two fp16 numbers, hi and lo / 2048.  A matrix whose norm is far
// below eps stays small: it is held times 2^k, with k from what its norm can grow to in `steps`, and S counts 2^-2k.
#include <math.h>

#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kNormThreads = 256;
struct ScaleParams {
  const void* g;
  double* partial;  // [batch][parts]
  __half *hi, *lo;
  float* scale;  // [batch]: X = 2^-k (hi + lo / 2048)
  unsigned int* arrived;
  float growth;
  int64_t height, width, stride, batch_stride, ld;  // ld: of hi and lo
  int parts;
  float eps;
};

// The values of one matrix in groups of eight, a block's share of them, four groups under way at a time: f(row, column, values)
template <typename T, bool kVector, typename F>
__device__ __forceinline__ void for_groups(const ScaleParams& p, const T* g, F f) {
  const uint32_t each = (uint32_t)((p.width + 7) / 8), step = gridDim.x * kNormThreads;
  const int64_t groups = p.height * (int64_t)each;
  for (int64_t i0 = blockIdx.x * kNormThreads + threadIdx.x; i0 < groups; i0 += 4ll * step) {
    float v[4][8];
    int64_t row[4], col[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = i0 + (int64_t)i * step;
      row[i] = groups <= 0xffffffffll ? (uint32_t)at / each : at / each;
      col[i] = (at - row[i] * each) * 8;
    }
    if (kVector && i0 + 3ll * step < groups) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load8(g + row[i] * p.stride + col[i], v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = i0 + (int64_t)i * step < groups && col[i] + j < p.width ? to_float(g[row[i] * p.stride + col[i] + j]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + (int64_t)i * step < groups) f(row[i], col[i], v[i]);
  }
}

// Sums of squares, in 64 bits: the entries may be anything that their type can hold.  Bound by memory.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kNormThreads) hc_square_sum_kernel(const __grid_constant__ ScaleParams p) {
  __shared__ double sums[kNormThreads / 32];
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  for_groups<T, kVector>(p, static_cast<const T*>(p.g) + blockIdx.y * p.batch_stride, [&](int64_t, int64_t, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[j & 3] = fma((double)v[j], (double)v[j], part[j & 3]);
  });
  double s = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; ++w) s += sums[w];
    p.partial[(int64_t)blockIdx.y * p.parts + blockIdx.x] = s;
  }
}

template <typename T, bool kVector>
__global__ void __launch_bounds__(kNormThreads) hc_scale_kernel(const __grid_constant__ ScaleParams p) {
  __shared__ double factor;
  __shared__ int exponent;
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < p.parts; i += 32) s += p.partial[(int64_t)blockIdx.y * p.parts + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) {
      const double norm = sqrt(s), room = (norm / (norm + (double)p.eps)) * (double)p.growth;
      int k = 0;
      while (k < 126 && room * exp2((double)(k + 1)) <= 1.0) ++k;
      factor = 1.0 / (norm + (double)p.eps);
      exponent = k;
      if (blockIdx.x == 0) p.scale[blockIdx.y] = exp2f((float)-k);
      if (blockIdx.x == 0 && blockIdx.y == 0) *p.arrived = 0;
    }
  }
  __syncthreads();
  // 2^k / (norm + eps) as a number of 24 bits times a power of two: products with entries stay in the range of fp32, and
  // are off by at most 1.5 2^-24
  int e;
  const float mantissa = (float)frexp(factor, &e);
  const int up = e + exponent, first = up / 2, second = up - up / 2;
  const float power1 = exp2f((float)max(-126, min(127, first))), power2 = exp2f((float)max(-126, min(127, second)));
  const int64_t at = (int64_t)blockIdx.y * p.height * p.ld;
  for_groups<T, kVector>(p, static_cast<const T*>(p.g) + blockIdx.y * p.batch_stride, [&](int64_t r, int64_t c, const float (&v)[8]) {
    float hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = v[j] * power1 * mantissa * power2;
      hi[j] = __half2float(__float2half_rn(x));
      lo[j] = (x - hi[j]) * 2048.0f;
    }
    // rows of hi and lo have room for whole groups
    store8(p.hi + at + r * p.ld + c, hi);
    store8(p.lo + at + r * p.ld + c, lo);
  });
}

// ---- small matrices ---------------------------------------------------------------------------------------------------
// The general form has its CTAs meet after every product, and each of them starts loading then.  Here one block takes a matrix through all steps in shared memory, short side first, with warp-wide 16 x 8 x 16 matrix instructions: they need
// neither tensor memory nor descriptors, and at this size what counts is the way from one product to the next.
constexpr int kSmallThreads = 512;

struct SmallParams {
  const void* g;
  __nv_bfloat16* out;
  int64_t stride, batch_stride;
  int height, width;  // of a matrix as it is given
  int side, length;   // short and long side
  int rows, pitch;    // short side rounded up to 16; halves from row to row of X
  int s_pitch;        // of S and the polynomial
  int steps;
  float a, b, c, eps, growth;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const __half* p, bool transposed) {
  const uint32_t at = smem_u32(p);
  if (transposed)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two neighbouring tiles, 16 rows from `row` and 16 columns from `col`, of a product over k: the first operand's rows lie along
// the sum; the second one is given as rows along it (kAcross: false) or as rows across it.
template <bool kAcross>
__device__ __forceinline__ void small_product(float (&d0)[4], float (&d1)[4], const __half* a, int a_pitch, const __half* b, int b_pitch, int row,
                                              int col, int k) {
  const int lane = threadIdx.x & 31;
  // the next operands are on their way while one pair is multiplied, and two sums take turns; not unrolled further: with all
  // tiles' loops in line the code outgrew the instruction cache (a step of 192 x 64: 6.0 us, 4.7 rolled up)
  float e0[4], e1[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) d0[j] = d1[j] = e0[j] = e1[j] = 0.0f;
  const __half* pa = a + (row + (lane & 15)) * a_pitch + (lane >> 4) * 8;
  const __half* pb = kAcross ? b + (lane & 15) * b_pitch + col + (lane >> 4) * 8 : b + (col + (lane & 7) + (lane >> 4) * 8) * b_pitch + ((lane >> 3) & 1) * 8;
  const int b_step = kAcross ? 16 * b_pitch : 16, n = k / 16;
  uint32_t fa[2][4], fb[2][4];
  ldmatrix4(fa[0], pa, false);
  ldmatrix4(fb[0], pb, kAcross);
#pragma unroll 1
  for (int i = 0; i < n; i += 2) {
    if (i + 1 < n) {
      ldmatrix4(fa[1], pa + (i + 1) * 16, false);
      ldmatrix4(fb[1], pb + (i + 1) * b_step, kAcross);
    }
    mma16816(d0, fa[0], fb[0][0], fb[0][1]);
    mma16816(d1, fa[0], fb[0][2], fb[0][3]);
    if (i + 1 >= n) break;
    if (i + 2 < n) {
      ldmatrix4(fa[0], pa + (i + 2) * 16, false);
      ldmatrix4(fb[0], pb + (i + 2) * b_step, kAcross);
    }
    mma16816(e0, fa[1], fb[1][0], fb[1][1]);
    mma16816(e1, fa[1], fb[1][2], fb[1][3]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    d0[j] += e0[j];
    d1[j] += e1[j];
  }
}

template <typename T>
__global__ void __launch_bounds__(kSmallThreads, 1) hc_newton_small_kernel(const __grid_constant__ SmallParams p) {
  extern __shared__ __align__(16) __half small[];
  __shared__ double sums[kSmallThreads / 32];
  __half* hi = small;
  __half* lo = hi + p.rows * p.pitch;
  __half* next = lo + p.rows * p.pitch;  // hi of the next step
  __half* s = next + p.rows * p.pitch;
  __half* q = s + p.rows * p.s_pitch;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool tall = p.height > p.width;
  const T* g = static_cast<const T*>(p.g) + blockIdx.x * p.batch_stride;
  const int count = p.height * p.width;
  // thread t has the values t, t + kSmallThreads, ... of the matrix
  const int rows_on = kSmallThreads / p.width, columns_on = kSmallThreads % p.width, r_first = threadIdx.x / p.width, c_first = threadIdx.x % p.width;
  double sum = 0.0;
  int r = r_first, c = c_first;
#pragma unroll 8
  for (int i = threadIdx.x; i < count; i += kSmallThreads) {
    const double v = (double)to_float(g[r * p.stride + c]);
    sum = fma(v, v, sum);
    r += rows_on;
    c += columns_on;
    if (c >= p.width) c -= p.width, ++r;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  if (p.side % 16 || p.length % 16)  // what rounds X up
    for (int i = threadIdx.x; i < p.rows * p.pitch * 3 / 2; i += kSmallThreads) reinterpret_cast<uint32_t*>(small)[i] = 0u;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kSmallThreads / 32; ++w) sum += sums[w];
  const double norm = sqrt(sum), room = (norm / (norm + (double)p.eps)) * (double)p.growth;
  int k = 0;
  while (k < 126 && room * exp2((double)(k + 1)) <= 1.0) ++k;
  const float scale = exp2f((float)-k);
  const double factor = exp2((double)k) / (norm + (double)p.eps);
  r = r_first, c = c_first;
#pragma unroll 8
  for (int i = threadIdx.x; i < count; i += kSmallThreads) {
    const float v = (float)((double)to_float(g[r * p.stride + c]) * factor);
    const __half h = __float2half_rn(v);
    const int at = tall ? c * p.pitch + r : r * p.pitch + c;
    hi[at] = h;
    lo[at] = __float2half_rn((v - __half2float(h)) * 2048.0f);
    r += rows_on;
    c += columns_on;
    if (c >= p.width) c -= p.width, ++r;
  }
  __syncthreads();
  const int row_tiles = p.rows / 16, s_tiles = row_tiles * row_tiles, length = (p.length + 15) / 16 * 16, x_tiles = row_tiles * (length / 16);
  const int r0 = lane / 4, c0 = (lane & 3) * 2;  // of a thread's part of a tile: rows r0 and r0 + 8, columns c0 and c0 + 1
  const float c1 = p.b * scale * scale, c2 = p.c * scale * scale * scale * scale;
  for (int step = 0; step < p.steps; ++step) {
    for (int t = warp; t < s_tiles; t += kSmallThreads / 32) {
      const int row = t / row_tiles * 16, col = t % row_tiles * 16;
      float d[2][4];
      small_product<false>(d[0], d[1], hi, p.pitch, hi, p.pitch, row, col, length);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __half* to = s + (row + r0 + (j >> 1) * 8) * p.s_pitch + col + c0;
        *reinterpret_cast<__half2*>(to + (j & 1) * 8) = __floats2half2_rn(d[j & 1][(j >> 1) * 2], d[j & 1][(j >> 1) * 2 + 1]);
      }
    }
    __syncthreads();
    for (int t = warp; t < s_tiles; t += kSmallThreads / 32) {
      const int row = t / row_tiles * 16, col = t % row_tiles * 16;
      float d[2][4];
      small_product<false>(d[0], d[1], s, p.s_pitch, s, p.s_pitch, row, col, p.rows);  // S is its own mirror image
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = (row + r0 + (j >> 1) * 8) * p.s_pitch + col + c0 + (j & 1) * 8;
        const float2 old = __half22float2(*reinterpret_cast<const __half2*>(s + at));
        const float* v = d[j & 1] + (j >> 1) * 2;
        *reinterpret_cast<__half2*>(q + at) = __floats2half2_rn(fmaf(c2, v[0], c1 * old.x), fmaf(c2, v[1], c1 * old.y));
      }
    }
    __syncthreads();
    const bool last = step == p.steps - 1;
#pragma unroll 1
    for (int t = warp; t < x_tiles; t += kSmallThreads / 32) {
      float d[2][4];
      small_product<true>(d[0], d[1], q, p.s_pitch, hi, p.pitch, t % row_tiles * 16, t / row_tiles * 16, p.rows);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = t % row_tiles * 16 + r0 + (j >> 1) * 8, col = t / row_tiles * 16 + c0 + (j & 1) * 8, at = row * p.pitch + col;
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(hi + at)), l = __half22float2(*reinterpret_cast<const __half2*>(lo + at));
        const float* v = d[j & 1] + (j >> 1) * 2;
        const float x0 = fmaf(p.a, fmaf(l.x, 1.0f / 2048.0f, h.x), v[0]), x1 = fmaf(p.a, fmaf(l.y, 1.0f / 2048.0f, h.y), v[1]);
        if (last) {
          __nv_bfloat16* out = p.out + (int64_t)blockIdx.x * count;
          if (row < p.side && col < p.length) out[tall ? col * p.width + row : row * p.width + col] = __float2bfloat16_rn(x0 * scale);
          if (row < p.side && col + 1 < p.length) out[tall ? (col + 1) * p.width + row : row * p.width + col + 1] = __float2bfloat16_rn(x1 * scale);
        } else {
          const __half2 nh = __floats2half2_rn(x0, x1);
          const float2 f = __half22float2(nh);
          *reinterpret_cast<__half2*>(next + at) = nh;
          *reinterpret_cast<__half2*>(lo + at) = __floats2half2_rn((x0 - f.x) * 2048.0f, (x1 - f.y) * 2048.0f);
        }
      }
    }
    __half* old = hi;
    hi = next;
    next = old;
    __syncthreads();
  }
}

}  // namespace dev

namespace {

struct Layout {
  int64_t ld, side, ld_side, parts;
  size_t x, s;  // bytes of one array of the size of X, and of S
  size_t total;
};
size_t round_up(size_t v) { return (v + 255) / 256 * 256; }
Layout layout_of(size_t batch, size_t height, size_t width) {
  Layout l;
  l.ld = (width + 7) / 8 * 8;
  l.side = height < width ? height : width;
  l.ld_side = (l.side + 7) / 8 * 8;
  // blocks: about eight an SM, and no more than have four groups a thread
  const size_t most = (height * (width + 7) / 8 + 4 * dev::kNormThreads - 1) / (4 * dev::kNormThreads), some = (1184 + batch - 1) / (batch ? batch : 1);
  l.parts = most < some ? most : some;
  l.x = round_up(batch * height * l.ld * 2);
  l.s = round_up(batch * l.side * l.ld_side * 2);
  l.total = round_up(batch * l.parts * 8) + round_up(batch * 4 + 4) + 3 * l.x + 2 * l.s;
  return l;
}

bool matrices_ok(size_t batch, size_t height, size_t width) {
  const size_t most = (size_t)1 << 24;
  return height > 0 && width > 0 && height < most && width < most && batch <= 65535 && batch <= ((size_t)1 << 48) / (height * width);
}

template <typename T, bool kVector>
void scale_of(const dev::ScaleParams& p, size_t batch, cudaStream_t stream) {
  const dim3 grid((unsigned)p.parts, (unsigned)batch);
  dev::hc_square_sum_kernel<T, kVector><<<grid, dev::kNormThreads, 0, stream>>>(p);
  dev::hc_scale_kernel<T, kVector><<<grid, dev::kNormThreads, 0, stream>>>(p);
}
template <typename T>
void scale(const dev::ScaleParams& p, size_t batch, cudaStream_t stream) {
  const bool vector = (reinterpret_cast<uintptr_t>(p.g) & 15u) == 0 && p.width % 8 == 0 && p.stride % 8 == 0 && (batch == 1 || p.batch_stride % 8 == 0);
  if (vector) scale_of<T, true>(p, batch, stream);
  else scale_of<T, false>(p, batch, stream);
}

// What `steps` steps do to a singular value that starts in [0, 1]: with s its square, a step takes it to |a + b s + c s s| times
// itself.  `growth`: at most how many times as large one of them gets (X of a small norm is held times 2^k by it).  False if X, S
// or the polynomial may leave the range of fp16 in which they are held: if a product begins with a singular value above 244, or with a
// b s + c s s above 60000.  The coefficients that the iteration is used with keep all of them below 4.
bool iteration_ok(int steps, double a, double b, double c, float* growth) {
  constexpr double kMost = 60000.0;
  *growth = 1.0f;
  double most = 1.0;  // the largest singular value there can be
  for (int i = 0; i < steps; ++i) {
    const double end = most * most;
    // largest absolute values over s in [0, end]: at the ends, or where a derivative is 0
    const auto factor = [&](double s) { return fabs(a + s * (b + s * c)); };
    const auto poly = [&](double s) { return fabs(s * (b + s * c)); };
    const auto value = [&](double s) { return sqrt(s) * factor(s); };
    double f = fmax(factor(0.0), factor(end)), q = poly(end), v = value(end);
    const double middle = -b / (2.0 * c);  // of both parabolas
    if (middle > 0.0 && middle < end) f = fmax(f, factor(middle)), q = fmax(q, poly(middle));
    const double root = 9.0 * b * b - 20.0 * a * c;  // a + 3 b s + 5 c s s = 0
    for (int sign = -1; sign <= 1; sign += 2) {
      const double s = c != 0.0 ? (-3.0 * b + sign * sqrt(root)) / (10.0 * c) : -a / (3.0 * b);
      if (s > 0.0 && s < end) v = fmax(v, value(s));
    }
    if (!(end <= kMost) || !(q <= kMost) || !(f < INFINITY)) return false;
    if (f > 1.0) *growth *= (float)f;
    most = v;
  }
  return true;
}

constexpr int kSmallSmem = 224 * 1024;

// The form for small matrices: where its tiles fit a warp's registers and shared memory, and a block is done with a matrix
// sooner than the general form goes through its three products.  A step of that takes 16 us and more; a block computes about
// 1.2 MFLOP a microsecond (five steps of 1 x 128 x 128 take 66 us here, of 1 x 144 x 144 92; of 1 x 145 x 145, the general form, 100).
bool small_plan(dev::SmallParams* p, size_t batch, size_t height, size_t width, int* smem) {
  const int64_t side = height < width ? height : width, length = height < width ? width : height;
  const int64_t rows = (side + 15) / 16 * 16, long_rows = (length + 15) / 16 * 16;
  if (long_rows > 4096) return false;
  // rows of 16 bytes more than a whole number of 32: eight rows of ldmatrix lie in different banks
  p->pitch = (int)long_rows + 8;
  p->s_pitch = (int)rows + 8;
  const int64_t bytes = (3 * rows * p->pitch + 2 * rows * p->s_pitch) * 2;
  if (bytes > kSmallSmem) return false;
  *smem = (int)bytes;
  const int64_t sms = device_info().sms > 0 ? device_info().sms : 1, waves = ((int64_t)batch + sms - 1) / sms;
  const double flop = 2.0 * rows * rows * (2.0 * long_rows + rows);
  if (waves * flop / 1.2e6 > 16.0) return false;
  p->height = (int)height, p->width = (int)width, p->side = (int)side, p->length = (int)length, p->rows = (int)rows;
  return true;
}
template <typename T>
cudaError_t run_small(const dev::SmallParams& p, size_t batch, int smem, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  const cudaError_t e = allow_smem(dev::hc_newton_small_kernel<T>, kSmallSmem, &allowed);
  if (e != cudaSuccess) return e;
  dev::hc_newton_small_kernel<T><<<(unsigned)batch, dev::kSmallThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace
}  // namespace hc

extern "C" {

size_t hc_orthogonalize_bytes(size_t batch, size_t height, size_t width) {
  return batch && hc::matrices_ok(batch, height, width) ? hc::layout_of(batch, height, width).total : 0;
}

int hc_orthogonalize(const void* g, int type, size_t batch, size_t height, size_t width, size_t stride, size_t batch_stride, void* out,
                     int steps, float a, float b, float c, float eps, void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  if (!element_type_ok(type) || !matrices_ok(batch, height, width) || stride < width || steps < 1 || steps > 100 || !(eps >= 0.0f)) return kErrArgument;
  if (stride > ((size_t)1 << 32) || batch_stride > ((size_t)1 << 56)) return kErrArgument;
  float growth;
  if (!iteration_ok(steps, a, b, c, &growth)) return kErrArgument;
  if (batch == 0) return kOk;
  if (!g || !out || !scratch || !lies_at(g, element_bytes(type)) || !lies_at(out, 2) || !lies_at(scratch, 256)) return kErrArgument;
  const Layout l = layout_of(batch, height, width);
  if (scratch_bytes < l.total) return kErrArgument;
  dev::SmallParams small;
  int smem = 0;
  if (small_plan(&small, batch, height, width, &smem)) {
    small.g = g;
    small.out = static_cast<__nv_bfloat16*>(out);
    small.stride = (int64_t)stride, small.batch_stride = (int64_t)batch_stride;
    small.steps = steps;
    small.a = a, small.b = b, small.c = c, small.eps = eps, small.growth = growth;
    const cudaError_t e = type == kF32 ? run_small<float>(small, batch, smem, stream)
                          : type == kBf16 ? run_small<__nv_bfloat16>(small, batch, smem, stream) : run_small<__half>(small, batch, smem, stream);
    return e == cudaSuccess ? kOk : kErrCuda;
  }
  unsigned char* at = static_cast<unsigned char*>(scratch);
  double* partial = reinterpret_cast<double*>(at);
  at += round_up(batch * l.parts * 8);
  float* scales = reinterpret_cast<float*>(at);
  unsigned int* arrived = reinterpret_cast<unsigned int*>(scales + batch);
  at += round_up(batch * 4 + 4);
  void* hi[2] = {at, at + l.x};
  void* lo = at + 2 * l.x;
  void* gram = at + 3 * l.x;
  void* poly = at + 3 * l.x + l.s;
  const dev::ScaleParams p = {g, partial, static_cast<__half*>(hi[0]), static_cast<__half*>(lo), scales, arrived, growth, (int64_t)height, (int64_t)width, (int64_t)stride,
                              (int64_t)batch_stride, l.ld, (int)l.parts, eps};
  if (type == kF32) scale<float>(p, batch, stream);
  else if (type == kBf16) scale<__nv_bfloat16>(p, batch, stream);
  else scale<__half>(p, batch, stream);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  const bool wide = height <= width;
  const int64_t x_stride = (int64_t)height * l.ld, s_stride = l.side * l.ld_side;
  GemmChain chain;
  memset(&chain, 0, sizeof(chain));
  chain.steps = steps;
  chain.arrived = arrived;
  const GemmOperand s = {gram, l.ld_side, s_stride, true}, q = {poly, l.ld_side, s_stride, true};
  GemmCall call;
  memset(&call, 0, sizeof(call));
  call.type = call.out_type = kF16;
  call.batch = (int64_t)batch;
  call.ca = a, call.cb = b, call.cc = c;
  call.scale = scales;
  chain.poly = call;
  chain.poly.m = chain.poly.n = chain.poly.k = l.side;
  chain.poly.a = chain.poly.b = s;
  chain.poly.in = {gram, l.ld_side, s_stride};
  chain.poly.out = {poly, l.ld_side, s_stride};
  for (int i = 0; i < 2; ++i) {  // from hi[i] to the other one
    GemmOperand x = {hi[i], l.ld, x_stride, wide};  // along its rows, or (tall) down its columns
    chain.gram[i] = call;
    chain.gram[i].m = chain.gram[i].n = l.side;
    chain.gram[i].k = wide ? width : height;
    chain.gram[i].a = chain.gram[i].b = x;
    chain.gram[i].out = {gram, l.ld_side, s_stride};
    x.k_major = !wide;
    GemmCall& u = chain.update[i];
    u = call;
    u.m = height;
    u.n = width;
    u.k = l.side;
    u.a = wide ? q : x;
    u.b = wide ? x : q;
    u.in = {hi[i], l.ld, x_stride};
    u.in2 = u.out2 = {lo, l.ld, x_stride};
    u.out = {hi[1 - i], l.ld, x_stride};
  }
  chain.last = chain.update[(steps - 1) & 1];
  chain.last.out = {out, (int64_t)width, (int64_t)(height * width)};
  chain.last.out2 = {nullptr, 0, 0};
  chain.last.out_type = kBf16;
  return launch_chain(chain, stream) == cudaSuccess ? kOk : kErrCuda;
}

}  // extern "C"
