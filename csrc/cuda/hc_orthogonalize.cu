// Newton-Schulz iteration of a batch of matrices: X = G / (|G| + eps), then X = a X + (b S + c S S) X with S = X X^T, or
// X = a X + X (b S + c S S) with S = X^T X where that is the smaller one.  Three products a step (hc_gemm.cu), of which
// the first two give symmetric matrices and compute one half.
//
// Operands are fp16: 11 bits, and no entry of X, S or the polynomial leaves its range once |X| <= 1.  What is rounded off
// X in directions that G hardly has would grow by `a` in every step (485 times in five); products with X carry none of it
// there, only the term a X does, so that term takes X from two fp16 numbers, hi and lo / 2048.  A matrix whose norm is far
// below eps stays small: it is held times 2^k, with k from what its norm can grow to in `steps`, and S counts 2^-2k.
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
  float growth;
  int64_t height, width, stride, batch_stride, ld;  // ld: of hi and lo
  int parts;
  int lanes;  // threads of a block that share a row, a power of two
  float eps;
};

// The values of one matrix in groups of eight, a block's share of them: f(row, column, values)
template <typename T, bool kVector, typename F>
__device__ __forceinline__ void for_groups(const ScaleParams& p, const T* g, F f) {
  const int rows = kNormThreads / p.lanes, lane = threadIdx.x & (p.lanes - 1);
  for (int64_t r = (int64_t)blockIdx.x * rows + threadIdx.x / p.lanes; r < p.height; r += (int64_t)p.parts * rows)
#pragma unroll 4
    for (int64_t c = lane * 8; c < p.width; c += p.lanes * 8) {
      float v[8];
      if (kVector) {
        load8(g + r * p.stride + c, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < p.width ? to_float(g[r * p.stride + c + j]) : 0.0f;
      }
      f(r, c, v);
    }
}

// Sums of squares, in 64 bits: the entries may be anything that their type can hold.  Bound by memory.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kNormThreads) hc_square_sum_kernel(const __grid_constant__ ScaleParams p) {
  __shared__ double sums[kNormThreads / 32];
  double s = 0.0;
  for_groups<T, kVector>(p, static_cast<const T*>(p.g) + blockIdx.y * p.batch_stride, [&](int64_t, int64_t, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fma((double)v[j], (double)v[j], s);
  });
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

}  // namespace dev

namespace {

struct Layout {
  int64_t ld, side, ld_side, parts;
  int lanes;
  size_t x, s;  // bytes of one array of the size of X, and of S
  size_t total;
};
size_t round_up(size_t v) { return (v + 255) / 256 * 256; }
Layout layout_of(size_t batch, size_t height, size_t width) {
  Layout l;
  l.ld = (width + 7) / 8 * 8;
  l.side = height < width ? height : width;
  l.ld_side = (l.side + 7) / 8 * 8;
  l.lanes = 1;
  while (l.lanes < dev::kNormThreads && (size_t)l.lanes * 8 < width) l.lanes *= 2;
  const size_t rows = dev::kNormThreads / l.lanes, most = (height + rows - 1) / rows, some = (1184 + batch - 1) / (batch ? batch : 1);
  l.parts = most < some ? most : some;  // about eight blocks an SM
  l.x = round_up(batch * height * l.ld * 2);
  l.s = round_up(batch * l.side * l.ld_side * 2);
  l.total = round_up(batch * l.parts * 8) + round_up(batch * 4) + 3 * l.x + 2 * l.s;
  return l;
}

bool matrices_ok(size_t batch, size_t height, size_t width) {
  const size_t most = (size_t)1 << 24;
  return height > 0 && width > 0 && height < most && width < most && batch <= 65535;
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
  if (batch == 0) return kOk;
  if (!g || !out || !scratch || (reinterpret_cast<uintptr_t>(scratch) & 255u)) return kErrArgument;
  const Layout l = layout_of(batch, height, width);
  if (scratch_bytes < l.total) return kErrArgument;
  unsigned char* at = static_cast<unsigned char*>(scratch);
  double* partial = reinterpret_cast<double*>(at);
  at += round_up(batch * l.parts * 8);
  float* scales = reinterpret_cast<float*>(at);
  at += round_up(batch * 4);
  void* hi[2] = {at, at + l.x};
  void* lo = at + 2 * l.x;
  void* gram = at + 3 * l.x;
  void* poly = at + 3 * l.x + l.s;
  float growth = 1.0f;
  for (int i = 0; i < steps; ++i) growth *= a > 1.0f || a < -1.0f ? (a < 0.0f ? -a : a) : 1.0f;
  const dev::ScaleParams p = {g, partial, static_cast<__half*>(hi[0]), static_cast<__half*>(lo), scales, growth, (int64_t)height, (int64_t)width, (int64_t)stride,
                              (int64_t)batch_stride, l.ld, (int)l.parts, l.lanes, eps};
  if (type == kF32) scale<float>(p, batch, stream);
  else if (type == kBf16) scale<__nv_bfloat16>(p, batch, stream);
  else scale<__half>(p, batch, stream);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  const bool wide = height <= width;
  const int64_t x_stride = (int64_t)height * l.ld, s_stride = l.side * l.ld_side;
  for (int i = 0; i < steps; ++i) {
    const GemmOperand x = {hi[i & 1], l.ld, x_stride, wide};  // along its rows, or (tall) down its columns
    const GemmOperand s = {gram, l.ld_side, s_stride, true}, q = {poly, l.ld_side, s_stride, true};
    GemmCall call;
    memset(&call, 0, sizeof(call));
    call.type = kF16;
    call.batch = (int64_t)batch;
    call.ca = a, call.cb = b, call.cc = c;
    call.scale = scales;
    call.mode = kGemmGram;
    call.m = call.n = l.side;
    call.k = wide ? width : height;
    call.a = call.b = x;
    call.out = {gram, l.ld_side, s_stride};
    call.out_type = kF16;
    if (launch_gemm(call, stream) != cudaSuccess) return kErrCuda;
    call.mode = kGemmPoly;
    call.k = l.side;
    call.a = call.b = s;
    call.in = call.out;
    call.out = {poly, l.ld_side, s_stride};
    if (launch_gemm(call, stream) != cudaSuccess) return kErrCuda;
    const bool last = i == steps - 1;
    call.mode = kGemmUpdate;
    call.m = height;
    call.n = width;
    GemmOperand y = x;
    y.k_major = !wide;
    call.a = wide ? q : y;
    call.b = wide ? y : q;
    call.in = {hi[i & 1], l.ld, x_stride};
    call.in2 = {lo, l.ld, x_stride};
    call.out = last ? GemmSide{out, (int64_t)width, (int64_t)(height * width)} : GemmSide{hi[(i + 1) & 1], l.ld, x_stride};
    call.out2 = last ? GemmSide{nullptr, 0, 0} : call.in2;
    call.out_type = last ? kBf16 : kF16;
    if (launch_gemm(call, stream) != cudaSuccess) return kErrCuda;
  }
  return kOk;
}

}  // extern "C"
