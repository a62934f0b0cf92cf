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
  float eps;
};

// sums of squares, in 64 bits: the entries may be anything that their type can hold
template <typename T>
__global__ void __launch_bounds__(kNormThreads) hc_square_sum_kernel(const __grid_constant__ ScaleParams p) {
  __shared__ double sums[kNormThreads / 32];
  const T* g = static_cast<const T*>(p.g) + blockIdx.y * p.batch_stride;
  double s = 0.0;
  for (int64_t r = blockIdx.x; r < p.height; r += p.parts)
    for (int64_t c = threadIdx.x; c < p.width; c += kNormThreads) {
      const double v = (double)to_float(g[r * p.stride + c]);
      s = fma(v, v, s);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; ++w) s += sums[w];
    p.partial[(int64_t)blockIdx.y * p.parts + blockIdx.x] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) hc_scale_kernel(const __grid_constant__ ScaleParams p) {
  __shared__ double total;
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < p.parts; i += 32) s += p.partial[(int64_t)blockIdx.y * p.parts + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) total = s;
  }
  __syncthreads();
  const double norm = sqrt(total), room = (norm / (norm + (double)p.eps)) * (double)p.growth;
  int k = 0;
  while (k < 126 && room * exp2((double)(k + 1)) <= 1.0) ++k;
  const double scale = exp2((double)k) / (norm + (double)p.eps);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.scale[blockIdx.y] = exp2f((float)-k);
  const T* g = static_cast<const T*>(p.g) + blockIdx.y * p.batch_stride;
  const int64_t at = (int64_t)blockIdx.y * p.height * p.ld;
  for (int64_t r = blockIdx.x; r < p.height; r += gridDim.x)
    for (int64_t c = threadIdx.x; c < p.width; c += kNormThreads) {
      const float v = (float)((double)to_float(g[r * p.stride + c]) * scale);
      const __half hi = __float2half_rn(v);
      p.hi[at + r * p.ld + c] = hi;
      p.lo[at + r * p.ld + c] = __float2half_rn((v - __half2float(hi)) * 2048.0f);
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
  l.parts = height < 64 ? height : 64;
  l.x = round_up(batch * height * l.ld * 2);
  l.s = round_up(batch * l.side * l.ld_side * 2);
  l.total = round_up(batch * l.parts * 8) + round_up(batch * 4) + 3 * l.x + 2 * l.s;
  return l;
}

bool matrices_ok(size_t batch, size_t height, size_t width) {
  const size_t most = (size_t)1 << 24;
  return height > 0 && width > 0 && height < most && width < most && batch <= 65535;
}

template <typename T>
void scale(const dev::ScaleParams& p, size_t batch, cudaStream_t stream) {
  dev::hc_square_sum_kernel<T><<<dim3((unsigned)p.parts, (unsigned)batch), dev::kNormThreads, 0, stream>>>(p);
  const int64_t rows = p.height < 1024 ? p.height : 1024;
  dev::hc_scale_kernel<T><<<dim3((unsigned)rows, (unsigned)batch), dev::kNormThreads, 0, stream>>>(p);
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
                              (int64_t)batch_stride, l.ld, (int)l.parts, eps};
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
