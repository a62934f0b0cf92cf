// act(x W^T + b) + residual and its backward pass: the products are hc_gemm.cu's, here is what lies around them.
#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

// ---- a few rows -----------------------------------------------------------------------------------------------------
// With up to eight rows the weights are read once and everything else is small: a warp takes two columns of the result,
// its lanes go along the sum in groups of eight and add up all rows' products, in fp32, joined over the warp at the end.
// Bound by reading W; the tensor cores would compute 128 rows for these few.
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

template <typename T, int R, bool kVector>
__global__ void __launch_bounds__(256) hc_few_rows_kernel(const __grid_constant__ FewRowsParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t first = (blockIdx.x * 8ll + (threadIdx.x >> 5)) * 2;
  if (first >= p.width) return;
  const bool two = first + 1 < p.width;
  const T* w0 = static_cast<const T*>(p.w) + first * p.ldw;
  const T* w1 = two ? w0 + p.ldw : w0;
  const T* x = static_cast<const T*>(p.x);
  float sum[2][R];
#pragma unroll
  for (int r = 0; r < R; ++r) sum[0][r] = sum[1][r] = 0.0f;
  if (kVector) {
    for (int64_t k = lane * 8; k < p.inner; k += 256) {
      float a[8], b[8], v[8];
      load8(w0 + k, a);
      load8(w1 + k, b);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < p.rows) {
          load8(x + r * p.ldx + k, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum[0][r] = fmaf(v[j], a[j], sum[0][r]);
            sum[1][r] = fmaf(v[j], b[j], sum[1][r]);
          }
        }
      }
    }
  } else {
    for (int64_t k = lane; k < p.inner; k += 32) {
      const float a = to_float(w0[k]), b = to_float(w1[k]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < p.rows) {
          const float v = to_float(x[r * p.ldx + k]);
          sum[0][r] = fmaf(v, a, sum[0][r]);
          sum[1][r] = fmaf(v, b, sum[1][r]);
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v = warp_sum(sum[c][r]);
      const int64_t n = first + c;
      if (lane == r && r < p.rows && n < p.width) {  // lane r stores row r
        if (p.bias) v += param_at(p.bias, p.bias_type, n);
        if (p.z) static_cast<T*>(p.z)[r * p.ldz + n] = from_float<T>(v);
        v = act_value(v, p.activation);
        if (p.residual) v += param_at(p.residual, p.out_type, r * p.ldr + n);
        param_put(p.out, p.out_type, r * p.ldo + n, v);
      }
    }
}

// ---- rows of the backward pass ----------------------------------------------------------------------------------------
// dz = dy act'(z), rounded for the products, and the sums of its columns.  A thread has eight columns, a block 256 and a
// share of the rows.  Bound by memory.
struct RowsBackwardParams {
  const void *dy, *z;
  void* dz;
  float* partial;  // [share][width]
  int64_t ldy, ldz, ldd, rows, width;
  int activation, shares;
};

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
// dW has few tiles and a long sum: parts of the sum go to different SMs, which leave fp32 matrices that are added here.
template <typename T>
__global__ void __launch_bounds__(256) hc_add_parts_kernel(const float* parts, int n, int64_t rows, int64_t width, int64_t ld, int64_t stride, T* out, int64_t ldo) {
  const int64_t groups = (width + 7) / 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * groups; i += gridDim.x * 256ll) {
    const int64_t r = i / groups, c = (i - r * groups) * 8;
    float s[8], v[8];
    load8(parts + r * ld + c, s);
    for (int k = 1; k < n; ++k) {
      load8(parts + k * stride + r * ld + c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
    T* to = out + r * ldo + c;
    if (c + 8 <= width && ((reinterpret_cast<uintptr_t>(to) & 15u) == 0)) {
      store8(to, s);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < width) to[j] = from_float<T>(s[j]);
    }
  }
}

}  // namespace dev

namespace {

constexpr size_t kMostSize = (size_t)1 << 26;  // of each side: a tile's sum then stays far below the limit of a wait
constexpr size_t kFewRows = 8;

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

template <typename T, int R>
void few_rows_of(const dev::FewRowsParams& p, bool vector, cudaStream_t stream) {
  const unsigned grid = (unsigned)((p.width + 15) / 16);
  if (vector) dev::hc_few_rows_kernel<T, R, true><<<grid, 256, 0, stream>>>(p);
  else dev::hc_few_rows_kernel<T, R, false><<<grid, 256, 0, stream>>>(p);
}
template <typename T>
void few_rows(const dev::FewRowsParams& p, bool vector, cudaStream_t stream) {
  if (p.rows == 1) few_rows_of<T, 1>(p, vector, stream);
  else if (p.rows == 2) few_rows_of<T, 2>(p, vector, stream);
  else if (p.rows <= 4) few_rows_of<T, 4>(p, vector, stream);
  else few_rows_of<T, 8>(p, vector, stream);
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

// scratch memory of a backward pass: sums of columns, sums of parts of the rows, dz
struct BackwardLayout {
  size_t sums, parts, total;
};
BackwardLayout backward_layout(size_t rows, size_t inner, size_t width, int keep_dz) {
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  const int parts = gemm_parts((int64_t)width, (int64_t)inner, (int64_t)rows);
  BackwardLayout l;
  l.sums = up((size_t)shares_of(rows, width, kActNone) * width * sizeof(float));  // the most there are
  l.parts = parts > 1 ? up((size_t)parts * width * ((inner + 7) / 8 * 8) * sizeof(float)) : 0;
  l.total = l.sums + l.parts + (keep_dz ? up(rows * ((width + 7) / 8 * 8) * 2) : 0);
  return l;
}

bool aligned_rows(const void* p, size_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 8 == 0; }

}  // namespace
}  // namespace hc

extern "C" {

int hc_linear(const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, const void* bias, int bias_type,
              const void* residual, size_t residual_stride, void* out, int out_type, size_t out_stride, void* z, size_t z_stride,
              int activation, size_t rows, size_t inner, size_t width, hc_stream_t stream) {
  using namespace hc;
  if (!product_type(type) || (out_type != kF32 && out_type != type) || !element_type_ok(bias_type)) return kErrArgument;
  if (activation < kActNone || activation > kActSilu || !sizes_ok(rows, inner, width)) return kErrArgument;
  if (!stride_ok(x_stride, inner) || !stride_ok(weight_stride, inner) || !stride_ok(out_stride, width)) return kErrArgument;
  if ((residual && !stride_ok(residual_stride, width)) || (z && !stride_ok(z_stride, width))) return kErrArgument;
  if (rows == 0) return kOk;
  if (!x || !weight || !out) return kErrArgument;
  if (rows <= kFewRows) {
    const dev::FewRowsParams p = {x, weight, bias, residual, out, z, (int64_t)x_stride, (int64_t)weight_stride, (int64_t)residual_stride,
                                  (int64_t)out_stride, (int64_t)z_stride, (int64_t)inner, (int64_t)width, (int)rows, out_type, bias_type, activation};
    const bool vector = inner % 8 == 0 && aligned_rows(x, x_stride) && aligned_rows(weight, weight_stride);
    if (type == kBf16) few_rows<__nv_bfloat16>(p, vector, stream);
    else few_rows<__half>(p, vector, stream);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
  }
  if (!gemm_operand_ok(x, x_stride) || !gemm_operand_ok(weight, weight_stride)) return kErrArgument;
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
  return launch_gemm(c, stream) == cudaSuccess ? kOk : kErrCuda;
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
  if (dbias || (products && keep_dz)) {
    const dev::RowsBackwardParams p = {dy, z, products && keep_dz ? const_cast<void*>(dz) : nullptr, dbias ? reinterpret_cast<float*>(at) : nullptr,
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
  if (dx) {
    c.m = rows, c.n = inner, c.k = width;
    c.a = {dz, (int64_t)dz_stride, 0, true};
    c.b = {weight, (int64_t)weight_stride, 0, false};
    c.out = {dx, (int64_t)dx_stride, 0};
    if (launch_gemm(c, stream) != cudaSuccess) return kErrCuda;
  }
  if (dweight) {
    c.m = width, c.n = inner, c.k = rows;
    c.a = {dz, (int64_t)dz_stride, 0, false};
    c.b = {x, (int64_t)x_stride, 0, false};
    c.out = {dweight, (int64_t)dweight_stride, 0};
    c.parts = gemm_parts(c.m, c.n, c.k);
    const int64_t ld = (int64_t)(inner + 7) / 8 * 8, stride = (int64_t)width * ld;
    float* sums = reinterpret_cast<float*>(at + l.sums);
    if (c.parts > 1) {
      c.out_type = kF32;
      c.out = {sums, ld, stride};
    }
    if (launch_gemm(c, stream) != cudaSuccess) return kErrCuda;
    if (c.parts > 1) {
      const int64_t groups = (int64_t)width * (ld / 8);
      const unsigned grid = (unsigned)((groups + 255) / 256 < 2368 ? (groups + 255) / 256 : 2368);
      if (type == kBf16)
        dev::hc_add_parts_kernel<<<grid, 256, 0, stream>>>(sums, c.parts, (int64_t)width, (int64_t)inner, ld, stride, static_cast<__nv_bfloat16*>(dweight), (int64_t)dweight_stride);
      else
        dev::hc_add_parts_kernel<<<grid, 256, 0, stream>>>(sums, c.parts, (int64_t)width, (int64_t)inner, ld, stride, static_cast<__half*>(dweight), (int64_t)dweight_stride);
      if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    }
  }
  return kOk;
}

}  // extern "C"
