// Layer norm over rows: y = (x - mean) rstd w + b, and its backward pass.
//
// A row is held in registers by T threads (a warp, or a block), K groups of eight values a thread, so x is read once:
// mean first, then the squares of what is left of it (no difference of large sums).  The backward pass reads x and dy
// once,
//   h = (x - mean) rstd,  dx = rstd (w dy - mean(w dy) - h mean(w dy h)),  dw = sum dy h,  db = sum dy,
// with the column sums of a thread's own columns in its registers over all rows that its block works on.  Rows whose
// length eight does not divide begin at one of eight places within an aligned group; a block takes rows that begin at
// the same place, so that its threads keep their columns (and their w) from row to row.  The sums of the blocks are
// added by a second kernel in a fixed order.  Both passes are bound by memory.
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

struct NormParams {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* out;       // y, or dx
  float* stats;    // [rows][2]: mean, rstd
  float* partial;  // backward: [block][2][width]
  int64_t rows, width;
  float eps;
  int param_type;
  int period;  // rows r, r + period, ... begin at the same place of an aligned group
};

// T threads a row, K groups of eight a thread; T = 32: one row a warp, 8 warps a block
template <typename X, typename Y, int T, int K>
__global__ void __launch_bounds__(T == 32 ? 256 : T) hc_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[T / 32];
  const int lane = T == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t team = T == 32 ? blockIdx.x * 8ll + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t teams = T == 32 ? gridDim.x * 8ll : gridDim.x;
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = team; row < p.rows; row += teams) {
    const int shift = (int)(row * p.width & 7);
    const X* x = static_cast<const X*>(p.x) + row * p.width;
    float v[K][8];
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load_group(x, ((int64_t)k * T + lane) * 8 - shift, p.width, v[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[k][j];
    }
    group_sum2<T>(sum, none, shared);
    const float mean = sum * inv;
    float squares = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t first = ((int64_t)k * T + lane) * 8 - shift;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = first + j >= 0 && first + j < p.width ? v[k][j] - mean : 0.0f;
        v[k][j] = c;
        squares = fmaf(c, c, squares);
      }
    }
    none = 0.0f;
    group_sum2<T>(squares, none, shared);
    const float rstd = 1.0f / sqrtf(fmaf(squares, inv, p.eps));
    Y* y = static_cast<Y*>(p.out) + row * p.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t first = ((int64_t)k * T + lane) * 8 - shift;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = first + j;
        const bool in = c >= 0 && c < p.width;
        const float w = p.weight && in ? param_at(p.weight, p.param_type, c) : 1.0f;
        const float b = p.bias && in ? param_at(p.bias, p.param_type, c) : 0.0f;
        v[k][j] = fmaf(v[k][j] * rstd, w, b);
      }
      store_group(y, first, p.width, v[k]);
    }
    if (p.stats && lane == 0) reinterpret_cast<float2*>(p.stats)[row] = make_float2(mean, rstd);
  }
}

template <typename X, typename Y, int T, int K>
__global__ void __launch_bounds__(T == 32 ? 256 : T) hc_norm_backward_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[T / 32];
  constexpr int kTeams = T == 32 ? 8 : 1;
  const int lane = T == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int place = blockIdx.x % p.period;  // rows place, place + period, ... are shared out among the blocks of this place
  const int64_t team = (int64_t)(blockIdx.x / p.period) * kTeams + (T == 32 ? threadIdx.x >> 5 : 0);
  const int64_t teams = (int64_t)(gridDim.x / p.period) * kTeams;
  const int shift = (int)(place * p.width & 7);
  const float inv = 1.0f / (float)p.width;
  float w[K][8], dw[K][8], db[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = ((int64_t)k * T + lane) * 8 - shift + j;
      w[k][j] = c < 0 || c >= p.width ? 0.0f : p.weight ? param_at(p.weight, p.param_type, c) : 1.0f;
      dw[k][j] = db[k][j] = 0.0f;
    }
  for (int64_t row = place + team * p.period; row < p.rows; row += teams * p.period) {
    const X* x = static_cast<const X*>(p.x) + row * p.width;
    const Y* dy = static_cast<const Y*>(p.dy) + row * p.width;
    const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
    float h[K][8], g[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t first = ((int64_t)k * T + lane) * 8 - shift;
      load_group(x, first, p.width, h[k]);
      load_group(dy, first, p.width, g[k]);
    }
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // outside the row g and w are 0 and h is whatever: nothing reaches a sum
        h[k][j] = (h[k][j] - st.x) * st.y;
        dw[k][j] = fmaf(g[k][j], h[k][j], dw[k][j]);
        db[k][j] += g[k][j];
        g[k][j] *= w[k][j];
        a += g[k][j];
        b = fmaf(g[k][j], h[k][j], b);
      }
    if (p.out) {
      group_sum2<T>(a, b, shared);
      a *= inv;
      b *= inv;
      X* dx = static_cast<X*>(p.out) + row * p.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int64_t first = ((int64_t)k * T + lane) * 8 - shift;
#pragma unroll
        for (int j = 0; j < 8; ++j) g[k][j] = st.y * (fmaf(-h[k][j], b, g[k][j]) - a);
        store_group(dx, first, p.width, g[k]);
      }
    }
  }
  if (!p.partial) return;
  float* mine = p.partial + (int64_t)blockIdx.x * 2 * p.width;
  if (T == 32) {  // the block's warps one after the other: a fixed order
    extern __shared__ float sums[];  // [2][K * 256]
    for (int warp = 0; warp < 8; ++warp) {
      if ((threadIdx.x >> 5) == warp) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at = (k * 8 + j) * 32 + lane;
            sums[at] = warp ? sums[at] + dw[k][j] : dw[k][j];
            sums[K * 256 + at] = warp ? sums[K * 256 + at] + db[k][j] : db[k][j];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < K * 256; i += 256) {
      const int64_t c = ((int64_t)(i / 256) * 32 + (i & 31)) * 8 - shift + (i / 32) % 8;
      if (c < 0 || c >= p.width) continue;
      mine[c] = sums[i];
      mine[p.width + c] = sums[K * 256 + i];
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = ((int64_t)k * T + lane) * 8 - shift + j;
        if (c < 0 || c >= p.width) continue;
        mine[c] = dw[k][j];
        mine[p.width + c] = db[k][j];
      }
  }
}

// Rows too long for the registers of a block: three passes over the row, of which the later ones find it in L2.
constexpr int kLong = 1024;
template <typename X, typename Y>
__global__ void __launch_bounds__(kLong) hc_norm_long_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[kLong / 32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const X* x = static_cast<const X*>(p.x) + row * p.width;
    Y* y = static_cast<Y*>(p.out) + row * p.width;
    const int64_t start = -(int64_t)(row * p.width & 7) + threadIdx.x * 8;
    float v[8], sum = 0.0f, squares = 0.0f, none = 0.0f;
    for (int64_t f = start; f < p.width; f += kLong * 8) {
      load_group(x, f, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j];
    }
    group_sum2<kLong>(sum, none, shared);
    const float mean = sum * inv;
    for (int64_t f = start; f < p.width; f += kLong * 8) {
      load_group(x, f, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = f + j >= 0 && f + j < p.width ? v[j] - mean : 0.0f;
        squares = fmaf(c, c, squares);
      }
    }
    none = 0.0f;
    group_sum2<kLong>(squares, none, shared);
    const float rstd = 1.0f / sqrtf(fmaf(squares, inv, p.eps));
    for (int64_t f = start; f < p.width; f += kLong * 8) {
      load_group(x, f, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = f + j;
        const bool in = c >= 0 && c < p.width;
        v[j] = fmaf((v[j] - mean) * rstd, p.weight && in ? param_at(p.weight, p.param_type, c) : 1.0f,
                    p.bias && in ? param_at(p.bias, p.param_type, c) : 0.0f);
      }
      store_group(y, f, p.width, v);
    }
    if (p.stats && threadIdx.x == 0) reinterpret_cast<float2*>(p.stats)[row] = make_float2(mean, rstd);
  }
}

template <typename X, typename Y>
__global__ void __launch_bounds__(kLong) hc_norm_long_dx_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 shared[kLong / 32];
  const float inv = 1.0f / (float)p.width;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const X* x = static_cast<const X*>(p.x) + row * p.width;
    const Y* dy = static_cast<const Y*>(p.dy) + row * p.width;
    X* dx = static_cast<X*>(p.out) + row * p.width;
    const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
    const int64_t start = -(int64_t)(row * p.width & 7) + threadIdx.x * 8;
    float v[8], g[8], a = 0.0f, b = 0.0f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      for (int64_t f = start; f < p.width; f += kLong * 8) {
        load_group(x, f, p.width, v);
        load_group(dy, f, p.width, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t c = f + j;
          v[j] = (v[j] - st.x) * st.y;
          if (p.weight && c >= 0 && c < p.width) g[j] *= param_at(p.weight, p.param_type, c);
          if (pass == 0) {
            a += g[j];
            b = fmaf(g[j], v[j], b);
          } else {
            g[j] = st.y * (fmaf(-v[j], b, g[j]) - a);
          }
        }
        if (pass == 1) store_group(dx, f, p.width, g);
      }
      if (pass == 0) {
        group_sum2<kLong>(a, b, shared);
        a *= inv;
        b *= inv;
      }
    }
  }
}

// column sums of a share of the rows (blockIdx.y), one thread a column
template <typename X, typename Y>
__global__ void __launch_bounds__(256) hc_norm_long_sums_kernel(const __grid_constant__ NormParams p) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= p.width) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
    const float g = to_float(static_cast<const Y*>(p.dy)[row * p.width + c]);
    dw = fmaf(g, (to_float(static_cast<const X*>(p.x)[row * p.width + c]) - st.x) * st.y, dw);
    db += g;
  }
  float* mine = p.partial + (int64_t)blockIdx.y * 2 * p.width;
  mine[c] = dw;
  mine[p.width + c] = db;
}

// adds up the partial sums of `n` blocks: 32 columns a block of 32 x 32 threads, always in the same order
__global__ void __launch_bounds__(1024) hc_norm_finish_kernel(const float* partial, int n, int64_t width, void* dweight,
                                                               void* dbias, int param_type) {
  __shared__ float sums[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < width)
    for (int b = threadIdx.y; b < n; b += 32) s += partial[((int64_t)b * 2 + blockIdx.y) * width + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = warp_sum(sums[threadIdx.x][threadIdx.y]);
  if (threadIdx.x == 0) {
    const int64_t at = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (at < width) param_put(blockIdx.y ? dbias : dweight, param_type, at, s);
  }
}

}  // namespace dev

namespace {

constexpr int64_t kLongestInRegisters = 8192;
constexpr int kBlocksPerSm = 4;

// threads and groups of eight a thread for rows of `width` values (with one group more where rows begin anywhere)
struct Shape {
  int threads, groups;
};
Shape shape_of(size_t width) {
  const int need = (int)((width + 7) / 8) + (width % 8 ? 1 : 0);
  if (need <= 128) return {32, (need + 31) / 32};
  if (need <= 256) return {128, 2};
  if (need <= 512) return {128, 4};
  return {256, 4};
}
int period_of(size_t width) { return width % 8 == 0 ? 1 : width % 4 == 0 ? 2 : width % 2 == 0 ? 4 : 8; }
bool in_registers(size_t width) { return width <= kLongestInRegisters - (width % 8 ? 8 : 0); }

int backward_blocks(size_t rows, size_t width) {
  const int sms = device_info().sms > 0 ? device_info().sms : 1;
  const int period = period_of(width);
  if (!in_registers(width)) return (int)(rows < 64 ? rows : 64);
  const size_t teams = shape_of(width).threads == 32 ? 8 : 1;
  size_t blocks = (rows + teams - 1) / teams;
  const size_t most = (size_t)sms * (shape_of(width).threads == 256 ? 2 : shape_of(width).threads == 128 ? 4 : 2);
  if (blocks > most) blocks = most;
  return (int)((blocks + period - 1) / period * period);
}

template <typename X, typename Y, int T, int K>
cudaError_t run_forward(const dev::NormParams& p, cudaStream_t stream) {
  const int64_t teams = T == 32 ? 8 : 1;
  int64_t blocks = (p.rows + teams - 1) / teams;
  if (blocks > 0x7fffffff) blocks = 0x7fffffff;
  dev::hc_norm_kernel<X, Y, T, K><<<(unsigned)blocks, T == 32 ? 256 : T, 0, stream>>>(p);
  return cudaGetLastError();
}
template <typename X, typename Y, int T, int K>
cudaError_t run_backward(const dev::NormParams& p, int blocks, cudaStream_t stream) {
  dev::hc_norm_backward_kernel<X, Y, T, K><<<blocks, T == 32 ? 256 : T, T == 32 ? K * 2048 : 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename X, typename Y>
cudaError_t forward(const dev::NormParams& p, cudaStream_t stream) {
  if (!in_registers(p.width)) {
    dev::hc_norm_long_kernel<X, Y><<<(unsigned)(p.rows < 65536 ? p.rows : 65536), dev::kLong, 0, stream>>>(p);
    return cudaGetLastError();
  }
  const Shape s = shape_of(p.width);
  if (s.threads == 32) {
    if (s.groups == 1) return run_forward<X, Y, 32, 1>(p, stream);
    if (s.groups == 2) return run_forward<X, Y, 32, 2>(p, stream);
    if (s.groups == 3) return run_forward<X, Y, 32, 3>(p, stream);
    return run_forward<X, Y, 32, 4>(p, stream);
  }
  if (s.threads == 128) return s.groups == 2 ? run_forward<X, Y, 128, 2>(p, stream) : run_forward<X, Y, 128, 4>(p, stream);
  return run_forward<X, Y, 256, 4>(p, stream);
}
template <typename X, typename Y>
cudaError_t backward(const dev::NormParams& p, int blocks, cudaStream_t stream) {
  if (!in_registers(p.width)) {
    if (p.out) dev::hc_norm_long_dx_kernel<X, Y><<<(unsigned)(p.rows < 65536 ? p.rows : 65536), dev::kLong, 0, stream>>>(p);
    if (p.partial) dev::hc_norm_long_sums_kernel<X, Y><<<dim3((unsigned)((p.width + 255) / 256), blocks), 256, 0, stream>>>(p);
    return cudaGetLastError();
  }
  const Shape s = shape_of(p.width);
  if (s.threads == 32) {
    if (s.groups == 1) return run_backward<X, Y, 32, 1>(p, blocks, stream);
    if (s.groups == 2) return run_backward<X, Y, 32, 2>(p, blocks, stream);
    if (s.groups == 3) return run_backward<X, Y, 32, 3>(p, blocks, stream);
    return run_backward<X, Y, 32, 4>(p, blocks, stream);
  }
  if (s.threads == 128) return s.groups == 2 ? run_backward<X, Y, 128, 2>(p, blocks, stream) : run_backward<X, Y, 128, 4>(p, blocks, stream);
  return run_backward<X, Y, 256, 4>(p, blocks, stream);
}

template <typename F>
cudaError_t by_types(int x, int y, F f) {
  using b = __nv_bfloat16;
  using h = __half;
  if (x == kF32) return y == kF32 ? f(float(), float()) : y == kBf16 ? f(float(), b()) : f(float(), h());
  if (x == kBf16) return y == kF32 ? f(b(), float()) : y == kBf16 ? f(b(), b()) : cudaErrorInvalidValue;
  return y == kF32 ? f(h(), float()) : y == kF16 ? f(h(), h()) : cudaErrorInvalidValue;
}

bool norm_arguments_ok(const void* x, int x_type, const void* y, int y_type, int param_type, size_t rows, size_t width) {
  if (!element_type_ok(x_type) || !element_type_ok(y_type) || !element_type_ok(param_type)) return false;
  if (x_type != kF32 && y_type != kF32 && x_type != y_type) return false;
  if (width == 0 || width > (1u << 30) || rows > (1ull << 40) || rows * width > (1ull << 60)) return false;
  return rows == 0 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0;
}

}  // namespace
}  // namespace hc

extern "C" {

int hc_layer_norm(const void* x, int x_type, const void* weight, const void* bias, int param_type, void* y, int y_type,
                  float* stats, size_t rows, size_t width, float eps, hc_stream_t stream) {
  if (!hc::norm_arguments_ok(x, x_type, y, y_type, param_type, rows, width) || !(eps >= 0.0f)) return hc::kErrArgument;
  if (rows == 0) return hc::kOk;
  if (!x || !y) return hc::kErrArgument;
  hc::dev::NormParams p = {x, nullptr, weight, bias, y, stats, nullptr, (int64_t)rows, (int64_t)width, eps, param_type, 1};
  const cudaError_t e = hc::by_types(x_type, y_type, [&](auto a, auto b) { return hc::forward<decltype(a), decltype(b)>(p, stream); });
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

size_t hc_layer_norm_backward_bytes(size_t rows, size_t width) {
  return rows && width ? (size_t)hc::backward_blocks(rows, width) * 2 * width * sizeof(float) : 0;
}

int hc_layer_norm_backward(const void* dy, int y_type, const void* x, int x_type, const void* weight, int param_type,
                           const float* stats, void* dx, void* dweight, void* dbias, size_t rows, size_t width,
                           void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  if (!hc::norm_arguments_ok(x, x_type, dy, y_type, param_type, rows, width) || (!dweight != !dbias)) return hc::kErrArgument;
  if (reinterpret_cast<uintptr_t>(dx) & 15u) return hc::kErrArgument;
  if (rows == 0) {
    if (!dweight) return hc::kOk;
    cudaError_t e = cudaMemsetAsync(dweight, 0, width * hc::element_bytes(param_type), stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, width * hc::element_bytes(param_type), stream);
    return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
  }
  if (!x || !dy || !stats) return hc::kErrArgument;
  if (!dx && !dweight) return hc::kOk;
  const int blocks = hc::backward_blocks(rows, width);
  if (dweight && (!scratch || scratch_bytes < hc_layer_norm_backward_bytes(rows, width))) return hc::kErrArgument;
  hc::dev::NormParams p = {x, dy, weight, nullptr, dx, const_cast<float*>(stats), dweight ? static_cast<float*>(scratch) : nullptr,
                           (int64_t)rows, (int64_t)width, 0.0f, param_type, hc::period_of(width)};
  cudaError_t e = hc::by_types(x_type, y_type, [&](auto a, auto b) { return hc::backward<decltype(a), decltype(b)>(p, blocks, stream); });
  if (e == cudaSuccess && dweight) {
    hc::dev::hc_norm_finish_kernel<<<dim3((unsigned)((width + 31) / 32), 2), dim3(32, 32), 0, stream>>>(
        p.partial, blocks, (int64_t)width, dweight, dbias, param_type);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

}  // extern "C"
