// Layer norm over rows: y = (x - mean) rstd w + b, and its backward pass.
//
// A row is held in registers by T threads (a warp, or a block), K groups of eight values a thread, so x is read once:
// mean first, then the squares of what is left of it (no difference of large sums).  The backward pass reads x and dy
// once,
//   h = (x - mean) rstd,  dx = rstd (w dy - mean(w dy) - h mean(w dy h)),  dw = sum dy h,  db = sum dy,
// with the column sums of a thread's own columns in its registers over all rows that its block works on.  Rows whose
// length eight does not divide begin at one of eight places within an aligned group; a block takes rows that begin at
// the same place, so that its threads keep their columns, whose w and b wait in shared memory.  Where a block shares a row,
// the next row is on its way while it works on this one.  The sums of the blocks are added by a second kernel in a fixed
// order.  Both passes are bound by memory.
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

// Eight values as they lie in memory
template <typename T>
struct Raw {
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  }
  __device__ __forceinline__ void load_some(const T* p, int64_t count) {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (2 * j < count ? q[2 * j] : 0u) | (2 * j + 1 < count ? q[2 * j + 1] : 0u) << 16;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) unpack2<T>(w[j], v[2 * j], v[2 * j + 1]);
  }
  __device__ __forceinline__ void keep(int from, int to) {  // zeros outside of [from, to)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < from || j >= to) w[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
  }
  // what was computed from the values is computed again behind this, not kept in registers
  __device__ __forceinline__ void touch() { asm volatile("" : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3])::"memory"); }
};
template <>
struct Raw<float> {
  float w[8];
  __device__ __forceinline__ void load(const float* p) { load8(p, w); }
  __device__ __forceinline__ void load_some(const float* p, int64_t count) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < count ? p[j] : 0.0f;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = w[j];
  }
  __device__ __forceinline__ void keep(int from, int to) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < from || j >= to) w[j] = 0.0f;
  }
  __device__ __forceinline__ void touch() {
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+f"(w[j])::"memory");
  }
};
// The group at `first` of a row whose first value is number `base` of `all`: whole, with the neighbouring rows' values, but
// nothing behind the last one; what is not the row's reads as 0.
template <typename T>
__device__ __forceinline__ void take(Raw<T>& raw, const T* x, int64_t base, int first, int64_t width, int64_t all) {
  if (first < width) {
    if (base + first + 8 <= all) raw.load(x + base + first);
    else raw.load_some(x + base + first, all - base - first);
  }
  if (first < 0 || first + 8 > width) raw.keep(max(-first, 0), (int)max(min(width - first, (int64_t)8), (int64_t)0));
}

template <int T>
struct Team {
  static constexpr int kThreads = T == 32 ? 128 : T;
  static constexpr int kTeams = kThreads / T;
  static constexpr int kBlocks = T == 32 ? 3 : 512 / T;  // that an SM holds at the least
  static constexpr bool kAhead = T > 32;  // a row ahead; with a row a warp there are warps enough
};

// T threads a row, K groups of eight a thread
template <typename X, typename Y, int T, int K>
__global__ void __launch_bounds__(Team<T>::kThreads, Team<T>::kBlocks) hc_norm_kernel(const __grid_constant__ NormParams p) {
  using G = Team<T>;
  __shared__ float2 shared[T / 32];
  extern __shared__ __align__(16) float params[];  // w and b by place: [2][K * T * 8]
  const int lane = T == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int place = blockIdx.x % p.period;
  const int64_t team = (int64_t)(blockIdx.x / p.period) * G::kTeams + (T == 32 ? threadIdx.x >> 5 : 0);
  const int64_t step = (int64_t)(gridDim.x / p.period) * G::kTeams * p.period, all = p.rows * p.width;
  const int shift = (int)(place * p.width & 7);
  const float inv = 1.0f / (float)p.width;
  int64_t row = place + team * p.period;
  Raw<X> raw[K], next[K];
  if (row < p.rows)
#pragma unroll
    for (int k = 0; k < K; ++k) take(raw[k], static_cast<const X*>(p.x), row * p.width, (k * T + lane) * 8 - shift, p.width, all);
  for (int i = threadIdx.x; i < K * T * 8; i += G::kThreads) {
    const int64_t c = i - shift;
    const bool in = c >= 0 && c < p.width;
    params[i] = !in ? 0.0f : p.weight ? param_at(p.weight, p.param_type, c) : 1.0f;
    params[K * T * 8 + i] = p.bias && in ? param_at(p.bias, p.param_type, c) : 0.0f;
  }
  __syncthreads();
  for (; row < p.rows; row += step) {
    if (G::kAhead && row + step < p.rows)
#pragma unroll
      for (int k = 0; k < K; ++k) take(next[k], static_cast<const X*>(p.x), (row + step) * p.width, (k * T + lane) * 8 - shift, p.width, all);
    float v[K][8];
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      raw[k].values(v[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[k][j];
    }
    group_sum2<T>(sum, none, shared);
    const float mean = sum * inv;
    float squares = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = (k * T + lane) * 8 - shift;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] -= mean;
      if (first < 0 || first + 8 > p.width) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (first + j < 0 || first + j >= p.width) v[k][j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) squares = fmaf(v[k][j], v[k][j], squares);
    }
    none = 0.0f;
    group_sum2<T>(squares, none, shared);
    const float rstd = 1.0f / sqrtf(fmaf(squares, inv, p.eps));
    Y* y = static_cast<Y*>(p.out) + row * p.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = (k * T + lane) * 8 - shift;
      if (first >= p.width) continue;
      float w[8], b[8];
      load8(params + (k * T + lane) * 8, w);
      load8(params + K * T * 8 + (k * T + lane) * 8, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = fmaf(v[k][j] * rstd, w[j], b[j]);
      store_group(y, first, p.width, v[k]);
    }
    if (p.stats && lane == 0) reinterpret_cast<float2*>(p.stats)[row] = make_float2(mean, rstd);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (G::kAhead) raw[k] = next[k];
      else if (row + step < p.rows) take(raw[k], static_cast<const X*>(p.x), (row + step) * p.width, (k * T + lane) * 8 - shift, p.width, all);
    }
  }
}

template <typename X, typename Y, int T, int K>
__global__ void __launch_bounds__(Team<T>::kThreads, Team<T>::kBlocks) hc_norm_backward_kernel(const __grid_constant__ NormParams p) {
  using G = Team<T>;
  __shared__ float2 shared[T / 32];
  extern __shared__ __align__(16) float params[];  // w by place: [K * T * 8]; with a row a warp behind it the sums [2][K * 256]
  const int lane = T == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int place = blockIdx.x % p.period;  // rows place, place + period, ... are shared out among the blocks of this place
  const int64_t team = (int64_t)(blockIdx.x / p.period) * G::kTeams + (T == 32 ? threadIdx.x >> 5 : 0);
  const int64_t step = (int64_t)(gridDim.x / p.period) * G::kTeams * p.period, all = p.rows * p.width;
  const int shift = (int)(place * p.width & 7);
  const float inv = 1.0f / (float)p.width;
  int64_t row = place + team * p.period;
  Raw<X> x[K], next_x[K];
  Raw<Y> dy[K], next_dy[K];
  float2 st = make_float2(0.0f, 0.0f), next_st = st;
  float dw[K][8], db[K][8];
  if (row < p.rows) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      take(x[k], static_cast<const X*>(p.x), row * p.width, (k * T + lane) * 8 - shift, p.width, all);
      take(dy[k], static_cast<const Y*>(p.dy), row * p.width, (k * T + lane) * 8 - shift, p.width, all);
    }
    st = reinterpret_cast<const float2*>(p.stats)[row];
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[k][j] = db[k][j] = 0.0f;
  for (int i = threadIdx.x; i < K * T * 8; i += G::kThreads) {
    const int64_t c = i - shift;
    params[i] = c < 0 || c >= p.width ? 0.0f : p.weight ? param_at(p.weight, p.param_type, c) : 1.0f;
  }
  __syncthreads();
  for (; row < p.rows; row += step) {
    const bool more = row + step < p.rows;
    if (G::kAhead && more) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        take(next_x[k], static_cast<const X*>(p.x), (row + step) * p.width, (k * T + lane) * 8 - shift, p.width, all);
        take(next_dy[k], static_cast<const Y*>(p.dy), (row + step) * p.width, (k * T + lane) * 8 - shift, p.width, all);
      }
      next_st = reinterpret_cast<const float2*>(p.stats)[row + step];
    }
    // outside the row dy and w are 0, and nothing that is not a number there reaches a sum of other columns
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float h[8], g[8], w[8];
      x[k].values(h);
      dy[k].values(g);
      load8(params + (k * T + lane) * 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[j] = (h[j] - st.x) * st.y;
        dw[k][j] = fmaf(g[j], h[j], dw[k][j]);
        db[k][j] += g[j];
        g[j] *= w[j];
        a += g[j];
        b = fmaf(g[j], h[j], b);
      }
    }
    if (p.out) {
      group_sum2<T>(a, b, shared);
      a *= inv;
      b *= inv;
      X* dx = static_cast<X*>(p.out) + row * p.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int first = (k * T + lane) * 8 - shift;
        if (first >= p.width) continue;
        float h[8], g[8], w[8];
        x[k].touch();
        dy[k].touch();
        x[k].values(h);
        dy[k].values(g);
        load8(params + (k * T + lane) * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = st.y * (fmaf(-(h[j] - st.x) * st.y, b, g[j] * w[j]) - a);
        store_group(dx, first, p.width, g);
      }
    }
    if (G::kAhead) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        x[k] = next_x[k];
        dy[k] = next_dy[k];
      }
      st = next_st;
    } else if (more) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        take(x[k], static_cast<const X*>(p.x), (row + step) * p.width, (k * T + lane) * 8 - shift, p.width, all);
        take(dy[k], static_cast<const Y*>(p.dy), (row + step) * p.width, (k * T + lane) * 8 - shift, p.width, all);
      }
      st = reinterpret_cast<const float2*>(p.stats)[row + step];
    }
  }
  if (!p.partial) return;
  float* mine = p.partial + (int64_t)blockIdx.x * 2 * p.width;
  if (T == 32) {  // the block's warps one after the other: a fixed order
    float* sums = params + K * 256;
    for (int warp = 0; warp < G::kTeams; ++warp) {
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
    for (int i = threadIdx.x; i < K * 256; i += G::kThreads) {
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

// Threads and groups of eight a thread for rows of `width` values (with one group more where rows begin anywhere): a warp while
// three groups a thread do, then two groups a thread, which leaves room in the registers for the row ahead.
struct Shape {
  int threads, groups;
};
Shape shape_of(size_t width) {
  const int need = (int)((width + 7) / 8) + (width % 8 ? 1 : 0);
  if (need <= 96) return {32, (need + 31) / 32};
  return {need <= 256 ? 128 : need <= 384 ? 192 : need <= 512 ? 256 : need <= 768 ? 384 : 512, 2};
}
int period_of(size_t width) { return width % 8 == 0 ? 1 : width % 4 == 0 ? 2 : width % 2 == 0 ? 4 : 8; }
bool in_registers(size_t width) { return width <= kLongestInRegisters - (width % 8 ? 8 : 0); }

// Blocks: those that the SMs hold stay for all rows, a whole number of them for each place of an aligned group
int norm_blocks(size_t rows, size_t width) {
  const int sms = device_info().sms > 0 ? device_info().sms : 1;
  if (!in_registers(width)) return (int)(rows < 64 ? rows : 64);
  const int period = period_of(width);
  const Shape s = shape_of(width);
  const size_t teams = s.threads == 32 ? 4 : 1, most = (size_t)sms * (s.threads == 32 ? 3 : 512 / s.threads) / period * period;
  const size_t blocks = (rows + teams * period - 1) / (teams * period) * period;
  return (int)(blocks < most ? blocks : most);
}

template <typename X, typename Y, int T, int K>
cudaError_t run_forward(const dev::NormParams& p, cudaStream_t stream) {
  constexpr int smem = 2 * K * T * 8 * 4;
  if (smem > 40 * 1024) {  // with what the kernel has besides, 48 KB need no permission
    const cudaError_t e = set_smem(dev::hc_norm_kernel<X, Y, T, K>, smem);
    if (e != cudaSuccess) return e;
  }
  dev::hc_norm_kernel<X, Y, T, K><<<norm_blocks(p.rows, p.width), dev::Team<T>::kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}
template <typename X, typename Y, int T, int K>
cudaError_t run_backward(const dev::NormParams& p, int blocks, cudaStream_t stream) {
  constexpr int smem = K * T * 8 * 4 + (T == 32 ? K * 2048 : 0);
  static_assert(smem <= 40 * 1024, "more needs the kernel's permission");
  dev::hc_norm_backward_kernel<X, Y, T, K><<<blocks, dev::Team<T>::kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

// f with the threads and groups as constants
template <typename F>
cudaError_t by_shape(size_t width, F f) {
  const Shape s = shape_of(width);
  if (s.threads == 32) return s.groups == 1 ? f.template run<32, 1>() : s.groups == 2 ? f.template run<32, 2>() : f.template run<32, 3>();
  if (s.threads == 128) return f.template run<128, 2>();
  if (s.threads == 192) return f.template run<192, 2>();
  if (s.threads == 256) return f.template run<256, 2>();
  return s.threads == 384 ? f.template run<384, 2>() : f.template run<512, 2>();
}
template <typename X, typename Y>
struct Forward {
  const dev::NormParams& p;
  cudaStream_t stream;
  template <int T, int K>
  cudaError_t run() {
    return run_forward<X, Y, T, K>(p, stream);
  }
};
template <typename X, typename Y>
struct Backward {
  const dev::NormParams& p;
  int blocks;
  cudaStream_t stream;
  template <int T, int K>
  cudaError_t run() {
    return run_backward<X, Y, T, K>(p, blocks, stream);
  }
};

template <typename X, typename Y>
cudaError_t forward(const dev::NormParams& p, cudaStream_t stream) {
  if (in_registers(p.width)) return by_shape(p.width, Forward<X, Y>{p, stream});
  dev::hc_norm_long_kernel<X, Y><<<(unsigned)(p.rows < 65536 ? p.rows : 65536), dev::kLong, 0, stream>>>(p);
  return cudaGetLastError();
}
template <typename X, typename Y>
cudaError_t backward(const dev::NormParams& p, int blocks, cudaStream_t stream) {
  if (in_registers(p.width)) return by_shape(p.width, Backward<X, Y>{p, blocks, stream});
  if (p.out) dev::hc_norm_long_dx_kernel<X, Y><<<(unsigned)(p.rows < 65536 ? p.rows : 65536), dev::kLong, 0, stream>>>(p);
  if (p.partial) dev::hc_norm_long_sums_kernel<X, Y><<<dim3((unsigned)((p.width + 255) / 256), blocks), 256, 0, stream>>>(p);
  return cudaGetLastError();
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
  hc::dev::NormParams p = {x, nullptr, weight, bias, y, stats, nullptr, (int64_t)rows, (int64_t)width, eps, param_type, hc::period_of(width)};
  const cudaError_t e = hc::by_types(x_type, y_type, [&](auto a, auto b) { return hc::forward<decltype(a), decltype(b)>(p, stream); });
  return e == cudaSuccess ? hc::kOk : hc::kErrCuda;
}

size_t hc_layer_norm_backward_bytes(size_t rows, size_t width) {
  return rows && width ? (size_t)hc::norm_blocks(rows, width) * 2 * width * sizeof(float) : 0;
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
  const int blocks = hc::norm_blocks(rows, width);
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
