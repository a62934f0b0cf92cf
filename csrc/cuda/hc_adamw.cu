// One AdamW step over many tensors in one launch, with the moments in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - (m / (sqrt(v) / sqrt(1 - b2^t) + eps)) lr / (1 - b1^t)
//
// Every operation is an fp32 operation of its own in this order; a 16-bit parameter is rounded once, to nearest.
//
// Moments in 8 bits: 256 values share the largest |m| and the largest sqrt(v) among them, in fp32.  m is held as a sign, 4 bits of
// exponent and 3 of fraction, sqrt(v), which has half of v's range of exponents, as 4 and 4, both relative to the largest.  With
// its exponent lowered by 111 such a number is the top of an fp32 number's bits, numbers below the lowest exponent among them as subnormals,
// so coding is an addition and a shift.  b2 = 0.999 moves v by 0.1 % a step, and a code step is 3 to 6 %: rounded to nearest v would
// stay where it is for ever, so both are rounded up or down at random, in proportion to what is lost.  The random bits are a hash of the
// value's number, the tensor's number, the step and a seed.  A sqrt(v) above 0 stays above 0, or the next step would divide by eps.
//
// With moments in 32 bits bound by memory: 28 bytes an element with fp32 parameters and gradients (124 million: 557 us, 6.25 TB/s).  With moments in 8 bits 16 bytes, and bound by the instructions: 99 an
// element, 75 % of the issue slots, DRAM 52 % (455 us).  A warp takes a block of 256 values, four neighbours a lane, twice, so a block's largest values are one reduction instruction each and nothing is shared
// between warps.  The tensors' addresses are arguments of the kernel (a table of 16 or of 448), so that a call copies nothing to the device.
#include <math.h>

#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

constexpr int kAdamUnit = 256;  // values of a warp, and of a block that shares its scales
constexpr int kAdamThreads = 256;

struct AdamEntry {
  void* param;
  const void* grad;
  void* m;
  void* v;
  float2* scales;
  int64_t n;
  uint32_t first;   // units before it
  uint32_t number;  // the tensor's number in the call
};
template <int N>
struct AdamParams {
  AdamEntry entry[N];
  int count;
  uint32_t units;
  double lr, b1d, b2d, decay;
  float b1, rest1, b2, rest2, eps;
  float keep, root, size;  // 1 - lr decay, 1 / sqrt(1 - b2^t), lr / (1 - b1^t), where step and lr are known to the host
  uint32_t key;            // of seed and step
  uint64_t seed;
  const int64_t* step_at;  // the step's number in device memory, or NULL
  const float* lr_at;
};

// A whole number with its bits spread: the last steps of MurmurHash3 (A. Appleby, public domain)
__host__ __device__ inline uint32_t adam_mixed(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x85EBCA6Bu;
  x = (x ^ (x >> 13)) * 0xC2B2AE35u;
  return x ^ (x >> 16);
}
__host__ __device__ inline uint32_t adam_key(uint64_t seed, int64_t step) { return adam_mixed((uint32_t)seed + (uint32_t)step * 0x9E3779B9u); }

// what the codes' largest number stands for before the scale, and the powers of two between a code's exponents and fp32's
constexpr float kTopM = 0.9375f, kTopV = 0.96875f;
__device__ __forceinline__ float adam_down() { return __uint_as_float((127u - 111u) << 23); }
__device__ __forceinline__ float adam_up() { return __uint_as_float((127u + 111u) << 23); }
constexpr uint32_t kLeastBits = (127u - 100u) << 23;  // 2^-100: a block whose largest value is below is held as zeros
constexpr uint32_t kInfBits = 0x7f800000u;
template <typename T>
__device__ __forceinline__ void unpack_pair(uint32_t w, float& a, float& b) {
  unpack2<T>(w, a, b);
}
template <>
__device__ __forceinline__ void unpack_pair<float>(uint32_t, float&, float&) {}  // floats are not packed
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  return pack2<T>(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<float>(float, float) {
  return 0;
}

// 2^111 over what the largest code stands for: the product is a power of two times the quotient rounded, so nothing is rounded twice
constexpr float kUpM = (float)(1.0 / 0.9375), kUpV = (float)(1.0 / 0.96875);
__device__ __forceinline__ float adam_m_of(uint32_t code, float scale) {
  const float size = (__uint_as_float((code & 127u) << 20) * (adam_up() * kUpM)) * scale;
  return __uint_as_float(__float_as_uint(size) ^ (code & 128u) << 24);
}
__device__ __forceinline__ float adam_root_of(uint32_t code, float scale) { return (__uint_as_float(code << 19) * (adam_up() * kUpV)) * scale; }
// code number j of a word
__device__ __forceinline__ uint32_t code_at(uint32_t word, int j, int bit, uint32_t mask) { return (bit >= 8 * j ? word << (bit - 8 * j) : word >> (8 * j - bit)) & mask; }
// four codes of m and of root(v)
__device__ __forceinline__ void adam_decode4(uint32_t cm, uint32_t cv, float2 scale, float* m, float* v) {
  const Pair up_m = pair(adam_up() * kUpM, adam_up() * kUpM), up_v = pair(adam_up() * kUpV, adam_up() * kUpV), sm = pair(scale.x, scale.x), sv = pair(scale.y, scale.y);
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    float a, b;
    parts((pair(__uint_as_float(code_at(cm, j, 20, 127u << 20)), __uint_as_float(code_at(cm, j + 1, 20, 127u << 20))) * up_m) * sm, a, b);
    m[j] = __uint_as_float(__float_as_uint(a) ^ code_at(cm, j, 24, 1u << 31));
    m[j + 1] = __uint_as_float(__float_as_uint(b) ^ code_at(cm, j + 1, 24, 1u << 31));
    const Pair root = (pair(__uint_as_float(code_at(cv, j, 19, 255u << 19)), __uint_as_float(code_at(cv, j + 1, 19, 255u << 19))) * up_v) * sv;
    parts(root * root, v[j], v[j + 1]);
  }
}
// the scale that stands for a block's largest value, and one over it, 0 where nothing is held: of zeros (below 2^-100), and of a block
// with something that is no number or infinite, which becomes NaN as a whole
__device__ __forceinline__ void adam_scale(uint32_t largest, float& scale, float& inverse) {
  const bool usable = largest >= kLeastBits && largest < kInfBits;
  scale = usable ? __uint_as_float(largest) : largest < kLeastBits ? 0.0f : __uint_as_float(0x7fc00000u);
  inverse = usable ? 1.0f / scale : 0.0f;
}

struct AdamNow {
  float keep, root, size;
  uint32_t key;
};

// m and v of this step and the parameter's new value
template <typename P>
__device__ __forceinline__ float adam_update(const P& p, const AdamNow& now, float x, float g, float& m, float& v, float& root_v) {
  m = m * p.b1 + g * p.rest1;
  v = v * p.b2 + (g * g) * p.rest2;
  root_v = __fsqrt_rn(v);
  return x * now.keep - __fdiv_rn(m, root_v * now.root + p.eps) * now.size;
}

template <typename T, bool kWide>
__device__ __forceinline__ void adam_load4(const T* p, float* v) {
  if (!kWide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = to_float(p[j]);
  } else if (sizeof(T) == 4) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    unpack_pair<T>(w.x, v[0], v[1]);
    unpack_pair<T>(w.y, v[2], v[3]);
  }
}
template <typename T, bool kWide>
__device__ __forceinline__ void adam_store4(T* p, const float* v) {
  if (!kWide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = from_float<T>(v[j]);
  } else if (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]));
  }
}

// A whole block of 256: four neighbours a lane, twice, so that a warp's pieces of each array are adjacent.  kWide: parameter and gradient lie at 16 bytes (the moments do in any case).
template <typename T, typename G, bool k8, bool kWide, typename P>
__device__ __forceinline__ void adam_unit_vector(const P& p, const AdamNow& now, const AdamEntry& e, int64_t at) {
  const int lane = threadIdx.x & 31;
  const int64_t i = at + lane * 4;
  T* param = static_cast<T*>(e.param) + i;
  const G* grad = static_cast<const G*>(e.grad) + i;
  float x[8], g[8], m[8], v[8], r[8];
  uint32_t cm[2], cv[2];
  float2 scale;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    adam_load4<T, kWide>(param + h * 128, x + h * 4);
    adam_load4<G, kWide>(grad + h * 128, g + h * 4);
    if (k8) {
      cm[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(e.m) + i + h * 128);
      cv[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(e.v) + i + h * 128);
    } else {
      adam_load4<float, true>(static_cast<const float*>(e.m) + i + h * 128, m + h * 4);
      adam_load4<float, true>(static_cast<const float*>(e.v) + i + h * 128, v + h * 4);
    }
  }
  if (k8) {
    scale = e.scales[at / kAdamUnit];
#pragma unroll
    for (int h = 0; h < 2; ++h) adam_decode4(cm[h], cv[h], scale, m + h * 4, v + h * 4);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = adam_update(p, now, x[j], g[j], m[j], v[j], r[j]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    adam_store4<T, kWide>(param + h * 128, x + h * 4);
    if (!k8) {
      adam_store4<float, true>(static_cast<float*>(e.m) + i + h * 128, m + h * 4);
      adam_store4<float, true>(static_cast<float*>(e.v) + i + h * 128, v + h * 4);
    }
  }
  if (!k8) return;
  uint32_t most_m = 0, most_v = 0, sign[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    sign[j] = __float_as_uint(m[j]) >> 24 & 128u;
    m[j] = fabsf(m[j]);
    most_m = max(most_m, __float_as_uint(m[j]));
    most_v = max(most_v, __float_as_uint(r[j]) & 0x7fffffffu);
  }
  most_m = __reduce_max_sync(0xffffffffu, most_m);
  most_v = __reduce_max_sync(0xffffffffu, most_v);
  float inverse_m, inverse_v;
  adam_scale(most_m, scale.x, inverse_m);
  adam_scale(most_v, scale.y, inverse_v);
  const uint32_t first = (uint32_t)i * 0x9E3779B1u + adam_mixed(now.key + e.number);
  const Pair im = pair(inverse_m, inverse_m), iv = pair(inverse_v, inverse_v), top_m = pair(kTopM, kTopM), top_v = pair(kTopV, kTopV), down = pair(adam_down(), adam_down());
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t word_m = 0, word_v = 0;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      float y[2], z[2];
      parts(((pair(m[h * 4 + j], m[h * 4 + j + 1]) * im) * top_m) * down, y[0], y[1]);
      parts(((pair(r[h * 4 + j], r[h * 4 + j + 1]) * iv) * top_v) * down, z[0], z[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t random = adam_mixed(first + (uint32_t)(h * 128 + j + k) * 0x9E3779B1u);
        const uint32_t a = min((__float_as_uint(y[k]) + (random << 4 & 0xffff0u) + 8u) >> 20, 127u);
        const uint32_t b = min((__float_as_uint(z[k]) + (random >> 13 & 0x7fff8u) + 4u) >> 19, 255u);
        word_m |= (a | sign[h * 4 + j + k]) << (8 * (j + k));
        word_v |= max(b, min(__float_as_uint(r[h * 4 + j + k]), 1u)) << (8 * (j + k));  // a root above 0 stays above it
      }
    }
    if (inverse_m == 0.0f) word_m = 0;  // of the whole block
    if (inverse_v == 0.0f) word_v = 0;
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(e.m) + i + h * 128) = word_m;
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(e.v) + i + h * 128) = word_v;
  }
  if (lane == 0) e.scales[at / kAdamUnit] = scale;
}

// The same value by value, for moments that begin anywhere and for a tensor's last values: lane l takes every 32nd.
template <typename T, typename G, bool k8, typename P>
__device__ __forceinline__ void adam_unit_single(const P& p, const AdamNow& now, const AdamEntry& e, int64_t at) {
  const int lane = threadIdx.x & 31;
  const int count = (int)min((int64_t)kAdamUnit, e.n - at);
  T* param = static_cast<T*>(e.param) + at;
  const G* grad = static_cast<const G*>(e.grad) + at;
  float x[8], g[8], m[8], v[8], r[8];
  float2 scale = make_float2(0.0f, 0.0f);
  if (k8) scale = e.scales[at / kAdamUnit];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = j * 32 + lane;
    const bool in = i < count;
    x[j] = in ? to_float(param[i]) : 0.0f;
    g[j] = in ? to_float(grad[i]) : 0.0f;
    if (k8) {
      m[j] = in ? adam_m_of(static_cast<const uint8_t*>(e.m)[at + i], scale.x) : 0.0f;
      const float root = in ? adam_root_of(static_cast<const uint8_t*>(e.v)[at + i], scale.y) : 0.0f;
      v[j] = root * root;
    } else {
      m[j] = in ? static_cast<const float*>(e.m)[at + i] : 0.0f;
      v[j] = in ? static_cast<const float*>(e.v)[at + i] : 0.0f;
    }
  }
  uint32_t most_m = 0, most_v = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = j * 32 + lane;
    x[j] = adam_update(p, now, x[j], g[j], m[j], v[j], r[j]);
    if (i >= count) continue;
    param[i] = from_float<T>(x[j]);
    if (!k8) {
      static_cast<float*>(e.m)[at + i] = m[j];
      static_cast<float*>(e.v)[at + i] = v[j];
    } else {
      most_m = max(most_m, __float_as_uint(m[j]) & 0x7fffffffu);
      most_v = max(most_v, __float_as_uint(r[j]) & 0x7fffffffu);
    }
  }
  if (!k8) return;
  most_m = __reduce_max_sync(0xffffffffu, most_m);
  most_v = __reduce_max_sync(0xffffffffu, most_v);
  float inverse_m, inverse_v;
  adam_scale(most_m, scale.x, inverse_m);
  adam_scale(most_v, scale.y, inverse_v);
  const uint32_t key = adam_mixed(now.key + e.number);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = j * 32 + lane;
    if (i >= count) continue;
    const uint32_t h = adam_mixed((uint32_t)(at + i) * 0x9E3779B1u + key);
    const float y = ((fabsf(m[j]) * inverse_m) * kTopM) * adam_down(), z = ((r[j] * inverse_v) * kTopV) * adam_down();
    uint32_t a = min((__float_as_uint(y) + (h << 4 & 0xffff0u) + 8u) >> 20, 127u) | (__float_as_uint(m[j]) >> 24 & 128u);
    uint32_t b = max(min((__float_as_uint(z) + (h >> 13 & 0x7fff8u) + 4u) >> 19, 255u), min(__float_as_uint(r[j]), 1u));
    a = inverse_m > 0.0f ? a : 0u;
    b = inverse_v > 0.0f ? b : 0u;
    static_cast<uint8_t*>(e.m)[at + i] = (uint8_t)a;
    static_cast<uint8_t*>(e.v)[at + i] = (uint8_t)b;
  }
  if (lane == 0) e.scales[at / kAdamUnit] = scale;
}

template <typename T, typename G, bool k8, int N>
__global__ void __launch_bounds__(kAdamThreads) hc_adamw_kernel(const __grid_constant__ AdamParams<N> p) {
  __shared__ AdamNow shared_now;
  AdamNow now = {p.keep, p.root, p.size, p.key};
  if (p.step_at || p.lr_at) {  // as the host computes them where it knows step and rate
    if (threadIdx.x == 0) {
      const double lr = p.lr_at ? (double)*p.lr_at : p.lr, t = p.step_at ? (double)*p.step_at : 0.0;
      shared_now = now;
      shared_now.keep = (float)(1.0 - lr * p.decay);
      if (p.step_at) {
        shared_now.root = (float)(1.0 / sqrt(1.0 - pow(p.b2d, t)));
        shared_now.size = (float)(lr / (1.0 - pow(p.b1d, t)));
        shared_now.key = adam_key(p.seed, *p.step_at);
      } else {
        shared_now.size = (float)(lr / p.b1d);  // b1d: 1 - b1^t
      }
    }
    __syncthreads();
    now = shared_now;
  }
  const uint32_t warps = gridDim.x * (kAdamThreads / 32);
  int t = 0;
  for (uint32_t unit = blockIdx.x * (kAdamThreads / 32) + (threadIdx.x >> 5); unit < p.units; unit += warps) {
    int high = p.count - 1;  // the last tensor whose first unit is not behind this one
    while (t < high) {
      const int mid = (t + high + 1) >> 1;
      if (p.entry[mid].first <= unit) t = mid;
      else high = mid - 1;
    }
    const AdamEntry& e = p.entry[t];
    const int64_t at = (int64_t)(unit - e.first) * kAdamUnit;
    const uintptr_t own = reinterpret_cast<uintptr_t>(e.param) | reinterpret_cast<uintptr_t>(e.grad), moments = reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v);
    if (at + kAdamUnit > e.n || moments & (k8 ? 3u : 15u)) adam_unit_single<T, G, k8>(p, now, e, at);
    else if (own & 15u) adam_unit_vector<T, G, k8, false>(p, now, e, at);
    else adam_unit_vector<T, G, k8, true>(p, now, e, at);
  }
}

// What moments in 8 bits stand for.  Four neighbours a thread, four times.
__global__ void __launch_bounds__(256) hc_adamw_values_kernel(const uint8_t* m, const uint8_t* v, const float2* scales, int64_t n, float* m_out, float* v_out, bool vector) {
  constexpr int kAtOnce = 4;
  for (int64_t first = blockIdx.x * (1024ll * kAtOnce); first < n; first += gridDim.x * (1024ll * kAtOnce)) {
    uint32_t cm[kAtOnce], cv[kAtOnce];
    float2 scale[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t i = first + k * 1024 + threadIdx.x * 4;
      if (!vector || i + 4 > n) continue;
      cm[k] = *reinterpret_cast<const uint32_t*>(m + i);
      cv[k] = *reinterpret_cast<const uint32_t*>(v + i);
      scale[k] = scales[i / kAdamUnit];
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t i = first + k * 1024 + threadIdx.x * 4;
      if (vector && i + 4 <= n) {
        float a[4], b[4];
        adam_decode4(cm[k], cv[k], scale[k], a, b);
        *reinterpret_cast<float4*>(m_out + i) = make_float4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<float4*>(v_out + i) = make_float4(b[0], b[1], b[2], b[3]);
      } else {
        for (int64_t j = i; j < i + 4 && j < n; ++j) {
          const float2 s = scales[j / kAdamUnit];
          const float root = adam_root_of(v[j], s.y);
          m_out[j] = adam_m_of(m[j], s.x);
          v_out[j] = root * root;
        }
      }
    }
  }
}

}  // namespace dev

namespace {

template <typename T, typename G, bool k8, int N>
cudaError_t run_adamw(const hc_adamw_tensor* tensors, size_t count, const dev::AdamParams<1>& common, cudaStream_t stream) {
  dev::AdamParams<N> p;
  p.lr = common.lr, p.b1d = common.b1d, p.b2d = common.b2d, p.decay = common.decay;
  p.b1 = common.b1, p.rest1 = common.rest1, p.b2 = common.b2, p.rest2 = common.rest2, p.eps = common.eps;
  p.keep = common.keep, p.root = common.root, p.size = common.size;
  p.key = common.key, p.seed = common.seed, p.step_at = common.step_at, p.lr_at = common.lr_at;
  size_t i = 0;
  while (i < count) {
    p.count = 0;
    int64_t units = 0;
    for (; i < count && p.count < N; ++i) {
      const hc_adamw_tensor& t = tensors[i];
      if (t.n == 0) continue;
      // a launch numbers its units in 31 bits: what is behind that goes to the next one
      const int64_t all = ((int64_t)t.n + dev::kAdamUnit - 1) / dev::kAdamUnit;
      if (units + all > 0x7fffffffll) break;
      p.entry[p.count++] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, reinterpret_cast<float2*>(t.scales), (int64_t)t.n, (uint32_t)units, t.number};
      units += all;
    }
    if (p.count == 0) {
      if (i < count) return cudaErrorInvalidValue;  // one tensor of more than 2^39 values
      break;
    }
    p.units = (uint32_t)units;
    static int resident[64];
    const int most = resident_ctas(dev::hc_adamw_kernel<T, G, k8, N>, dev::kAdamThreads, 0, resident);
    if (most <= 0) return cudaErrorInvalidConfiguration;
    const int64_t blocks = (units + dev::kAdamThreads / 32 - 1) / (dev::kAdamThreads / 32);
    dev::hc_adamw_kernel<T, G, k8, N><<<(unsigned)(blocks < most ? blocks : most), dev::kAdamThreads, 0, stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
template <typename T, typename G>
cudaError_t adamw_of(const hc_adamw_tensor* tensors, size_t count, int bits, const dev::AdamParams<1>& common, cudaStream_t stream) {
  // arguments of a kernel are copied at every launch: 1 KB of them, or 25
  if (count <= 16) return bits == 8 ? run_adamw<T, G, true, 16>(tensors, count, common, stream) : run_adamw<T, G, false, 16>(tensors, count, common, stream);
  return bits == 8 ? run_adamw<T, G, true, 448>(tensors, count, common, stream) : run_adamw<T, G, false, 448>(tensors, count, common, stream);
}

}  // namespace
}  // namespace hc

extern "C" {

int hc_adamw(const hc_adamw_tensor* tensors, size_t count, int param_type, int grad_type, int bits, double lr, const float* lr_at, double beta1, double beta2,
             double eps, double weight_decay, int64_t step, const int64_t* step_at, uint64_t seed, hc_stream_t stream) {
  using namespace hc;
  if (!element_type_ok(param_type) || !element_type_ok(grad_type) || (param_type != kF32 && param_type != grad_type) || (bits != 8 && bits != 32)) return kErrArgument;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0 && weight_decay >= 0.0) || (!lr_at && !(lr >= 0.0)) || (!step_at && step < 1)) return kErrArgument;
  if (!lies_at(lr_at, 4) || !lies_at(step_at, 8) || (count && !tensors)) return kErrArgument;
  const size_t state = bits == 8 ? 1 : 4;
  for (size_t i = 0; i < count; ++i) {
    const hc_adamw_tensor& t = tensors[i];
    if (t.n == 0) continue;
    if (t.n > (1ull << 39) - 256 || !t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (bits == 8 && !t.scales)) return kErrArgument;
    if (!lies_at(t.param, element_bytes(param_type)) || !lies_at(t.grad, element_bytes(grad_type)) || !lies_at(t.exp_avg, state) || !lies_at(t.exp_avg_sq, state) ||
        (bits == 8 && !lies_at(t.scales, 8)))
      return kErrArgument;
  }
  dev::AdamParams<1> c;
  memset(&c, 0, sizeof(c));
  c.lr = lr, c.b2d = beta2, c.decay = weight_decay;
  c.b1 = (float)beta1, c.rest1 = (float)(1.0 - beta1), c.b2 = (float)beta2, c.rest2 = (float)(1.0 - beta2), c.eps = (float)eps;
  c.seed = seed, c.step_at = step_at, c.lr_at = lr_at;
  c.keep = (float)(1.0 - lr * weight_decay);
  if (step_at) {
    c.b1d = beta1;
  } else {
    c.b1d = 1.0 - pow(beta1, (double)step);
    c.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    c.size = (float)(lr / c.b1d);
    c.key = dev::adam_key(seed, step);
  }
  cudaError_t e;
  using b = __nv_bfloat16;
  using h = __half;
  if (param_type == kF32)
    e = grad_type == kF32 ? adamw_of<float, float>(tensors, count, bits, c, stream)
                          : grad_type == kBf16 ? adamw_of<float, b>(tensors, count, bits, c, stream) : adamw_of<float, h>(tensors, count, bits, c, stream);
  else
    e = param_type == kBf16 ? adamw_of<b, b>(tensors, count, bits, c, stream) : adamw_of<h, h>(tensors, count, bits, c, stream);
  return e == cudaSuccess ? kOk : kErrCuda;
}

int hc_adamw_values(const uint8_t* exp_avg, const uint8_t* exp_avg_sq, const float* scales, size_t n, float* m, float* v, hc_stream_t stream) {
  using namespace hc;
  if (n > (1ull << 39)) return kErrArgument;
  if (n == 0) return kOk;
  if (!exp_avg || !exp_avg_sq || !scales || !m || !v || !lies_at(scales, 8) || !lies_at(m, 4) || !lies_at(v, 4)) return kErrArgument;
  const bool vector = lies_at(exp_avg, 4) && lies_at(exp_avg_sq, 4) && lies_at(m, 16) && lies_at(v, 16);
  const size_t blocks = (n + 4095) / 4096, most = (size_t)(device_info().sms > 0 ? device_info().sms : 1) * 8;
  dev::hc_adamw_values_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(exp_avg, exp_avg_sq, reinterpret_cast<const float2*>(scales), (int64_t)n, m, v,
                                                                                           vector);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // extern "C"
