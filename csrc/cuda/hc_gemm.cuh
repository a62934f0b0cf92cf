// Matrix products of 16-bit operands on the tensor cores, with what the operators do to the result before it is stored.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hc_train.cuh"

namespace hc {
enum GemmMode : int {
  kGemmLinear = 0,  // out = act(acc + bias) + residual; z = acc + bias
  kGemmGram = 1,    // out = acc, symmetric
  kGemmPoly = 2,    // out = b c1 + c acc, symmetric (c1: the operand itself)
  kGemmUpdate = 3,  // x = a (hi + lo / 2048) + acc; out hi and lo again, or bf16
};
enum Activation : int { kActNone = 0, kActGeluTanh = 1, kActRelu = 2, kActSilu = 3 };

namespace dev {

// Activations of two values at a time.  GELU (tanh form) and SiLU are z sigmoid(v), with v = 2 sqrt(2 / pi) (z + 0.044715 z^3)
// or z; sigmoid(v) = 1 / (1 + e) with e = exp(-v).  Each value has its own exp and reciprocal: with one reciprocal for both, of
// the product of their sums, a value's last bits depended on its neighbour, and a NaN made the neighbour one.  z is raised to where
// e is about 2^60 and the function within 1e-16 of 0: minus infinity times 0 would not be a number.
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kGelu1 = 1.5957691216057308f, kGelu3 = 0.044715f * 1.5957691216057308f;
constexpr float kGeluLeast = -7.5f, kSiluLeast = -41.5f;  // v = -42.1, -41.5

__device__ __forceinline__ float act_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float act_min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// sigmoid of both v, given v times -log2(e)
__device__ __forceinline__ Pair sigmoid_pair(Pair exponent) {
  float a, b;
  parts(exponent, a, b);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(a));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(b));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(a + 1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(b + 1.0f));
  return pair(a, b);
}
template <int kAct>
__device__ __forceinline__ void activate_pair(float& x, float& y) {
  if (kAct == kActRelu) {
    x = act_max_nan(x, 0.0f);
    y = act_max_nan(y, 0.0f);
  } else if (kAct == kActGeluTanh || kAct == kActSilu) {
    const float least = kAct == kActSilu ? kSiluLeast : kGeluLeast;
    const Pair z = pair(act_max_nan(x, least), act_max_nan(y, least));
    Pair v = z * pair(-kLog2E, -kLog2E);
    if (kAct == kActGeluTanh) v = z * fma2(z * z, pair(-kGelu3 * kLog2E, -kGelu3 * kLog2E), pair(-kGelu1 * kLog2E, -kGelu1 * kLog2E));
    parts(z * sigmoid_pair(v), x, y);
  }
}
// g times the activation's slope at z: s + z s (1 - s) v'.  Beyond +-7.5 (41.5) it is 0 and 1 to within 1e-16.
template <int kAct>
__device__ __forceinline__ Pair slope_pair(Pair g, float x, float y) {
  if (kAct == kActNone) return g;
  if (kAct == kActRelu) {  // chosen, not multiplied: an infinite g has no part where the slope is 0
    float a, b;
    parts(g, a, b);
    return pair(x > 0.0f ? a : x != x ? x : 0.0f, y > 0.0f ? b : y != y ? y : 0.0f);
  }
  const float least = kAct == kActSilu ? kSiluLeast : kGeluLeast;
  const Pair z = pair(act_min_nan(act_max_nan(x, least), -least), act_min_nan(act_max_nan(y, least), -least));
  Pair v = z * pair(-kLog2E, -kLog2E), zdv = z;
  if (kAct == kActGeluTanh) {
    const Pair square = z * z;
    v = z * fma2(square, pair(-kGelu3 * kLog2E, -kGelu3 * kLog2E), pair(-kGelu1 * kLog2E, -kGelu1 * kLog2E));
    zdv = z * fma2(square, pair(3.0f * kGelu3, 3.0f * kGelu3), pair(kGelu1, kGelu1));
  }
  const Pair s = sigmoid_pair(v), minus = s * pair(-1.0f, -1.0f);
  return g * fma2(zdv, fma2(minus, s, s), s);
}

// fp16 products take an fp32 gradient times 2^k (sign 1), and their results times 2^-k (sign -1), with k from the bits of the largest
// finite |gradient|, which comes to [2^13, 2^14): times a slope it stays in range, and 2^-38 of it is still a number.
__device__ __forceinline__ float gradient_power(const unsigned int* most, int sign) {
  const int exponent = (int)(*most >> 23);
  const int k = *most ? min(127 + 13 - exponent, 100) : 0;  // from -114
  return __int_as_float((127 + sign * k) << 23);
}

}  // namespace dev

// An operand is stored as rows of adjacent elements.  kMajor: its rows are those of the product (or its columns, for the
// second operand) and lie along the sum; otherwise the sum runs over its rows.
struct GemmOperand {
  const void* data;
  int64_t ld;      // elements from row to row, a multiple of 8
  int64_t stride;  // elements from matrix to matrix of a batch
  bool k_major;
};
// What an epilogue reads or writes beside the accumulator: m rows of n values
struct GemmSide {
  void* data;
  int64_t ld;
  int64_t stride;
};
struct GemmCall {
  int type;  // of the operands
  int64_t m, n, k, batch;
  int parts;  // over 1 (kGemmLinear without anything behind it, batch 1): as many results, each of a part of the sum, as a batch
  bool precise;  // the sum is wanted with fp32's precision, not only with that of a 16-bit result of `type`
  GemmOperand a, b;
  GemmSide out, out2;  // result; z, or lo
  GemmSide in, in2;    // residual, c1 or hi; lo
  int out_type;        // kF32, kBf16, kF16
  const void* bias;
  int bias_type;
  int activation;
  float ca, cb, cc;
  const float* scale;  // of each matrix of a batch (kGemmPoly, kGemmUpdate): X is that times what is stored
  const unsigned int* most;  // kGemmLinear without anything behind it: see gradient_power, whose inverse the result is taken times; or NULL
};

// Into how many parts the sum of a product is best shared out (1: none).
int gemm_parts(int64_t m, int64_t n, int64_t k);
// act(a b + bias) + residual
cudaError_t launch_gemm(const GemmCall& call, cudaStream_t stream);
// The products of a Newton-Schulz iteration in one launch: step i takes gram[i % 2], poly and update[i % 2], the last one `last`.
struct GemmChain {
  GemmCall gram[2], poly, update[2], last;
  int steps;
  unsigned int* arrived;  // a word of device memory that is 0 when the launch begins
};
cudaError_t launch_chain(const GemmChain& chain, cudaStream_t stream);
bool gemm_operand_ok(const void* data, int64_t ld);

}  // namespace hc
