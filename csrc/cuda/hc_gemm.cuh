// Matrix products of 16-bit operands on the tensor cores, with what the operators do to the result before it is stored.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace hc {
namespace dev {
__device__ __forceinline__ float sigmoid(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
}  // namespace dev

enum GemmMode : int {
  kGemmLinear = 0,  // out = act(acc + bias) + residual; z = acc + bias
  kGemmGram = 1,    // out = acc, symmetric
  kGemmPoly = 2,    // out = b c1 + c acc, symmetric (c1: the operand itself)
  kGemmUpdate = 3,  // x = a (hi + lo / 2048) + acc; out hi and lo again, or bf16
};
enum Activation : int { kActNone = 0, kActGeluTanh = 1, kActRelu = 2, kActSilu = 3 };

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
  int mode;
  int type;  // of the operands
  int64_t m, n, k, batch;
  int parts;  // over 1 (kGemmLinear without anything behind it, batch 1): as many results, each of a part of the sum, as a batch
  GemmOperand a, b;
  GemmSide out, out2;  // result; z, or lo
  GemmSide in, in2;    // residual, c1 or hi; lo
  int out_type;        // kF32, kBf16, kF16
  const void* bias;
  int bias_type;
  int activation;
  float ca, cb, cc;
  const float* scale;  // of each matrix of a batch (kGemmPoly, kGemmUpdate): X is that times what is stored
};

// Into how many parts the sum of a product with fp32 results is best shared out (1: none).
int gemm_parts(int64_t m, int64_t n, int64_t k);
cudaError_t launch_gemm(const GemmCall& call, cudaStream_t stream);
bool gemm_operand_ok(const void* data, int64_t ld);

}  // namespace hc
