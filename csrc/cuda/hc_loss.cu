// Softmax cross entropy of x W^T over a vocabulary, with the gradients of x and W, in pieces of the vocabulary: the logits are never stored.
//
//   l_iv = x_i . w_v,  lse_i = log sum_v exp l_iv,  loss_i = lse_i - l_i,token
//   G_iv = a_i (exp(l_iv - lse_i) - [v = token_i]),  dx = G W,  dW = G^T x         (a: the upstream gradient of a row)
//
// Forward, one product whose epilogue keeps each row's largest logit and sum of exponentials over a stretch of columns (hc_gemm.cu), its token's logit apart: 8 bytes for 32
// to 128 logits, joined by a second kernel.  Backward, a piece of the vocabulary at a time: its logits are formed again, G leaves the
// epilogue in 16 bits, and two products take it up: dx is summed over the pieces in fp32, the piece of dW is done.  That is four products where three
// would do with the logits kept; kept in 16 bits they would be wrong by 2^-9 of themselves, and G by as much times the logit.  G rounded to 16 bits is what any
// product of it needs; fp16, which holds nothing below 2^-24, gets G times a power of two that takes the largest |a| to 2^13.
//
// Sums over columns, rows and pieces have a fixed order.
#include "hc_gemm.cuh"
#include "hc_host.cuh"
#include "hc_train.cuh"
#include "homcomp_train.h"

namespace hc {
namespace dev {

enum Reduction : int { kNone = 0, kSum = 1, kMean = 2 };

// A row's loss and lse from its token's logit z and what the others come to, their largest and their sum of exponentials relative to it: with d = log sum of the others - z, loss = log(1 + exp d).  The token
// has no part in the sum: of a row that is sure of its token little is left, which a sum that begins with the token's 1, or lse, rounded at its own size, no longer has.  A row with an infinite logit,
// or a NaN, has a NaN among its sums (or as z); where all others are -inf their sum is 0.
__device__ __forceinline__ void loss_of_row(float most, float sum, int64_t row, const float* picked, const int64_t* tokens, int64_t ignore, int64_t vocab, float* lse, float* kept,
                                            float* losses) {
  const float none = __int_as_float(0x7fc00000), others = most + logf(sum);
  const int64_t token = tokens[row];
  if (token == ignore || token < 0 || token >= vocab) {
    lse[row] = sum == 0.0f ? none : others;
    kept[row] = token == ignore ? 0.0f : none;
    if (losses) losses[row] = kept[row];
    return;
  }
  const float z = picked[row], d = (most - z) + logf(sum), above = log1pf(expf(-fabsf(d)));
  lse[row] = z < INFINITY ? (d > 0.0f ? others : z) + above : none;
  kept[row] = z < INFINITY ? d > 0.0f ? d + above : above : none;
  if (losses) losses[row] = kept[row];
}

// Joins the stretches of 32 rows: warp w takes every 32nd, a lane a row.
__global__ void __launch_bounds__(1024) hc_loss_join_kernel(const float2* sums, int64_t stretches, int64_t rows, const float* picked, const int64_t* tokens, int64_t ignore,
                                                             int64_t vocab, float* lse, float* kept, float* losses) {
  __shared__ float2 shared[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x * 32ll + lane;
  float most = -INFINITY, sum = 0.0f;
  const auto take = [&](float2 v) {
    const float top = fmaxf(most, v.x), ref = top == -INFINITY ? 0.0f : top;
    sum = sum * exp2f((most - ref) * kLog2E) + v.y * exp2f((v.x - ref) * kLog2E);
    most = top;
  };
  if (row < rows) {
#pragma unroll 4
    for (int64_t s = warp; s < stretches; s += 32) take(sums[s * rows + row]);
  }
  shared[warp][lane] = make_float2(most, sum);
  __syncthreads();
  if (warp != 0 || row >= rows) return;
  for (int w = 1; w < 32; ++w) take(shared[w][lane]);
  loss_of_row(most, sum, row, picked, tokens, ignore, vocab, lse, kept, losses);
}

// The same of few rows, a block each, whose stretches lie one after the other.  Its launch overlaps the products' (1 row of 768, 50257 tokens: 19.6 us a call, 20.6 without).
__global__ void __launch_bounds__(1024) hc_loss_join_row_kernel(const float2* sums, int64_t stretches, const float* picked, const int64_t* tokens, int64_t ignore, int64_t vocab, float* lse,
                                                                 float* kept, float* losses) {
  __shared__ float tops[32], totals[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  constexpr int kAtOnce = 4;
  grid_dependency_wait();
  float most = -INFINITY, sum = 0.0f;
  const auto joined = [](float& most, float& sum, float m, float s) {
    const float top = fmaxf(most, m), ref = top == -INFINITY ? 0.0f : top;
    sum = sum * exp2f((most - ref) * kLog2E) + s * exp2f((m - ref) * kLog2E);
    most = top;
  };
  for (int64_t i = threadIdx.x; i < stretches; i += 1024 * kAtOnce) {
    float2 v[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) v[k] = i + k * 1024 < stretches ? sums[row * stretches + i + k * 1024] : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) joined(most, sum, v[k].x, v[k].y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_down_sync(0xffffffffu, most, o), s = __shfl_down_sync(0xffffffffu, sum, o);
    joined(most, sum, m, s);
  }
  if (lane == 0) tops[warp] = most, totals[warp] = sum;
  __syncthreads();
  if (warp != 0) return;
  most = tops[lane], sum = totals[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_down_sync(0xffffffffu, most, o), s = __shfl_down_sync(0xffffffffu, sum, o);
    joined(most, sum, m, s);
  }
  if (lane != 0) return;
  loss_of_row(most, sum, row, picked, tokens, ignore, vocab, lse, kept, losses);
}

// their sum, or their mean over the rows that have a token, whose number is kept for the backward pass
__global__ void __launch_bounds__(1024) hc_loss_reduce_kernel(const float* losses, const int64_t* tokens, int64_t ignore, int64_t rows, int reduction, float* loss, float* count) {
  __shared__ double sums[32];
  __shared__ long long counts[32];
  double sum = 0.0;
  long long kept = 0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    sum += losses[i];
    kept += tokens[i] != ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    kept += __shfl_xor_sync(0xffffffffu, kept, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[threadIdx.x >> 5] = sum;
    counts[threadIdx.x >> 5] = kept;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 32; ++w) {
    sum += sums[w];
    kept += counts[w];
  }
  *count = (float)kept;
  if (reduction != kNone) *loss = (float)(reduction == kMean ? sum / (double)kept : sum);
}

// Each row's weight in the gradient, and the bits of the largest of them.  Where all rows weigh the same G is formed with weights of 1 and the results are taken times `factor`: of a token that a row
// hardly expects G is then -1 to within p, and what rounding G costs is less.  G at a row's token, -(1 - p), is made of its loss: exp(logit - lse), which is off by lse's rounding and by what the two passes'
// sums differ by, has nothing left of 1 - p where the row is sure of its token.
__global__ void __launch_bounds__(256) hc_loss_weights_kernel(const float* dloss, const int64_t* tokens, int64_t ignore, int64_t rows, int64_t vocab, int reduction,
                                                              const float* losses, const float* count, float* weight, float* picked, unsigned int* most, float* factor) {
  unsigned int largest = 0;
  // where no row has a token nothing is taken times an upstream gradient, which may be no number
  if (blockIdx.x == 0 && threadIdx.x == 0 && factor) *factor = *count > 0.0f ? reduction == kSum ? dloss[0] : dloss[0] / *count : 0.0f;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows; i += gridDim.x * 256ll) {
    const int64_t token = tokens[i];
    float a = 0.0f;
    if (token != ignore) {
      a = reduction == kNone ? dloss[i] : 1.0f;
      if (token < 0 || token >= vocab) a = __int_as_float(0x7fc00000);
    }
    weight[i] = a;
    picked[i] = token != ignore ? a * expm1f(-losses[i]) : 0.0f;
    const unsigned int bits = __float_as_uint(a) & 0x7fffffffu;
    if (bits < 0x7f800000u) largest = max(largest, bits);
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (most && (threadIdx.x & 31) == 0 && largest) atomicMax(most, largest);
}

// dx in its own type, from the parts of its sum, which is times 2^k (gradient_power) and, over `factor`, of weights of 1.  Rows without a token get zeros, also where `factor` is no number.
template <typename T>
__global__ void __launch_bounds__(256) hc_loss_dx_kernel(const float* sum, int64_t from_stride, int parts, int64_t rows, int64_t width, const unsigned int* most, const float* factor,
                                                         const int64_t* tokens, int64_t ignore, T* dx, int64_t stride) {
  const float power = (most ? gradient_power(most, -1) : 1.0f) * (factor ? *factor : 1.0f);
  const int64_t groups = (width + 7) / 8;
  const bool vector = stride % 8 == 0 && (reinterpret_cast<uintptr_t>(dx) & 15u) == 0;
  for (int64_t k = blockIdx.x * 256ll + threadIdx.x; k < rows * groups; k += gridDim.x * 256ll) {
    const int64_t r = k / groups, c = (k - r * groups) * 8;
    float v[8];
    load8(sum + r * from_stride + c, v);
    for (int part = 1; part < parts; ++part) {
      float w[8];
      load8(sum + (part * rows + r) * from_stride + c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += w[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tokens[r] == ignore ? 0.0f : v[j] * power;
    if (vector && c + 8 <= width) {
      store8(dx + r * stride + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < width) dx[r * stride + c + j] = from_float<T>(v[j]);
    }
  }
}

}  // namespace dev

namespace {

constexpr size_t kMostSide = (size_t)1 << 26;
constexpr size_t kMostBytes = 256;
// G of a piece takes no more than this, or 1024 columns.  8192 x 768 x 50257, both passes: 3030 us with at most 48 MiB, 2690 with 64, 2475 with 128, 2390 with 256, 2293 with 384, 2255 in one piece.
constexpr size_t kPieceBytes = (size_t)384 << 20;

size_t up(size_t v, size_t unit) { return (v + unit - 1) / unit * unit; }
bool loss_sizes_ok(size_t rows, size_t inner, size_t vocab) { return inner > 0 && vocab > 0 && inner < kMostSide && vocab < kMostSide && rows < kMostSide; }

int64_t stretches_of(size_t rows, size_t inner, size_t vocab) { return rows <= HC_LINEAR_FEW_ROWS ? (int64_t)(vocab + 15) / 16 : gemm_loss_stretches(rows, vocab, inner); }
size_t forward_bytes(size_t rows, size_t inner, size_t vocab) {
  if (!rows) return 0;
  return up((size_t)stretches_of(rows, inner, vocab) * rows * sizeof(float2), 256) + up(rows * sizeof(float), 256);
}

// Into how many parts the sum of dx's product with a piece is shared out, each of which is summed over the pieces in an array of its own: 96 tiles of 256 x 256 on 74 pairs of SMs leave a third of
// them idle, 288 thirds of tiles do not.
constexpr int kMostParts = 4;
int dx_parts_of(size_t rows, size_t inner, size_t piece) {
  int best = 1;
  double least = 0;
  for (int parts = 1; parts <= kMostParts && piece >= (size_t)parts * 1024; ++parts) {
    // what a part writes and reads, some 3000 bytes a cycle, passes beside the products but for a quarter of it
    const double cost = (double)gemm_cost(rows, inner, piece, parts) + (parts - 1) * (rows * inner * 8.0 / 3000.0 * 0.25);
    if (least == 0 || cost < least) {
      least = cost;
      best = parts;
    }
  }
  return best;
}

// The pieces of the vocabulary: as many columns as the tiles of the three products fill the SMs best with, by their reckoned times.
size_t piece_of(size_t rows, size_t inner, size_t vocab) {
  size_t most = kPieceBytes / (rows * 2) / 256 * 256;
  if (most < 1024) most = 1024;
  if (most >= vocab) return vocab;
  size_t best = most;
  double least = 0;
  for (size_t piece = most; piece >= 1024 && piece * 4 > most; piece -= 256) {
    const auto cost = [&](size_t n) { return (double)(gemm_cost(rows, n, inner, 1) + gemm_cost(rows, inner, n, dx_parts_of(rows, inner, n)) + gemm_cost(n, inner, rows, 1)); };
    const size_t whole = vocab / piece, rest = vocab % piece;
    const double all = whole * (cost(piece) + 15000.0) + (rest ? cost(rest) + 15000.0 : 0.0);
    if (least == 0 || all < least) {
      least = all;
      best = piece;
    }
  }
  return best;
}
struct LossLayout {
  int parts;  // of dx
  size_t piece, g, dx, weight, picked, most, total;  // offsets, G at 0
};
LossLayout backward_layout(size_t rows, size_t inner, size_t vocab) {
  LossLayout l;
  l.piece = piece_of(rows, inner, vocab);
  l.parts = dx_parts_of(rows, inner, l.piece);
  l.dx = up(rows * up(l.piece, 8) * 2, 256);
  l.weight = l.dx + up((size_t)l.parts * rows * up(inner, 8) * sizeof(float), 256);
  l.picked = l.weight + up(rows * sizeof(float), 256);
  l.most = l.picked + up(rows * sizeof(float), 256);
  l.total = l.most + kMostBytes;
  return l;
}

bool operands_ok(const void* x, size_t x_stride, const void* weight, size_t weight_stride, size_t inner, bool anywhere) {
  return x && weight && x_stride >= inner && weight_stride >= inner && x_stride < ((size_t)1 << 32) && weight_stride < ((size_t)1 << 32) &&
         (anywhere ? lies_at(x, 2) && lies_at(weight, 2) : gemm_operand_ok(x, (int64_t)x_stride) && gemm_operand_ok(weight, (int64_t)weight_stride));
}

}  // namespace
}  // namespace hc

extern "C" {

size_t hc_linear_cross_entropy_bytes(size_t rows, size_t inner, size_t vocab) { return hc::loss_sizes_ok(rows, inner, vocab) ? hc::forward_bytes(rows, inner, vocab) : 0; }

int hc_linear_cross_entropy(const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, const int64_t* tokens, int64_t ignore, int reduction, float* loss,
                            float* stats, size_t rows, size_t inner, size_t vocab, void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  if ((type != kBf16 && type != kF16) || reduction < 0 || reduction > 2 || !loss_sizes_ok(rows, inner, vocab)) return kErrArgument;
  if (!lies_at(loss, 4) || !lies_at(stats, 4) || !lies_at(tokens, 8) || (!loss && (rows || reduction)) || !stats) return kErrArgument;
  float *losses = reduction == dev::kNone ? loss : nullptr, *lse = stats, *kept = stats + rows, *count = stats + 2 * rows;
  if (rows) {
    if (!tokens || !operands_ok(x, x_stride, weight, weight_stride, inner, rows <= HC_LINEAR_FEW_ROWS)) return kErrArgument;
    if (!scratch || !lies_at(scratch, 256) || scratch_bytes < forward_bytes(rows, inner, vocab)) return kErrArgument;
    GemmCall c;
    memset(&c, 0, sizeof(c));
    c.type = type;
    c.m = rows, c.n = vocab, c.k = inner, c.batch = 1;
    c.a = {x, (int64_t)x_stride, 0, true};
    c.b = {weight, (int64_t)weight_stride, 0, true};
    const int64_t stretches = stretches_of(rows, inner, vocab);
    unsigned char* at = static_cast<unsigned char*>(scratch);
    c.loss.sums = reinterpret_cast<float2*>(at);
    c.loss.stretches = stretches;
    at += up((size_t)stretches * rows * sizeof(float2), 256);
    c.loss.picked = reinterpret_cast<float*>(at);
    c.loss.tokens = tokens;
    c.loss.ignore = ignore;
    const bool few = rows <= HC_LINEAR_FEW_ROWS;
    if ((few ? launch_few_rows_loss(c, stream) : launch_loss_sums(c, stream)) != cudaSuccess) return kErrCuda;
    const float2* sums = c.loss.sums;
    const float* picked = c.loss.picked;
    if (few) {
      if (launch_with(dev::hc_loss_join_row_kernel, (int64_t)rows, 1, 1024, 0, stream, true, sums, stretches, picked, tokens, ignore, (int64_t)vocab, lse, kept, losses) != cudaSuccess) return kErrCuda;
    } else {
      dev::hc_loss_join_kernel<<<(unsigned)((rows + 31) / 32), 1024, 0, stream>>>(sums, stretches, (int64_t)rows, picked, tokens, ignore, (int64_t)vocab, lse, kept, losses);
    }
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  }
  if (reduction == dev::kNone) return kOk;
  dev::hc_loss_reduce_kernel<<<1, 1024, 0, stream>>>(kept, tokens, ignore, (int64_t)rows, reduction, loss, count);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

size_t hc_linear_cross_entropy_backward_bytes(size_t rows, size_t inner, size_t vocab) {
  return hc::loss_sizes_ok(rows, inner, vocab) && rows ? hc::backward_layout(rows, inner, vocab).total : 0;
}

int hc_linear_cross_entropy_backward(const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, const int64_t* tokens, int64_t ignore, int reduction,
                                     const float* stats, const float* dloss, void* dx, size_t dx_stride, void* dweight, size_t dweight_stride, size_t rows, size_t inner, size_t vocab,
                                     void* scratch, size_t scratch_bytes, hc_stream_t stream) {
  using namespace hc;
  if ((type != kBf16 && type != kF16) || reduction < 0 || reduction > 2 || !loss_sizes_ok(rows, inner, vocab)) return kErrArgument;
  if ((dx && (dx_stride < inner || dx_stride >= ((size_t)1 << 32))) || (dweight && (dweight_stride < inner || dweight_stride >= ((size_t)1 << 32)))) return kErrArgument;
  if (!lies_at(stats, 4) || !lies_at(dloss, 4) || !lies_at(dx, 2) || !lies_at(dweight, 2) || !lies_at(tokens, 8)) return kErrArgument;
  if (rows == 0)
    return !dweight || cudaMemset2DAsync(dweight, dweight_stride * 2, 0, inner * 2, vocab, stream) == cudaSuccess ? kOk : kErrCuda;
  if (!dx && !dweight) return kOk;
  if (!tokens || !stats || !dloss || !operands_ok(x, x_stride, weight, weight_stride, inner, false)) return kErrArgument;
  const LossLayout l = backward_layout(rows, inner, vocab);
  if (!scratch || !lies_at(scratch, 256) || scratch_bytes < l.total) return kErrArgument;
  unsigned char* at = static_cast<unsigned char*>(scratch);
  float *dx_sum = reinterpret_cast<float*>(at + l.dx), *row_weight = reinterpret_cast<float*>(at + l.weight), *picked = reinterpret_cast<float*>(at + l.picked);
  unsigned int* most = type == kF16 ? reinterpret_cast<unsigned int*>(at + l.most) : nullptr;
  float* factor = reduction != dev::kNone ? reinterpret_cast<float*>(at + l.most + 4) : nullptr;
  if (most && cudaMemsetAsync(most, 0, sizeof(*most), stream) != cudaSuccess) return kErrCuda;
  const size_t blocks = (rows + 255) / 256;
  dev::hc_loss_weights_kernel<<<(unsigned)(blocks < 256 ? blocks : 256), 256, 0, stream>>>(dloss, tokens, ignore, (int64_t)rows, (int64_t)vocab, reduction, stats + rows, stats + 2 * rows,
                                                                                     row_weight, picked, most, factor);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  const int64_t dx_ld = (int64_t)up(inner, 8);
  for (size_t first = 0; first < vocab; first += l.piece) {
    const size_t n = vocab - first < l.piece ? vocab - first : l.piece;
    const uint16_t* w = static_cast<const uint16_t*>(weight) + first * weight_stride;
    const int64_t g_ld = (int64_t)up(n, 8);
    GemmCall c;
    memset(&c, 0, sizeof(c));
    c.type = c.out_type = type;
    c.batch = 1;
    c.most = most;
    c.m = rows, c.n = n, c.k = inner;
    c.a = {x, (int64_t)x_stride, 0, true};
    c.b = {w, (int64_t)weight_stride, 0, true};
    c.out = {at, g_ld, 0};
    c.loss.tokens = tokens;
    c.loss.ignore = ignore;
    c.loss.first = (int64_t)first;
    c.loss.lse = stats;
    c.loss.weight = row_weight;
    c.loss.picked = picked;
    if (launch_loss_grad(c, stream) != cudaSuccess) return kErrCuda;
    c.factor = factor;
    if (dweight) {
      c.m = n, c.n = inner, c.k = rows;
      c.a = {at, g_ld, 0, false};
      c.b = {x, (int64_t)x_stride, 0, false};
      c.out = {static_cast<uint16_t*>(dweight) + first * dweight_stride, (int64_t)dweight_stride, 0};
      if (launch_gemm(c, stream) != cudaSuccess) return kErrCuda;
    }
    if (dx) {
      c.m = rows, c.n = inner, c.k = n;
      c.a = {at, g_ld, 0, true};
      c.b = {w, (int64_t)weight_stride, 0, false};
      c.out_type = kF32;
      c.out = {dx_sum, dx_ld, (int64_t)rows * dx_ld};
      c.parts = l.parts;
      c.most = nullptr;
      c.factor = nullptr;
      if (first) c.in = c.out;
      if (launch_gemm(c, stream) != cudaSuccess) return kErrCuda;
    }
  }
  if (!dx) return kOk;
  const size_t dx_blocks = (rows * (up(inner, 8) / 8) + 255) / 256;
  const unsigned grid = (unsigned)(dx_blocks < 2368 ? dx_blocks : 2368);
  if (type == kBf16)
    dev::hc_loss_dx_kernel<<<grid, 256, 0, stream>>>(dx_sum, dx_ld, l.parts, (int64_t)rows, (int64_t)inner, most, factor, tokens, ignore, static_cast<__nv_bfloat16*>(dx), (int64_t)dx_stride);
  else
    dev::hc_loss_dx_kernel<<<grid, 256, 0, stream>>>(dx_sum, dx_ld, l.parts, (int64_t)rows, (int64_t)inner, most, factor, tokens, ignore, static_cast<__half*>(dx), (int64_t)dx_stride);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // extern "C"
