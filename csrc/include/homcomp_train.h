// homcomp-b200: operators of a training step, for the code on either side of the compressed gradient exchange.
//
// All pointers are device pointers unless named otherwise.  Calls only enqueue work on `stream`: they never allocate,
// never synchronise and keep nothing between calls, so they may be captured into a graph and replayed.  What scratch
// memory a call needs is given by the caller, 256-byte aligned; two calls that can run at the same time (two streams,
// two graphs) need two of them.  All functions return 0 or a hc::Status code: 4 for arguments that the call does not
// take, 5 for an error of the CUDA runtime.
//
// A pointer that does not begin where its elements may is refused.  What a call writes does not overlap what it reads, its scratch memory
// or its other results.
//
// Types: 0 fp32, 1 bf16, 2 fp16.  Strides count elements from one row to the next; the elements of a row are adjacent.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* hc_stream_t;  // same type as cudaStream_t

// ---- layer norm ---------------------------------------------------------------------------------------------------
// y = (x - mean(x)) * rstd * weight + bias over rows of `width` values, rstd = 1 / sqrt(var(x) + eps).
// x, y (and dy, dx): `rows` rows, one after the other (stride = width), 16-byte aligned; weight / bias: NULL for 1 / 0.
// stats: 2 floats a row (mean, rstd), 8-byte aligned, for the backward pass, or NULL.
int hc_layer_norm(const void* x, int x_type, const void* weight, const void* bias, int param_type, void* y, int y_type,
                  float* stats, size_t rows, size_t width, float eps, hc_stream_t stream);
// dx, and dweight / dbias (both or neither; sums over the rows in fp32, in a fixed order).  dx may be NULL.
size_t hc_layer_norm_backward_bytes(size_t rows, size_t width);
int hc_layer_norm_backward(const void* dy, int y_type, const void* x, int x_type, const void* weight, int param_type,
                           const float* stats, void* dx, void* dweight, void* dbias, size_t rows, size_t width,
                           void* scratch, size_t scratch_bytes, hc_stream_t stream);

// ---- log probabilities of given tokens ------------------------------------------------------------------------------
// Per row of `vocab` logits: log p(token), the entropy of p, and the `top` (0 to 64) most likely tokens, most likely
// first, the lowest index first among equals.  A row whose token is `ignore` gives 0, 0, and tokens of -1; a token
// outside the vocabulary gives NaN, as does a row with a NaN or +inf or with nothing above -inf (tokens -1).
// stats: 3 floats a row (maximum, log of the sum above it, entropy) for the backward pass, or NULL.
int hc_token_logprobs(const void* logits, int type, size_t rows, size_t vocab, size_t stride, const int64_t* tokens,
                      int64_t ignore, int top, float* logprobs, float* entropy, int64_t* top_tokens, float* top_logprobs,
                      float* stats, hc_stream_t stream);
// dlogits = a (1[token] - p) - b p (log p + entropy) with a = dlogprobs, b = dentropy of the row (NULL: 0).
int hc_token_logprobs_backward(const void* logits, int type, size_t rows, size_t vocab, size_t stride,
                               const int64_t* tokens, int64_t ignore, const float* stats, const float* dlogprobs,
                               const float* dentropy, void* dlogits, size_t dstride, hc_stream_t stream);

// ---- products ---------------------------------------------------------------------------------------------------------
// Operands are bf16 or fp16 (`type` 1 or 2), sums fp32, in the tensor core over up to 1024 terms for fp32 results and up to 8192 (fp16) or 65536
// (bf16) for 16-bit ones, whose rounding is four times and more what that loses.  x [rows][inner], weight [width][inner], out [rows][width], each side
// below 2^26.
#define HC_LINEAR_FEW_ROWS 16
// A product of more than HC_LINEAR_FEW_ROWS rows, and the products of a backward pass, read their operands in 16-byte pieces: data
// 16-byte aligned, strides multiples of 8.  Fewer rows, and their weights, may begin anywhere.
// Results and what is added to them may lie anywhere.  Where a result's stride is its width rounded up to eight, what lies
// behind its rows is padding and may be overwritten; behind rows of any other stride nothing is.
//
// activation: 0 none, 1 GELU (tanh form), 2 ReLU, 3 SiLU.
// out = act(x weight^T + bias) + residual; out_type 0 or `type`, residual (NULL: none) of out_type, bias (NULL: none)
// of bias_type.  z: what the activation is applied to, of `type`, for the backward pass, or NULL.
// hc_align_rows copies rows of 16-bit values that begin anywhere to where a product can read them.
int hc_align_rows(const void* from, size_t from_stride, size_t rows, size_t width, void* to, size_t to_stride, hc_stream_t stream);
// Scratch memory (hc_linear_bytes for the current device, 256-byte aligned) takes the parts of a sum that is shared out; 0: none.
size_t hc_linear_bytes(size_t rows, size_t inner, size_t width);
int hc_linear(const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, const void* bias, int bias_type,
              const void* residual, size_t residual_stride, void* out, int out_type, size_t out_stride, void* z, size_t z_stride,
              int activation, size_t rows, size_t inner, size_t width, void* scratch, size_t scratch_bytes, hc_stream_t stream);
// Backward pass: dz = dy act'(z), rounded to `type` for the products (of an fp32 dy and fp16 operands times a power of two, which its largest
// finite value gives, and which the results are freed of); dx = dz weight, dweight = dz^T x (of `type`) and dbias =
// the sums of dz's columns before rounding (of bias_type), each NULL where it is not wanted.  dy is of dy_type, 0 or `type`.
// keep_dz: dz is written to the scratch memory; 0 where dy itself is dz and a product can read it (no activation, dy of
// `type`, its rows as operands have to lie).  Sums over rows are formed in a fixed order.
size_t hc_linear_backward_bytes(size_t rows, size_t inner, size_t width, int keep_dz);
int hc_linear_backward(const void* dy, int dy_type, size_t dy_stride, const void* z, size_t z_stride, int activation, int keep_dz,
                       const void* x, size_t x_stride, const void* weight, size_t weight_stride, int type, void* dx, size_t dx_stride,
                       void* dweight, size_t dweight_stride, void* dbias, int bias_type, size_t rows, size_t inner, size_t width,
                       void* scratch, size_t scratch_bytes, hc_stream_t stream);

// ---- orthogonalised updates ---------------------------------------------------------------------------------------------
// Newton-Schulz iteration: X = G / (|G| + eps); `steps` times X = a X + (b S + c S S) X with S = X X^T (or its mirror image
// from the right where a matrix is taller than wide).  G: `batch` matrices [height][width] of `type`, rows `stride` and
// matrices `batch_stride` elements apart; out: the same matrices in bf16 without gaps.  Products take fp16 operands; X
// itself is carried in two fp16 numbers (22 bits), for what is rounded off it grows by up to `a` a step.  Coefficients that could
// take a singular value in [0, 1], in all steps but the last, above 244, or b s + c s s of its square s above 60000, are refused.
size_t hc_orthogonalize_bytes(size_t batch, size_t height, size_t width);
int hc_orthogonalize(const void* g, int type, size_t batch, size_t height, size_t width, size_t stride, size_t batch_stride, void* out,
                     int steps, float a, float b, float c, float eps, void* scratch, size_t scratch_bytes, hc_stream_t stream);

// The kernels' waits are bounded (2 s).  Where one ran out the call's results are wrong.  Synchronises the device and returns 3 if that
// happened since the status was last cleared, 0 if not.
int hc_train_status(int clear);

#ifdef __cplusplus
}
#endif
