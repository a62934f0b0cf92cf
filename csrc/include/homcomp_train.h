// homcomp-b200: operators of a training step, for the code on either side of the compressed gradient exchange.
//
// All pointers are device pointers unless named otherwise.  Calls only enqueue work on `stream`: they never allocate,
// never synchronise and keep nothing between calls, so they may be captured into a graph and replayed.  What scratch
// memory a call needs is given by the caller, 256-byte aligned; two calls that can run at the same time (two streams,
// two graphs) need two of them.  All functions return 0 or a hc::Status code: 4 for arguments that the call does not
// take, 5 for an error of the CUDA runtime.
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
// stats: 2 floats a row (mean, rstd) for the backward pass, or NULL.
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

#ifdef __cplusplus
}
#endif
