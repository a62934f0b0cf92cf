// The training step's operators on torch tensors, with their gradients.
//
// A call of a small size costs what the host spends on it, and most of that, where the front end was Python over ctypes,
// was the front end: forward and backward pass of a layer norm took the host 115 us, of which torch's autograd engine has 53.
// This module checks arguments, allocates results and scratch memory on the current stream's pool, and calls the functions
// of homcomp_train.h, whose addresses it is given when it is loaded (so that it runs whichever build of the library is loaded).
// It is built by g++ against torch's headers and links nothing of the library.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <string>
#include <tuple>
#include <unordered_map>

#include "homcomp_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::tensor_list;
using OptTensor = std::optional<Tensor>;

struct Api {
  decltype(&hc_layer_norm) layer_norm;
  decltype(&hc_layer_norm_backward_bytes) layer_norm_backward_bytes;
  decltype(&hc_layer_norm_backward) layer_norm_backward;
  decltype(&hc_token_logprobs) token_logprobs;
  decltype(&hc_token_logprobs_backward) token_logprobs_backward;
  decltype(&hc_align_rows) align_rows;
  decltype(&hc_linear_bytes) linear_bytes;
  decltype(&hc_linear) linear;
  decltype(&hc_linear_backward_bytes) linear_backward_bytes;
  decltype(&hc_linear_backward) linear_backward;
  decltype(&hc_orthogonalize_bytes) orthogonalize_bytes;
  decltype(&hc_orthogonalize) orthogonalize;
} api;

void bind_all(const std::unordered_map<std::string, uintptr_t>& at) {
#define HC_BIND(name) api.name = reinterpret_cast<decltype(api.name)>(at.at("hc_" #name))
  HC_BIND(layer_norm);
  HC_BIND(layer_norm_backward_bytes);
  HC_BIND(layer_norm_backward);
  HC_BIND(token_logprobs);
  HC_BIND(token_logprobs_backward);
  HC_BIND(align_rows);
  HC_BIND(linear_bytes);
  HC_BIND(linear);
  HC_BIND(linear_backward_bytes);
  HC_BIND(linear_backward);
  HC_BIND(orthogonalize_bytes);
  HC_BIND(orthogonalize);
#undef HC_BIND
}

// ---- types, checks, memory ------------------------------------------------------------------------------------------
constexpr int kNoType = -1;
int type_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : kNoType;
}
at::ScalarType scalar_of(int type) { return type == 0 ? at::kFloat : type == 1 ? at::kBFloat16 : at::kHalf; }
int type_of(const Tensor& t) { return type_of(t.scalar_type()); }
int type_of(const OptTensor& t) { return t ? type_of(*t) : 0; }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The kernels run outside of torch's dispatcher: a tangent would be lost without a word, and a recording of a call would hold its
// results' allocation and nothing that fills them.
void not_recorded() {
  bool recorded = at::tracer::impl::is_dispatch_enabled();
  using Modes = c10::impl::TorchDispatchModeTLS;
  if (Modes::any_modes_set())
    for (int8_t i = 0; i < static_cast<int8_t>(c10::impl::TorchDispatchModeKey::NUM_MODE_KEYS); ++i)
      recorded = recorded || Modes::get_mode(static_cast<c10::impl::TorchDispatchModeKey>(i)).has_value();
  TORCH_CHECK_NOT_IMPLEMENTED(!recorded, "the operators of a training step cannot be recorded (torch.jit.trace, make_fx, fake tensors)");
}
void ordinary(const char* name, const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet others({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                        DispatchKey::FuncTorchVmapMode, DispatchKey::Batched, DispatchKey::ZeroTensor});
  TORCH_CHECK_NOT_IMPLEMENTED(!t.key_set().has_any(others), name, ": vmap, functional transforms and tensor subclasses are not implemented for the operators of a training step");
  TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), name,
                              ": forward-mode derivatives are not implemented for the operators of a training step");
}
void ordinary(const char* name, const OptTensor& t) {
  if (t) ordinary(name, *t);
}
// A view may stand for the negative of what lies in its memory (the imaginary part of a conjugate does; gradients may)
Tensor held(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
OptTensor held(const OptTensor& t) { return t ? OptTensor(held(*t)) : t; }
void floating(const char* name, const Tensor& t) {
  TORCH_CHECK_VALUE(type_of(t) != kNoType, name, ": expected a float32, bfloat16 or float16 tensor");
  TORCH_CHECK_VALUE(t.is_cuda(), name, ": expected a CUDA tensor");
}
void beside(const char* name, const Tensor& t, const Tensor& other) {
  TORCH_CHECK_VALUE(t.device() == other.device(), name, " is on ", t.device(), ", not on ", other.device());
}
void vector(const char* name, const Tensor& t, int64_t n, const Tensor& other) {
  floating(name, t);
  beside(name, t, other);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, ": expected ", n, " values in one dimension, got shape ", t.sizes());
}

void check(int status, const char* what) {
  static const char* names[] = {"", "capacity", "truncated", "timeout", "argument", "cuda", "peer"};
  TORCH_CHECK(status == 0, what, " failed: status ", status, " (", status > 0 && status < 7 ? names[status] : "?", ")");
}
hc_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<hc_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}
Tensor scratch_of(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
// without gaps and 16-byte aligned, copied only if it is not so
Tensor packed(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}
OptTensor contiguous(const OptTensor& t) { return t ? OptTensor(t->contiguous()) : t; }

int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }
// A tensor of shape (rows, width), or `shape`, whose rows are `apart` elements apart: not a view, which autograd would not let
// be changed in place, but with memory for all of its last row.
Tensor empty_apart(int64_t rows, int64_t width, int64_t apart, const at::TensorOptions& options, at::IntArrayRef shape = {}) {
  Tensor t = at::empty({rows, apart}, options);
  at::DimVector sizes(shape);
  if (shape.empty()) sizes = {rows, width};
  at::DimVector strides(sizes.size(), 1);
  for (int64_t i = (int64_t)sizes.size() - 2, s = apart; i >= 0; s *= std::max<int64_t>(sizes[i], 1), --i) strides[i] = s;
  t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides);
  return t;
}
// A matrix whose rows begin at 16-byte boundaries, with gaps where eight does not divide `width`; as `shape` where that is given
Tensor empty_rows(int64_t rows, int64_t width, const at::TensorOptions& options, at::IntArrayRef shape = {}) {
  if (padded(width) == width) return shape.empty() ? at::empty({rows, width}, options) : at::empty(shape, options);
  return empty_apart(rows, width, padded(width), options, shape);
}
int64_t any_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : padded(t.size(1)); }
// rows whose elements are adjacent and that do not overlap
bool rows_adjacent(const Tensor& t) { return (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)); }
// as the products read it: such rows that begin at 16-byte boundaries
bool is_operand(const Tensor& t) { return rows_adjacent(t) && row_stride(t) % 8 == 0 && aligned(t); }
Tensor operand(const Tensor& t) {
  if (is_operand(t)) return t;
  Tensor copy = empty_rows(t.size(0), t.size(1), t.options());
  if (!rows_adjacent(t)) return copy.copy_(t);
  const c10::cuda::CUDAGuard guard(t.device());
  check(api.align_rows(t.data_ptr(), any_stride(t), t.size(0), t.size(1), copy.data_ptr(), padded(t.size(1)), stream_of(t)), "linear");
  return copy;
}
Tensor adjacent(const Tensor& t) { return rows_adjacent(t) ? t : t.contiguous(); }
Tensor matrix(const Tensor& t, int64_t width) { return t.dim() == 2 ? t : t.reshape({-1, width}); }

bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const OptTensor& t) { return t && t->requires_grad(); }

// Gradients are formed outside of autograd: a graph of them may be asked for, but not gone through.
tensor_list once(tensor_list grads, bool graph) {
  if (!graph) return grads;
  const at::AutoGradMode with_graph(true);
  tensor_list given;
  for (const Tensor& g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>("these gradients have no gradients of their own", (int64_t)given.size());
  given = (*error)(std::move(given));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = given[i++];
  return grads;
}

// ---- layer norm -----------------------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, int out, Tensor* stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor y = at::empty(x.sizes(), x.options().dtype(scalar_of(out)));
  if (stats) *stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  check(api.layer_norm(x.data_ptr(), type_of(x), ptr(weight), ptr(bias), weight ? type_of(weight) : type_of(bias), y.data_ptr(), out,
                       stats ? static_cast<float*>(stats->data_ptr()) : nullptr, rows, width, (float)eps, stream_of(x)),
        "layer_norm");
  return y;
}

struct LayerNorm : Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& given, const OptTensor& weight, const OptTensor& bias, double eps, int64_t out) {
    const Tensor x = packed(given);
    const OptTensor w = contiguous(weight), b = contiguous(bias);
    Tensor stats;
    Tensor y = norm_forward(x, w, b, eps, (int)out, &stats);
    ctx->save_for_backward({x, w ? *w : Tensor(), stats});
    ctx->saved_data["param_type"] = (int64_t)(w ? type_of(w) : type_of(b));
    ctx->saved_data["inputs"] = (int64_t)(weight ? 1 : 0) + (bias ? 2 : 0);
    return y;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
    not_recorded();
    ordinary("gradient", grads[0]);
    const int64_t inputs = ctx->saved_data["inputs"].toInt();
    const int param_type = (int)ctx->saved_data["param_type"].toInt();
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t width = x.size(-1), rows = x.numel() / width;
    // edges are numbered by the tensors that there are
    const bool want_x = ctx->needs_input_grad(0), want_w = (inputs & 1) && ctx->needs_input_grad(1),
               want_b = (inputs & 2) && ctx->needs_input_grad((inputs & 1) ? 2 : 1), sums = want_w || want_b;
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const Tensor dy = packed(held(grads[0]));
    const Tensor dx = want_x ? at::empty(x.sizes(), x.options()) : Tensor();
    const at::TensorOptions params = x.options().dtype(scalar_of(param_type));
    const Tensor dw = sums ? at::empty({width}, params) : Tensor(), db = sums ? at::empty({width}, params) : Tensor();
    const size_t need = sums ? api.layer_norm_backward_bytes(rows, width) : 0;
    const Tensor scratch = scratch_of(need, x);
    check(api.layer_norm_backward(dy.data_ptr(), type_of(dy), x.data_ptr(), type_of(x), ptr(weight), param_type, static_cast<float*>(stats.data_ptr()),
                                  ptr(dx), ptr(dw), ptr(db), rows, width, ptr(scratch), need, stream_of(x)),
          "layer_norm backward");
    return once({dx, want_w ? dw : Tensor(), want_b ? db : Tensor(), Tensor(), Tensor()}, graph);
  }
};

Tensor layer_norm(const Tensor& x_, const OptTensor& weight_, const OptTensor& bias_, double eps, int out) {
  not_recorded();
  ordinary("x", x_);
  ordinary("weight", weight_);
  ordinary("bias", bias_);
  const Tensor x = held(x_);
  const OptTensor weight = held(weight_), bias = held(bias_);
  floating("x", x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "layer_norm: x has no columns");
  if (out == kNoType) out = type_of(x);
  TORCH_CHECK_VALUE(out >= 0 && out <= 2 && (out == type_of(x) || out == 0 || type_of(x) == 0), "layer_norm: no result of that type of ", x.scalar_type(), " rows");
  if (weight) vector("weight", *weight, x.size(-1), x);
  if (bias) vector("bias", *bias, x.size(-1), x);
  TORCH_CHECK_VALUE(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "layer_norm: weight and bias have different types");
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps is negative");
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias))) return LayerNorm::apply(x, weight, bias, eps, (int64_t)out);
  return norm_forward(packed(x), contiguous(weight), contiguous(bias), eps, out, nullptr);
}

// ---- products -------------------------------------------------------------------------------------------------------
Tensor linear_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t act, int out, at::IntArrayRef shape,
                      Tensor* z) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
  Tensor y = empty_rows(m, n, x.options().dtype(scalar_of(out)), shape);
  if (z && act) *z = empty_rows(m, n, x.options());
  const size_t need = api.linear_bytes(m, k, n);
  const Tensor scratch = scratch_of(need, x);
  check(api.linear(x.data_ptr(), row_stride(x), weight.data_ptr(), row_stride(weight), type_of(x), ptr(bias), type_of(bias), ptr(residual),
                   residual ? any_stride(*residual) : 0, y.data_ptr(), out, padded(n), z ? ptr(*z) : nullptr, padded(n), (int)act, m, k, n, ptr(scratch), need,
                   stream_of(x)),
        "linear");
  return y;
}
// operands as the call with m rows reads them
Tensor for_rows(const Tensor& t, int64_t m) { return m > HC_LINEAR_FEW_ROWS ? operand(t) : adjacent(t); }

struct Linear : Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& given, const Tensor& given_weight, const OptTensor& bias, const OptTensor& residual, int64_t act,
                        int64_t out) {
    const int64_t k = given_weight.size(1), n = given_weight.size(0);
    const Tensor flat = matrix(given, k);
    const Tensor x = for_rows(flat, flat.size(0)), weight = for_rows(given_weight, flat.size(0));
    at::DimVector shape(given.sizes());
    shape.back() = n;
    const OptTensor r = residual ? OptTensor(adjacent(matrix(*residual, n))) : residual;
    Tensor z;
    Tensor y = linear_forward(x, weight, contiguous(bias), r, act, (int)out, shape, &z);
    ctx->save_for_backward({x, weight, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["inputs"] = (int64_t)(bias ? 1 : 0) + (residual ? 2 : 0);
    ctx->saved_data["bias_type"] = (int64_t)type_of(bias);
    ctx->saved_data["shape"] = given.sizes().vec();
    return y;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &z = saved[2];
    const int64_t act = ctx->saved_data["act"].toInt(), inputs = ctx->saved_data["inputs"].toInt();
    const int bias_type = (int)ctx->saved_data["bias_type"].toInt();
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = (inputs & 1) && ctx->needs_input_grad(2),
               want_r = (inputs & 2) && ctx->needs_input_grad((inputs & 1) ? 3 : 2);
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    Tensor dx, dw, db;
    if (want_x || want_w || want_b) {
      not_recorded();
      ordinary("gradient", grads[0]);
      const Tensor dy = adjacent(matrix(held(grads[0]), n));
      // dz is written where dy itself is not what the products can read
      const int keep = act || dy.scalar_type() != x.scalar_type() || !is_operand(dy);
      const auto shape = ctx->saved_data["shape"].toIntVector();
      if (want_x) dx = empty_rows(m, k, x.options(), shape);
      if (want_w) dw = empty_rows(n, k, x.options());
      if (want_b) db = at::empty({n}, x.options().dtype(scalar_of(bias_type)));
      const Tensor w = want_x ? operand(weight) : weight, a = want_w ? operand(x) : x;
      const size_t need = m ? api.linear_backward_bytes(m, k, n, keep) : 0;
      const Tensor scratch = scratch_of(need, x);
      check(api.linear_backward(dy.data_ptr(), type_of(dy), row_stride(dy), ptr(z), padded(n), (int)act, keep, a.data_ptr(), row_stride(a), w.data_ptr(),
                                row_stride(w), type_of(x), ptr(dx), padded(k), ptr(dw), padded(k), ptr(db), bias_type, m, k, n, ptr(scratch), need,
                                stream_of(x)),
            "linear backward");
    }
    return once({dx, dw, db, want_r ? grads[0] : Tensor(), Tensor(), Tensor()}, graph);
  }
};

Tensor linear(const Tensor& x_, const Tensor& weight_, const OptTensor& bias_, int64_t act, const OptTensor& residual_, int out) {
  not_recorded();
  ordinary("x", x_);
  ordinary("weight", weight_);
  ordinary("bias", bias_);
  ordinary("residual", residual_);
  const Tensor x = held(x_), weight = held(weight_);
  const OptTensor bias = held(bias_), residual = held(residual_);
  floating("x", x);
  floating("weight", weight);
  beside("weight", weight, x);
  const int type = type_of(x);
  TORCH_CHECK_VALUE(type != 0 && type_of(weight) == type, "linear: x and weight are both bfloat16 or both float16, got ", x.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK_VALUE(x.dim() > 0 && weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.numel() > 0, "linear: no product of x ", x.sizes(), " and weight ", weight.sizes());
  const int64_t n = weight.size(0), k = weight.size(1), m = x.numel() / k;
  TORCH_CHECK_VALUE(std::max(m, std::max(n, k)) < (1 << 26), "linear: every side is below 2^26");
  if (bias) vector("bias", *bias, n, x);
  at::DimVector shape(x.sizes());
  shape.back() = n;
  if (residual) {
    floating("residual", *residual);
    beside("residual", *residual, x);
    TORCH_CHECK_VALUE(residual->sizes().equals(shape), "linear: residual has shape ", residual->sizes(), ", the result ", at::IntArrayRef(shape));
    TORCH_CHECK_VALUE(out == kNoType || out == type_of(*residual), "linear: the result has the residual's type");
    out = type_of(*residual);
  }
  if (out == kNoType) out = type;
  TORCH_CHECK_VALUE(out == 0 || out == type, "linear: the result is float32 or of x's type");
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias) || wants(residual))) return Linear::apply(x, weight, bias, residual, act, (int64_t)out);
  const OptTensor r = residual ? OptTensor(adjacent(matrix(*residual, n))) : residual;
  return linear_forward(for_rows(matrix(x, k), m), for_rows(weight, m), contiguous(bias), r, act, out, shape, nullptr);
}

// ---- log probabilities ----------------------------------------------------------------------------------------------
struct Rows {
  Tensor logprobs, entropy, top_tokens, top_logprobs, stats;
};
Rows logprobs_forward(const Tensor& logits, const Tensor& tokens, at::IntArrayRef shape, int64_t top, int64_t ignore, bool keep) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t rows = logits.size(0);
  const at::TensorOptions f = logits.options().dtype(at::kFloat);
  Rows r;
  r.logprobs = at::empty(shape, f);
  r.entropy = at::empty(shape, f);
  if (top) {
    at::DimVector with_top(shape);
    with_top.push_back(top);
    r.top_tokens = at::empty(with_top, logits.options().dtype(at::kLong));
    r.top_logprobs = at::empty(with_top, f);
  }
  if (keep) r.stats = at::empty({rows, 3}, f);
  check(api.token_logprobs(logits.data_ptr(), type_of(logits), rows, logits.size(1), any_stride(logits), static_cast<int64_t*>(tokens.data_ptr()), ignore, (int)top,
                           static_cast<float*>(r.logprobs.data_ptr()), static_cast<float*>(r.entropy.data_ptr()), static_cast<int64_t*>(ptr(r.top_tokens)),
                           static_cast<float*>(ptr(r.top_logprobs)), static_cast<float*>(ptr(r.stats)), stream_of(logits)),
        "token_logprobs");
  return r;
}
// rows that do not overlap, as those of expand() do
Tensor logit_rows(const Tensor& logits) {
  const int64_t vocab = logits.size(-1);
  return adjacent(matrix(logits.stride(-1) != 1 && vocab > 1 ? logits.contiguous() : logits, vocab));
}

struct TokenLogprobs : Function<TokenLogprobs> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& given, const Tensor& given_tokens, int64_t top, int64_t ignore) {
    const Tensor logits = logit_rows(given), tokens = given_tokens.contiguous();
    Rows r = logprobs_forward(logits, tokens, given_tokens.sizes(), top, ignore, true);
    ctx->save_for_backward({logits, tokens, r.stats});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["shape"] = given.sizes().vec();
    ctx->set_materialize_grads(false);
    if (!top) return {r.logprobs, r.entropy};
    ctx->mark_non_differentiable({r.top_tokens, r.top_logprobs});
    return {r.logprobs, r.entropy, r.top_tokens, r.top_logprobs};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2];
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    not_recorded();
    for (int i = 0; i < 2; ++i)
      if (grads[i].defined()) ordinary("gradient", grads[i]);
    const c10::cuda::CUDAGuard guard(logits.device());
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const int64_t rows = logits.size(0), vocab = logits.size(1), stride = any_stride(logits);
    const Tensor a = grads[0].defined() ? held(grads[0]).contiguous() : Tensor(), b = grads[1].defined() ? held(grads[1]).contiguous() : Tensor();
    // rows that begin at the same places of 16-byte groups as the logits', so that both move in whole groups; a product whose
    // rows were padded to such groups gets its gradient padded alike
    const int64_t at = vocab + (stride - vocab) % 8;
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Tensor d = empty_apart(rows, vocab, at, logits.options(), shape);
    check(api.token_logprobs_backward(logits.data_ptr(), type_of(logits), rows, vocab, stride, static_cast<int64_t*>(tokens.data_ptr()),
                                      ctx->saved_data["ignore"].toInt(), static_cast<float*>(stats.data_ptr()), static_cast<float*>(ptr(a)),
                                      static_cast<float*>(ptr(b)), d.data_ptr(), at, stream_of(logits)),
          "token_logprobs backward");
    return once({d, Tensor(), Tensor(), Tensor()}, graph);
  }
};

std::tuple<Tensor, Tensor, OptTensor, OptTensor> token_logprobs(const Tensor& logits_, const Tensor& tokens_, int64_t top, int64_t ignore) {
  not_recorded();
  ordinary("logits", logits_);
  ordinary("tokens", tokens_);
  const Tensor logits = held(logits_), tokens = held(tokens_);
  floating("logits", logits);
  TORCH_CHECK_VALUE(logits.dim() > 0 && logits.size(-1) > 0, "token_logprobs: logits have no vocabulary");
  const int64_t vocab = logits.size(-1), rows = logits.numel() / vocab;
  TORCH_CHECK_VALUE(vocab <= 0x7fffffff && rows <= 0x7fffffff, "token_logprobs: a vocabulary and rows of at most 2^31 - 1");
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong && tokens.device() == logits.device(), "token_logprobs: expected int64 tokens on the device of the logits");
  TORCH_CHECK_VALUE(tokens.sizes().equals(logits.sizes().slice(0, logits.dim() - 1)), "token_logprobs: tokens of shape ", tokens.sizes(), " for logits of shape ", logits.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= std::min<int64_t>(64, vocab), "token_logprobs: top is from 0 to ", std::min<int64_t>(64, vocab));
  if (at::GradMode::is_enabled() && wants(logits)) {
    const tensor_list r = TokenLogprobs::apply(logits, tokens, top, ignore);
    return {r[0], r[1], top ? OptTensor(r[2]) : std::nullopt, top ? OptTensor(r[3]) : std::nullopt};
  }
  const Rows r = logprobs_forward(logit_rows(logits), tokens.contiguous(), tokens.sizes(), top, ignore, false);
  return {r.logprobs, r.entropy, top ? OptTensor(r.top_tokens) : std::nullopt, top ? OptTensor(r.top_logprobs) : std::nullopt};
}

// ---- orthogonalised updates -----------------------------------------------------------------------------------------
Tensor orthogonalize(const Tensor& update_, int64_t steps, double a, double b, double c, double eps) {
  not_recorded();
  ordinary("update", update_);
  const Tensor update = held(update_);
  floating("update", update);
  TORCH_CHECK_VALUE(update.dim() >= 2 && update.size(-1) > 0 && update.size(-2) > 0, "orthogonalize: expected matrices, got shape ", update.sizes());
  TORCH_CHECK_VALUE(steps >= 1 && steps <= 100 && eps >= 0, "orthogonalize: 1 to 100 steps, eps not negative");
  const at::NoGradGuard no_grad;
  const int64_t height = update.size(-2), width = update.size(-1), batch = update.numel() / (height * width);
  TORCH_CHECK_VALUE(batch <= 65535 && std::max(height, width) < (1 << 24), "orthogonalize: at most 65535 matrices with sides below 2^24");
  Tensor g = update.dim() == 3 ? update.detach() : update.detach().reshape({batch, height, width});
  if ((g.stride(2) != 1 && width > 1) || (height > 1 && g.stride(1) < width)) g = g.contiguous();
  const c10::cuda::CUDAGuard guard(g.device());
  Tensor out = at::empty(update.sizes(), update.options().dtype(at::kBFloat16));
  const size_t need = api.orthogonalize_bytes(batch, height, width);
  const Tensor scratch = scratch_of(need, g);
  const int status = api.orthogonalize(g.data_ptr(), type_of(g), batch, height, width, height > 1 ? g.stride(1) : width, batch > 1 ? g.stride(0) : 0, out.data_ptr(),
                                       (int)steps, (float)a, (float)b, (float)c, (float)eps, ptr(scratch), need, stream_of(g));
  TORCH_CHECK_VALUE(status != 4, "orthogonalize: coefficients (", a, ", ", b, ", ", c, ") may carry the iteration beyond the range of float16 in ", steps, " steps");
  check(status, "orthogonalize");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind_all);
  m.def("layer_norm", &layer_norm);
  m.def("linear", &linear);
  m.def("token_logprobs", &token_logprobs);
  m.def("orthogonalize", &orthogonalize);
}
