// torch.ops.vlak registration of the rotation ops (csrc/rotary.cu): schemas of
// this library's own, CUDA implementations that validate, allocate and call
// the C ABI on the current stream, and their autograd formulas.

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <vector>

#include "vlak_b200.h"
#include "vlak_torch.h"

namespace {

using at::Tensor;
using vlak_torch::check_status;
using vlak_torch::dtype_code;
using vlak_torch::new_empty;
using vlak_torch::raise_pending_device_error;
using vlak_torch::refuse_tangents;
using OptTensor = std::optional<Tensor>;
using Tensors = std::vector<Tensor>;

bool present(const OptTensor& t) { return t.has_value() && t->defined(); }

// The kernels read any (b, m, h) strides but want the entries contiguous.
Tensor unit_last(const Tensor& t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); }

// Checks shared by the ops; fills the token grid, positions and frequencies.
// `keep` holds the tensors whose memory the arguments point into.
vlak_rotary_args rotary_args(const Tensor& q, const OptTensor& k, const Tensor& positions,
                             const Tensor& inv_freq, bool interleaved, double amplitude,
                             const char* op, Tensors& keep) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4, op, ": expected 4D CUDA heads (B, M, heads, head_dim)");
  const int dt = dtype_code(q.scalar_type());
  TORCH_CHECK(dt == VLAK_F32 || dt == VLAK_F16 || dt == VLAK_BF16, op, ": unsupported dtype ",
              q.scalar_type());
  const int64_t B = q.size(0), M = q.size(1), D = q.size(3);
  if (present(k)) {
    TORCH_CHECK(k->is_cuda() && k->device() == q.device(), op, ": q and k must be on one CUDA device");
    TORCH_CHECK(k->scalar_type() == q.scalar_type(), op, ": q and k must have one dtype");
    TORCH_CHECK(k->dim() == 4 && k->size(0) == B && k->size(1) == M && k->size(3) == D, op,
                ": k must be (B, M, heads, head_dim) with the B, M and head_dim of q");
  }
  TORCH_CHECK(positions.device() == q.device() && inv_freq.device() == q.device(), op,
              ": positions and inv_freq must be on the device of q");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, op,
              ": positions must be int32 or int64");
  TORCH_CHECK((positions.dim() == 1 && positions.size(0) == M) ||
                  (positions.dim() == 2 && (positions.size(0) == B || positions.size(0) == 1) &&
                   positions.size(1) == M),
              op, ": positions must be (B, M), (1, M) or (M,)");
  TORCH_CHECK(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1, op,
              ": inv_freq must be a float64 vector");
  keep.push_back(inv_freq.contiguous());
  vlak_rotary_args a{};
  a.positions = positions.data_ptr();
  a.pos_dtype = positions.scalar_type() == at::kLong ? VLAK_I64 : VLAK_I32;
  a.pos_stride[0] = positions.dim() == 1 || positions.size(0) != B ? 0 : positions.stride(0);
  a.pos_stride[1] = positions.stride(-1);
  a.inv_freq = static_cast<const double*>(keep[0].data_ptr());
  a.B = B;
  a.M = M;
  a.D = D;
  a.rotary_dim = 2 * inv_freq.size(0);
  a.amplitude = amplitude;
  a.interleaved = interleaved;
  a.dtype = dt;
  a.weight_dtype = dt;
  a.n_tensors = present(k) ? 2 : 1;
  return a;
}

void set_heads(vlak_rotary_tensor& t, const Tensor& x) {
  t.x = x.data_ptr();
  t.H = x.size(2);
  for (int d = 0; d < 3; ++d) t.x_stride[d] = x.stride(d);
}

void set_weights(vlak_rotary_args& a, const Tensor& q, const OptTensor& k, const Tensor& q_weight,
                 const OptTensor& k_weight, const char* op, Tensors& keep) {
  TORCH_CHECK(present(k) == present(k_weight), op, ": k and k_weight come together");
  for (int i = 0; i < a.n_tensors; ++i) {
    const Tensor& w = i == 0 ? q_weight : *k_weight;
    TORCH_CHECK(w.device() == q.device(), op, ": weights must be on the device of q");
    TORCH_CHECK(w.dim() == 1 && w.size(0) == a.D, op, ": weights must be (head_dim,)");
    TORCH_CHECK(w.scalar_type() == q_weight.scalar_type() &&
                    (w.scalar_type() == at::kFloat || w.scalar_type() == q.scalar_type()),
                op, ": weights must both be float32 or of the dtype of q");
    keep.push_back(w.contiguous());
    a.t[i].weight = keep.back().data_ptr();
  }
  a.weight_dtype = dtype_code(q_weight.scalar_type());
}

Tensor empty_heads(const Tensor& x) { return new_empty(x, x.sizes(), x.scalar_type()); }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

Tensors rotary(const Tensor& q, const OptTensor& k, const Tensor& positions,
               const Tensor& inv_freq, bool interleaved, double amplitude, bool inverse) {
  const char* op = "vlak::rotary";
  raise_pending_device_error(op);
  Tensors keep, out;
  vlak_rotary_args a = rotary_args(q, k, positions, inv_freq, interleaved, amplitude, op, keep);
  a.inverse = inverse;
  c10::cuda::CUDAGuard guard(q.device());
  for (int i = 0; i < a.n_tensors; ++i) {
    keep.push_back(unit_last(i == 0 ? q : *k));
    set_heads(a.t[i], keep.back());
    out.push_back(empty_heads(keep.back()));
    a.t[i].y = out.back().data_ptr();
  }
  check_status(vlak_rotary(&a, stream()), op);
  return out;
}

Tensors qk_norm_rotary(const Tensor& q, const OptTensor& k, const Tensor& q_weight,
                       const OptTensor& k_weight, const Tensor& positions,
                       const Tensor& inv_freq, double eps, bool interleaved, double amplitude) {
  const char* op = "vlak::qk_norm_rotary";
  raise_pending_device_error(op);
  Tensors keep, out;
  vlak_rotary_args a = rotary_args(q, k, positions, inv_freq, interleaved, amplitude, op, keep);
  a.eps = eps;
  c10::cuda::CUDAGuard guard(q.device());
  set_weights(a, q, k, q_weight, k_weight, op, keep);
  for (int i = 0; i < a.n_tensors; ++i) {
    keep.push_back(unit_last(i == 0 ? q : *k));
    set_heads(a.t[i], keep.back());
    out.push_back(empty_heads(keep.back()));
    a.t[i].y = out.back().data_ptr();
  }
  check_status(vlak_qk_norm_rotary_fwd(&a, stream()), op);
  return out;
}

// [dq, (dk,) dq_weight, (dk_weight)]
Tensors qk_norm_rotary_bwd(const Tensor& grad_q, const OptTensor& grad_k, const Tensor& q,
                           const OptTensor& k, const Tensor& q_weight, const OptTensor& k_weight,
                           const Tensor& positions, const Tensor& inv_freq, double eps,
                           bool interleaved, double amplitude) {
  const char* op = "vlak::qk_norm_rotary_bwd";
  raise_pending_device_error(op);
  Tensors keep, out, dw;
  vlak_rotary_args a = rotary_args(q, k, positions, inv_freq, interleaved, amplitude, op, keep);
  a.eps = eps;
  TORCH_CHECK(present(k) == present(grad_k), op, ": k and grad_k come together");
  c10::cuda::CUDAGuard guard(q.device());
  set_weights(a, q, k, q_weight, k_weight, op, keep);
  for (int i = 0; i < a.n_tensors; ++i) {
    const Tensor& x = i == 0 ? q : *k;
    const Tensor& g = i == 0 ? grad_q : *grad_k;
    TORCH_CHECK(g.device() == q.device() && g.scalar_type() == q.scalar_type() &&
                    g.sizes() == x.sizes(),
                op, ": a gradient must have the device, dtype and shape of its heads");
    keep.push_back(unit_last(x));
    set_heads(a.t[i], keep.back());
    keep.push_back(unit_last(g));
    a.t[i].grad = keep.back().data_ptr();
    for (int d = 0; d < 3; ++d) a.t[i].grad_stride[d] = keep.back().stride(d);
    out.push_back(empty_heads(x));
    a.t[i].y = out.back().data_ptr();
    dw.push_back(new_empty(q, {a.D}, q_weight.scalar_type()));
    a.t[i].grad_weight = dw.back().data_ptr();
  }
  int64_t bytes = 0;
  check_status(vlak_qk_norm_rotary_workspace_size(&a, &bytes), op);
  // from the caching allocator on the current stream: reused only by work
  // queued behind this call there, and a captured graph's own while it lives
  const Tensor ws = new_empty(q, {bytes}, at::kByte);
  check_status(vlak_qk_norm_rotary_bwd(&a, ws.data_ptr(), bytes, stream()), op);
  out.insert(out.end(), dw.begin(), dw.end());
  return out;
}

// ---------------------------------------------------------------------------
// autograd

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

Tensors call_rotary(const Tensor& q, const OptTensor& k, const Tensor& positions,
                    const Tensor& inv_freq, bool interleaved, double amplitude, bool inverse) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vlak::rotary", "")
                       .typed<decltype(rotary)>();
  return op.call(q, k, positions, inv_freq, interleaved, amplitude, inverse);
}
Tensors call_norm(const Tensor& q, const OptTensor& k, const Tensor& qw, const OptTensor& kw,
                  const Tensor& positions, const Tensor& inv_freq, double eps, bool interleaved,
                  double amplitude) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vlak::qk_norm_rotary", "")
                       .typed<decltype(qk_norm_rotary)>();
  return op.call(q, k, qw, kw, positions, inv_freq, eps, interleaved, amplitude);
}
Tensors call_norm_bwd(const Tensor& gq, const OptTensor& gk, const Tensor& q, const OptTensor& k,
                      const Tensor& qw, const OptTensor& kw, const Tensor& positions,
                      const Tensor& inv_freq, double eps, bool interleaved, double amplitude) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vlak::qk_norm_rotary_bwd", "")
                       .typed<decltype(qk_norm_rotary_bwd)>();
  return op.call(gq, gk, q, k, qw, kw, positions, inv_freq, eps, interleaved, amplitude);
}

bool wants_grad(const OptTensor& t) { return present(t) && t->requires_grad(); }
Tensor or_none(const OptTensor& t) { return t.value_or(Tensor()); }
// There is no gradient of the frequencies: where one would be recorded, say so.
void refuse_frequency_grad(const Tensor& inv_freq, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled() || !inv_freq.requires_grad(), op,
                              " has no gradient of inv_freq; pass inv_freq.detach()");
}

// Gradient of the rotation: the same op with the turn reversed, on the
// gradients that arrived (one of the outputs may be unused). It goes through
// the dispatcher, so it can itself be differentiated.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Variable& q,
                               const std::optional<Variable>& k, const Variable& positions,
                               const Variable& inv_freq, bool interleaved, double amplitude,
                               bool inverse) {
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["inverse"] = inverse;
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_rotary(q, k, positions, inv_freq, interleaved, amplitude, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    const double amplitude = ctx->saved_data["amplitude"].toDouble();
    const bool inverse = !ctx->saved_data["inverse"].toBool();
    const bool with_q = g[0].defined() && ctx->needs_input_grad(0);
    const bool with_k = g.size() > 1 && g[1].defined() && ctx->needs_input_grad(1);
    variable_list out(7);
    if (!with_q && !with_k) return out;
    const Tensors d = call_rotary(with_q ? g[0] : g[1],
                                  with_q && with_k ? OptTensor(g[1]) : std::nullopt, saved[0],
                                  saved[1], interleaved, amplitude, inverse);
    if (with_q) out[0] = d[0];
    if (with_k) out[1] = d.back();
    return out;
  }
};

Tensors rotary_autograd(const Tensor& q, const OptTensor& k, const Tensor& positions,
                        const Tensor& inv_freq, bool interleaved, double amplitude,
                        bool inverse) {
  refuse_tangents({q, or_none(k), inv_freq}, "vlak::rotary");
  refuse_frequency_grad(inv_freq, "vlak::rotary");
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k)))
    return RotaryFunction::apply(q, k, positions, inv_freq, interleaved, amplitude, inverse);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_rotary(q, k, positions, inv_freq, interleaved, amplitude, inverse);
}

struct NormRotaryFunction : torch::autograd::Function<NormRotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Variable& q,
                               const std::optional<Variable>& k, const Variable& qw,
                               const std::optional<Variable>& kw, const Variable& positions,
                               const Variable& inv_freq, double eps, bool interleaved,
                               double amplitude) {
    ctx->save_for_backward({q, k.value_or(Variable()), qw, kw.value_or(Variable()), positions,
                            inv_freq});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView below;
    return call_norm(q, k, qw, kw, positions, inv_freq, eps, interleaved, amplitude);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    const double amplitude = ctx->saved_data["amplitude"].toDouble();
    variable_list out(9);
    const bool with_q = g[0].defined();
    const bool with_k = g.size() > 1 && g[1].defined();
    if (!with_q && !with_k) return out;
    const int f = with_q ? 0 : 1;  // the first (or only) tensor of the call
    const bool both = with_q && with_k;
    const Tensors d = call_norm_bwd(g[f], both ? OptTensor(g[1]) : std::nullopt, s[f],
                                    both ? OptTensor(s[1]) : std::nullopt, s[2 + f],
                                    both ? OptTensor(s[3]) : std::nullopt, s[4], s[5], eps,
                                    interleaved, amplitude);
    if (with_q) {
      out[0] = d[0];
      out[2] = both ? d[2] : d[1];
    }
    if (with_k) {
      out[1] = both ? d[1] : d[0];
      out[3] = d.back();
    }
    return out;
  }
};

Tensors qk_norm_rotary_autograd(const Tensor& q, const OptTensor& k, const Tensor& qw,
                                const OptTensor& kw, const Tensor& positions,
                                const Tensor& inv_freq, double eps, bool interleaved,
                                double amplitude) {
  refuse_tangents({q, or_none(k), qw, or_none(kw), inv_freq}, "vlak::qk_norm_rotary");
  refuse_frequency_grad(inv_freq, "vlak::qk_norm_rotary");
  if (at::GradMode::is_enabled() &&
      (wants_grad(q) || wants_grad(k) || wants_grad(qw) || wants_grad(kw)))
    return NormRotaryFunction::apply(q, k, qw, kw, positions, inv_freq, eps, interleaved, amplitude);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_norm(q, k, qw, kw, positions, inv_freq, eps, interleaved, amplitude);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(vlak, m) {
  m.def(
      "rotary(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, bool interleaved=False, "
      "float amplitude=1., bool inverse=False) -> Tensor[]");
  m.def(
      "qk_norm_rotary(Tensor q, Tensor? k, Tensor q_weight, Tensor? k_weight, Tensor positions, "
      "Tensor inv_freq, float eps=1e-6, bool interleaved=False, float amplitude=1.) -> Tensor[]");
  m.def(
      "qk_norm_rotary_bwd(Tensor grad_q, Tensor? grad_k, Tensor q, Tensor? k, Tensor q_weight, "
      "Tensor? k_weight, Tensor positions, Tensor inv_freq, float eps=1e-6, "
      "bool interleaved=False, float amplitude=1.) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(vlak, CUDA, m) {
  m.impl("rotary", &rotary);
  m.impl("qk_norm_rotary", &qk_norm_rotary);
  m.impl("qk_norm_rotary_bwd", &qk_norm_rotary_bwd);
}

TORCH_LIBRARY_IMPL(vlak, Autograd, m) {
  m.impl("rotary", &rotary_autograd);
  m.impl("qk_norm_rotary", &qk_norm_rotary_autograd);
  m.impl("qk_norm_rotary_bwd", torch::autograd::autogradNotImplementedFallback());
}
