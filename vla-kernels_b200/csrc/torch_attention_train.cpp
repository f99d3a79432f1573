// torch.ops.vlak registration of GQA attention for training: the forward op
// that also returns the rows' log-sums, the backward op (csrc/attention_bwd.cu)
// and the differentiable op that ties them together.

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <vector>

#include "vlak_b200.h"
#include "vlak_torch.h"

namespace {

using at::Tensor;
using vlak_torch::check_status;
using vlak_torch::new_empty;
using vlak_torch::raise_pending_device_error;
using OptTensor = std::optional<Tensor>;

bool present(const OptTensor& t) { return t.has_value() && t->defined(); }

// Expanded tensors (a stride of 0 over more than one entry) are written out:
// a tensor map steps over memory.
Tensor stepped(const Tensor& t) {
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.stride(d) == 0 && t.size(d) > 1) return t.contiguous();
  return t;
}

// The masks of a call: checked, and laid out as the kernels read them.
struct Masks {
  Tensor lengths, mask;
};
Masks check_masks(const vlak_attn_gqa_args& a, const Tensor& q, const OptTensor& lengths,
                  const OptTensor& attn_mask, int64_t prefix_len, int64_t dead_start,
                  int64_t dead_end, const char* op) {
  Masks m;
  TORCH_CHECK(!(present(lengths) && present(attn_mask)), op, ": lengths or attn_mask, not both");
  if (present(lengths) || present(attn_mask))
    TORCH_CHECK(prefix_len < 0 && dead_start == 0 && dead_end == 0, op,
                ": the analytic mask goes with neither lengths nor attn_mask");
  if (present(lengths)) {
    TORCH_CHECK(lengths->device() == q.device(), op, ": lengths must be on the device of q");
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == a.B, op, ": lengths must be (B,)");
    TORCH_CHECK(lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong, op,
                ": lengths must be int32 or int64");
    m.lengths = lengths->contiguous();
  }
  if (present(attn_mask)) {
    TORCH_CHECK(attn_mask->device() == q.device(), op, ": attn_mask must be on the device of q");
    TORCH_CHECK(attn_mask->scalar_type() == at::kBool, op, ": attn_mask must be bool");
    TORCH_CHECK(attn_mask->dim() == 3 && attn_mask->size(0) == a.B && attn_mask->size(1) == a.M &&
                    attn_mask->size(2) == a.N,
                op, ": attn_mask must be (B, M, N)");
    m.mask = attn_mask->stride(2) == 1 || a.N <= 1 ? *attn_mask : attn_mask->contiguous();
  }
  return m;
}

vlak_attn_train_args train_args(const vlak_attn_gqa_args& a, const Masks& m) {
  vlak_attn_train_args t{};
  t.attn = a;
  if (m.lengths.defined()) {
    t.lengths = m.lengths.data_ptr();
    t.lengths_dtype = m.lengths.scalar_type() == at::kLong ? VLAK_I64 : VLAK_I32;
  }
  if (m.mask.defined()) {
    t.mask = m.mask.data_ptr();
    t.mask_stride_b = m.mask.stride(0);
    t.mask_stride_m = m.mask.stride(1);
  }
  return t;
}

void set_o(vlak_attn_gqa_args& a, const Tensor& o) {
  a.o = o.data_ptr();
  for (int d = 0; d < 3; ++d) a.o_stride[d] = o.stride(d);
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// o, its rows' log-sums, and (for a backward pass) its low bytes
std::tuple<Tensor, Tensor, Tensor> forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                           double scale, int64_t prefix_len, int64_t dead_start,
                                           int64_t dead_end, const OptTensor& lengths,
                                           const OptTensor& attn_mask, bool for_backward) {
  const char* op = "fused_attention_gqa_train";
  raise_pending_device_error(op);
  const Tensor q = stepped(q_in), k = stepped(k_in), v = stepped(v_in);
  vlak_attn_gqa_args a = vlak_torch::gqa_args(q, k, v, scale, prefix_len, dead_start, dead_end, op);
  const Masks m = check_masks(a, q, lengths, attn_mask, prefix_len, dead_start, dead_end, op);
  c10::cuda::CUDAGuard guard(q.device());
  check_status(vlak_attn_gqa_check(&a, nullptr, nullptr), op);
  Tensor o = new_empty(q, {a.B, a.M, a.H, 64}, q.scalar_type());
  Tensor lse = new_empty(q, {a.B, a.M, a.H}, at::kFloat);
  Tensor o_low;
  set_o(a, o);
  vlak_attn_train_args t = train_args(a, m);
  t.lse = lse.data_ptr<float>();
  if (for_backward) {
    o_low = new_empty(q, {a.B, a.M, a.H, 64}, at::kChar);
    t.o_low = o_low.data_ptr();
  }
  // workspaces: from the caching allocator on the current stream, so reused only
  // by work queued behind this call there, and a captured graph's own while it lives
  int64_t bytes = 0;
  check_status(vlak_attn_gqa_train_workspace_size(&t, &bytes), op);
  Tensor ws;
  if (bytes > 0) ws = new_empty(q, {bytes}, at::kByte);
  check_status(vlak_attn_gqa_train_fwd(&t, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream()), op);
  return {o, lse, o_low};
}

std::tuple<Tensor, Tensor, Tensor> fwd_lse(const Tensor& q, const Tensor& k, const Tensor& v,
                                           double scale, int64_t prefix_len, int64_t dead_start,
                                           int64_t dead_end, const OptTensor& lengths,
                                           const OptTensor& attn_mask) {
  return forward(q, k, v, scale, prefix_len, dead_start, dead_end, lengths, attn_mask, true);
}

// [dq, dk, dv], or [dq] without with_kv
std::vector<Tensor> bwd(const Tensor& grad_o_in, const Tensor& q_in, const Tensor& k_in,
                        const Tensor& v_in, const Tensor& o_in, const Tensor& lse,
                        const Tensor& o_low, double scale,
                        int64_t prefix_len, int64_t dead_start, int64_t dead_end,
                        const OptTensor& lengths, const OptTensor& attn_mask, bool with_kv) {
  const char* op = "fused_attention_gqa_bwd";
  raise_pending_device_error(op);
  const Tensor q = stepped(q_in), k = stepped(k_in), v = stepped(v_in);
  vlak_attn_gqa_args a = vlak_torch::gqa_args(q, k, v, scale, prefix_len, dead_start, dead_end, op);
  const Masks m = check_masks(a, q, lengths, attn_mask, prefix_len, dead_start, dead_end, op);
  for (const Tensor* t : {&grad_o_in, &o_in})
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kBFloat16 &&
                    t->sizes() == q.sizes(),
                op, ": grad_o and o must be bf16 on the device of q, of its shape");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.dim() == 3 &&
                  lse.size(0) == a.B && lse.size(1) == a.M && lse.size(2) == a.H &&
                  lse.is_contiguous(),
              op, ": lse must be the contiguous float32 (B, M, H) of the forward call");
  TORCH_CHECK(o_low.device() == q.device() && o_low.scalar_type() == at::kChar &&
                  o_low.sizes() == q.sizes() && o_low.is_contiguous(),
              op, ": o_low must be the contiguous int8 tensor of the forward call");
  c10::cuda::CUDAGuard guard(q.device());
  // a gradient arrives in whatever layout its consumer left it in
  auto tma_ready = [](const Tensor& t) {
    bool ready = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d)
      ready = ready && t.stride(d) % 8 == 0 && (t.stride(d) != 0 || t.size(d) <= 1);
    return ready ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  const Tensor grad_o = tma_ready(grad_o_in), o = tma_ready(o_in);
  set_o(a, o);
  check_status(vlak_attn_gqa_check(&a, nullptr, nullptr), op);
  std::vector<Tensor> out{new_empty(q, {a.B, a.M, a.H, 64}, q.scalar_type())};
  vlak_attn_train_args t = train_args(a, m);
  t.lse = lse.data_ptr<float>();
  t.o_low = o_low.data_ptr();
  t.grad_o = grad_o.data_ptr();
  for (int d = 0; d < 3; ++d) t.grad_o_stride[d] = grad_o.stride(d);
  t.dq = out[0].data_ptr();
  if (with_kv) {
    out.push_back(new_empty(q, {a.B, a.N, a.Hkv, 64}, q.scalar_type()));
    out.push_back(new_empty(q, {a.B, a.N, a.Hkv, 64}, q.scalar_type()));
    t.dk = out[1].data_ptr();
    t.dv = out[2].data_ptr();
  }
  int64_t bytes = 0;
  check_status(vlak_attn_gqa_bwd_workspace_size(&t, &bytes), op);
  const Tensor ws = new_empty(q, {bytes}, at::kByte);
  check_status(vlak_attn_gqa_bwd(&t, ws.data_ptr(), bytes, stream()), op);
  return out;
}

Tensor train(const Tensor& q, const Tensor& k, const Tensor& v, double scale, int64_t prefix_len,
             int64_t dead_start, int64_t dead_end, const OptTensor& lengths,
             const OptTensor& attn_mask) {
  return std::get<0>(
      forward(q, k, v, scale, prefix_len, dead_start, dead_end, lengths, attn_mask, false));
}

// ---------------------------------------------------------------------------
// autograd

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

template <typename F>
auto typed_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

struct TrainFunction : torch::autograd::Function<TrainFunction> {
  static Variable forward(AutogradContext* ctx, const Variable& q, const Variable& k,
                          const Variable& v, double scale, int64_t prefix_len, int64_t dead_start,
                          int64_t dead_end, const std::optional<Variable>& lengths,
                          const std::optional<Variable>& attn_mask) {
    static auto op = typed_op<decltype(fwd_lse)>("vlak::fused_attention_gqa_fwd_lse");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse, o_low] = op.call(q, k, v, scale, prefix_len, dead_start, dead_end, lengths, attn_mask);
    ctx->save_for_backward({q, k, v, o, lse, o_low, lengths.value_or(Variable()),
                            attn_mask.value_or(Variable())});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["prefix_len"] = prefix_len;
    ctx->saved_data["dead_start"] = dead_start;
    ctx->saved_data["dead_end"] = dead_end;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static auto op = typed_op<decltype(bwd)>("vlak::fused_attention_gqa_bwd");
    const auto s = ctx->get_saved_variables();
    auto optional = [](const Variable& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    const bool with_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const std::vector<Tensor> d =
        op.call(g[0], s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble(),
                ctx->saved_data["prefix_len"].toInt(), ctx->saved_data["dead_start"].toInt(),
                ctx->saved_data["dead_end"].toInt(), optional(s[6]), optional(s[7]), with_kv);
    variable_list out(9);
    out[0] = d[0];
    if (with_kv) {
      out[1] = d[1];
      out[2] = d[2];
    }
    return out;
  }
};

Tensor train_autograd(const Tensor& q, const Tensor& k, const Tensor& v, double scale,
                      int64_t prefix_len, int64_t dead_start, int64_t dead_end,
                      const OptTensor& lengths, const OptTensor& attn_mask) {
  vlak_torch::refuse_tangents({q, k, v}, "fused_attention_gqa_train");
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return TrainFunction::apply(q, k, v, scale, prefix_len, dead_start, dead_end, lengths, attn_mask);
  static auto op = typed_op<decltype(train)>("vlak::fused_attention_gqa_train");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, scale, prefix_len, dead_start, dead_end, lengths, attn_mask);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(vlak, m) {
  m.def(
      "fused_attention_gqa_train(Tensor q, Tensor k, Tensor v, float scale=-1., "
      "int prefix_len=-1, int dead_start=0, int dead_end=0, Tensor? lengths=None, "
      "Tensor? attn_mask=None) -> Tensor");
  m.def(
      "fused_attention_gqa_fwd_lse(Tensor q, Tensor k, Tensor v, float scale=-1., "
      "int prefix_len=-1, int dead_start=0, int dead_end=0, Tensor? lengths=None, "
      "Tensor? attn_mask=None) -> (Tensor, Tensor, Tensor)");
  m.def(
      "fused_attention_gqa_bwd(Tensor grad_o, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, "
      "Tensor o_low, "
      "float scale=-1., int prefix_len=-1, int dead_start=0, int dead_end=0, "
      "Tensor? lengths=None, Tensor? attn_mask=None, bool with_kv=True) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(vlak, CUDA, m) {
  m.impl("fused_attention_gqa_train", &train);
  m.impl("fused_attention_gqa_fwd_lse", &fwd_lse);
  m.impl("fused_attention_gqa_bwd", &bwd);
}

TORCH_LIBRARY_IMPL(vlak, Autograd, m) {
  m.impl("fused_attention_gqa_train", &train_autograd);
  m.impl("fused_attention_gqa_fwd_lse", torch::autograd::autogradNotImplementedFallback());
  m.impl("fused_attention_gqa_bwd", torch::autograd::autogradNotImplementedFallback());
}
