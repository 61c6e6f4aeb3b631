/*
 * vsloss_vocab_torch.h -- header-only libtorch (C++) binding of the losses over a set of classes (vsloss.h):
 * vsl::top_logits(), vsl::topk_distillation_loss(), vsl::linear_cross_entropy().  torch::Tensor in, torch::Tensor out,
 * differentiable once (backwards only), stream-ordered on the current HIP stream of the tensors' device, no host synchronisation.  The
 * Python package's vocab_losses module calls these functions: a loss of a few rows takes some ten microseconds on the
 * device, and an autograd node that runs without the interpreter is half of what such a call costs the host.
 *
 * Malformed arguments throw c10::ValueError, errors of the library std::runtime_error.
 */
#ifndef VSLOSS_VOCAB_TORCH_H
#define VSLOSS_VOCAB_TORCH_H

#include <tuple>

#include "vsloss_torch.h"

namespace vsl {
namespace vocab_detail {

inline int type_of(const torch::Tensor& t) {
  return t.scalar_type() == torch::kFloat32 ? VSL_TYPE_F32 : t.scalar_type() == torch::kBFloat16 ? VSL_TYPE_BF16 : VSL_TYPE_F16;
}

/* float32, bfloat16 and float16 as they are, float64 as float32 */
inline torch::Tensor floating(const torch::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.defined() && t.is_cuda(), name, " must be a GPU tensor (there is no CPU implementation)");
  const auto type = t.scalar_type();
  if (type == torch::kFloat32 || type == torch::kBFloat16 || type == torch::kFloat16) return t;
  TORCH_CHECK_VALUE(type == torch::kFloat64, name, " must be float32, bfloat16 or float16, not ", type);
  return t.to(torch::kFloat32);
}

inline void on(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", not on ", like.device());
}

/* [..., n] as [rows, n] whose rows may be strided and whose elements are not */
inline torch::Tensor matrix(torch::Tensor t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, " needs a last dimension of at least 1");
  if (t.dim() != 2) {
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    t = t.reshape({rows, t.size(-1)});
  }
  return t.stride(1) != 1 || t.stride(0) < t.size(1) ? t.contiguous() : t;
}
inline int64_t row_stride(const torch::Tensor& t) { return std::max(t.stride(0), t.size(1)); }

/* a float32 vector with one entry per row, or an undefined tensor */
inline torch::Tensor per_row(const std::optional<torch::Tensor>& t, const char* name, torch::IntArrayRef shape,
                             const torch::Tensor& like) {
  if (!t || !t->defined()) return {};
  on(*t, name, like);
  TORCH_CHECK_VALUE(t->sizes() == shape, name, " must have the shape of the rows, ", shape, ", not ", t->sizes());
  return t->detach().to(torch::kFloat32).reshape({-1}).contiguous();
}

inline double temperature_of(double value) {
  const float t = (float)value;   /* as the library holds it: float32's 1e-4 is a little below the double one */
  TORCH_CHECK_VALUE(t >= 1e-4f && t <= 1e4f, "temperature must lie in 1e-4..1e4, not ", value);
  return value;
}

inline int reduction_of(const std::string& name) {
  if (name == "mean") return VSL_REDUCE_MEAN;
  if (name == "sum") return VSL_REDUCE_SUM;
  TORCH_CHECK_VALUE(name == "none", "reduction must be 'none', 'sum' or 'mean', not '", name, "'");
  return VSL_REDUCE_NONE;
}

/* Whether a call needs an autograd node.  A tangent of torch's forward mode would be lost without a word: it is refused. */
inline bool differentiable(std::initializer_list<const torch::Tensor*> tensors) {
  for (const torch::Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      throw std::runtime_error("libvsloss: the losses over a set of classes have no forward-mode derivative");
  if (!torch::GradMode::is_enabled()) return false;
  for (const torch::Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

/* autograd's functions take a tensor that is not there as no value, never as an undefined tensor */
inline std::optional<torch::Tensor> given(const torch::Tensor& t) { return t.defined() ? std::make_optional(t) : std::nullopt; }
inline torch::Tensor bytes(size_t n, const torch::Tensor& like) {
  return torch::empty({(int64_t)n}, like.options().dtype(torch::kUInt8));
}
inline torch::Tensor floats(torch::IntArrayRef shape, const torch::Tensor& like) {
  return torch::empty(shape, like.options().dtype(torch::kFloat32));
}
inline void* ptr(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* at(const torch::Tensor& t, size_t byte) { return (float*)((char*)t.data_ptr() + byte); }
inline void* stream_of(const torch::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

/* Stands over a gradient that was asked for with create_graph: there is no second derivative to give. */
class FirstDerivativeOnly : public torch::autograd::Function<FirstDerivativeOnly> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext*, const torch::Tensor& grad, const torch::Tensor&) { return grad; }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    throw std::runtime_error("libvsloss: the losses over a set of classes are differentiable once");
  }
};
/* `of`: every tensor that the gradient depends on and that may itself want one */
inline torch::Tensor once(torch::Tensor grad, std::initializer_list<const torch::Tensor*> of) {
  if (torch::GradMode::is_enabled() && grad.defined())
    for (const torch::Tensor* t : of)
      if (t->defined() && t->requires_grad()) return FirstDerivativeOnly::apply(grad, *t);
  return grad;
}

/* ---- distillation.  kept: statistics of the rows and, behind them, the divisor of the mean; the workspace and, where they
 * are summed, the row losses share that allocation: all are small beside the logits. */
struct DistillConfig {
  double temperature;
  int64_t reduction;
};

inline vsl_distill_desc distill_desc(const torch::Tensor& x, const torch::Tensor& values, const torch::Tensor& indices,
                                     const torch::Tensor& lse, const torch::Tensor& weights, const DistillConfig& c) {
  vsl_distill_desc d{};
  d.rows = x.size(0);
  d.vocab = x.size(1);
  d.stride = row_stride(x);
  d.k = (int32_t)values.size(1);
  d.type = type_of(x);
  d.value_type = type_of(values);
  d.index_bytes = (int32_t)indices.element_size();
  d.reduction = (int32_t)c.reduction;
  d.temperature = (float)c.temperature;
  d.logits = x.data_ptr();
  d.teacher_values = values.data_ptr();
  d.teacher_indices = indices.data_ptr();
  d.teacher_lse = (const float*)ptr(lse);
  d.weights = (const float*)ptr(weights);
  return d;
}

inline std::pair<torch::Tensor, torch::Tensor> distill_forward(const torch::Tensor& x, const torch::Tensor& values,
                                                               const torch::Tensor& indices, const torch::Tensor& lse,
                                                               const torch::Tensor& weights, const DistillConfig& c) {
  const c10::DeviceGuard guard(x.device());
  const vsl_distill_desc d = distill_desc(x, values, indices, lse, weights, c);
  const size_t rows = (size_t)d.rows, need = vsl_distill_workspace_bytes(&d);
  const size_t stats = 4 * VSL_DISTILL_STATS * rows, head = (stats + 4 + 255) / 256 * 256;
  const bool none = c.reduction == VSL_REDUCE_NONE;
  torch::Tensor kept = bytes(head + need + 4 * rows, x), out = none ? floats({d.rows}, x) : floats({}, x);
  float* loss = out.data_ptr<float>();
  check(vsl_distill_fwd(&d, none ? loss : at(kept, head + need), none ? nullptr : loss, none ? nullptr : at(kept, stats),
                        at(kept, 0), at(kept, head), need, stream_of(x)));
  return {out, kept};
}

class Distill : public torch::autograd::Function<Distill> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& values,
                               const torch::Tensor& indices, const std::optional<torch::Tensor>& lse,
                               const std::optional<torch::Tensor>& given, const DistillConfig& c) {
    const torch::Tensor weights = given.value_or(torch::Tensor());
    auto [out, kept] = distill_forward(x, values, indices, lse.value_or(torch::Tensor()), weights, c);
    ctx->save_for_backward({x, values, indices, weights, kept});
    ctx->saved_data["temperature"] = c.temperature;
    ctx->saved_data["reduction"] = c.reduction;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();   /* a hook may have moved them: the descriptor is made anew */
    const torch::Tensor &x = saved[0], &kept = saved[4];
    const c10::DeviceGuard guard(x.device());
    const vsl_distill_desc d = distill_desc(x, saved[1], saved[2], {}, saved[3],
                                            {ctx->saved_data["temperature"].toDouble(), ctx->saved_data["reduction"].toInt()});
    const torch::Tensor g = grads[0].contiguous();
    torch::Tensor grad = torch::empty(x.sizes(), x.options());
    check(vsl_distill_bwd(&d, at(kept, 0), at(kept, 4 * VSL_DISTILL_STATS * (size_t)d.rows), g.data_ptr<float>(), grad.data_ptr(),
                          d.vocab, stream_of(x)));
    return {once(grad, {&x, &grads[0]}), {}, {}, {}, {}, {}};
  }
};

/* ---- linear cross entropy.  kept: statistics of the rows and, behind them, the divisor of the mean. */
struct LinearCeConfig {
  int64_t ignore_index, reduction;
  double z_loss;
};

inline vsl_linear_ce_desc linear_ce_desc(const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& bias,
                                         const torch::Tensor& target, const LinearCeConfig& c) {
  vsl_linear_ce_desc d{};
  d.rows = hidden.size(0);
  d.vocab = weight.size(0);
  d.dim = hidden.size(1);
  d.hidden_stride = row_stride(hidden);
  d.weight_stride = row_stride(weight);
  d.ignore_index = c.ignore_index;
  d.type = type_of(hidden);
  d.reduction = (int32_t)c.reduction;
  d.z_loss = (float)c.z_loss;
  d.hidden = hidden.data_ptr();
  d.weight = weight.data_ptr();
  d.bias = ptr(bias);
  d.target = target.data_ptr<int64_t>();
  return d;
}

inline std::pair<torch::Tensor, torch::Tensor> linear_ce_forward(const torch::Tensor& hidden, const torch::Tensor& weight,
                                                                 const torch::Tensor& bias, const torch::Tensor& target,
                                                                 const LinearCeConfig& c) {
  const c10::DeviceGuard guard(hidden.device());
  const vsl_linear_ce_desc d = linear_ce_desc(hidden, weight, bias, target, c);
  const size_t need = vsl_linear_ce_fwd_workspace_bytes(&d);
  const bool none = c.reduction == VSL_REDUCE_NONE;
  torch::Tensor kept = floats({2 * d.rows + 1}, hidden), out = none ? floats({d.rows}, hidden) : floats({}, hidden);
  torch::Tensor work = bytes(need + (none ? 0 : 4 * (size_t)d.rows), hidden);   /* summed row losses are scratch behind it */
  float* loss = out.data_ptr<float>();
  check(vsl_linear_ce_fwd(&d, none ? loss : at(work, need), at(kept, 0), none ? nullptr : loss,
                          none ? nullptr : at(kept, 8 * (size_t)d.rows), work.data_ptr(), need, stream_of(hidden)));
  return {out, kept};
}

class LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& hidden, const torch::Tensor& weight,
                               const std::optional<torch::Tensor>& given, const torch::Tensor& target,
                               const LinearCeConfig& c) {
    const torch::Tensor bias = given.value_or(torch::Tensor());
    auto [out, kept] = linear_ce_forward(hidden, weight, bias, target, c);
    ctx->save_for_backward({hidden, weight, bias, target, kept});
    ctx->saved_data["ignore_index"] = c.ignore_index;
    ctx->saved_data["reduction"] = c.reduction;
    ctx->saved_data["z_loss"] = c.z_loss;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &hidden = saved[0], &weight = saved[1], &bias = saved[2], &kept = saved[4];
    const c10::DeviceGuard guard(hidden.device());
    const vsl_linear_ce_desc d = linear_ce_desc(hidden, weight, bias, saved[3],
                                                {ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["reduction"].toInt(),
                                                 ctx->saved_data["z_loss"].toDouble()});
    const torch::Tensor g = grads[0].contiguous();
    torch::Tensor out[3];
    uint32_t mask = 0;
    for (int i = 0; i < 3; ++i) {
      if (!saved[i].defined() || !ctx->needs_input_grad(i)) continue;
      out[i] = torch::empty(saved[i].sizes(), saved[i].options());
      mask |= 1u << i;
    }
    const size_t need = vsl_linear_ce_bwd_workspace_bytes(&d, mask);
    torch::Tensor work = bytes(need, hidden);
    check(vsl_linear_ce_bwd(&d, at(kept, 0), at(kept, 8 * (size_t)d.rows), g.data_ptr<float>(), ptr(out[0]), ptr(out[1]),
                            ptr(out[2]), work.data_ptr(), need, stream_of(hidden)));
    for (auto& t : out) t = once(t, {&hidden, &weight, &bias, &grads[0]});
    return {out[0], out[1], out[2], {}, {}};
  }
};

}  // namespace vocab_detail

/* The k largest logits of every row, larger first, their classes (int32) and the rows' log sum exp(logits / temperature). */
inline std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> top_logits(const torch::Tensor& logits, int64_t k,
                                                                          double temperature = 1.0) {
  using namespace vocab_detail;
  const torch::NoGradGuard no_grad;
  const torch::Tensor z = floating(logits, "logits"), x = matrix(z, "logits");
  const c10::DeviceGuard guard(x.device());
  TORCH_CHECK_VALUE(k >= 1 && k <= std::min<int64_t>(x.size(1), VSL_MAX_TOP), "k must lie in 1..min(classes, ", VSL_MAX_TOP,
                    "), not ", k);
  std::vector<int64_t> shape(z.sizes().begin(), z.sizes().end() - 1);
  vsl_top_desc d{};
  d.rows = x.size(0);
  d.vocab = x.size(1);
  d.stride = row_stride(x);
  d.k = (int32_t)k;
  d.type = type_of(x);
  d.temperature = (float)temperature_of(temperature);
  d.logits = x.data_ptr();
  torch::Tensor lse = floats(shape, x);
  shape.push_back(k);
  torch::Tensor values = torch::empty(shape, x.options()), indices = torch::empty(shape, x.options().dtype(torch::kInt32));
  const size_t need = vsl_top_logits_workspace_bytes(&d);
  torch::Tensor work = bytes(need, x);
  check(vsl_top_logits(&d, values.data_ptr(), indices.data_ptr<int32_t>(), lse.data_ptr<float>(), work.data_ptr(), need,
                       stream_of(x)));
  return {values, indices, lse};
}

/* temperature^2 * KL(teacher || student) from the teacher's top logits; gradient of `logits`. */
inline torch::Tensor topk_distillation_loss(const torch::Tensor& logits, const torch::Tensor& teacher_values,
                                            const torch::Tensor& teacher_indices,
                                            const std::optional<torch::Tensor>& teacher_lse = {}, double temperature = 1.0,
                                            const std::optional<torch::Tensor>& weights = {},
                                            const std::string& reduction = "mean") {
  using namespace vocab_detail;
  const torch::Tensor z = floating(logits, "logits");
  torch::Tensor values = floating(teacher_values, "teacher_values").detach(), indices = teacher_indices;
  on(values, "teacher_values", z);
  on(indices, "teacher_indices", z);
  TORCH_CHECK_VALUE(indices.scalar_type() == torch::kInt32 || indices.scalar_type() == torch::kInt64,
                    "teacher_indices must be int32 or int64, not ", indices.scalar_type());
  const torch::Tensor x = matrix(z, "logits");
  const auto shape = z.sizes().slice(0, z.dim() - 1);
  TORCH_CHECK_VALUE(values.dim() >= 1 && values.sizes() == indices.sizes() && values.sizes().slice(0, values.dim() - 1) == shape,
                    "teacher_values and teacher_indices must both be [..., k] over the rows of logits");
  const int64_t k = values.size(-1);
  TORCH_CHECK_VALUE(k >= 1 && k <= std::min<int64_t>(x.size(1), VSL_MAX_TOP), "the teacher's k must lie in 1..min(classes, ",
                    VSL_MAX_TOP, "), not ", k);
  values = values.reshape({x.size(0), k}).contiguous();
  indices = indices.reshape({x.size(0), k}).contiguous();
  const torch::Tensor lse = per_row(teacher_lse, "teacher_lse", shape, z), w = per_row(weights, "weights", shape, z);
  const DistillConfig c{temperature_of(temperature), reduction_of(reduction)};
  torch::Tensor loss = differentiable({&x}) ? Distill::apply(x, values, indices, given(lse), given(w), c)
                                            : distill_forward(x, values, indices, lse, w, c).first;
  return c.reduction == VSL_REDUCE_NONE && shape.size() != 1 ? loss.reshape(shape) : loss;
}

/* Cross entropy of hidden @ weight.T + bias against target, in pieces of the vocabulary, with the gradients of all three. */
inline torch::Tensor linear_cross_entropy(const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& target,
                                          const std::optional<torch::Tensor>& bias = {}, int64_t ignore_index = -100,
                                          double z_loss = 0.0, const std::string& reduction = "mean") {
  using namespace vocab_detail;
  const torch::Tensor h = floating(hidden, "hidden"), w = floating(weight, "weight");
  on(w, "weight", h);
  on(target, "target", h);
  TORCH_CHECK_VALUE(w.dim() == 2 && h.dim() >= 1 && w.size(1) == h.size(-1) && w.size(0) >= 1,
                    "hidden must be [..., dim] and weight [classes, dim], not ", h.sizes(), " and ", w.sizes());
  TORCH_CHECK_VALUE(w.scalar_type() == h.scalar_type(), "hidden and weight must have one type, not ", h.scalar_type(), " and ",
                    w.scalar_type());
  torch::Tensor b;
  if (bias && bias->defined()) {
    b = floating(*bias, "bias");
    on(b, "bias", h);
    TORCH_CHECK_VALUE(b.dim() == 1 && b.size(0) == w.size(0) && b.scalar_type() == h.scalar_type(),
                      "bias must be [classes] of hidden's type");
    b = b.contiguous();
  }
  const auto shape = h.sizes().slice(0, h.dim() - 1);
  TORCH_CHECK_VALUE(c10::isIntegralType(target.scalar_type(), /*includeBool=*/false) && target.sizes() == shape,
                    "target must be whole numbers over the rows of hidden, ", shape);
  TORCH_CHECK_VALUE(z_loss >= 0.0 && z_loss <= 1e30, "z_loss must be finite and not negative");
  const torch::Tensor t = target.to(torch::kInt64).reshape({-1}).contiguous(), hm = matrix(h, "hidden"), wm = matrix(w, "weight");
  const LinearCeConfig c{ignore_index, reduction_of(reduction), z_loss};
  torch::Tensor loss = differentiable({&hm, &wm, &b}) ? LinearCrossEntropy::apply(hm, wm, given(b), t, c)
                                                      : linear_ce_forward(hm, wm, b, t, c).first;
  return c.reduction == VSL_REDUCE_NONE && shape.size() != 1 ? loss.reshape(shape) : loss;
}

}  // namespace vsl

#endif
