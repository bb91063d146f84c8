// PyTorch operators over the C entry points of the row norm and the dense layers (include/flashcart_hip.h), with their
// autograd formulas; those in 8 bits have none.
#include "node_ops.h"

using namespace fct;

namespace {

const Tensor& or_none(const optional<Tensor>& t) {
  static const Tensor none;
  return t ? *t : none;
}
// (an absent optional tensor takes no place among the inputs whose gradients are asked for)
bool has(const optional<Tensor>& t) { return t && t->defined(); }
const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
Tensor take_optional(const char* name, const optional<Tensor>& t, at::ScalarType type, const Tensor& first) {
  return t && t->defined() ? take(name, *t, type, first) : Tensor();
}
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::empty(sizes, like.options().dtype(type));
}
Tensor none_like(const Tensor& t) { return at::empty({0}, t.options()); }
struct Workspace {
  Tensor memory;
  void* at = nullptr;
  Workspace(const Tensor& like, int64_t size, const char* what) {
    if (size < 0) check(-size, what);
    if (size == 0) return;
    memory = fresh({size}, at::kByte, like);
    at = memory.mutable_data_ptr();
  }
};

// ---- root-mean-square norm with the residual's addition ----

struct Rows {
  Tensor x, residual, weight;
  int32_t code;
  int64_t n, width;
};
Rows norm_rows(const char* what, const Tensor& x_, const optional<Tensor>& residual_, const optional<Tensor>& weight_) {
  Rows r;
  r.code = code_of("x", x_);
  const auto type = x_.scalar_type();
  r.x = take("x", x_, type, x_);
  TORCH_CHECK_VALUE(r.x.dim() > 0 && r.x.size(-1) > 0, what, ": x must be (..., width) and not of width 0, got ",
                    r.x.sizes(), ".");
  r.width = r.x.size(-1);
  r.n = r.x.numel() / r.width;
  r.residual = take_optional("residual", residual_, type, r.x);
  TORCH_CHECK_VALUE(!r.residual.defined() || r.residual.sizes() == r.x.sizes(), what, ": residual and x ", r.x.sizes(),
                    " differ in shape.");
  r.weight = take_optional("weight", weight_, type, r.x);
  TORCH_CHECK_VALUE(!r.weight.defined() || r.weight.sizes() == at::IntArrayRef({r.width}), what,
                    ": the weight must be (", r.width, "), as x is wide.");
  return r;
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_add(const Tensor& x, const optional<Tensor>& residual,
                                                const optional<Tensor>& weight, double eps, bool save) {
  const Rows r = norm_rows("rms_norm_add", x, residual, weight);
  const c10::DeviceGuard guard(r.x.device());
  Tensor y = at::empty(r.x.sizes(), r.x.options());
  Tensor total = r.residual.defined() ? at::empty(r.x.sizes(), r.x.options()) : none_like(r.x);
  Tensor rstd = fresh({save ? r.n : 0}, at::kFloat, r.x);
  check(api.row_norm_fwd(r.code, r.n, r.width, r.x.const_data_ptr(), data(r.residual), data(r.weight), (float)eps,
                         r.residual.defined() ? total.mutable_data_ptr() : nullptr, y.mutable_data_ptr(),
                         save ? rstd.mutable_data_ptr<float>() : nullptr, stream_of(r.x)),
        "fc_row_norm_fwd");
  return {y, total, rstd};
}

std::tuple<Tensor, Tensor> rms_norm_add_bwd(const Tensor& grad_, const optional<Tensor>& grad_total_, const Tensor& total_,
                                            const optional<Tensor>& weight_, const Tensor& rstd_, bool need_x,
                                            bool need_weight) {
  const Rows r = norm_rows("rms_norm_add_bwd", total_, grad_total_, weight_);
  TORCH_CHECK_VALUE(grad_.sizes() == r.x.sizes(), "rms_norm_add_bwd: grad ", grad_.sizes(), " and the rows ", r.x.sizes(),
                    " differ in shape.");
  const Tensor grad = take("grad", grad_, r.x.scalar_type(), r.x), rstd = take("rstd", rstd_, at::kFloat, r.x);
  TORCH_CHECK_VALUE(rstd.numel() == r.n, "rms_norm_add_bwd: rstd holds ", rstd.numel(), " values, not the ", r.n,
                    " of a forward pass with save=True.");
  const c10::DeviceGuard guard(r.x.device());
  Tensor dx = need_x ? at::empty(r.x.sizes(), r.x.options()) : none_like(r.x);
  Tensor dw = !need_weight ? none_like(r.x)
              : r.n == 0   ? at::zeros({r.width}, r.x.options())
                           : at::empty({r.width}, r.x.options());
  if (r.n == 0) return {dx, dw};
  const int64_t size = api.row_norm_bwd_workspace(r.code, r.n, r.width, need_weight);
  const Workspace ws(r.x, size, "fc_row_norm_bwd_workspace");
  check(api.row_norm_bwd(r.code, r.n, r.width, grad.const_data_ptr(), data(r.residual), r.x.const_data_ptr(),
                         data(r.weight), rstd.const_data_ptr<float>(), need_x ? dx.mutable_data_ptr() : nullptr,
                         need_weight ? dw.mutable_data_ptr() : nullptr, ws.at, size, stream_of(r.x)),
        "fc_row_norm_bwd");
  return {dx, dw};
}

struct RmsNormBwdNode : torch::autograd::Function<RmsNormBwdNode> {
  static variable_list forward(AutogradContext*, const Tensor& grad, const optional<Tensor>& grad_total,
                               const Tensor& total, const optional<Tensor>& weight, const Tensor& rstd, bool need_x, bool need_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatched<decltype(rms_norm_add_bwd)>("flashcart::rms_norm_add_bwd");
    auto [dx, dw] = op.call(grad, grad_total, total, weight, rstd, need_x, need_weight);
    return {dx, dw};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "second derivatives of rms_norm_add are not provided (its backward pass was run "
                                       "with create_graph=True).");
  }
};
std::tuple<Tensor, Tensor> rms_norm_add_bwd_autograd(const Tensor& grad, const optional<Tensor>& grad_total,
                                                     const Tensor& total, const optional<Tensor>& weight,
                                                     const Tensor& rstd, bool need_x, bool need_weight) {
  if (records({&grad, &or_none(grad_total), &total, &or_none(weight)})) {
    auto g = RmsNormBwdNode::apply(grad, grad_total, total, weight, rstd, need_x, need_weight);
    return {g[0], g[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(rms_norm_add_bwd, grad, grad_total, total, weight, rstd, need_x, need_weight);
}

struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual,
                               const optional<Tensor>& weight, double eps, bool save) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatched<decltype(rms_norm_add)>("flashcart::rms_norm_add");
    auto [y, total, rstd] = op.call(x, residual, weight, eps, save);
    ctx->save_for_backward({has(residual) ? total : x, or_none(weight), rstd});
    ctx->saved_data["save"] = save;
    ctx->saved_data["residual"] = has(residual);
    ctx->saved_data["weight"] = has(weight);
    ctx->set_materialize_grads(false);
    if (has(residual)) ctx->mark_non_differentiable({rstd});
    else ctx->mark_non_differentiable({total, rstd});
    return {y, total, rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const bool residual = ctx->saved_data["residual"].toBool(), weight = ctx->saved_data["weight"].toBool();
    const bool nx = ctx->needs_input_grad(0), nr = residual && ctx->needs_input_grad(1),
               nw = weight && ctx->needs_input_grad(1 + residual);
    variable_list out(5);
    if (!grad[0].defined()) {  // the total alone, if that
      if (nx) out[0] = grad[1];
      if (nr) out[1] = grad[1];
      return out;
    }
    TORCH_CHECK(ctx->saved_data["save"].toBool(),
                "rms_norm_add was called with save=False: its gradients cannot be formed.");
    const auto kept = ctx->get_saved_variables();
    auto [dx, dw] = rms_norm_add_bwd_autograd(grad[0], grad[1].defined() ? optional<Tensor>(grad[1]) : optional<Tensor>(),
                                              kept[0], weight ? optional<Tensor>(kept[1]) : optional<Tensor>(), kept[2],
                                              nx || nr, nw);
    if (nx) out[0] = dx;
    if (nr) out[1] = dx;
    if (nw) out[2] = dw;
    return out;
  }
};
std::tuple<Tensor, Tensor, Tensor> rms_norm_add_autograd(const Tensor& x, const optional<Tensor>& residual,
                                                         const optional<Tensor>& weight, double eps, bool save) {
  if (records({&x, &or_none(residual), &or_none(weight)})) {
    auto out = RmsNormNode::apply(x, residual, weight, eps, save);
    return {out[0], out[1], out[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(rms_norm_add, x, residual, weight, eps, save);
}

// ---- 8 bits: no gradients ----

void refuse_gradients(const char* what, std::initializer_list<const Tensor*> inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!records(inputs), what, " has no derivatives, and an argument asks for them: call it under "
                              "torch.no_grad(), or on detached tensors.");
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_add_quantized(const Tensor& x, const optional<Tensor>& residual,
                                                          const optional<Tensor>& weight, double eps) {
  const Rows r = norm_rows("rms_norm_add_quantized", x, residual, weight);
  const c10::DeviceGuard guard(r.x.device());
  auto shape = r.x.sizes().vec();
  shape.pop_back();
  Tensor q = fresh(r.x.sizes(), at::kFloat8_e4m3fn, r.x);
  Tensor scale = fresh(shape, at::kFloat, r.x);
  Tensor total = r.residual.defined() ? at::empty(r.x.sizes(), r.x.options()) : none_like(r.x);
  check(api.row_norm_quantize(r.code, 1, r.n, r.width, r.x.const_data_ptr(), data(r.residual), data(r.weight), (float)eps,
                              r.residual.defined() ? total.mutable_data_ptr() : nullptr, q.mutable_data_ptr(),
                              scale.mutable_data_ptr<float>(), stream_of(r.x)),
        "fc_row_norm_quantize");
  return {q, scale, total};
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_add_quantized_autograd(const Tensor& x, const optional<Tensor>& residual,
                                                                   const optional<Tensor>& weight, double eps) {
  refuse_gradients("rms_norm_add_quantized", {&x, &or_none(residual), &or_none(weight)});
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(rms_norm_add_quantized, x, residual, weight, eps);
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  const Rows r = norm_rows("quantize_rows", x, {}, {});
  const c10::DeviceGuard guard(r.x.device());
  auto shape = r.x.sizes().vec();
  shape.pop_back();
  Tensor q = fresh(r.x.sizes(), at::kFloat8_e4m3fn, r.x);
  Tensor scale = fresh(shape, at::kFloat, r.x);
  check(api.row_norm_quantize(r.code, 0, r.n, r.width, r.x.const_data_ptr(), nullptr, nullptr, 0.f, nullptr,
                              q.mutable_data_ptr(), scale.mutable_data_ptr<float>(), stream_of(r.x)),
        "fc_row_norm_quantize");
  return {q, scale};
}
std::tuple<Tensor, Tensor> quantize_rows_autograd(const Tensor& x) {
  refuse_gradients("quantize_rows", {&x});
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(quantize_rows, x);
}

// ---- dense layers ----

constexpr int64_t kNoAct = 3;

fc_dense_desc dense_desc(const char* what, int32_t code, const Tensor& x, const Tensor& weight, bool groups, int64_t act,
                         double act_scale, double scale) {
  fc_dense_desc d{};
  d.dtype = code;
  const int64_t dims = groups ? 3 : 2;
  TORCH_CHECK_VALUE(weight.dim() == dims && weight.numel() > 0, what, ": the weight must be ",
                    groups ? "(groups, out, in)" : "(out, in)", " and not empty, got ", weight.sizes(), ".");
  const int64_t in = weight.size(-1), out = weight.size(-2);
  TORCH_CHECK_VALUE(x.dim() > 0 && (!groups || x.dim() == 2) && x.size(-1) == in, what, ": rows ", x.sizes(),
                    " do not match a weight ", weight.sizes(), ".");
  TORCH_CHECK_VALUE(act >= 0 && act <= kNoAct, what, ": act must be 0 (silu), 1 (sigmoid), 2 (gelu) or 3 (none), got ",
                    act, ".");
  const int64_t most = int64_t(1) << 20, several = groups ? weight.size(0) : 0;
  TORCH_CHECK_VALUE(in <= most && out <= most && several <= (1 << 16) && (several + 1) * out < (1 << 30), what,
                    ": a weight of ", weight.sizes(), " is too large.");
  d.act = (int32_t)act;
  d.in = (int32_t)in;
  d.out = (int32_t)out;
  d.groups = (int32_t)several;
  d.act_scale = (float)act_scale;
  d.scale = (float)scale;
  return d;
}
std::vector<int64_t> dense_shape(const Tensor& x, int64_t out) {
  auto shape = x.sizes().vec();
  shape.back() = out;
  return shape;
}
Tensor take_bias(const char* what, const optional<Tensor>& bias_, const fc_dense_desc& d, at::ScalarType type,
                 const Tensor& x) {
  const Tensor bias = take_optional("bias", bias_, type, x);
  if (bias.defined()) {
    const bool ok = d.groups > 0 ? bias.sizes() == at::IntArrayRef({d.groups, d.out}) : bias.sizes() == at::IntArrayRef({d.out});
    TORCH_CHECK_VALUE(ok, what, ": the bias must be ", d.groups > 0 ? "(groups, out)" : "(out)", ", got ", bias.sizes(), ".");
  }
  return bias;
}
Tensor take_residual(const char* what, const optional<Tensor>& residual_, at::IntArrayRef shape, at::ScalarType type,
                     const Tensor& x) {
  const Tensor residual = take_optional("residual", residual_, type, x);
  TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == shape, what, ": the residual must be ", shape, ", as the output is.");
  return residual;
}
Tensor take_offsets(const char* what, const optional<Tensor>& offsets_, const fc_dense_desc& d, const Tensor& x) {
  if (!offsets_ || !offsets_->defined()) return Tensor();
  const Tensor& o = *offsets_;
  TORCH_CHECK_TYPE(o.scalar_type() == at::kLong || o.scalar_type() == at::kInt, "`offsets` must be int64 or int32, got ",
                   o.scalar_type(), ".");
  TORCH_CHECK_VALUE(o.sizes() == at::IntArrayRef({d.groups + 1}), what, ": offsets must be (", d.groups + 1, "), got ",
                    o.sizes(), ".");
  return take("offsets", o.scalar_type() == at::kInt ? o.to(at::kLong) : o, at::kLong, x);
}

std::tuple<Tensor, Tensor> node_dense(const Tensor& x_, const Tensor& weight_, const optional<Tensor>& bias_,
                                      const optional<Tensor>& residual_, const optional<Tensor>& offsets_, int64_t act,
                                      double act_scale, double scale, bool save) {
  const bool groups = offsets_ && offsets_->defined();
  const char* const what = groups ? "grouped_dense" : "dense";
  fc_dense_desc d = dense_desc(what, code_of("x", x_), x_, weight_, groups, act, act_scale, scale);
  const auto type = x_.scalar_type();
  const Tensor x = take("x", x_, type, x_), weight = take("weight", weight_, type, x);
  const Tensor bias = take_bias(what, bias_, d, type, x), offsets = take_offsets(what, offsets_, d, x);
  const auto shape = dense_shape(x, d.out);
  const Tensor residual = take_residual(what, residual_, shape, type, x);
  TORCH_CHECK_VALUE(!groups || !residual.defined(), "grouped_dense takes no residual.");
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.numel() / d.in;
  d.aligned = aligned({&x, &weight});
  const int64_t size = api.node_dense_fwd_workspace(&d, n);
  const int64_t kept = save ? api.node_dense_saved(&d, n) : 0;
  if (kept < 0) check(-kept, "fc_node_dense_saved");
  const Workspace ws(x, size, "fc_node_dense_fwd_workspace");
  Tensor y = at::empty(shape, x.options()), saved = fresh({kept}, at::kByte, x);
  check(api.node_dense_fwd(&d, n, x.const_data_ptr(), weight.const_data_ptr(), data(bias), data(residual),
                           (const int64_t*)data(offsets), y.mutable_data_ptr(),
                           kept ? saved.mutable_data_ptr() : nullptr, ws.at, size, stream_of(x)),
        "fc_node_dense_fwd");
  return {y, saved};
}

std::tuple<Tensor, Tensor, Tensor> node_dense_bwd(const Tensor& grad_, const Tensor& x_, const Tensor& weight_,
                                                  const Tensor& saved_, const optional<Tensor>& offsets_, int64_t act,
                                                  double act_scale, double scale, bool need_x, bool need_weight,
                                                  bool need_bias) {
  const bool groups = offsets_ && offsets_->defined();
  const char* const what = groups ? "grouped_dense_bwd" : "dense_bwd";
  fc_dense_desc d = dense_desc(what, code_of("x", x_), x_, weight_, groups, act, act_scale, scale);
  const auto type = x_.scalar_type();
  const Tensor x = take("x", x_, type, x_), weight = take("weight", weight_, type, x), grad = take("grad", grad_, type, x);
  const Tensor offsets = take_offsets(what, offsets_, d, x);
  TORCH_CHECK_VALUE(grad.sizes() == at::IntArrayRef(dense_shape(x, d.out)), what, ": grad ", grad.sizes(),
                    " does not match rows ", x.sizes(), " and a weight ", weight.sizes(), ".");
  Tensor saved = take("saved", saved_, at::kByte, x);
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.numel() / d.in, kept = api.node_dense_saved(&d, n);
  if (kept < 0) check(-kept, "fc_node_dense_saved");
  TORCH_CHECK_VALUE(saved.numel() == kept, what, ": saved holds ", saved.numel(), " bytes, not the ", kept,
                    " of a forward pass with save=True.");
  if ((uintptr_t)saved.const_data_ptr() & 15) saved = saved.clone();
  d.aligned = aligned({&grad, &x, &weight});
  auto result = [&](at::IntArrayRef shape, bool need) {
    if (!need) return none_like(x);
    return n == 0 ? at::zeros(shape, x.options()) : at::empty(shape, x.options());
  };
  Tensor gx = result(x.sizes(), need_x), gw = result(weight.sizes(), need_weight);
  Tensor gb = result(groups ? at::IntArrayRef({d.groups, d.out}) : at::IntArrayRef({d.out}), need_bias);
  if (n > 0) {
    const int64_t size = api.node_dense_bwd_workspace(&d, n, need_x, need_weight, need_bias);
    const Workspace ws(x, size, "fc_node_dense_bwd_workspace");
    check(api.node_dense_bwd(&d, n, grad.const_data_ptr(), x.const_data_ptr(), weight.const_data_ptr(),
                             kept ? saved.const_data_ptr() : nullptr, (const int64_t*)data(offsets),
                             need_x ? gx.mutable_data_ptr() : nullptr, need_weight ? gw.mutable_data_ptr() : nullptr,
                             need_bias ? gb.mutable_data_ptr() : nullptr, ws.at, size, stream_of(x)),
          "fc_node_dense_bwd");
  }
  return {gx, gw, gb};
}

struct DenseBwdNode : torch::autograd::Function<DenseBwdNode> {
  static variable_list forward(AutogradContext*, const Tensor& grad, const Tensor& x, const Tensor& weight,
                               const Tensor& saved, const optional<Tensor>& offsets, int64_t act, double act_scale,
                               double scale, bool need_x, bool need_weight, bool need_bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatched<decltype(node_dense_bwd)>("flashcart::node_dense_bwd");
    auto [gx, gw, gb] = op.call(grad, x, weight, saved, offsets, act, act_scale, scale, need_x, need_weight, need_bias);
    return {gx, gw, gb};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "second derivatives of dense layers are not provided (their backward pass was run "
                                       "with create_graph=True).");
  }
};
std::tuple<Tensor, Tensor, Tensor> node_dense_bwd_autograd(const Tensor& grad, const Tensor& x, const Tensor& weight,
                                                           const Tensor& saved, const optional<Tensor>& offsets,
                                                           int64_t act, double act_scale, double scale, bool need_x,
                                                           bool need_weight, bool need_bias) {
  if (records({&grad, &x, &weight})) {
    auto g = DenseBwdNode::apply(grad, x, weight, saved, offsets, act, act_scale, scale, need_x, need_weight,
                                 need_bias);
    return {g[0], g[1], g[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(node_dense_bwd, grad, x, weight, saved, offsets, act, act_scale, scale, need_x, need_weight, need_bias);
}

struct DenseNode : torch::autograd::Function<DenseNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                               const optional<Tensor>& residual, const optional<Tensor>& offsets, int64_t act,
                               double act_scale, double scale, bool save) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatched<decltype(node_dense)>("flashcart::node_dense");
    auto [y, saved] = op.call(x, weight, bias, residual, offsets, act, act_scale, scale, save);
    ctx->save_for_backward({x, weight, saved, or_none(offsets)});
    ctx->saved_data["bias"] = has(bias);
    ctx->saved_data["residual"] = has(residual);
    ctx->saved_data["groups"] = has(offsets);
    ctx->saved_data["act"] = act;
    ctx->saved_data["scales"] = std::vector<double>{act_scale, scale};
    ctx->saved_data["save"] = save;
    ctx->mark_non_differentiable({saved});
    ctx->set_materialize_grads(false);
    return {y, saved};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const bool bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = bias && ctx->needs_input_grad(2);
    variable_list out(9);
    if (!grad[0].defined()) return out;
    if (residual && ctx->needs_input_grad(2 + bias)) out[3] = grad[0];
    if (!(nx || nw || nb)) return out;
    TORCH_CHECK(ctx->saved_data["save"].toBool(),
                "a dense layer was called with save=False: its gradients cannot be formed.");
    const auto kept = ctx->get_saved_variables();
    const auto scales = ctx->saved_data["scales"].toDoubleVector();
    const optional<Tensor> offsets = ctx->saved_data["groups"].toBool() ? optional<Tensor>(kept[3]) : optional<Tensor>();
    auto [gx, gw, gb] = node_dense_bwd_autograd(grad[0], kept[0], kept[1], kept[2], offsets, ctx->saved_data["act"].toInt(),
                                                scales[0], scales[1], nx, nw, nb);
    if (nx) out[0] = gx;
    if (nw) out[1] = gw;
    if (nb) out[2] = gb;
    return out;
  }
};
std::tuple<Tensor, Tensor> node_dense_autograd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                                               const optional<Tensor>& residual, const optional<Tensor>& offsets,
                                               int64_t act, double act_scale, double scale, bool save) {
  if (records({&x, &weight, &or_none(bias), &or_none(residual)})) {
    auto out = DenseNode::apply(x, weight, bias, residual, offsets, act, act_scale, scale, save);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(node_dense, x, weight, bias, residual, offsets, act, act_scale, scale, save);
}

Tensor quantized_dense(const Tensor& x_, const Tensor& x_scale_, const Tensor& weight_, const Tensor& weight_scale_,
                       const optional<Tensor>& bias_, const optional<Tensor>& residual_, int64_t act, double act_scale,
                       double scale, at::ScalarType dtype) {
  const char* const what = "quantized_dense";
  TORCH_CHECK_TYPE(dtype == at::kBFloat16 || dtype == at::kHalf, "`dtype` must be bfloat16 or float16, got ", dtype, ".");
  const int32_t code = dtype == at::kBFloat16 ? FC_BF16 : FC_F16;
  const Tensor x = take("x", x_, at::kFloat8_e4m3fn, x_), weight = take("weight", weight_, at::kFloat8_e4m3fn, x);
  fc_dense_desc d = dense_desc(what, code, x, weight, false, act, act_scale, scale);
  const Tensor x_scale = take("x_scale", x_scale_, at::kFloat, x), weight_scale = take("weight_scale", weight_scale_, at::kFloat, x);
  TORCH_CHECK_VALUE(x_scale.sizes() == x.sizes().slice(0, x.dim() - 1) && weight_scale.sizes() == at::IntArrayRef({d.out}), what,
                    ": scales ", x_scale.sizes(), " and ", weight_scale.sizes(), " are not one for each row of x ", x.sizes(),
                    " and of the weight ", weight.sizes(), ".");
  const Tensor bias = take_bias(what, bias_, d, dtype, x);
  const auto shape = dense_shape(x, d.out);
  const Tensor residual = take_residual(what, residual_, shape, dtype, x);
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.numel() / d.in;
  d.aligned = aligned({&x, &weight});
  const int64_t size = api.quantized_dense_workspace(&d, n);
  const Workspace ws(x, size, "fc_quantized_dense_workspace");
  Tensor y = fresh(shape, dtype, x);
  check(api.quantized_dense(&d, n, x.const_data_ptr(), x_scale.const_data_ptr<float>(), weight.const_data_ptr(),
                            weight_scale.const_data_ptr<float>(), data(bias), data(residual), y.mutable_data_ptr(),
                            ws.at, size, stream_of(x)),
        "fc_quantized_dense");
  return y;
}
Tensor quantized_dense_autograd(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale,
                                const optional<Tensor>& bias, const optional<Tensor>& residual, int64_t act,
                                double act_scale, double scale, at::ScalarType dtype) {
  refuse_gradients("quantized_dense", {&x, &x_scale, &weight, &weight_scale, &or_none(bias), &or_none(residual)});
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(quantized_dense, x, x_scale, weight, weight_scale, bias, residual, act, act_scale, scale, dtype);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(flashcart, m) {
  m.def("rms_norm_add(Tensor x, Tensor? residual, Tensor? weight, float eps, bool save) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_add_bwd(Tensor grad, Tensor? grad_total, Tensor total, Tensor? weight, Tensor rstd, bool need_x, "
        "bool need_weight) -> (Tensor, Tensor)");
  m.def("rms_norm_add_quantized(Tensor x, Tensor? residual, Tensor? weight, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("quantize_rows(Tensor x) -> (Tensor, Tensor)");
  m.def("node_dense(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, Tensor? offsets, int act, float act_scale, "
        "float scale, bool save) -> (Tensor, Tensor)");
  m.def("node_dense_bwd(Tensor grad, Tensor x, Tensor weight, Tensor saved, Tensor? offsets, int act, float act_scale, "
        "float scale, bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
  m.def("quantized_dense(Tensor x, Tensor x_scale, Tensor weight, Tensor weight_scale, Tensor? bias, Tensor? residual, "
        "int act, float act_scale, float scale, ScalarType dtype) -> Tensor");
}

// (on the CPU they end in their own error)
#define FCT_DENSE_IMPLS(m)                                                  \
  m.impl("rms_norm_add", TORCH_FN(rms_norm_add));                           \
  m.impl("rms_norm_add_bwd", TORCH_FN(rms_norm_add_bwd));                   \
  m.impl("rms_norm_add_quantized", TORCH_FN(rms_norm_add_quantized));       \
  m.impl("quantize_rows", TORCH_FN(quantize_rows));                         \
  m.impl("node_dense", TORCH_FN(node_dense));                               \
  m.impl("node_dense_bwd", TORCH_FN(node_dense_bwd));                       \
  m.impl("quantized_dense", TORCH_FN(quantized_dense));
TORCH_LIBRARY_IMPL(flashcart, CUDA, m) { FCT_DENSE_IMPLS(m) }
TORCH_LIBRARY_IMPL(flashcart, CPU, m) { FCT_DENSE_IMPLS(m) }

TORCH_LIBRARY_IMPL(flashcart, Autograd, m) {
  m.impl("rms_norm_add", TORCH_FN(rms_norm_add_autograd));
  m.impl("rms_norm_add_bwd", TORCH_FN(rms_norm_add_bwd_autograd));
  m.impl("rms_norm_add_quantized", TORCH_FN(rms_norm_add_quantized_autograd));
  m.impl("quantize_rows", TORCH_FN(quantize_rows_autograd));
  m.impl("node_dense", TORCH_FN(node_dense_autograd));
  m.impl("node_dense_bwd", TORCH_FN(node_dense_bwd_autograd));
  m.impl("quantized_dense", TORCH_FN(quantized_dense_autograd));
}
