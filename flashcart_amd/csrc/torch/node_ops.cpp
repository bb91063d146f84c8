// PyTorch operators over the C entry points of the node-wise kernels (include/flashcart_hip.h): embedding, gated
// feed-forward block, residual dropout, with their autograd formulas. They are C++ and not Python because a training step
// of small tensors is bound by the host: its backward pass runs in the autograd engine's thread, where Python code costs
// several times what the kernels take (forward and backward of 903 elements: 110 us from Python, 40 us of them the
// engine's own).
//
// The kernels' library is opened by fct_bind (the same file that the Python package binds), nothing is linked.
#include "node_ops.h"

fct::Api fct::api{};

using namespace fct;

namespace {

// ---- embedding ----

Tensor embedding(const Tensor& ids_, const Tensor& table_, double scale, int64_t /*padding*/) {
  const int32_t code = code_of("table", table_);
  const Tensor table = take("table", table_, table_.scalar_type(), table_);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0,
                    "embedding: the table must be (rows, width) and not empty, got ", table.sizes(), ".");
  const Tensor ids = take_ids(ids_, table);
  const c10::DeviceGuard guard(table.device());
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  Tensor out = at::empty(shape, table.options());
  check(api.embedding_fwd(code, ids.numel(), table.size(0), table.size(1), ids.const_data_ptr<int64_t>(),
                          table.const_data_ptr(), (float)scale, out.mutable_data_ptr(), stream_of(table)),
        "fc_embedding_fwd");
  return out;
}

Tensor embedding_bwd(const Tensor& grad_, const Tensor& ids_, int64_t rows, double scale, int64_t padding) {
  const int32_t code = code_of("grad", grad_);
  const Tensor grad = take("grad", grad_, grad_.scalar_type(), grad_), ids = take_ids(ids_, grad);
  TORCH_CHECK_VALUE(grad.dim() == ids.dim() + 1 && grad.sizes().slice(0, ids.dim()) == ids.sizes(),
                    "embedding_bwd: grad ", grad.sizes(), " does not match ids ", ids.sizes(), ".");
  const c10::DeviceGuard guard(grad.device());
  const int64_t n = ids.numel(), width = grad.size(-1), size = api.embedding_bwd_workspace(code, n, rows, width);
  Tensor out = at::empty({rows, width}, grad.options()), ws = bytes(grad, size, "fc_embedding_bwd_workspace");
  check(api.embedding_bwd(code, n, rows, width, ids.const_data_ptr<int64_t>(), grad.const_data_ptr(), (float)scale,
                          padding, out.mutable_data_ptr(), ws.mutable_data_ptr(), size, stream_of(grad)),
        "fc_embedding_bwd");
  return out;
}

struct EmbeddingBwdNode : torch::autograd::Function<EmbeddingBwdNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& ids, int64_t rows, double scale,
                        int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = rows;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    FCT_DISPATCHED(embedding_bwd, grad, ids, rows, scale, padding);
  }
  // The table's gradient is linear in `grad`: the rows that an id adds to, looked up in the cotangent; zero for the
  // padding row and for ids outside the table, which add to none.
  static variable_list backward(AutogradContext* ctx, variable_list cot) {
    static const auto op = dispatched<decltype(embedding)>("flashcart::embedding");
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t rows = ctx->saved_data["rows"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const Tensor out = op.call(ids.clamp(0, rows - 1), cot[0], ctx->saved_data["scale"].toDouble(), padding);
    const Tensor dead = ids.lt(0).logical_or(ids.ge(rows)).logical_or(ids.eq(padding));
    return {out.masked_fill(dead.unsqueeze(-1), 0), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor embedding_bwd_autograd(const Tensor& grad, const Tensor& ids, int64_t rows, double scale, int64_t padding) {
  if (records({&grad})) return EmbeddingBwdNode::apply(grad, ids, rows, scale, padding);
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(embedding_bwd, grad, ids, rows, scale, padding);
}

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale, int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    FCT_DISPATCHED(embedding, ids, table, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    return {Tensor(),
            embedding_bwd_autograd(grad[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                                   ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt()),
            Tensor(), Tensor()};
  }
};
Tensor embedding_autograd(const Tensor& ids, const Tensor& table, double scale, int64_t padding) {
  if (records({&table})) return EmbeddingNode::apply(ids, table, scale, padding);
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(embedding, ids, table, scale, padding);
}

// ---- residual dropout ----

Tensor dropout_add(const Tensor& x_, const optional<Tensor>& residual_, double p, const Tensor& rng_) {
  const int32_t code = code_of("x", x_);
  const Tensor x = take("x", x_, x_.scalar_type(), x_);
  Tensor residual;
  if (residual_ && residual_->defined()) {
    TORCH_CHECK_VALUE(residual_->sizes() == x.sizes(), "dropout_add: residual ", residual_->sizes(), " and x ",
                      x.sizes(), " differ in shape.");
    residual = take("residual", *residual_, x.scalar_type(), x);
  }
  TORCH_CHECK_VALUE(rng_.numel() == 2, "dropout_add: rng must hold a seed and an offset, got ", rng_.sizes(), ".");
  TORCH_CHECK_VALUE(p >= 0 && p <= 1, "dropout_add: p must be in [0, 1], got ", p, ".");
  const Tensor rng = take("rng", rng_, at::kLong, x);
  const c10::DeviceGuard guard(x.device());
  Tensor out = at::empty(x.sizes(), x.options());
  check(api.dropout_add(code, x.numel(), x.const_data_ptr(), residual.defined() ? residual.const_data_ptr() : nullptr, p,
                        rng.const_data_ptr<int64_t>(), out.mutable_data_ptr(), stream_of(x)),
        "fc_dropout_add");
  return out;
}

Tensor dropout_add_autograd(const Tensor& x, const optional<Tensor>& residual, double p, const Tensor& rng);

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual, double p,
                        const Tensor& rng) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({rng});
    ctx->saved_data["p"] = p;
    FCT_DISPATCHED(dropout_add, x, residual, p, rng);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    Tensor gx, gr;
    if (ctx->needs_input_grad(0))
      gx = dropout_add_autograd(grad[0], {}, ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0]);
    if (ctx->needs_input_grad(1)) gr = grad[0];
    return {gx, gr, Tensor(), Tensor()};
  }
};
Tensor dropout_add_autograd(const Tensor& x, const optional<Tensor>& residual, double p, const Tensor& rng) {
  const Tensor r = residual ? *residual : Tensor();
  if (records({&x, &r})) return DropoutNode::apply(x, residual, p, rng);
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(dropout_add, x, residual, p, rng);
}

// Seed and offset of one call; `state` goes on to the next offset. A call that the backward pass runs again would get other
// numbers than the first time. (Asked here, when it runs, so that it holds in compiled functions too.)
Tensor dropout_draw(Tensor& state) {
  TORCH_CHECK(torch::autograd::get_current_graph_task_id() == -1,
              "random numbers of a dropout call were asked for during a backward pass, as activation checkpointing does when "
              "it runs a call again: those of the first run cannot be drawn again. Take rng = layer.draw() outside the "
              "checkpointed function and pass it in.");
  TORCH_CHECK_VALUE(state.scalar_type() == at::kLong && state.sizes() == at::IntArrayRef({2}),
                    "dropout_draw: the state must be an int64 seed and offset, got ", state.scalar_type(), " ",
                    state.sizes(), ".");
  Tensor rng = state.clone();  // (kept for the backward pass)
  state.select(0, 1).add_(1);
  return rng;
}

// ---- gated feed-forward block ----

fc_ffn_desc ffn_desc(const char* what, const Tensor& x, const Tensor& w_in, const Tensor& w_out, int64_t act,
                     double act_scale, double scale_in, double scale_out) {
  fc_ffn_desc d{};
  d.dtype = code_of("x", x);
  TORCH_CHECK_VALUE(w_in.dim() == 2 && w_out.dim() == 2 && w_in.size(0) == 2 * w_out.size(1) &&
                        w_in.size(1) == w_out.size(0),
                    what, ": w_in ", w_in.sizes(), " and w_out ", w_out.sizes(),
                    " are not (2 hidden, width) and (width, hidden).");
  TORCH_CHECK_VALUE(w_out.size(0) > 0 && w_out.size(1) > 0 && x.dim() > 0 && x.size(-1) == w_out.size(0), what, ": rows ",
                    x.sizes(), " do not match weights of width ", w_out.size(0), ", hidden ", w_out.size(1), ".");
  TORCH_CHECK_VALUE(act >= 0 && act <= 2, what, ": act must be 0 (silu), 1 (sigmoid) or 2 (gelu), got ", act, ".");
  TORCH_CHECK_VALUE(w_out.numel() < (int64_t(1) << 40) && w_out.size(0) < (1 << 30) && w_out.size(1) < (1 << 30), what,
                    ": weights of ", w_out.sizes(), " are too large.");
  d.act = (int32_t)act;
  d.width = (int32_t)w_out.size(0);
  d.hidden = (int32_t)w_out.size(1);
  d.act_scale = (float)act_scale;
  d.scale_in = (float)scale_in;
  d.scale_out = (float)scale_out;
  return d;
}
std::tuple<Tensor, Tensor> gated_feed_forward(const Tensor& x_, const Tensor& w_in_, const Tensor& w_out_, int64_t act,
                                              double act_scale, double scale_in, double scale_out, bool save) {
  fc_ffn_desc d = ffn_desc("gated_feed_forward", x_, w_in_, w_out_, act, act_scale, scale_in, scale_out);
  const auto type = x_.scalar_type();
  const Tensor x = take("x", x_, type, x_), w_in = take("w_in", w_in_, type, x), w_out = take("w_out", w_out_, type, x);
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.numel() / d.width;
  d.aligned = aligned({&x, &w_in, &w_out});
  const int64_t size = api.ffn_fwd_workspace(&d, n, save);
  Tensor y = at::empty(x.sizes(), x.options()), ws = bytes(x, size, "fc_ffn_fwd_workspace");
  Tensor saved = bytes(x, save ? api.ffn_saved(&d, n) : 0, "fc_ffn_saved");
  check(api.ffn_fwd(&d, n, x.const_data_ptr(), w_in.const_data_ptr(), w_out.const_data_ptr(), y.mutable_data_ptr(),
                    save && n ? saved.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), size, stream_of(x)),
        "fc_ffn_fwd");
  return {y, saved};
}

std::tuple<Tensor, Tensor, Tensor> gated_feed_forward_bwd(const Tensor& grad_, const Tensor& x_, const Tensor& w_in_,
                                                          const Tensor& w_out_, const Tensor& saved_, int64_t act,
                                                          double act_scale, double scale_in, double scale_out,
                                                          bool need_x, bool need_w_in, bool need_w_out) {
  fc_ffn_desc d = ffn_desc("gated_feed_forward_bwd", x_, w_in_, w_out_, act, act_scale, scale_in, scale_out);
  TORCH_CHECK_VALUE(grad_.sizes() == x_.sizes(), "gated_feed_forward_bwd: grad ", grad_.sizes(), " and x ", x_.sizes(),
                    " differ in shape.");
  const auto type = x_.scalar_type();
  const Tensor x = take("x", x_, type, x_), grad = take("grad", grad_, type, x), w_in = take("w_in", w_in_, type, x),
               w_out = take("w_out", w_out_, type, x);
  Tensor saved = take("saved", saved_, at::kByte, x);
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.numel() / d.width, kept = api.ffn_saved(&d, n);
  if (kept < 0) check(-kept, "fc_ffn_saved");
  TORCH_CHECK_VALUE(saved.numel() == kept, "gated_feed_forward_bwd: saved holds ", saved.numel(), " bytes, not the ", kept,
                    " of a forward pass with save=True.");
  if ((uintptr_t)saved.const_data_ptr() & 15) saved = saved.clone();
  d.aligned = aligned({&grad, &x, &w_in, &w_out});
  auto result = [&](const Tensor& t, bool need) {
    if (!need) return at::empty({0}, t.options());
    return n == 0 ? at::zeros(t.sizes(), t.options()) : at::empty(t.sizes(), t.options());
  };
  Tensor gx = result(x, need_x), gwi = result(w_in, need_w_in), gwo = result(w_out, need_w_out);
  if (n > 0) {
    const int64_t size = api.ffn_bwd_workspace(&d, n, need_x, need_w_in, need_w_out);
    Tensor ws = bytes(x, size, "fc_ffn_bwd_workspace");
    check(api.ffn_bwd(&d, n, grad.const_data_ptr(), x.const_data_ptr(), w_in.const_data_ptr(), w_out.const_data_ptr(),
                      saved.const_data_ptr(), need_x ? gx.mutable_data_ptr() : nullptr,
                      need_w_in ? gwi.mutable_data_ptr() : nullptr, need_w_out ? gwo.mutable_data_ptr() : nullptr,
                      ws.mutable_data_ptr(), size, stream_of(x)),
          "fc_ffn_bwd");
  }
  return {gx, gwi, gwo};
}

struct FeedForwardBwdNode : torch::autograd::Function<FeedForwardBwdNode> {
  static variable_list forward(AutogradContext*, const Tensor& grad, const Tensor& x, const Tensor& w_in,
                               const Tensor& w_out, const Tensor& saved, int64_t act, double act_scale, double scale_in,
                               double scale_out, bool need_x, bool need_w_in, bool need_w_out) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatched<decltype(gated_feed_forward_bwd)>("flashcart::gated_feed_forward_bwd");
    auto [gx, gwi, gwo] = op.call(grad, x, w_in, w_out, saved, act, act_scale, scale_in, scale_out, need_x, need_w_in,
                                  need_w_out);
    return {gx, gwi, gwo};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "second derivatives of gated_feed_forward are not provided (its backward pass was "
                                       "run with create_graph=True).");
  }
};
std::tuple<Tensor, Tensor, Tensor> gated_feed_forward_bwd_autograd(const Tensor& grad, const Tensor& x,
                                                                   const Tensor& w_in, const Tensor& w_out,
                                                                   const Tensor& saved, int64_t act, double act_scale,
                                                                   double scale_in, double scale_out, bool need_x,
                                                                   bool need_w_in, bool need_w_out) {
  if (records({&grad, &x, &w_in, &w_out})) {
    auto g = FeedForwardBwdNode::apply(grad, x, w_in, w_out, saved, act, act_scale, scale_in, scale_out, need_x,
                                       need_w_in, need_w_out);
    return {g[0], g[1], g[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(gated_feed_forward_bwd, grad, x, w_in, w_out, saved, act, act_scale, scale_in, scale_out, need_x,
                 need_w_in, need_w_out);
}

struct FeedForwardNode : torch::autograd::Function<FeedForwardNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_in, const Tensor& w_out,
                               int64_t act, double act_scale, double scale_in, double scale_out, bool save) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = dispatched<decltype(gated_feed_forward)>("flashcart::gated_feed_forward");
    auto [y, saved] = op.call(x, w_in, w_out, act, act_scale, scale_in, scale_out, save);
    ctx->save_for_backward({x, w_in, w_out, saved});
    ctx->saved_data["act"] = act;
    ctx->saved_data["scales"] = std::vector<double>{act_scale, scale_in, scale_out};
    ctx->saved_data["save"] = save;
    ctx->mark_non_differentiable({saved});
    ctx->set_materialize_grads(false);  // (no zeros the size of `saved` as its gradient)
    return {y, saved};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const bool nx = ctx->needs_input_grad(0), ni = ctx->needs_input_grad(1), no = ctx->needs_input_grad(2);
    variable_list none(8);
    if (!grad[0].defined() || !(nx || ni || no)) return none;
    TORCH_CHECK(ctx->saved_data["save"].toBool(),
                "gated_feed_forward was called with save=False: its gradients cannot be formed.");
    const auto kept = ctx->get_saved_variables();
    const auto scales = ctx->saved_data["scales"].toDoubleVector();
    auto [gx, gwi, gwo] =
        gated_feed_forward_bwd_autograd(grad[0], kept[0], kept[1], kept[2], kept[3], ctx->saved_data["act"].toInt(),
                                        scales[0], scales[1], scales[2], nx, ni, no);
    if (nx) none[0] = gx;
    if (ni) none[1] = gwi;
    if (no) none[2] = gwo;
    return none;
  }
};
std::tuple<Tensor, Tensor> gated_feed_forward_autograd(const Tensor& x, const Tensor& w_in, const Tensor& w_out,
                                                       int64_t act, double act_scale, double scale_in,
                                                       double scale_out, bool save) {
  if (records({&x, &w_in, &w_out})) {
    auto out = FeedForwardNode::apply(x, w_in, w_out, act, act_scale, scale_in, scale_out, save);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  FCT_DISPATCHED(gated_feed_forward, x, w_in, w_out, act, act_scale, scale_in, scale_out, save);
}

}  // namespace

// Opens the kernels' library and takes its entry points; 0, or 1 where one is missing.
extern "C" int fct_bind(const char* path) {
  void* lib = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!lib) return 1;
  bool ok = true;
  auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(lib, name));
    ok = ok && f != nullptr;
  };
  get(api.status_string, "fc_status_string");
  get(api.embedding_fwd, "fc_embedding_fwd");
  get(api.embedding_bwd_workspace, "fc_embedding_bwd_workspace");
  get(api.embedding_bwd, "fc_embedding_bwd");
  get(api.dropout_add, "fc_dropout_add");
  get(api.ffn_saved, "fc_ffn_saved");
  get(api.ffn_fwd_workspace, "fc_ffn_fwd_workspace");
  get(api.ffn_fwd, "fc_ffn_fwd");
  get(api.ffn_bwd_workspace, "fc_ffn_bwd_workspace");
  get(api.ffn_bwd, "fc_ffn_bwd");
  get(api.node_dense_saved, "fc_node_dense_saved");
  get(api.node_dense_fwd_workspace, "fc_node_dense_fwd_workspace");
  get(api.node_dense_fwd, "fc_node_dense_fwd");
  get(api.node_dense_bwd_workspace, "fc_node_dense_bwd_workspace");
  get(api.node_dense_bwd, "fc_node_dense_bwd");
  get(api.quantized_dense_workspace, "fc_quantized_dense_workspace");
  get(api.quantized_dense, "fc_quantized_dense");
  get(api.row_norm_fwd, "fc_row_norm_fwd");
  get(api.row_norm_quantize, "fc_row_norm_quantize");
  get(api.row_norm_bwd_workspace, "fc_row_norm_bwd_workspace");
  get(api.row_norm_bwd, "fc_row_norm_bwd");
  return ok ? 0 : 1;
}

TORCH_LIBRARY_FRAGMENT(flashcart, m) {
  m.def("embedding(Tensor ids, Tensor table, float scale, int padding) -> Tensor");
  m.def("embedding_bwd(Tensor grad, Tensor ids, int rows, float scale, int padding) -> Tensor");
  m.def("dropout_add(Tensor x, Tensor? residual, float p, Tensor rng) -> Tensor");
  m.def("dropout_draw(Tensor(a!) state) -> Tensor");
  m.def("gated_feed_forward(Tensor x, Tensor w_in, Tensor w_out, int act, float act_scale, float scale_in, "
        "float scale_out, bool save) -> (Tensor, Tensor)");
  m.def("gated_feed_forward_bwd(Tensor grad, Tensor x, Tensor w_in, Tensor w_out, Tensor saved, int act, "
        "float act_scale, float scale_in, float scale_out, bool need_x, bool need_w_in, bool need_w_out) -> "
        "(Tensor, Tensor, Tensor)");
}

// (on the CPU they end in their own error, dropout_draw aside)
#define FCT_IMPLS(m)                                         \
  m.impl("embedding", TORCH_FN(embedding));                  \
  m.impl("embedding_bwd", TORCH_FN(embedding_bwd));          \
  m.impl("dropout_add", TORCH_FN(dropout_add));              \
  m.impl("dropout_draw", TORCH_FN(dropout_draw));            \
  m.impl("gated_feed_forward", TORCH_FN(gated_feed_forward)); \
  m.impl("gated_feed_forward_bwd", TORCH_FN(gated_feed_forward_bwd));
TORCH_LIBRARY_IMPL(flashcart, CUDA, m) { FCT_IMPLS(m) }
TORCH_LIBRARY_IMPL(flashcart, CPU, m) { FCT_IMPLS(m) }

TORCH_LIBRARY_IMPL(flashcart, Autograd, m) {
  m.impl("embedding", TORCH_FN(embedding_autograd));
  m.impl("embedding_bwd", TORCH_FN(embedding_bwd_autograd));
  m.impl("dropout_add", TORCH_FN(dropout_add_autograd));
  m.impl("gated_feed_forward", TORCH_FN(gated_feed_forward_autograd));
  m.impl("gated_feed_forward_bwd", TORCH_FN(gated_feed_forward_bwd_autograd));
}
