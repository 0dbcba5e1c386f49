// flagos:: ops of a training step around the matrix products: rotary
// positions without a table, the norms around a block with its gate and
// residual add, softmax over spans of keys, and the clipping of gradients.
// Autograd is registered natively beside them.
#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>

#include "fused_common.h"
#include "layer_ops.h"

namespace flb200::aten {
namespace {

// ------------------------------------------------------------------ rotary --
struct HeadsView {
  int64_t B, H, S, D, sb, sh, ss;
};
HeadsView Heads(const at::Tensor& t, int64_t unsqueeze_dim) {
  const int h = unsqueeze_dim == 1 ? 1 : 2, s = 3 - h;
  return {t.size(0), t.size(h), t.size(s), t.size(3), t.stride(0), t.stride(h), t.stride(s)};
}

// A result laid out as t where that keeps its heads whole: of overlapping
// views (windows of one row, say) the densest layout has another dim innermost.
at::Tensor HeadsLike(const at::Tensor& t) {
  at::Tensor o = at::empty_like(t);
  return o.size(-1) <= 1 || o.stride(-1) == 1 ? o : at::empty(t.sizes(), t.options());
}

std::tuple<at::Tensor, at::Tensor> Rotary(const at::Tensor& q_in, const at::Tensor& k_in,
                                          const at::Tensor& positions, const at::Tensor& inv_freq, double scale,
                                          bool interleaved, int64_t unsqueeze_dim, bool inverse) {
  const char* op = "flagos::rotary";
  const int code = FloatCode(q_in, op);
  SameDevice(q_in, k_in, op);
  SameDevice(q_in, positions, op);
  SameDevice(q_in, inv_freq, op);
  TORCH_CHECK(k_in.scalar_type() == q_in.scalar_type(), op, ": q and k must share a dtype");
  TORCH_CHECK(q_in.dim() == 4 && k_in.dim() == 4, op, ": q and k must be 4-D");
  TORCH_CHECK(unsqueeze_dim == 1 || unsqueeze_dim == 2, op,
              ": unsqueeze_dim must be 1 ([B,H,S,D]) or 2 ([B,S,H,D])");
  const auto unit = [](const at::Tensor& t) {
    return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
  };
  at::Tensor q = unit(q_in), k = unit(k_in);
  const HeadsView lq = Heads(q, unsqueeze_dim), lk = Heads(k, unsqueeze_dim);
  TORCH_CHECK(lq.B == lk.B && lq.S == lk.S && lq.D == lk.D, op, ": q and k disagree");
  TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, op,
              ": positions must be int32 or int64, got ", positions.scalar_type());
  TORCH_CHECK((positions.dim() == 1 || (positions.dim() == 2 && (positions.size(0) == lq.B || positions.size(0) == 1))) &&
                  positions.size(-1) == lq.S,
              op, ": positions must be [seq] or [batch, seq]");
  TORCH_CHECK(inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1 && inv_freq.size(0) >= 1 &&
                  2 * inv_freq.size(0) <= lq.D && 2 * inv_freq.size(0) <= FL_B200_ROTARY_MAX,
              op, ": inv_freq must be float32 [n] with 2 n <= head_dim and at most ",
              std::to_string(FL_B200_ROTARY_MAX));
  TORCH_CHECK(std::isfinite(scale), op, ": scale must be finite");
  const int64_t pb = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
  at::Tensor freq = inv_freq.contiguous();
  at::Tensor qo = HeadsLike(q), ko = HeadsLike(k);
  const HeadsView oq = Heads(qo, unsqueeze_dim), ok = Heads(ko, unsqueeze_dim);
  if (q.numel() == 0 && k.numel() == 0) return {qo, ko};
  GpuGuard g(q);
  CheckB200(fl_b200_rotary(q.data_ptr(), qo.data_ptr(), lq.H, lq.sb, lq.sh, lq.ss, oq.sb, oq.sh, oq.ss,
                           k.data_ptr(), ko.data_ptr(), lk.H, lk.sb, lk.sh, lk.ss, ok.sb, ok.sh, ok.ss,
                           positions.data_ptr(), pb, positions.stride(-1), B200Dtype(positions.scalar_type()),
                           freq.data_ptr<float>(), 2 * freq.size(0), (float)scale, interleaved, inverse, lq.B,
                           lq.S, lq.D, code, StreamOf(q)),
            op);
  return {qo, ko};
}

// ----------------------------------------------------------- sandwich norm --
// How many of x's rows share a row of the gate: the gate is [cols], or has
// x's dims with sizes that agree up to some dim and are 1 after it.
int64_t RowsPerGate(const at::Tensor& x, const at::Tensor& gate, const char* op) {
  const int64_t rows = x.size(-1) ? x.numel() / x.size(-1) : 0;
  if (gate.dim() == 1) return std::max<int64_t>(rows, 1);
  int64_t per = 1;
  int64_t d = x.dim() - 2;
  for (; d >= 0 && gate.size(d) == 1; --d) per *= x.size(d);
  for (; d >= 0; --d)
    TORCH_CHECK(gate.size(d) == x.size(d), op,
                ": gate must be [hidden], or x's shape with the last dims before hidden 1");
  return std::max<int64_t>(per, 1);
}
void SandwichArgs(const at::Tensor& x, const at::Tensor& like, const at::Tensor& post, const at::Tensor& pre,
                  const std::optional<at::Tensor>& gate, double eps, double scale, double offset, const char* op) {
  SameDevice(x, like, op);
  SameDevice(x, post, op);
  SameDevice(x, pre, op);
  TORCH_CHECK(x.dim() >= 1 && x.sizes() == like.sizes() && x.scalar_type() == like.scalar_type(), op,
              ": x and the residual must match");
  for (const at::Tensor* w : {&post, &pre})
    TORCH_CHECK(w->scalar_type() == x.scalar_type() && w->dim() == 1 && w->size(0) == x.size(-1), op,
                ": weights must be [hidden] tensors of x's dtype");
  TORCH_CHECK(eps >= 0 && std::isfinite(eps) && std::isfinite(scale) && std::isfinite(offset), op,
              ": eps, scale and weight_offset must be finite, eps at least 0");
  if (gate.has_value() && gate->defined()) {
    SameDevice(x, *gate, op);
    TORCH_CHECK(gate->scalar_type() == x.scalar_type() && (gate->dim() == 1 || gate->dim() == x.dim()) &&
                    gate->size(-1) == x.size(-1),
                op, ": gate must be [hidden], or x's shape with the last dims before hidden 1, of x's dtype");
  }
}

std::tuple<at::Tensor, at::Tensor> SandwichNorm(const at::Tensor& x_in, const at::Tensor& res_in,
                                                const at::Tensor& post_in, const at::Tensor& pre_in,
                                                const std::optional<at::Tensor>& gate_in, double eps,
                                                double scale, double offset) {
  const char* op = "flagos::sandwich_norm";
  const int code = FloatCode(x_in, op);
  SandwichArgs(x_in, res_in, post_in, pre_in, gate_in, eps, scale, offset, op);
  at::Tensor x, res, gate;
  const RowsView rx = Rows(x_in, x), rr = Rows(res_in, res);
  at::Tensor post = post_in.contiguous(), pre = pre_in.contiguous();
  int64_t per = 1;
  if (gate_in.has_value() && gate_in->defined()) {
    per = RowsPerGate(x_in, *gate_in, op);
    gate = gate_in->contiguous();
  }
  at::Tensor y = at::empty(x_in.sizes(), x.options()), h = at::empty(x_in.sizes(), x.options());
  if (y.numel() == 0) return {y, h};
  GpuGuard g(x);
  CheckB200(fl_b200_sandwich_norm(x.data_ptr(), rx.ld, res.data_ptr(), rr.ld, post.data_ptr(), pre.data_ptr(),
                                  gate.defined() ? gate.data_ptr() : nullptr, per, y.data_ptr(), h.data_ptr(),
                                  rx.rows, rx.cols, (float)eps, (float)scale, (float)offset, code, StreamOf(x)),
            op);
  return {y, h};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> SandwichNormBackward(
    const at::Tensor& dy_in, const std::optional<at::Tensor>& dh_in, const at::Tensor& x_in, const at::Tensor& h_in,
    const at::Tensor& post_in, const at::Tensor& pre_in, const std::optional<at::Tensor>& gate_in, double eps,
    double scale, double offset) {
  const char* op = "flagos::sandwich_norm_backward";
  const int code = FloatCode(x_in, op);
  SandwichArgs(x_in, h_in, post_in, pre_in, gate_in, eps, scale, offset, op);
  SandwichArgs(x_in, dy_in, post_in, pre_in, gate_in, eps, scale, offset, op);
  at::Tensor x, h, dy, dh, gate;
  const RowsView rx = Rows(x_in, x), rh = Rows(h_in, h), ry = Rows(dy_in, dy);
  RowsView rd{0, 0, 0};
  if (dh_in.has_value() && dh_in->defined()) {
    SandwichArgs(x_in, *dh_in, post_in, pre_in, gate_in, eps, scale, offset, op);
    rd = Rows(*dh_in, dh);
  }
  at::Tensor post = post_in.contiguous(), pre = pre_in.contiguous();
  int64_t per = 1;
  at::Tensor dgate;
  if (gate_in.has_value() && gate_in->defined()) {
    per = RowsPerGate(x_in, *gate_in, op);
    gate = gate_in->contiguous();
    dgate = at::empty(gate_in->sizes(), x.options());
  } else {
    dgate = at::empty({0}, x.options());
  }
  at::Tensor dx = at::empty(x_in.sizes(), x.options()), dres = at::empty(x_in.sizes(), x.options());
  at::Tensor dpost = at::empty({x_in.size(-1)}, x.options()), dpre = at::empty({x_in.size(-1)}, x.options());
  GpuGuard g(x);
  if (x_in.numel() == 0 && dgate.numel()) dgate.zero_();
  const int64_t rows = x_in.size(-1) ? x_in.numel() / x_in.size(-1) : 0;
  const size_t nws = fl_b200_sandwich_norm_bwd_workspace_size(rows, rx.cols);
  at::Tensor ws = at::empty({(int64_t)std::max<size_t>(nws, 16)}, x.options().dtype(at::kByte));
  CheckB200(fl_b200_sandwich_norm_bwd(
                dy.data_ptr(), ry.ld, dh.defined() ? dh.data_ptr() : nullptr, rd.ld, x.data_ptr(), rx.ld,
                h.data_ptr(), rh.ld, post.data_ptr(), pre.data_ptr(), gate.defined() ? gate.data_ptr() : nullptr,
                per, dx.data_ptr(), dres.data_ptr(), dpost.data_ptr(), dpre.data_ptr(),
                gate.defined() ? dgate.data_ptr() : nullptr, rows, rx.cols, (float)eps, (float)scale,
                (float)offset, code, ws.data_ptr(), nws, StreamOf(x)),
            op);
  return {dx, dres, dpost, dpre, dgate};
}

// ------------------------------------------------------------ span softmax --
// int32 data over (batch, query) as a tensor and its strides.
at::Tensor PerQuery(const at::Tensor& t, int64_t B, int64_t Q, int64_t tail, int64_t* sb, int64_t* sq,
                    const char* name, const char* op) {
  TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
  at::Tensor u = tail ? t : t.unsqueeze(-1);
  if (u.dim() == 2) u = u.unsqueeze(0);
  TORCH_CHECK(u.dim() == 3 && (u.size(0) == B || u.size(0) == 1) && u.size(1) == Q && (!tail || u.size(2) == tail),
              op, ": ", name, " must be [queries", tail ? ", 2" : "", "] or [batch, queries", tail ? ", 2]" : "]");
  if (tail && u.stride(2) != 1) u = u.contiguous();
  *sb = u.size(0) == 1 ? 0 : u.stride(0);
  *sq = u.stride(1);
  return u;
}
// The scores' sizes as [B, H, Q, K].
struct Scores {
  int64_t B, H, Q, K;
};
Scores ScoresOf(const at::Tensor& x, const char* op) {
  TORCH_CHECK(x.dim() >= 2 && x.dim() <= 4, op, ": x must be [Q, K], [H, Q, K] or [B, H, Q, K]");
  return {x.dim() == 4 ? x.size(0) : 1, x.dim() >= 3 ? x.size(-3) : 1, x.size(-2), x.size(-1)};
}
float Cap(std::optional<double> cap, const char* op) {
  if (!cap.has_value()) return 0.f;
  TORCH_CHECK((float)*cap > 1e-30f && (float)*cap < 1e30f, op, ": cap must be positive and finite, got ",
              std::to_string(*cap));
  return (float)*cap;
}

at::Tensor SpanSoftmax(const at::Tensor& x_in, const at::Tensor& spans_in, double scale, std::optional<double> cap,
                       const std::optional<at::Tensor>& slopes_in, const std::optional<at::Tensor>& pos_in,
                       std::optional<at::ScalarType> dtype) {
  const char* op = "flagos::span_softmax";
  const int ci = FloatCode(x_in, op);
  const at::ScalarType ot = dtype.value_or(x_in.scalar_type());
  const int co = B200Dtype(ot);
  TORCH_CHECK(co == ci || co == FL_B200_F32, op, ": output dtype must be the input's or float32");
  const Scores s = ScoresOf(x_in, op);
  SameDevice(x_in, spans_in, op);
  TORCH_CHECK(std::isfinite(scale), op, ": scale must be finite");
  const float cp = Cap(cap, op);
  int64_t sb, sq, pb = 0, pq = 0;
  at::Tensor spans = PerQuery(spans_in, s.B, s.Q, 2, &sb, &sq, "spans", op), pos, slopes;
  if (pos_in.has_value() && pos_in->defined()) {
    SameDevice(x_in, *pos_in, op);
    pos = PerQuery(*pos_in, s.B, s.Q, 0, &pb, &pq, "positions", op);
  }
  if (slopes_in.has_value() && slopes_in->defined()) {
    SameDevice(x_in, *slopes_in, op);
    TORCH_CHECK(slopes_in->scalar_type() == at::kFloat && slopes_in->dim() == 1 && slopes_in->size(0) == s.H, op,
                ": slopes must be a float32 [heads] tensor");
    slopes = slopes_in->contiguous();
  }
  at::Tensor x;
  const RowsView r = Rows(x_in, x);
  at::Tensor out = at::empty(x_in.sizes(), x.options().dtype(ot));
  if (out.numel() == 0) return out;
  GpuGuard g(x);
  CheckB200(fl_b200_span_softmax(x.data_ptr(), r.ld, spans.data_ptr<int32_t>(), sb, sq,
                                 pos.defined() ? pos.data_ptr<int32_t>() : nullptr, pb, pq,
                                 slopes.defined() ? slopes.data_ptr<float>() : nullptr, out.data_ptr(), s.K,
                                 r.rows, s.K, s.H, s.Q, (float)scale, cp, ci, co, StreamOf(x)),
            op);
  return out;
}

at::Tensor SpanSoftmaxBackward(const at::Tensor& dy_in, const at::Tensor& y_in, const at::Tensor& x_in,
                               const at::Tensor& spans_in, double scale, std::optional<double> cap) {
  const char* op = "flagos::span_softmax_backward";
  const int cx = FloatCode(x_in, op), cy = FloatCode(y_in, op);
  TORCH_CHECK(cy == cx || cy == FL_B200_F32, op, ": y must have x's dtype or float32");
  SameDevice(x_in, y_in, op);
  SameDevice(x_in, dy_in, op);
  SameDevice(x_in, spans_in, op);
  TORCH_CHECK(dy_in.sizes() == y_in.sizes() && dy_in.scalar_type() == y_in.scalar_type() &&
                  y_in.sizes() == x_in.sizes(),
              op, ": dy, y and x must match");
  const Scores s = ScoresOf(y_in, op);
  TORCH_CHECK(std::isfinite(scale), op, ": scale must be finite");
  const float cp = Cap(cap, op);
  int64_t sb, sq;
  at::Tensor spans = PerQuery(spans_in, s.B, s.Q, 2, &sb, &sq, "spans", op);
  at::Tensor dx = at::empty(x_in.sizes(), x_in.options());
  if (dx.numel() == 0) return dx;
  at::Tensor dy, y, x;
  const RowsView rd = Rows(dy_in, dy), ry = Rows(y_in, y);
  int64_t ldx = s.K;
  if (cp > 0.f) ldx = Rows(x_in, x).ld;
  GpuGuard g(y);
  CheckB200(fl_b200_span_softmax_bwd(dy.data_ptr(), rd.ld, y.data_ptr(), ry.ld, cp > 0.f ? x.data_ptr() : nullptr,
                                     ldx, spans.data_ptr<int32_t>(), sb, sq, dx.data_ptr(), s.K, ry.rows, s.K, s.H,
                                     s.Q, (float)scale, cp, cy, cx, StreamOf(y)),
            op);
  return dx;
}

// ------------------------------------------------------- gradient clipping --
// The list's addresses, counts and types.
struct GradList {
  std::vector<const void*> in;
  std::vector<void*> out;
  std::vector<int64_t> numel;
  std::vector<int> dtype;
  explicit GradList(size_t n) {
    in.reserve(n), out.reserve(n), numel.reserve(n), dtype.reserve(n);
  }
  void add(const at::Tensor& t) {
    in.push_back(t.const_data_ptr());
    numel.push_back(t.numel());
    dtype.push_back(B200Dtype(t.scalar_type()));
  }
};
// Tensors may come here without the dispatcher: nothing but memory of the
// first one's GPU is taken.
void CheckGrad(const at::Tensor& t, const at::Tensor& first, const char* op) {
  TORCH_CHECK(t.defined() && (t.is_cuda() || t.is_privateuseone()) && t.layout() == at::kStrided && !t.is_neg(), op,
              ": dense tensors on a GPU expected");
  SameDevice(first, t, op);
  (void)FloatCode(t, op);
}
int NormKind(double norm_type, const char* op) {
  TORCH_CHECK(norm_type == 2.0 || norm_type == INFINITY, op, ": norm_type must be 2 or inf, got ",
              std::to_string(norm_type));
  return norm_type == 2.0 ? 0 : 1;
}
at::Tensor GradWorkspace(const at::Tensor& t, int64_t count) {
  return at::empty({(int64_t)std::max<size_t>(fl_b200_grad_norm_workspace_size(count), 16)},
                   t.options().dtype(at::kByte));
}

std::tuple<std::vector<at::Tensor>, at::Tensor> ClipGrads(at::TensorList grads, double max_norm, double norm_type) {
  std::vector<at::Tensor> out;
  out.reserve(grads.size());
  for (const at::Tensor& t : grads) out.push_back(at::empty_like(t));
  at::Tensor norm = ClipGradsOut(grads, max_norm, norm_type, out);
  return {out, norm};
}

// ------------------------------------------------------------- autograd --
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradients' own gradients where a graph of them is wanted: there are
// none, which is said when they are asked for.
#define FLB_NO_SECOND(name)                                        \
  static variable_list backward(AutogradContext*, variable_list) { \
    TORCH_CHECK(false, name ": there is no second derivative");    \
  }

using RotaryFn = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                    const at::Tensor&, double, bool, int64_t, bool);
const c10::TypedOperatorHandle<RotaryFn>& RotaryOp() { return FLB_OP(RotaryFn, "flagos::rotary"); }

// Linear in q and k: the gradient is the same op the other way round, which
// carries its own gradient.
struct RotaryGrad : torch::autograd::Function<RotaryGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                               const at::Tensor& positions, const at::Tensor& inv_freq, double scale,
                               bool interleaved, int64_t unsqueeze_dim, bool inverse) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [qo, ko] = RotaryOp().call(q, k, positions, inv_freq, scale, interleaved, unsqueeze_dim, inverse);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["unsqueeze_dim"] = unsqueeze_dim;
    ctx->saved_data["inverse"] = inverse;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool need_q = ctx->needs_input_grad(0) && grads[0].defined();
    const bool need_k = ctx->needs_input_grad(1) && grads[1].defined();
    variable_list out(8);
    if (!need_q && !need_k) return out;
    const auto saved = ctx->get_saved_variables();
    const int64_t dim = ctx->saved_data["unsqueeze_dim"].toInt();
    // the one without a gradient goes along without heads
    const at::Tensor& some = need_q ? grads[0] : grads[1];
    const at::Tensor none = some.narrow(dim == 1 ? 1 : 2, 0, 0);
    auto [dq, dk] = RotaryOp().call(need_q ? grads[0] : none, need_k ? grads[1] : none, saved[0], saved[1],
                                    ctx->saved_data["scale"].toDouble(), ctx->saved_data["interleaved"].toBool(),
                                    dim, !ctx->saved_data["inverse"].toBool());
    if (need_q) out[0] = dq;
    if (need_k) out[1] = dk;
    return out;
  }
};
std::tuple<at::Tensor, at::Tensor> RotaryAutograd(const at::Tensor& q, const at::Tensor& k,
                                                  const at::Tensor& positions, const at::Tensor& inv_freq,
                                                  double scale, bool interleaved, int64_t unsqueeze_dim,
                                                  bool inverse) {
  NoTangent(q, "flagos::rotary");
  NoTangent(k, "flagos::rotary");
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(!inv_freq.requires_grad(), "flagos::rotary: inv_freq has no gradient");
    if (q.requires_grad() || k.requires_grad()) {
      auto out = RotaryGrad::apply(q, k, positions, inv_freq, scale, interleaved, unsqueeze_dim, inverse);
      return {out[0], out[1]};
    }
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return RotaryOp().call(q, k, positions, inv_freq, scale, interleaved, unsqueeze_dim, inverse);
}

using SandwichFn = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                      const at::Tensor&, const std::optional<at::Tensor>&, double,
                                                      double, double);
using Five = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
using SandwichBackwardFn = Five(const at::Tensor&, const std::optional<at::Tensor>&, const at::Tensor&,
                                const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                const std::optional<at::Tensor>&, double, double, double);

struct SandwichGradGrad : torch::autograd::Function<SandwichGradGrad> {
  static variable_list forward(AutogradContext*, const at::Tensor& dy, const std::optional<at::Tensor>& dh,
                               const at::Tensor& x, const at::Tensor& h, const at::Tensor& post,
                               const at::Tensor& pre, const std::optional<at::Tensor>& gate, double eps,
                               double scale, double offset) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [a, b, c, d, e] = FLB_OP(SandwichBackwardFn, "flagos::sandwich_norm_backward")
                               .call(dy, dh, x, h, post, pre, gate, eps, scale, offset);
    return {a, b, c, d, e};
  }
  FLB_NO_SECOND("flagos::sandwich_norm")
};
Five SandwichBackwardAutograd(const at::Tensor& dy, const std::optional<at::Tensor>& dh, const at::Tensor& x,
                              const at::Tensor& h, const at::Tensor& post, const at::Tensor& pre,
                              const std::optional<at::Tensor>& gate, double eps, double scale, double offset) {
  const auto wants = [](const std::optional<at::Tensor>& t) {
    return t.has_value() && t->defined() && t->requires_grad();
  };
  if (at::GradMode::is_enabled() && (dy.requires_grad() || wants(dh) || x.requires_grad() || h.requires_grad() ||
                                     post.requires_grad() || pre.requires_grad() || wants(gate))) {
    auto out = SandwichGradGrad::apply(dy, dh, x, h, post, pre, gate, eps, scale, offset);
    return {out[0], out[1], out[2], out[3], out[4]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(SandwichBackwardFn, "flagos::sandwich_norm_backward")
      .call(dy, dh, x, h, post, pre, gate, eps, scale, offset);
}
struct SandwichGrad : torch::autograd::Function<SandwichGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual,
                               const at::Tensor& post, const at::Tensor& pre,
                               const std::optional<at::Tensor>& gate, double eps, double scale, double offset) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, h] = FLB_OP(SandwichFn, "flagos::sandwich_norm").call(x, residual, post, pre, gate, eps, scale, offset);
    ctx->set_materialize_grads(false);
    const bool gated = gate.has_value() && gate->defined();
    ctx->save_for_backward({x, h, post, pre, gated ? *gate : at::Tensor()});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["offset"] = offset;
    return {y, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(8);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor dy = grads[0].defined() ? grads[0] : at::zeros_like(saved[0]);
    const std::optional<at::Tensor> dh = grads[1].defined() ? std::optional<at::Tensor>(grads[1]) : std::nullopt;
    const std::optional<at::Tensor> gate =
        saved[4].defined() ? std::optional<at::Tensor>(saved[4]) : std::nullopt;
    const auto call = at::GradMode::is_enabled() ? SandwichBackwardAutograd : SandwichNormBackward;
    auto [dx, dres, dpost, dpre, dgate] =
        call(dy, dh, saved[0], saved[1], saved[2], saved[3], gate, ctx->saved_data["eps"].toDouble(),
             ctx->saved_data["scale"].toDouble(), ctx->saved_data["offset"].toDouble());
    const at::Tensor all[] = {dx, dres, dpost, dpre, dgate};
    for (int i = 0; i < (gate.has_value() ? 5 : 4); ++i)
      if (ctx->needs_input_grad(i)) out[i] = all[i];
    return out;
  }
};
std::tuple<at::Tensor, at::Tensor> SandwichAutograd(const at::Tensor& x, const at::Tensor& residual,
                                                    const at::Tensor& post, const at::Tensor& pre,
                                                    const std::optional<at::Tensor>& gate, double eps, double scale,
                                                    double offset) {
  bool grad = false;
  for (const at::Tensor* t : {&x, &residual, &post, &pre}) {
    NoTangent(*t, "flagos::sandwich_norm");
    grad |= t->requires_grad();
  }
  if (gate.has_value() && gate->defined()) {
    NoTangent(*gate, "flagos::sandwich_norm");
    grad |= gate->requires_grad();
  }
  if (at::GradMode::is_enabled() && grad) {
    auto out = SandwichGrad::apply(x, residual, post, pre, gate, eps, scale, offset);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(SandwichFn, "flagos::sandwich_norm").call(x, residual, post, pre, gate, eps, scale, offset);
}

using SpanFn = at::Tensor(const at::Tensor&, const at::Tensor&, double, std::optional<double>,
                          const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                          std::optional<at::ScalarType>);
using SpanBackwardFn = at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, double,
                                  std::optional<double>);

struct SpanGradGrad : torch::autograd::Function<SpanGradGrad> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& dy, const at::Tensor& y, const at::Tensor& x,
                            const at::Tensor& spans, double scale, std::optional<double> cap) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return FLB_OP(SpanBackwardFn, "flagos::span_softmax_backward").call(dy, y, x, spans, scale, cap);
  }
  FLB_NO_SECOND("flagos::span_softmax")
};
at::Tensor SpanBackwardAutograd(const at::Tensor& dy, const at::Tensor& y, const at::Tensor& x,
                                const at::Tensor& spans, double scale, std::optional<double> cap) {
  if (at::GradMode::is_enabled() && (dy.requires_grad() || y.requires_grad() || x.requires_grad()))
    return SpanGradGrad::apply(dy, y, x, spans, scale, cap);
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(SpanBackwardFn, "flagos::span_softmax_backward").call(dy, y, x, spans, scale, cap);
}
// Saves y, and x only where the cap's slope needs it (else an empty tensor of
// x's type stands for it: the gradient takes its dtype).
struct SpanGrad : torch::autograd::Function<SpanGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& spans, double scale,
                            std::optional<double> cap, const std::optional<at::Tensor>& slopes,
                            const std::optional<at::Tensor>& positions, std::optional<at::ScalarType> dtype) {
    at::AutoDispatchBelowADInplaceOrView guard;
    at::Tensor y = FLB_OP(SpanFn, "flagos::span_softmax").call(x, spans, scale, cap, slopes, positions, dtype);
    ctx->save_for_backward({y, spans, cap.has_value() ? x : at::Tensor()});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    ctx->saved_data["dtype"] = x.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    const auto saved = ctx->get_saved_variables();
    const auto cap = ctx->saved_data["cap"].toOptional<double>();
    // (without a cap x is not read: y's shape in x's type says what dx is)
    at::Tensor x = saved[2];
    if (!x.defined()) {
      const auto type = ctx->saved_data["dtype"].toScalarType();
      x = type == saved[0].scalar_type() ? saved[0].detach()
                                         : at::empty({1}, saved[0].options().dtype(type)).expand(saved[0].sizes());
    }
    const auto call = at::GradMode::is_enabled() ? SpanBackwardAutograd : SpanSoftmaxBackward;
    out[0] = call(grads[0], saved[0], x, saved[1], ctx->saved_data["scale"].toDouble(), cap);
    return out;
  }
};
at::Tensor SpanAutograd(const at::Tensor& x, const at::Tensor& spans, double scale, std::optional<double> cap,
                        const std::optional<at::Tensor>& slopes, const std::optional<at::Tensor>& positions,
                        std::optional<at::ScalarType> dtype) {
  NoTangent(x, "flagos::span_softmax");
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(!slopes.has_value() || !slopes->defined() || !slopes->requires_grad(),
                "flagos::span_softmax: slopes have no gradient");
    if (x.requires_grad()) return SpanGrad::apply(x, spans, scale, cap, slopes, positions, dtype);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(SpanFn, "flagos::span_softmax").call(x, spans, scale, cap, slopes, positions, dtype);
}

}  // namespace

// Tensors whose elements fill their memory in some order are taken as they lie.
at::Tensor GradNorm(at::TensorList grads, double norm_type) {
  const char* op = "flagos::grad_norm";
  const int kind = NormKind(norm_type, op);
  TORCH_CHECK(!grads.empty(), op, ": no tensors");
  GradList l(grads.size());
  std::vector<at::Tensor> keep;
  for (const at::Tensor& t : grads) {
    CheckGrad(t, grads[0], op);
    if (t.is_non_overlapping_and_dense()) {
      l.add(t);
    } else {
      keep.push_back(t.contiguous());
      l.add(keep.back());
    }
  }
  GpuGuard g(grads[0]);
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  at::Tensor ws = GradWorkspace(grads[0], l.in.size());
  CheckB200(fl_b200_grad_norm(l.in.data(), l.numel.data(), l.dtype.data(), l.in.size(), kind,
                              norm.data_ptr<float>(), ws.data_ptr(), ws.numel(), StreamOf(grads[0])),
            op);
  return norm;
}

at::Tensor ClipGradsOut(at::TensorList grads, double max_norm, double norm_type, at::TensorList out) {
  const char* op = "flagos::clip_grads";
  const int kind = NormKind(norm_type, op);
  TORCH_CHECK(!grads.empty(), op, ": no tensors");
  TORCH_CHECK(max_norm >= 0, op, ": max_norm must be at least 0, got ", std::to_string(max_norm));
  TORCH_CHECK(out.size() == grads.size(), op, ": one output for each tensor");
  GradList l(grads.size());
  std::vector<std::pair<size_t, at::Tensor>> copies;
  for (size_t i = 0; i < grads.size(); ++i) {
    const at::Tensor &t = grads[i], &o = out[i];
    CheckGrad(t, grads[0], op);
    if (!t.is_same(o)) {
      CheckGrad(o, grads[0], op);
      TORCH_CHECK(o.sizes() == t.sizes() && o.scalar_type() == t.scalar_type(), op,
                  ": each output must have its tensor's shape and dtype");
    }
    if (o.is_non_overlapping_and_dense() && (t.is_same(o) || t.strides() == o.strides())) {
      l.add(t);
      l.out.push_back(o.mutable_data_ptr());
    } else {  // a dense copy, clipped in place and copied to where it belongs
      TORCH_CHECK(at::has_internal_overlap(o) != at::MemOverlap::Yes, op,
                  ": an output whose elements share memory (an expanded tensor) cannot be written");
      copies.emplace_back(i, t.clone(at::MemoryFormat::Contiguous));
      l.add(copies.back().second);
      l.out.push_back(copies.back().second.mutable_data_ptr());
    }
  }
  GpuGuard g(grads[0]);
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  at::Tensor ws = GradWorkspace(grads[0], l.in.size());
  CheckB200(fl_b200_clip_grads(l.in.data(), l.out.data(), l.numel.data(), l.dtype.data(), l.in.size(),
                               (float)max_norm, kind, norm.data_ptr<float>(), ws.data_ptr(), ws.numel(),
                               StreamOf(grads[0])),
            op);
  for (const at::Tensor& o : out)  // autograd is told that they were written
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  at::NoGradGuard no_grad;
  for (const auto& [i, c] : copies) out[i].copy_(c);
  return norm;
}

TORCH_LIBRARY_FRAGMENT(flagos, m) {
  m.def("rotary(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, float scale=1.0, "
        "bool interleaved=False, int unsqueeze_dim=1, bool inverse=False) -> (Tensor, Tensor)");
  m.def("sandwich_norm(Tensor x, Tensor residual, Tensor post_weight, Tensor pre_weight, Tensor? gate, "
        "float eps, float scale=1.0, float weight_offset=0.0) -> (Tensor, Tensor)");
  m.def("sandwich_norm_backward(Tensor dy, Tensor? dh, Tensor x, Tensor h, Tensor post_weight, "
        "Tensor pre_weight, Tensor? gate, float eps, float scale=1.0, float weight_offset=0.0) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("span_softmax(Tensor x, Tensor spans, float scale=1.0, float? cap=None, Tensor? slopes=None, "
        "Tensor? positions=None, ScalarType? dtype=None) -> Tensor");
  m.def("span_softmax_backward(Tensor dy, Tensor y, Tensor x, Tensor spans, float scale=1.0, "
        "float? cap=None) -> Tensor");
  m.def("grad_norm(Tensor[] grads, float norm_type=2.0) -> Tensor");
  m.def("clip_grads(Tensor[] grads, float max_norm, float norm_type=2.0) -> (Tensor[], Tensor)");
  m.def("clip_grads_out(Tensor[] grads, float max_norm, float norm_type, Tensor(a!)[] out) -> Tensor");
}

#define FLB_LAYER_IMPLS(m)                                \
  m.impl("rotary", Rotary);                               \
  m.impl("sandwich_norm", SandwichNorm);                  \
  m.impl("sandwich_norm_backward", SandwichNormBackward); \
  m.impl("span_softmax", SpanSoftmax);                    \
  m.impl("span_softmax_backward", SpanSoftmaxBackward);   \
  m.impl("grad_norm", GradNorm);                          \
  m.impl("clip_grads", ClipGrads);                        \
  m.impl("clip_grads_out", ClipGradsOut);

TORCH_LIBRARY_IMPL(flagos, PrivateUse1, m) { FLB_LAYER_IMPLS(m) }
TORCH_LIBRARY_IMPL(flagos, CUDA, m) { FLB_LAYER_IMPLS(m) }
TORCH_LIBRARY_IMPL(flagos, Autograd, m) {
  m.impl("rotary", RotaryAutograd);
  m.impl("sandwich_norm", SandwichAutograd);
  m.impl("sandwich_norm_backward", SandwichBackwardAutograd);
  m.impl("span_softmax", SpanAutograd);
  m.impl("span_softmax_backward", SpanBackwardAutograd);
  // Of gradients, which have no history: not differentiable.
  m.impl("grad_norm", torch::CppFunction::makeFallthrough());
  m.impl("clip_grads", torch::CppFunction::makeFallthrough());
  m.impl("clip_grads_out", torch::CppFunction::makeFallthrough());
}

}  // namespace flb200::aten
