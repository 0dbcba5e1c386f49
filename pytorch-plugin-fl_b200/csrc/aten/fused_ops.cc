// flagos:: fused ops -- the kernels the HF hooks call in place of the
// HuggingFace formulas (transformers models/qwen3/modeling_qwen3.py:59-64,
// 81-82, 138-181, 209-213, 248-268).  Registered for the flagos device and for plain
// CUDA tensors (the memory is the same kind); each op allocates its outputs
// on the input's device and launches on that device's current stream.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "fused_common.h"

namespace flb200::aten {
namespace {

int Rounding(c10::string_view r) {
  if (r == "fused") return FL_B200_ROUND_FUSED;
  if (r == "chain") return FL_B200_ROUND_CHAIN;
  TORCH_CHECK(false, "flagos: rounding must be 'fused' or 'chain', got '", std::string(r), "'");
}

// ---------------------------------------------------------------- RMSNorm --
at::Tensor RmsNorm(const at::Tensor& x_in, const at::Tensor& weight, double eps,
                   c10::string_view rounding) {
  const char* op = "flagos::rms_norm";
  const int code = FloatCode(x_in, op);
  SameDevice(x_in, weight, op);
  TORCH_CHECK(weight.scalar_type() == x_in.scalar_type() && weight.dim() == 1 &&
                  weight.numel() == x_in.size(-1),
              op, ": weight must be a [hidden] tensor of x's dtype");
  at::Tensor x;
  const RowsView r = Rows(x_in, x);
  at::Tensor w = weight.contiguous();
  at::Tensor out = at::empty(x.sizes(), x.options());
  GpuGuard g(x);
  CheckB200(fl_b200_rms_norm_fwd(x.data_ptr(), r.ld, w.data_ptr(), out.data_ptr(), r.cols,
                                 r.rows, r.cols, (float)eps, code, Rounding(rounding),
                                 StreamOf(x)),
            op);
  return out;
}

std::tuple<at::Tensor, at::Tensor> AddRmsNorm(const at::Tensor& x_in, const at::Tensor& res_in,
                                              const at::Tensor& weight, double eps,
                                              c10::string_view rounding) {
  const char* op = "flagos::add_rms_norm";
  const int code = FloatCode(x_in, op);
  SameDevice(x_in, res_in, op);
  SameDevice(x_in, weight, op);
  TORCH_CHECK(x_in.sizes() == res_in.sizes() && x_in.scalar_type() == res_in.scalar_type(),
              op, ": x and residual must match");
  TORCH_CHECK(weight.scalar_type() == x_in.scalar_type() && weight.numel() == x_in.size(-1),
              op, ": weight must be a [hidden] tensor of x's dtype");
  at::Tensor x = x_in.contiguous(), y = res_in.contiguous(), w = weight.contiguous();
  at::Tensor h = at::empty(x.sizes(), x.options());
  at::Tensor out = at::empty(x.sizes(), x.options());
  const int64_t cols = x.size(-1), rows = cols ? x.numel() / cols : 0;
  GpuGuard g(x);
  CheckB200(fl_b200_add_rms_norm_fwd(x.data_ptr(), y.data_ptr(), h.data_ptr(), w.data_ptr(),
                                     out.data_ptr(), rows, cols, (float)eps, code,
                                     Rounding(rounding), StreamOf(x)),
            op);
  return {out, h};
}

// ------------------------------------------------------------------- RoPE --
struct Bhsd {
  int64_t B, H, S, D, sb, sh, ss;
};
Bhsd Layout(const at::Tensor& t, int64_t unsqueeze_dim, const char* op) {
  TORCH_CHECK(t.dim() == 4, op, ": q/k must be 4-D");
  TORCH_CHECK(t.stride(3) == 1, op, ": the head dim must be contiguous");
  if (unsqueeze_dim == 1)  // [B, H, S, D]
    return {t.size(0), t.size(1), t.size(2), t.size(3), t.stride(0), t.stride(1), t.stride(2)};
  TORCH_CHECK(unsqueeze_dim == 2, op, ": unsqueeze_dim must be 1 ([B,H,S,D]) or 2 ([B,S,H,D])");
  return {t.size(0), t.size(2), t.size(1), t.size(3), t.stride(0), t.stride(2), t.stride(1)};
}

// cos/sin as [S, D], [B, S, D] or [B, 1, S, D]: strides over (b, s).
std::pair<int64_t, int64_t> TableStrides(const at::Tensor& c, int64_t B, int64_t S, int64_t D,
                                         const char* op) {
  at::Tensor t = c.dim() == 4 ? c.squeeze(1) : c;
  TORCH_CHECK(t.stride(-1) == 1 || D == 1, op, ": cos/sin last dim must be contiguous");
  if (t.dim() == 2) {
    TORCH_CHECK(t.size(0) == S && t.size(1) == D, op, ": cos/sin shape mismatch");
    return {0, t.stride(0)};
  }
  TORCH_CHECK(t.dim() == 3 && t.size(1) == S && t.size(2) == D && (t.size(0) == B || t.size(0) == 1),
              op, ": cos/sin must be [S, D], [B, S, D] or [B, 1, S, D]");
  return {t.size(0) == 1 ? 0 : t.stride(0), t.stride(1)};
}

std::tuple<at::Tensor, at::Tensor> RopeImpl(const at::Tensor& q, const at::Tensor& k,
                                            const at::Tensor* wq, const at::Tensor* wk,
                                            const at::Tensor& cos, const at::Tensor& sin,
                                            double eps, int64_t unsqueeze_dim,
                                            c10::string_view rounding, const char* op) {
  const int code = FloatCode(q, op);
  SameDevice(q, k, op);
  SameDevice(q, cos, op);
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && cos.scalar_type() == q.scalar_type() &&
                  sin.scalar_type() == q.scalar_type(),
              op, ": q, k, cos and sin must share a dtype");
  const Bhsd lq = Layout(q, unsqueeze_dim, op), lk = Layout(k, unsqueeze_dim, op);
  TORCH_CHECK(lq.B == lk.B && lq.S == lk.S && lq.D == lk.D, op, ": q and k disagree");
  const auto cs = TableStrides(cos, lq.B, lq.S, lq.D, op);
  TORCH_CHECK(TableStrides(sin, lq.B, lq.S, lq.D, op) == cs, op,
              ": cos and sin must share a layout");
  at::Tensor qo = at::empty_like(q), ko = at::empty_like(k);
  const Bhsd oq = Layout(qo, unsqueeze_dim, op), ok = Layout(ko, unsqueeze_dim, op);
  GpuGuard g(q);
  int st;
  if (wq) {
    TORCH_CHECK(wq->numel() == lq.D && wk->numel() == lq.D &&
                    wq->scalar_type() == q.scalar_type() && wk->scalar_type() == q.scalar_type(),
                op, ": q/k norm weights must be [head_dim] tensors of q's dtype");
    at::Tensor wqc = wq->contiguous(), wkc = wk->contiguous();
    st = fl_b200_rms_norm_rope(q.data_ptr(), qo.data_ptr(), lq.H, lq.sb, lq.sh, lq.ss, oq.sb,
                               oq.sh, oq.ss, wqc.data_ptr(), k.data_ptr(), ko.data_ptr(), lk.H,
                               lk.sb, lk.sh, lk.ss, ok.sb, ok.sh, ok.ss, wkc.data_ptr(),
                               cos.data_ptr(), sin.data_ptr(), cs.first, cs.second, lq.B, lq.S,
                               lq.D, (float)eps, code, Rounding(rounding), StreamOf(q));
  } else {
    st = fl_b200_rope_qk(q.data_ptr(), qo.data_ptr(), lq.H, lq.sb, lq.sh, lq.ss, oq.sb, oq.sh,
                         oq.ss, k.data_ptr(), ko.data_ptr(), lk.H, lk.sb, lk.sh, lk.ss, ok.sb,
                         ok.sh, ok.ss, cos.data_ptr(), sin.data_ptr(), cs.first, cs.second,
                         lq.B, lq.S, lq.D, code, Rounding(rounding), StreamOf(q));
  }
  CheckB200(st, op);
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor> RopeQk(const at::Tensor& q, const at::Tensor& k,
                                          const at::Tensor& cos, const at::Tensor& sin,
                                          int64_t unsqueeze_dim, c10::string_view rounding) {
  return RopeImpl(q, k, nullptr, nullptr, cos, sin, 0.0, unsqueeze_dim, rounding,
                  "flagos::rope_qk");
}

std::tuple<at::Tensor, at::Tensor> RmsNormRope(const at::Tensor& q, const at::Tensor& k,
                                               const at::Tensor& q_weight,
                                               const at::Tensor& k_weight,
                                               const at::Tensor& cos, const at::Tensor& sin,
                                               double eps, int64_t unsqueeze_dim,
                                               c10::string_view rounding) {
  return RopeImpl(q, k, &q_weight, &k_weight, cos, sin, eps, unsqueeze_dim, rounding,
                  "flagos::rms_norm_rope");
}

// ----------------------------------------------------------------- SwiGLU --
at::Tensor Swiglu(const at::Tensor& gate_in, const at::Tensor& up_in, c10::string_view rounding) {
  const char* op = "flagos::swiglu";
  const int code = FloatCode(gate_in, op);
  SameDevice(gate_in, up_in, op);
  TORCH_CHECK(gate_in.sizes() == up_in.sizes() && gate_in.scalar_type() == up_in.scalar_type(),
              op, ": gate and up must match");
  at::Tensor g, u;
  const RowsView rg = Rows(gate_in, g), ru = Rows(up_in, u);
  at::Tensor out = at::empty(g.sizes(), g.options());
  GpuGuard guard(g);
  CheckB200(fl_b200_swiglu(g.data_ptr(), rg.ld, u.data_ptr(), ru.ld, out.data_ptr(), rg.cols,
                           rg.rows, rg.cols, code, Rounding(rounding), StreamOf(g)),
            op);
  return out;
}

std::tuple<at::Tensor, at::Tensor> SwigluResidual(const at::Tensor& gate, const at::Tensor& up,
                                                  const at::Tensor& x, const at::Tensor& y,
                                                  c10::string_view rounding) {
  const char* op = "flagos::swiglu_residual";
  const int code = FloatCode(gate, op);
  TORCH_CHECK(gate.sizes() == up.sizes() && x.sizes() == y.sizes() &&
                  gate.scalar_type() == up.scalar_type() && x.scalar_type() == gate.scalar_type() &&
                  y.scalar_type() == gate.scalar_type(),
              op, ": gate/up and x/y must match pairwise and share a dtype");
  TORCH_CHECK(gate.dim() >= 1 && x.dim() >= 1 && gate.numel() / std::max<int64_t>(gate.size(-1), 1) ==
                  x.numel() / std::max<int64_t>(x.size(-1), 1),
              op, ": gate and x must have the same number of rows");
  at::Tensor g = gate.contiguous(), u = up.contiguous(), xc = x.contiguous(), yc = y.contiguous();
  at::Tensor act = at::empty(g.sizes(), g.options()), h = at::empty(xc.sizes(), xc.options());
  const int64_t rows = g.size(-1) ? g.numel() / g.size(-1) : 0;
  GpuGuard guard(g);
  CheckB200(fl_b200_swiglu_residual(g.data_ptr(), u.data_ptr(), act.data_ptr(), g.size(-1),
                                    xc.data_ptr(), yc.data_ptr(), h.data_ptr(), xc.size(-1), rows,
                                    code, Rounding(rounding), StreamOf(g)),
            op);
  return {act, h};
}

// ---------------------------------------------------------- causal softmax --
at::Tensor CausalSoftmax(const at::Tensor& x_in, int64_t offset, std::optional<at::ScalarType> dtype) {
  const char* op = "flagos::causal_softmax";
  const int ci = FloatCode(x_in, op);
  const at::ScalarType ot = dtype.value_or(x_in.scalar_type());
  const int co = B200Dtype(ot);
  TORCH_CHECK(co == ci || co == FL_B200_F32, op, ": output dtype must be the input's or float32");
  TORCH_CHECK(x_in.dim() >= 2, op, ": x must be [..., q_len, k_len]");
  at::Tensor x;
  const RowsView r = Rows(x_in, x);
  at::Tensor out = at::empty(x.sizes(), x.options().dtype(ot));
  GpuGuard g(x);
  CheckB200(fl_b200_softmax_lastdim(x.data_ptr(), r.ld, out.data_ptr(), r.cols, r.rows, r.cols,
                                    ci, co, 1, x.size(-2), offset, StreamOf(x)),
            op);
  return out;
}

// ---------------------------------------------------- masked softmax --
// HF eager attention's `softmax(w * scaling + mask, dtype=float32)
// .to(query.dtype)` (modeling_qwen3.py eager_attention_forward) in one
// launch.  x is [B, H, Q, K] (or fewer leading dims); the mask has x's dtype
// and broadcasts to x (HF's is [B, 1, Q, K]).
at::Tensor MaskedSoftmax(const at::Tensor& x_in, const std::optional<at::Tensor>& mask_in,
                         double scale, std::optional<at::ScalarType> dtype,
                         c10::string_view rounding) {
  const char* op = "flagos::masked_softmax";
  const int ci = FloatCode(x_in, op);
  const at::ScalarType ot = dtype.value_or(x_in.scalar_type());
  const int co = B200Dtype(ot);
  TORCH_CHECK(co == ci || co == FL_B200_F32, op, ": output dtype must be the input's or float32");
  TORCH_CHECK(x_in.dim() >= 2 && x_in.dim() <= 4, op,
              ": x must be [Q, K], [H, Q, K] or [B, H, Q, K]");
  at::Tensor x4 = x_in;
  while (x4.dim() < 4) x4 = x4.unsqueeze(0);
  const int64_t H = x4.size(1), Q = x4.size(2), K = x4.size(3);
  at::Tensor x;
  const RowsView r = Rows(x4, x);
  at::Tensor mask;
  int64_t sb = 0, sh = 0, sq = 0;
  if (mask_in.has_value() && mask_in->defined()) {
    SameDevice(x_in, *mask_in, op);
    TORCH_CHECK(mask_in->scalar_type() == x_in.scalar_type(), op, ": mask must have x's dtype, got ",
                mask_in->scalar_type());
    mask = mask_in->expand(x4.sizes());
    if (K > 1 && mask.stride(3) != 1) mask = mask.contiguous();
    sb = mask.stride(0);
    sh = mask.stride(1);
    sq = mask.stride(2);
  }
  at::Tensor out = at::empty(x4.sizes(), x.options().dtype(ot));
  if (out.numel() == 0) return out.view(x_in.sizes());
  GpuGuard g(x);
  CheckB200(fl_b200_softmax_masked(x.data_ptr(), r.ld, mask.defined() ? mask.data_ptr() : nullptr,
                                   sb, sh, sq, out.data_ptr(), K, r.rows, K, H, Q, (float)scale,
                                   ci, co, Rounding(rounding), StreamOf(x)),
            op);
  return out.view(x_in.sizes());
}

// -------------------------------------------------------------- backward --
// The backward ops the autograd formulas of the fused ops call
// (torch_fl/autograd.py).  fp32 math, one rounding to the output dtype.
std::tuple<at::Tensor, at::Tensor> RmsNormBackward(const at::Tensor& dy_in,
                                                   const at::Tensor& x_in,
                                                   const at::Tensor& weight, double eps) {
  const char* op = "flagos::rms_norm_backward";
  const int code = FloatCode(x_in, op);
  SameDevice(x_in, dy_in, op);
  SameDevice(x_in, weight, op);
  TORCH_CHECK(dy_in.sizes() == x_in.sizes() && dy_in.scalar_type() == x_in.scalar_type(), op,
              ": dy and x must match");
  TORCH_CHECK(weight.scalar_type() == x_in.scalar_type() && weight.dim() == 1 &&
                  weight.numel() == x_in.size(-1),
              op, ": weight must be a [hidden] tensor of x's dtype");
  at::Tensor x, dy;
  const RowsView r = Rows(x_in, x), rd = Rows(dy_in, dy);
  at::Tensor w = weight.contiguous();
  at::Tensor dx = at::empty(x.sizes(), x.options());
  at::Tensor dw = at::empty({r.cols}, w.options());
  GpuGuard g(x);
  const size_t nws = fl_b200_rms_norm_bwd_workspace_size(r.rows, r.cols);
  at::Tensor ws = at::empty({(int64_t)std::max<size_t>(nws, 16)}, x.options().dtype(at::kByte));
  CheckB200(fl_b200_rms_norm_bwd(dy.data_ptr(), rd.ld, x.data_ptr(), r.ld, w.data_ptr(),
                                 dx.data_ptr(), r.cols, dw.data_ptr(), r.rows, r.cols, (float)eps,
                                 code, ws.data_ptr(), nws, StreamOf(x)),
            op);
  return {dx, dw};
}

std::tuple<at::Tensor, at::Tensor> SwigluBackward(const at::Tensor& dout, const at::Tensor& gate,
                                                  const at::Tensor& up) {
  const char* op = "flagos::swiglu_backward";
  const int code = FloatCode(gate, op);
  SameDevice(gate, up, op);
  SameDevice(gate, dout, op);
  TORCH_CHECK(gate.sizes() == up.sizes() && gate.sizes() == dout.sizes() &&
                  up.scalar_type() == gate.scalar_type() &&
                  dout.scalar_type() == gate.scalar_type(),
              op, ": dout, gate and up must match");
  at::Tensor d = dout.contiguous(), g = gate.contiguous(), u = up.contiguous();
  at::Tensor dg = at::empty(g.sizes(), g.options()), du = at::empty(u.sizes(), u.options());
  GpuGuard guard(g);
  CheckB200(fl_b200_swiglu_bwd(d.data_ptr(), g.data_ptr(), u.data_ptr(), dg.data_ptr(),
                               du.data_ptr(), g.numel(), code, StreamOf(g)),
            op);
  return {dg, du};
}

at::Tensor SoftmaxBackward(const at::Tensor& dy_in, const at::Tensor& y_in,
                           std::optional<at::ScalarType> dtype, double scale) {
  const char* op = "flagos::softmax_backward";
  const int ci = FloatCode(y_in, op);
  SameDevice(y_in, dy_in, op);
  TORCH_CHECK(dy_in.sizes() == y_in.sizes() && dy_in.scalar_type() == y_in.scalar_type(), op,
              ": dy and y must match");
  const at::ScalarType ot = dtype.value_or(y_in.scalar_type());
  const int co = B200Dtype(ot);
  TORCH_CHECK(co == ci || (ci == FL_B200_F32 && (co == FL_B200_BF16 || co == FL_B200_F16)), op,
              ": output dtype must be y's, or 16-bit with float32 y");
  at::Tensor y, dy;
  const RowsView r = Rows(y_in, y), rd = Rows(dy_in, dy);
  at::Tensor dx = at::empty(y.sizes(), y.options().dtype(ot));
  GpuGuard g(y);
  CheckB200(fl_b200_softmax_bwd_scaled(dy.data_ptr(), rd.ld, y.data_ptr(), r.ld, dx.data_ptr(),
                                       r.cols, r.rows, r.cols, (float)scale, ci, co, StreamOf(y)),
            op);
  return dx;
}

// ------------------------------------------------- rows of the vocabulary --
// A teacher's top logits, the distillation loss on them, and the
// verification of drafted tokens.
std::tuple<at::Tensor, at::Tensor> Topk(const at::Tensor& x_in, int64_t k) {
  const char* op = "flagos::topk";
  const int code = FloatCode(x_in, op);
  TORCH_CHECK(x_in.dim() >= 1, op, ": x must have at least one dim");
  TORCH_CHECK(k >= 0 && k <= x_in.size(-1) && k <= FL_B200_TOPK_MAX, op, ": k must lie in [0, ",
              std::to_string(std::min<int64_t>(x_in.size(-1), FL_B200_TOPK_MAX)), "], got ", std::to_string(k));
  at::Tensor x;
  const RowsView r = Rows(x_in, x);
  std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = k;
  at::Tensor values = at::empty(sizes, x.options());
  at::Tensor indices = at::empty(sizes, x.options().dtype(at::kLong));
  GpuGuard g(x);
  CheckB200(fl_b200_topk_lastdim(x.data_ptr(), r.ld, r.rows, r.cols, k, values.data_ptr(),
                                 indices.data_ptr<int64_t>(), code, StreamOf(x)),
            op);
  return {values, indices};
}

at::Tensor TopkBackward(const at::Tensor& dvalues, const at::Tensor& indices, int64_t cols) {
  const char* op = "flagos::topk_backward";
  const int code = FloatCode(dvalues, op);
  SameDevice(dvalues, indices, op);
  TORCH_CHECK(dvalues.dim() >= 1 && dvalues.sizes() == indices.sizes() &&
                  indices.scalar_type() == at::kLong,
              op, ": dvalues and int64 indices must match");
  const int64_t k = dvalues.size(-1);
  TORCH_CHECK(cols >= k && k <= FL_B200_TOPK_MAX, op, ": at most min(cols, ",
              std::to_string(FL_B200_TOPK_MAX), ") values a row");
  at::Tensor d = dvalues.contiguous(), i = indices.contiguous();
  std::vector<int64_t> sizes(d.sizes().begin(), d.sizes().end());
  int64_t rows = 1;
  for (size_t n = 0; n + 1 < sizes.size(); ++n) rows *= sizes[n];
  sizes.back() = cols;
  at::Tensor dx = at::empty(sizes, d.options());
  GpuGuard g(d);
  CheckB200(fl_b200_topk_bwd(d.data_ptr(), i.data_ptr<int64_t>(), dx.data_ptr(), rows, cols, k, code,
                             StreamOf(d)),
            op);
  return dx;
}

// The student's rows and the teacher's lists of one call, checked.
struct Distill {
  at::Tensor x, t, ids;
  RowsView rx, rt, ri;
  int code, t_code, ids_code;
  at::IntArrayRef lead;  // logits' leading dims: the loss's shape
};
Distill DistillArgs(const at::Tensor& logits, const at::Tensor& teacher, const at::Tensor& ids,
                    double temperature, const char* op) {
  Distill d;
  d.code = FloatCode(logits, op);
  d.t_code = FloatCode(teacher, op);
  SameDevice(logits, teacher, op);
  SameDevice(logits, ids, op);
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, op,
              ": teacher_ids must be int32 or int64, got ", ids.scalar_type());
  d.ids_code = B200Dtype(ids.scalar_type());
  TORCH_CHECK(logits.dim() >= 1 && teacher.dim() == logits.dim() && teacher.sizes() == ids.sizes(), op,
              ": logits [..., vocab] with teacher_logits and teacher_ids [..., k] expected");
  d.lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK(teacher.sizes().slice(0, teacher.dim() - 1) == d.lead, op,
              ": teacher_logits' leading dims must be the logits'");
  TORCH_CHECK(teacher.size(-1) <= FL_B200_DISTILL_MAX, op, ": at most ", std::to_string(FL_B200_DISTILL_MAX),
              " teacher logits a row, got ", std::to_string(teacher.size(-1)));
  TORCH_CHECK(logits.size(-1) > 0 || logits.numel() == 0, op, ": an empty vocabulary");
  TORCH_CHECK((float)temperature > 1e-37f && (float)temperature <= 3e38f, op,
              ": temperature must be positive and finite, got ", std::to_string(temperature));
  d.rx = Rows(logits, d.x);
  d.rt = Rows(teacher, d.t);
  d.ri = Rows(ids, d.ids);
  int64_t rows = 1;
  for (int64_t n : d.lead) rows *= n;
  d.rx.rows = rows;
  TORCH_CHECK(rows == 0 || d.rx.cols > 0, op, ": an empty vocabulary");
  return d;
}

// Row weights (or dloss) of the loss's shape, or one that broadcasts to it,
// as a pointer and one stride over the rows; undefined: every row 1.
const float* RowWeights(const std::optional<at::Tensor>& w, const Distill& d, at::Tensor& keep,
                        int64_t& stride, const char* name, const char* op) {
  stride = 0;
  if (!w.has_value() || !w->defined()) return nullptr;
  SameDevice(d.x, *w, op);
  TORCH_CHECK(w->scalar_type() == at::kFloat, op, ": ", name, " must be float32, got ", w->scalar_type());
  if (w->sizes() == d.lead && w->is_contiguous()) {
    keep = *w;
    stride = d.rx.rows > 1 ? 1 : 0;
    return keep.data_ptr<float>();
  }
  keep = w->expand(d.lead).reshape({d.rx.rows});
  stride = d.rx.rows > 1 ? keep.stride(0) : 0;
  return keep.data_ptr<float>();
}

std::tuple<at::Tensor, at::Tensor> DistillTopk(const at::Tensor& logits, const at::Tensor& teacher,
                                               const at::Tensor& ids, double temperature) {
  const char* op = "flagos::distill_topk";
  const Distill d = DistillArgs(logits, teacher, ids, temperature, op);
  at::Tensor loss = at::empty(d.lead, d.x.options().dtype(at::kFloat));
  at::Tensor stats = at::empty({d.rx.rows, 2}, loss.options());
  GpuGuard g(d.x);
  CheckB200(fl_b200_distill_topk_fwd(d.x.data_ptr(), d.rx.ld, d.t.data_ptr(), d.rt.ld, d.t_code,
                                     d.ids.data_ptr(), d.ri.ld, d.ids_code, d.rx.rows, d.rx.cols,
                                     d.t.size(-1), (float)temperature, loss.data_ptr<float>(),
                                     stats.data_ptr<float>(), d.code, StreamOf(d.x)),
            op);
  return {loss, stats};
}

std::tuple<at::Tensor, at::Tensor> DistillTopkBackward(const at::Tensor& dloss, const at::Tensor& logits,
                                                       const at::Tensor& stats, const at::Tensor& teacher,
                                                       const at::Tensor& ids, double temperature,
                                                       bool need_logits, bool need_teacher) {
  const char* op = "flagos::distill_topk_backward";
  const Distill d = DistillArgs(logits, teacher, ids, temperature, op);
  SameDevice(logits, stats, op);
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == d.rx.rows &&
                  stats.size(1) == 2 && stats.is_contiguous(),
              op, ": stats must be the forward's [rows, 2] float32 tensor");
  at::Tensor w;
  int64_t ws;
  const float* wp = RowWeights(dloss, d, w, ws, "dloss", op);
  at::Tensor dx = need_logits ? at::empty(logits.sizes(), d.x.options()) : at::empty({0}, d.x.options());
  at::Tensor dt = need_teacher ? at::empty(teacher.sizes(), d.t.options()) : at::empty({0}, d.t.options());
  GpuGuard g(d.x);
  CheckB200(fl_b200_distill_topk_bwd(wp, ws, d.x.data_ptr(), d.rx.ld, stats.data_ptr<float>(),
                                     d.t.data_ptr(), d.rt.ld, d.t_code, d.ids.data_ptr(), d.ri.ld,
                                     d.ids_code, need_logits ? dx.data_ptr() : nullptr, d.rx.cols,
                                     need_teacher ? dt.data_ptr() : nullptr, d.rx.rows, d.rx.cols,
                                     d.t.size(-1), (float)temperature, d.code, StreamOf(d.x)),
            op);
  return {dx, dt};
}

std::tuple<at::Tensor, at::Tensor> DistillTopkGrad(const at::Tensor& logits, const at::Tensor& teacher,
                                                   const at::Tensor& ids, double temperature,
                                                   const std::optional<at::Tensor>& row_weight) {
  const char* op = "flagos::distill_topk_grad";
  const Distill d = DistillArgs(logits, teacher, ids, temperature, op);
  at::Tensor w;
  int64_t ws;
  const float* wp = RowWeights(row_weight, d, w, ws, "row_weight", op);
  at::Tensor loss = at::empty(d.lead, d.x.options().dtype(at::kFloat));
  at::Tensor stats = at::empty({d.rx.rows, 2}, loss.options());
  at::Tensor dx = at::empty(logits.sizes(), d.x.options());
  GpuGuard g(d.x);
  CheckB200(fl_b200_distill_topk_grad(d.x.data_ptr(), d.rx.ld, d.t.data_ptr(), d.rt.ld, d.t_code,
                                      d.ids.data_ptr(), d.ri.ld, d.ids_code, wp, ws, d.rx.rows,
                                      d.rx.cols, d.t.size(-1), (float)temperature,
                                      loss.data_ptr<float>(), stats.data_ptr<float>(), dx.data_ptr(),
                                      d.rx.cols, d.code, StreamOf(d.x)),
            op);
  return {loss, dx};
}

std::tuple<at::Tensor, at::Tensor> VerifyDraft(const at::Tensor& draft_ids, const at::Tensor& target,
                                               const std::optional<at::Tensor>& draft,
                                               const at::Tensor& uniform,
                                               const std::optional<at::Tensor>& draft_lens) {
  const char* op = "flagos::verify_draft";
  const int code = FloatCode(target, op);
  SameDevice(target, draft_ids, op);
  SameDevice(target, uniform, op);
  TORCH_CHECK(draft_ids.dim() == 2 && draft_ids.scalar_type() == at::kLong, op,
              ": draft_ids must be an int64 [batch, drafts] tensor");
  const int64_t B = draft_ids.size(0), K = draft_ids.size(1);
  TORCH_CHECK(target.dim() == 3 && target.size(0) == B && target.size(1) == K + 1, op,
              ": target_probs must be [batch, drafts + 1, vocab]");
  const int64_t V = target.size(2);
  TORCH_CHECK(B == 0 || V > 0, op, ": an empty vocabulary");
  TORCH_CHECK(uniform.dim() == 2 && uniform.size(0) == B && uniform.size(1) == K + 1 &&
                  uniform.scalar_type() == at::kFloat,
              op, ": uniform must be a float32 [batch, drafts + 1] tensor");
  const auto unit = [](const at::Tensor& t) {
    return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
  };
  at::Tensor ids = unit(draft_ids), p = unit(target), u = unit(uniform), q, lens;
  if (draft.has_value() && draft->defined()) {
    SameDevice(target, *draft, op);
    TORCH_CHECK(draft->scalar_type() == target.scalar_type() && draft->dim() == 3 &&
                    draft->size(0) == B && draft->size(1) == K && draft->size(2) == V,
                op, ": draft_probs must be [batch, drafts, vocab] of target_probs' dtype");
    q = unit(*draft);
  }
  if (draft_lens.has_value() && draft_lens->defined()) {
    SameDevice(target, *draft_lens, op);
    TORCH_CHECK(draft_lens->scalar_type() == at::kLong && draft_lens->dim() == 1 &&
                    draft_lens->size(0) == B,
                op, ": draft_lens must be an int64 [batch] tensor");
    lens = draft_lens->contiguous();
  }
  at::Tensor tokens = at::empty({B, K + 1}, ids.options()), accepted = at::empty({B}, ids.options());
  GpuGuard g(p);
  // (without a single drafted token q has no rows, and none is read)
  CheckB200(fl_b200_verify_draft(ids.data_ptr<int64_t>(), ids.stride(0), p.data_ptr(), p.stride(0),
                                 p.stride(1), q.defined() ? q.data_ptr() : nullptr,
                                 q.defined() ? q.stride(0) : 0, q.defined() ? q.stride(1) : 0,
                                 u.data_ptr<float>(), u.stride(0),
                                 lens.defined() ? lens.data_ptr<int64_t>() : nullptr, B, K, V,
                                 tokens.data_ptr<int64_t>(), accepted.data_ptr<int64_t>(), code,
                                 StreamOf(p)),
            op);
  return {tokens, accepted};
}

// ------------------------------------------------------------- autograd --
// Of topk and distill_topk, registered natively: a decode step's or a small
// batch's call is bound by the host, and a formula registered from Python
// costs it 5 us, needed or not.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using TopkFn = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, int64_t);
using TopkBackwardFn = at::Tensor(const at::Tensor&, const at::Tensor&, int64_t);
using DistillFn = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&,
                                                     const at::Tensor&, double);
using DistillBackwardFn = std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&,
                                                             const at::Tensor&, const at::Tensor&,
                                                             const at::Tensor&, double, bool, bool);

// dx = dvalues at the indices, 0 elsewhere: linear in dvalues, whose own
// gradient is dx's, gathered (0 where an index lies outside the row).
struct TopkGradGrad : torch::autograd::Function<TopkGradGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& dvalues, const at::Tensor& indices,
                            int64_t cols) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({indices});
    ctx->saved_data["cols"] = cols;
    return FLB_OP(TopkBackwardFn, "flagos::topk_backward").call(dvalues, indices, cols);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t cols = ctx->saved_data["cols"].toInt();
    const at::Tensor indices = ctx->get_saved_variables()[0];
    const at::Tensor taken = grads[0].gather(-1, indices.clamp(0, std::max<int64_t>(cols - 1, 0)));
    return {at::where(indices.ge(0).logical_and(indices.lt(cols)), taken, at::zeros_like(taken)),
            at::Tensor(), at::Tensor()};
  }
};
at::Tensor TopkBackwardAutograd(const at::Tensor& dvalues, const at::Tensor& indices, int64_t cols) {
  if (at::GradMode::is_enabled() && dvalues.requires_grad()) return TopkGradGrad::apply(dvalues, indices, cols);
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(TopkBackwardFn, "flagos::topk_backward").call(dvalues, indices, cols);
}
struct TopkGrad : torch::autograd::Function<TopkGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, int64_t k) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [values, indices] = FLB_OP(TopkFn, "flagos::topk").call(x, k);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({indices});
    ctx->save_for_backward({indices});
    ctx->saved_data["cols"] = x.size(-1);
    return {values, indices};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
    const auto call = at::GradMode::is_enabled() ? TopkBackwardAutograd : TopkBackward;
    return {call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["cols"].toInt()), at::Tensor()};
  }
};
std::tuple<at::Tensor, at::Tensor> TopkAutograd(const at::Tensor& x, int64_t k) {
  NoTangent(x, "flagos::topk");
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto out = TopkGrad::apply(x, k);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(TopkFn, "flagos::topk").call(x, k);
}

// The gradients where a graph of them is wanted: there is no second
// derivative, which is said when it is asked for.
struct DistillGradGrad : torch::autograd::Function<DistillGradGrad> {
  static variable_list forward(AutogradContext*, const at::Tensor& dloss, const at::Tensor& logits,
                               const at::Tensor& stats, const at::Tensor& teacher, const at::Tensor& ids,
                               double temperature, bool need_logits, bool need_teacher) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [dx, dt] = FLB_OP(DistillBackwardFn, "flagos::distill_topk_backward")
                        .call(dloss, logits, stats, teacher, ids, temperature, need_logits, need_teacher);
    return {dx, dt};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "flagos::distill_topk: there is no second derivative");
  }
};
std::tuple<at::Tensor, at::Tensor> DistillTopkBackwardAutograd(
    const at::Tensor& dloss, const at::Tensor& logits, const at::Tensor& stats, const at::Tensor& teacher,
    const at::Tensor& ids, double temperature, bool need_logits, bool need_teacher) {
  if (at::GradMode::is_enabled() &&
      (dloss.requires_grad() || logits.requires_grad() || teacher.requires_grad())) {
    auto out = DistillGradGrad::apply(dloss, logits, stats, teacher, ids, temperature, need_logits, need_teacher);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(DistillBackwardFn, "flagos::distill_topk_backward")
      .call(dloss, logits, stats, teacher, ids, temperature, need_logits, need_teacher);
}

// Both operands' gradients from the forward's row statistics, which have none.
struct DistillGrad : torch::autograd::Function<DistillGrad> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& teacher,
                               const at::Tensor& ids, double temperature) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [loss, stats] = FLB_OP(DistillFn, "flagos::distill_topk").call(logits, teacher, ids, temperature);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({stats});
    ctx->save_for_backward({logits, teacher, ids, stats});
    ctx->saved_data["temperature"] = temperature;
    return {loss, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool logits = ctx->needs_input_grad(0), teacher = ctx->needs_input_grad(1);
    variable_list none(4);
    if (!grads[0].defined() || (!logits && !teacher)) return none;
    const auto saved = ctx->get_saved_variables();
    const auto call = at::GradMode::is_enabled() ? DistillTopkBackwardAutograd : DistillTopkBackward;
    auto [dx, dt] = call(grads[0], saved[0], saved[3], saved[1], saved[2],
                         ctx->saved_data["temperature"].toDouble(), logits, teacher);
    if (logits) none[0] = dx;
    if (teacher) none[1] = dt;
    return none;
  }
};
std::tuple<at::Tensor, at::Tensor> DistillTopkAutograd(const at::Tensor& logits, const at::Tensor& teacher,
                                                       const at::Tensor& ids, double temperature) {
  NoTangent(logits, "flagos::distill_topk");
  NoTangent(teacher, "flagos::distill_topk");
  if (at::GradMode::is_enabled() && (logits.requires_grad() || teacher.requires_grad())) {
    auto out = DistillGrad::apply(logits, teacher, ids, temperature);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return FLB_OP(DistillFn, "flagos::distill_topk").call(logits, teacher, ids, temperature);
}

}  // namespace

TORCH_LIBRARY(flagos, m) {
  m.def("rms_norm(Tensor x, Tensor weight, float eps, str rounding='fused') -> Tensor");
  m.def("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps, "
        "str rounding='fused') -> (Tensor, Tensor)");
  m.def("rope_qk(Tensor q, Tensor k, Tensor cos, Tensor sin, int unsqueeze_dim=1, "
        "str rounding='fused') -> (Tensor, Tensor)");
  m.def("rms_norm_rope(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, "
        "Tensor sin, float eps, int unsqueeze_dim=1, str rounding='fused') -> (Tensor, Tensor)");
  m.def("swiglu(Tensor gate, Tensor up, str rounding='fused') -> Tensor");
  m.def("swiglu_residual(Tensor gate, Tensor up, Tensor x, Tensor y, str rounding='fused') "
        "-> (Tensor, Tensor)");
  m.def("causal_softmax(Tensor x, int offset=0, ScalarType? dtype=None) -> Tensor");
  m.def("rms_norm_backward(Tensor dy, Tensor x, Tensor weight, float eps) -> (Tensor, Tensor)");
  m.def("swiglu_backward(Tensor dout, Tensor gate, Tensor up) -> (Tensor, Tensor)");
  m.def("softmax_backward(Tensor dy, Tensor y, ScalarType? dtype=None, float scale=1.0) -> Tensor");
  m.def("masked_softmax(Tensor x, Tensor? mask=None, float scale=1.0, ScalarType? dtype=None, "
        "str rounding='fused') -> Tensor");
  m.def("topk(Tensor x, int k) -> (Tensor, Tensor)");
  m.def("topk_backward(Tensor dvalues, Tensor indices, int cols) -> Tensor");
  m.def("distill_topk(Tensor logits, Tensor teacher_logits, Tensor teacher_ids, "
        "float temperature=1.0) -> (Tensor, Tensor)");
  m.def("distill_topk_backward(Tensor dloss, Tensor logits, Tensor stats, Tensor teacher_logits, "
        "Tensor teacher_ids, float temperature=1.0, bool need_logits=True, "
        "bool need_teacher=False) -> (Tensor, Tensor)");
  m.def("distill_topk_grad(Tensor logits, Tensor teacher_logits, Tensor teacher_ids, "
        "float temperature=1.0, Tensor? row_weight=None) -> (Tensor, Tensor)");
  m.def("verify_draft(Tensor draft_ids, Tensor target_probs, Tensor? draft_probs, Tensor uniform, "
        "Tensor? draft_lens=None) -> (Tensor, Tensor)");
}

#define FLB_FUSED_IMPLS(m)                          \
  m.impl("rms_norm", RmsNorm);                      \
  m.impl("add_rms_norm", AddRmsNorm);               \
  m.impl("rope_qk", RopeQk);                        \
  m.impl("rms_norm_rope", RmsNormRope);             \
  m.impl("swiglu", Swiglu);                         \
  m.impl("swiglu_residual", SwigluResidual);        \
  m.impl("causal_softmax", CausalSoftmax);          \
  m.impl("rms_norm_backward", RmsNormBackward);     \
  m.impl("swiglu_backward", SwigluBackward);        \
  m.impl("softmax_backward", SoftmaxBackward);      \
  m.impl("masked_softmax", MaskedSoftmax);          \
  m.impl("topk", Topk);                             \
  m.impl("topk_backward", TopkBackward);            \
  m.impl("distill_topk", DistillTopk);              \
  m.impl("distill_topk_backward", DistillTopkBackward); \
  m.impl("distill_topk_grad", DistillTopkGrad);     \
  m.impl("verify_draft", VerifyDraft);

TORCH_LIBRARY_IMPL(flagos, PrivateUse1, m) { FLB_FUSED_IMPLS(m) }
TORCH_LIBRARY_IMPL(flagos, CUDA, m) { FLB_FUSED_IMPLS(m) }
TORCH_LIBRARY_IMPL(flagos, Autograd, m) {
  m.impl("topk", TopkAutograd);
  m.impl("topk_backward", TopkBackwardAutograd);
  m.impl("distill_topk", DistillTopkAutograd);
  m.impl("distill_topk_backward", DistillTopkBackwardAutograd);
  // Not differentiable: their results have no history.  (Without a word here
  // PyTorch boxes every call to say so on a backward.)
  m.impl("distill_topk_grad", torch::CppFunction::makeFallthrough());
  m.impl("verify_draft", torch::CppFunction::makeFallthrough());
}

}  // namespace flb200::aten
