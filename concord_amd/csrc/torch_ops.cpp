// torch_ops.cpp -- layer norm, attention and distillation as autograd nodes
// over the C entries of concord_amd.h.
//
// A training step calls these operators many times on few tokens' work, and
// the launches of a small one take less time than an autograd node written in
// Python takes to run (layer norm of 16384 x 384, forward and backward: 23 us
// of kernels; when they took 34, a pass from Python took 127 us, from C++ 65): the
// nodes are C++ for that reason alone.  They check arguments, hand out memory from torch's allocator on the
// current stream and call the entries; the C++ exceptions thrown here become
// Python's (ValueError, TypeError, RuntimeError).
#include "torch_ops.h"

namespace {

// ---- layer norm -----------------------------------------------------------------
const char* const kNorm = "layer_norm";

int norm_check(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  TORCH_CHECK_TYPE(dtype_of(x) >= 0, "layer_norm: x must be float32, bfloat16 or float16 (got ", x.scalar_type(), ")");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: x needs a last dimension of at least 1");
  int wdtype = -1;
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    const char* name = p == &weight ? "weight" : "bias";
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == x.size(-1), "layer_norm: ", name, " must have shape (", x.size(-1),
                      ",), got ", p->sizes());
    const int d = dtype_of(*p);
    TORCH_CHECK_TYPE(d >= 0 && (wdtype < 0 || d == wdtype),
                     "layer_norm: weight and bias must share one of float32, bfloat16, float16");
    TORCH_CHECK_VALUE(p->device() == x.device(), "layer_norm: ", name, " is on ", p->device(), ", x on ", x.device());
    wdtype = d;
  }
  need_gpu(x, kNorm, "x");
  return wdtype < 0 ? CONCORD_F32 : wdtype;
}

// y; with `stats` (fp32 [2, rows]) mean and 1 / deviation too
Tensor norm_forward(const Rows& x, const Tensor& like, const Tensor& weight, const Tensor& bias, int wdtype, double eps,
                    const Tensor& stats) {
  const int64_t width = like.size(-1), rows = like.numel() / width;
  Tensor y = at::empty(like.sizes(), like.options());
  float* mean = stats.defined() && rows ? stats.data_ptr<float>() : nullptr;
  check(concord_layernorm_fwd(ptr(x.t), x.ld, dtype_of(like), ptr(weight), ptr(bias), wdtype, rows, width, (float)eps,
                              ptr(y), width, mean, mean ? mean + rows : nullptr, stream_of(like)),
        kNorm);
  return y;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_,
                        int64_t wdtype, double eps) {
    const Tensor weight = value(weight_), bias = value(bias_);
    const int64_t width = x.size(-1), rows = x.numel() / width;
    const Rows r = rows_of(x, rows, width);
    Tensor stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    Tensor y = norm_forward(r, x, weight, bias, (int)wdtype, eps, stats);
    ctx->save_for_backward({r.t, weight, stats});
    ctx->saved_data["wdtype"] = wdtype;
    ctx->saved_data["has_bias"] = bias.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once(kNorm);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &dy = grads[0];
    const c10::OptionalDeviceGuard guard(dy.device());
    const int64_t width = dy.size(-1), rows = dy.numel() / width, wdtype = ctx->saved_data["wdtype"].toInt();
    const Tensor weight = saved[1].defined() ? saved[1].contiguous() : Tensor(), stats = packed(saved[2]);
    const auto wtype = wdtype == CONCORD_F32 ? at::kFloat : wdtype == CONCORD_BF16 ? at::kBFloat16 : at::kHalf;
    came_back(x, dy.scalar_type(), dy.numel(), dy, kNorm, "x");
    came_back(stats, at::kFloat, 2 * rows, dy, kNorm, "statistics");
    if (weight.defined()) came_back(weight, wtype, width, dy, kNorm, "weight");
    const Rows r = rows_of(x, rows, width), g = rows_of(dy, rows, width);
    Tensor dx = at::empty(dy.sizes(), x.options()), dw, db, ws;
    // (numbered among the tensors that were given)
    const size_t at_bias = weight.defined() ? 2 : 1;
    if (weight.defined() && ctx->needs_input_grad(1)) dw = at::empty({width}, x.options().dtype(wtype));
    if (ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(at_bias))
      db = at::empty({width}, x.options().dtype(wtype));
    size_t need = 0;
    if (dw.defined() || db.defined()) {
      need = concord_layernorm_workspace_bytes(rows, width);
      ws = bytes(need, x);
    }
    float* mean = stats.data_ptr<float>();
    check(concord_layernorm_bwd(ptr(g.t), g.ld, ptr(r.t), r.ld, dtype_of(x), ptr(weight), (int)wdtype, mean, mean + rows,
                                rows, width, ptr(dx), width, ptr(dw), ptr(db), ptr(ws), need, stream_of(x)),
          "layer_norm backward");
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, double eps) {
  Tensor weight = value(weight_), bias = value(bias_);
  no_tangent(kNorm, {&x, &weight, &bias});
  const int wdtype = norm_check(x, weight, bias);
  const c10::OptionalDeviceGuard guard(x.device());
  if (weight.defined()) weight = weight.contiguous();
  if (bias.defined()) bias = bias.contiguous();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LayerNormNode::apply(x, maybe(weight), maybe(bias), (int64_t)wdtype, eps);
  const int64_t width = x.size(-1);
  return norm_forward(rows_of(x, x.numel() / width, width), x, weight, bias, wdtype, eps, Tensor());
}

// ---- attention --------------------------------------------------------------------
const char* const kAttn = "attention";

void attn_check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts, const Tensor& k_starts,
                double scale) {
  for (const Tensor* t : {&q, &k, &v}) {
    const char* name = t == &q ? "q" : t == &k ? "k" : "v";
    TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16, "attention: ", name, " must be bfloat16 (got ", t->scalar_type(),
                     ")");
    TORCH_CHECK_VALUE(t->dim() == q.dim() && (t->dim() == 3 || t->dim() == 4),
                      "attention: q, k and v must all be [token, head, dim] or [batch, token, head, dim]");
    TORCH_CHECK_VALUE(t->device() == q.device(), "attention: ", name, " is on ", t->device(), ", q on ", q.device());
  }
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "attention: k ", k.sizes(), " and v ", v.sizes(), " differ");
  const int64_t h = q.size(-2), hk = k.size(-2), d = q.size(-1);
  TORCH_CHECK_VALUE(k.size(-1) == d && d % 8 == 0 && d >= 8 && d <= 128,
                    "attention: q and k need one head dimension, a multiple of 8 up to 128 (got ", d, " and ", k.size(-1),
                    ")");
  TORCH_CHECK_VALUE(h >= 1 && hk >= 1 && h % hk == 0, "attention: ", h, " query heads do not share ", hk,
                    " key heads evenly");
  TORCH_CHECK_VALUE(scale > 0 && std::isfinite(scale), "attention: the scale must be positive (got ", scale, ")");
  if (q.dim() == 4) {
    TORCH_CHECK_VALUE(!starts.defined() && !k_starts.defined(),
                      "attention: starts are for [token, head, dim] tensors");
    TORCH_CHECK_VALUE(q.size(0) == k.size(0), "attention: ", q.size(0), " sequences of queries, ", k.size(0), " of keys");
  } else {
    TORCH_CHECK_VALUE(starts.defined() || !k_starts.defined(), "attention: k_starts without starts");
    for (const Tensor* s : {&starts, &k_starts}) {
      if (!s->defined()) continue;
      TORCH_CHECK_VALUE(s->scalar_type() == at::kInt && s->dim() == 1 && s->numel() >= 1 && s->device() == q.device(),
                        "attention: ", s == &starts ? "starts" : "k_starts", " must be a 1-d int32 tensor on ", q.device(),
                        ", one value longer than the count of sequences");
    }
    TORCH_CHECK_VALUE(!k_starts.defined() || k_starts.numel() == starts.numel(),
                      "attention: starts and k_starts count different sequences");
    TORCH_CHECK_VALUE(!starts.defined() || k_starts.defined() || q.size(0) == k.size(0),
                      "attention: k_starts is needed where q and k have different token counts");
  }
  need_gpu(q, kAttn, "q");
}

// the part of the arguments that both passes share
concord_attn_args attn_args(const Operand& q, const Operand& k, const Operand& v, const Operand& out,
                            const Tensor& lse, const Tensor& low, const Tensor& starts, const Tensor& k_starts,
                            bool causal, double scale) {
  concord_attn_args a{};
  a.q = (const uint16_t*)ptr(q.t), a.q_t = q.token, a.q_h = q.head;
  a.k = (const uint16_t*)ptr(k.t), a.k_t = k.token, a.k_h = k.head;
  a.v = (const uint16_t*)ptr(v.t), a.v_t = v.token, a.v_h = v.head;
  const int64_t h = q.t.size(-2), d = q.t.size(-1), hk = k.t.size(-2);
  a.out = (uint16_t*)ptr(out.t), a.o_t = out.token, a.o_h = out.head;
  a.lse = (float*)ptr(lse), a.out_low = (int8_t*)ptr(low);
  a.starts = (const int32_t*)ptr(starts), a.k_starts = (const int32_t*)ptr(k_starts);
  const int64_t batch = q.t.dim() == 4 ? q.t.size(0) : 1;
  a.B = starts.defined() ? starts.numel() - 1 : batch;
  a.TQ = batch * q.t.size(-3), a.TK = batch * k.t.size(-3);
  a.H = (int32_t)h, a.HK = (int32_t)hk, a.D = (int32_t)d, a.causal = causal, a.scale = (float)scale;
  return a;
}

// the result as an operand
Operand fresh(const Tensor& out) { return {out, out.size(-2) * out.size(-1), out.size(-1)}; }

void attn_forward(const concord_attn_args& a, const Tensor& q) {
  const size_t need = concord_attention_fwd_workspace_bytes(&a);
  const Tensor ws = need ? bytes(need, q) : Tensor();
  check(concord_attention_fwd(&a, ptr(ws), need, stream_of(q)), kAttn);
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const MaybeTensor& starts_, const MaybeTensor& k_starts_, bool causal, double scale) {
    const Tensor starts = value(starts_), k_starts = value(k_starts_);
    const Operand oq = operand(q), ok = operand(k), ov = operand(v);
    Tensor out = at::empty(q.sizes(), q.options());
    Tensor lse = at::empty({q.numel() / q.size(-1)}, q.options().dtype(at::kFloat));
    Tensor low = at::empty(q.sizes(), q.options().dtype(at::kChar));
    const concord_attn_args a = attn_args(oq, ok, ov, fresh(out), lse, low, starts, k_starts, causal, scale);
    attn_forward(a, q);
    ctx->save_for_backward({oq.t, ok.t, ov.t, out, lse, low, starts, k_starts});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once(kAttn);
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &dout = grads[0];
    const c10::OptionalDeviceGuard guard(dout.device());
    const Tensor lse = packed(s[4]), low = packed(s[5]), starts = packed(s[6]), k_starts = packed(s[7]);
    const double scale = ctx->saved_data["scale"].toDouble();
    TORCH_CHECK(q.sizes() == dout.sizes() && s[3].sizes() == dout.sizes(), "attention: the saved q and out came back as ",
                q.sizes(), " and ", s[3].sizes());
    attn_check(q, k, v, starts, k_starts, scale);
    came_back(s[3], at::kBFloat16, q.numel(), dout, kAttn, "out");
    came_back(lse, at::kFloat, q.numel() / q.size(-1), dout, kAttn, "lse");
    came_back(low, at::kChar, q.numel(), dout, kAttn, "low part of out");
    const Operand oq = operand(q), ok = operand(k), ov = operand(v), out = operand(s[3]), g = operand(dout);
    concord_attn_args a =
        attn_args(oq, ok, ov, out, lse, low, starts, k_starts, ctx->saved_data["causal"].toBool(), scale);
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    Tensor dv = at::empty(k.sizes(), k.options());
    a.dout = (const uint16_t*)ptr(g.t), a.do_t = g.token, a.do_h = g.head;
    a.dq = (uint16_t*)ptr(dq), a.dk = (uint16_t*)ptr(dk), a.dv = (uint16_t*)ptr(dv);
    a.dq_t = (int64_t)a.H * a.D, a.dk_t = a.dv_t = (int64_t)a.HK * a.D;
    a.dq_h = a.dk_h = a.dv_h = a.D;
    const size_t need = concord_attention_workspace_bytes(&a);
    const Tensor ws = bytes(need, q);
    check(concord_attention_bwd(&a, ptr(ws), need, stream_of(q)), "attention backward");
    return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& starts_,
                 const MaybeTensor& k_starts_, bool causal, std::optional<double> scale_) {
  const Tensor starts = starts_ ? starts_->contiguous() : Tensor();
  const Tensor k_starts = k_starts_ ? k_starts_->contiguous() : Tensor();
  const double scale = scale_ ? *scale_ : q.dim() && q.size(-1) ? 1.0 / std::sqrt((double)q.size(-1)) : 1.0;
  no_tangent(kAttn, {&q, &k, &v});
  attn_check(q, k, v, starts, k_starts, scale);
  const c10::OptionalDeviceGuard guard(q.device());
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v)))
    return AttentionNode::apply(q, k, v, maybe(starts), maybe(k_starts), causal, scale);
  Tensor out = at::empty(q.sizes(), q.options());
  const concord_attn_args a =
      attn_args(operand(q), operand(k), operand(v), fresh(out), Tensor(), Tensor(), starts, k_starts, causal, scale);
  attn_forward(a, q);
  return out;
}

// ---- distillation -------------------------------------------------------------------
const char* const kDistill = "distill_loss";
constexpr int64_t kMaxTop = 1024;

void distill_check(const Tensor& z, const Tensor& t, const Tensor& i, double temperature) {
  TORCH_CHECK_TYPE(dtype_of(z) >= 0 && dtype_of(t) >= 0,
                   "distill_loss: logits and teacher_logits must be float32, bfloat16 or float16");
  TORCH_CHECK_TYPE(i.scalar_type() == at::kLong || i.scalar_type() == at::kInt,
                   "distill_loss: teacher_index must be int64 or int32 (got ", i.scalar_type(), ")");
  TORCH_CHECK_VALUE(z.dim() >= 1 && z.size(-1) >= 1, "distill_loss: logits need a vocabulary of at least 1");
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.sizes() == i.sizes() && t.sizes().slice(0, t.dim() - 1) == z.sizes().slice(0, z.dim() - 1),
                    "distill_loss: logits ", z.sizes(), ", teacher_logits ", t.sizes(), " and teacher_index ", i.sizes(),
                    " do not name the same rows");
  TORCH_CHECK_VALUE(t.size(-1) <= kMaxTop, "distill_loss: at most ", kMaxTop, " teacher logits a row (got ", t.size(-1), ")");
  TORCH_CHECK_VALUE(temperature > 0 && std::isfinite(temperature), "distill_loss: the temperature must be positive (got ",
                    temperature, ")");
  for (const Tensor* p : {&t, &i})
    TORCH_CHECK_VALUE(p->device() == z.device(), "distill_loss: ", p == &t ? "teacher_logits" : "teacher_index", " is on ",
                      p->device(), ", logits on ", z.device());
  need_gpu(z, kDistill, "logits");
}

// the rows of a call: logits, the teacher's values in 32 bits, places in 64
struct DistillRows {
  Rows z, t, i;
  int64_t rows, vocab;
  int32_t top;
  DistillRows(const Tensor& logits, const Tensor& teacher, const Tensor& index) {
    vocab = logits.size(-1), rows = logits.numel() / vocab, top = (int32_t)teacher.size(-1);
    z = rows_of(logits, rows, vocab);
    t = rows_of(teacher.to(at::kFloat), rows, top);
    i = rows_of(index.to(at::kLong), rows, top);
  }
};

Tensor distill_forward(const DistillRows& r, const Tensor& like, double temperature, const Tensor& stats) {
  Tensor loss = at::empty(like.sizes().slice(0, like.dim() - 1), like.options().dtype(at::kFloat));
  const size_t need = concord_distill_workspace_bytes(r.rows, r.vocab);
  const Tensor ws = need ? bytes(need, like) : Tensor();
  check(concord_distill_fwd(ptr(r.z.t), r.z.ld, dtype_of(like), r.rows, r.vocab, (const float*)ptr(r.t.t), r.t.ld,
                            (const int64_t*)ptr(r.i.t), r.i.ld, r.top, (float)temperature, loss.data_ptr<float>(),
                            (float*)ptr(stats), ptr(ws), need, stream_of(like)),
        kDistill);
  return loss;
}

struct DistillNode : torch::autograd::Function<DistillNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher, const Tensor& index,
                        double temperature) {
    const DistillRows r(logits, teacher, index);
    Tensor stats = at::empty({r.rows, 4}, logits.options().dtype(at::kFloat));
    Tensor loss = distill_forward(r, logits, temperature, stats);
    ctx->save_for_backward({r.z.t, r.t.t, r.i.t, stats});
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->saved_data["top"] = (int64_t)r.top;
    ctx->saved_data["type"] = (int64_t)logits.scalar_type();
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once(kDistill);
    const auto s = ctx->get_saved_variables();
    const Tensor& dloss = grads[0];
    const c10::OptionalDeviceGuard guard(dloss.device());
    const Tensor stats = packed(s[3]);
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t rows = dloss.numel(), vocab = shape.back(), top = ctx->saved_data["top"].toInt();
    came_back(s[0], (at::ScalarType)ctx->saved_data["type"].toInt(), rows * vocab, dloss, kDistill, "logits");
    came_back(s[1], at::kFloat, rows * top, dloss, kDistill, "teacher_logits");
    came_back(s[2], at::kLong, rows * top, dloss, kDistill, "teacher_index");
    came_back(stats, at::kFloat, rows * 4, dloss, kDistill, "statistics");
    const Rows z = rows_of(s[0], rows, vocab), t = rows_of(s[1], rows, top), i = rows_of(s[2], rows, top);
    // one value for all rows (a sum's or a mean's gradient) stays one value
    bool one = dloss.numel() > 0;
    for (int64_t d = 0; d < dloss.dim(); ++d) one = one && (dloss.stride(d) == 0 || dloss.size(d) == 1);
    const Rows g = one ? Rows{dloss, 0} : rows_of(dloss, rows, 1);
    Tensor dz = at::empty(shape, z.t.options());
    check(concord_distill_bwd((const float*)ptr(g.t), g.ld, ptr(z.t), z.ld, dtype_of(z.t), rows, vocab,
                              (const float*)ptr(t.t), t.ld, (const int64_t*)ptr(i.t), i.ld, (int32_t)top,
                              (float)ctx->saved_data["temperature"].toDouble(), stats.data_ptr<float>(), ptr(dz), vocab,
                              stream_of(z.t)),
          "distill_loss backward");
    return {dz, Tensor(), Tensor(), Tensor()};
  }
};

Tensor distill_loss(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature) {
  no_tangent(kDistill, {&logits});
  distill_check(logits, teacher, index, temperature);
  const c10::OptionalDeviceGuard guard(logits.device());
  const Tensor t = teacher.detach();
  if (at::GradMode::is_enabled() && wants_grad(logits)) return DistillNode::apply(logits, t, index, temperature);
  return distill_forward(DistillRows(logits, t, index), logits, temperature, Tensor());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm);
  m.def("attention", &attention);
  m.def("distill_loss", &distill_loss);
  for (auto add : concord_ops::registrars()) add(m);
}
