// torch_ops_block.cpp -- embedding, norms of queries and keys with the position
// rotation, and activations kept in 8 bits, as autograd nodes over the C entries
// of concord_amd.h (in C++ for the reason that torch_ops.cpp gives).
#include "torch_ops.h"

#include <cstring>

namespace {

// A node's settings as one saved entry: each has a name to look up and a box to
// allocate, and a step makes and reads them all.
const char* const kSettings = "settings";
int64_t bits_of(double v) {
  int64_t r;
  std::memcpy(&r, &v, sizeof r);
  return r;
}
double double_of(int64_t v) {
  double r;
  std::memcpy(&r, &v, sizeof r);
  return r;
}

// ---- embedding ------------------------------------------------------------------
const char* const kEmbedding = "embedding";

bool is_int64(const Tensor& t) { return t.scalar_type() == at::kLong; }

void embedding_check(const Tensor& tokens, const Tensor& weight, double scale, at::ScalarType dtype) {
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
                   "embedding: tokens must be int64 or int32 (got ", tokens.scalar_type(), ")");
  TORCH_CHECK_TYPE(dtype_of(weight) >= 0, "embedding: weight must be float32, bfloat16 or float16 (got ",
                   weight.scalar_type(), ")");
  TORCH_CHECK_TYPE(dtype == at::kFloat || dtype == at::kBFloat16 || dtype == at::kHalf,
                   "embedding: dtype must be float32, bfloat16 or float16 (got ", dtype, ")");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 1, "embedding: weight must be [vocabulary, width] (got ",
                    weight.sizes(), ")");
  // (as the kernels hold it: 0 times an infinite scale would not be the zero of a token outside the table)
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "embedding: the scale must be finite in 32 bits (got ", scale, ")");
  TORCH_CHECK_VALUE(tokens.device() == weight.device(), "embedding: tokens are on ", tokens.device(), ", weight on ",
                    weight.device());
  need_gpu(weight, kEmbedding, "weight");
}

Tensor embedding_forward(const Tensor& tokens, const Tensor& weight, double scale, at::ScalarType dtype) {
  const int64_t vocab = weight.size(0), width = weight.size(1);
  auto shape = tokens.sizes().vec();
  shape.push_back(width);
  const Rows w = rows_of(weight, vocab, width);
  Tensor y = at::empty(shape, weight.options().dtype(dtype));
  check(concord_embedding_fwd(ptr(tokens), is_int64(tokens), tokens.numel(), ptr(w.t), w.ld, dtype_of(weight), vocab, width,
                              (float)scale, ptr(y), width, dtype_of(y), stream_of(y)),
        kEmbedding);
  return y;
}

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, double scale, int64_t dtype) {
    ctx->save_for_backward({tokens});
    ctx->saved_data[kSettings] = std::vector<int64_t>{(int64_t)tokens.scalar_type(), weight.size(0),
                                                      (int64_t)weight.scalar_type(), bits_of(scale)};
    return embedding_forward(tokens, weight, scale, (at::ScalarType)dtype);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once(kEmbedding);
    const Tensor& dy = grads[0];
    const c10::OptionalDeviceGuard guard(dy.device());
    const Tensor tokens = ctx->get_saved_variables()[0].contiguous();
    const auto settings = ctx->saved_data[kSettings].toIntVector();
    const int64_t vocab = settings[1], width = dy.size(-1), n = dy.numel() / width;
    came_back(tokens, (at::ScalarType)settings[0], n, dy, kEmbedding, "tokens");
    const Rows g = rows_of(dy, n, width);
    Tensor dw = at::empty({vocab, width}, dy.options().dtype((at::ScalarType)settings[2]));
    const size_t need = concord_embedding_workspace_bytes(n, vocab, width);
    const Tensor ws = bytes(need, dy);
    check(concord_embedding_bwd(ptr(tokens), is_int64(tokens), n, ptr(g.t), g.ld, dtype_of(dy), vocab, width,
                                (float)double_of(settings[3]), ptr(dw), width, dtype_of(dw), ptr(ws), need,
                                stream_of(dy)),
          "embedding backward");
    return {dw, Tensor(), Tensor(), Tensor()};
  }
};

Tensor embedding(const Tensor& tokens_, const Tensor& weight, double scale, std::optional<at::ScalarType> dtype_) {
  const at::ScalarType dtype = dtype_ ? *dtype_ : weight.scalar_type();
  no_tangent(kEmbedding, {&weight});
  embedding_check(tokens_, weight, scale, dtype);
  const c10::OptionalDeviceGuard guard(weight.device());
  const Tensor tokens = tokens_.contiguous();
  if (at::GradMode::is_enabled() && wants_grad(weight)) return EmbeddingNode::apply(weight, tokens, scale, (int64_t)dtype);
  return embedding_forward(tokens, weight, scale, dtype);
}

// ---- norms of queries and keys, with the position rotation -----------------------
const char* const kQk = "qk_norm_rope";

struct QkSettings {
  double base, eps;
  int64_t rotary;
  bool adjacent;
};

at::ScalarType qk_check(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight, const Tensor& positions,
              const QkSettings& s) {
  for (const Tensor* t : {&q, &k}) {
    const char* name = t == &q ? "q" : "k";
    TORCH_CHECK_TYPE(dtype_of(*t) >= 0 && t->scalar_type() == q.scalar_type(),
                     "qk_norm_rope: q and k must share one of float32, bfloat16, float16 (got ", t->scalar_type(), " for ",
                     name, ")");
    TORCH_CHECK_VALUE(t->dim() == q.dim() && (t->dim() == 3 || t->dim() == 4),
                      "qk_norm_rope: q and k must both be [token, head, dim] or [batch, token, head, dim]");
    TORCH_CHECK_VALUE(t->device() == q.device(), "qk_norm_rope: ", name, " is on ", t->device(), ", q on ", q.device());
  }
  const int64_t d = q.size(-1);
  TORCH_CHECK_VALUE(k.size(-1) == d && d >= 8 && d <= 256 && d % 8 == 0,
                    "qk_norm_rope: q and k need one head dimension, a multiple of 8 up to 256 (got ", d, " and ", k.size(-1),
                    ")");
  TORCH_CHECK_VALUE(q.sizes().slice(0, q.dim() - 2) == k.sizes().slice(0, q.dim() - 2), "qk_norm_rope: q ", q.sizes(), " and k ",
                    k.sizes(), " are of different tokens");
  TORCH_CHECK_VALUE(q.size(-2) >= 1 && k.size(-2) >= 1, "qk_norm_rope: q and k need a head");
  TORCH_CHECK_VALUE(s.rotary >= 0 && s.rotary <= d && s.rotary % 8 == 0,
                    "qk_norm_rope: rotary_dim must be a multiple of 8 up to ", d, " (got ", s.rotary, ")");
  TORCH_CHECK_VALUE(s.base > 0 && s.base < 1e300, "qk_norm_rope: the base must be positive (got ", s.base, ")");
  // (as the kernels hold it: an infinite one would make every row zeros, one that is lost a row of zeros NaN)
  const float eps = (float)s.eps;
  TORCH_CHECK_VALUE(s.eps >= 0 && std::isfinite(eps) && (eps > 0 || s.eps == 0),
                    "qk_norm_rope: eps must be 0 or a positive number of 32 bits (got ", s.eps, ")");
  at::ScalarType wtype = at::kFloat;
  bool given = false;
  for (const Tensor* w : {&q_weight, &k_weight}) {
    if (!w->defined()) continue;
    const char* name = w == &q_weight ? "q_weight" : "k_weight";
    TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == d, "qk_norm_rope: ", name, " must have shape (", d, ",), got ", w->sizes());
    TORCH_CHECK_TYPE(dtype_of(*w) >= 0 && (!given || w->scalar_type() == wtype),
                     "qk_norm_rope: q_weight and k_weight must share one of float32, bfloat16, float16");
    TORCH_CHECK_VALUE(w->device() == q.device(), "qk_norm_rope: ", name, " is on ", w->device(), ", q on ", q.device());
    wtype = w->scalar_type(), given = true;
  }
  if (positions.defined()) {
    TORCH_CHECK_TYPE(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt,
                     "qk_norm_rope: positions must be int64 or int32 (got ", positions.scalar_type(), ")");
    const auto tokens = q.sizes().slice(0, q.dim() - 2);
    TORCH_CHECK_VALUE(positions.sizes() == tokens || positions.sizes() == tokens.slice(tokens.size() - 1),
                      "qk_norm_rope: positions ", positions.sizes(), " do not fit the tokens ", tokens);
    TORCH_CHECK_VALUE(positions.device() == q.device(), "qk_norm_rope: positions are on ", positions.device(), ", q on ",
                      q.device());
  }
  need_gpu(q, kQk, "q");
  return wtype;
}

// the part of the arguments that both passes share (q_weight, k_weight and positions contiguous)
concord_qk_args qk_args(const Operand& q, const Operand& k, const Tensor& q_weight, const Tensor& k_weight,
                        const Tensor& positions, const QkSettings& s) {
  concord_qk_args a{};
  a.q = ptr(q.t), a.q_t = q.token, a.q_h = q.head;
  a.k = ptr(k.t), a.k_t = k.token, a.k_h = k.head;
  a.q_weight = ptr(q_weight), a.k_weight = ptr(k_weight);
  const int64_t batch = q.t.dim() == 4 ? q.t.size(0) : 1;
  a.seq = q.t.size(-3), a.T = batch * a.seq;
  a.H = (int32_t)q.t.size(-2), a.HK = (int32_t)k.t.size(-2), a.D = (int32_t)q.t.size(-1), a.R = (int32_t)s.rotary;
  a.adjacent = s.adjacent;
  a.positions = a.T ? ptr(positions) : nullptr;
  if (positions.defined()) a.pos_seq = positions.numel(), a.pos64 = is_int64(positions);
  a.dtype = dtype_of(q.t);
  a.wtype = q_weight.defined() ? dtype_of(q_weight) : k_weight.defined() ? dtype_of(k_weight) : CONCORD_F32;
  a.base = s.base, a.eps = (float)s.eps;
  return a;
}

std::vector<Tensor> qk_forward(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                               const Tensor& positions, const QkSettings& s) {
  const Operand oq = operand(q), ok = operand(k);
  concord_qk_args a = qk_args(oq, ok, q_weight, k_weight, positions, s);
  Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  a.q_out = ptr(yq), a.k_out = ptr(yk);
  check(concord_qk_norm_rope_fwd(&a, stream_of(q)), kQk);
  return {yq, yk};
}

struct QkNormRopeNode : torch::autograd::Function<QkNormRopeNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const MaybeTensor& q_weight_,
                               const MaybeTensor& k_weight_, const MaybeTensor& positions_, double base, double eps,
                               int64_t rotary, bool adjacent) {
    const Tensor q_weight = value(q_weight_), k_weight = value(k_weight_), positions = value(positions_);
    ctx->save_for_backward({q, k, q_weight, k_weight, positions});
    ctx->saved_data[kSettings] = std::vector<int64_t>{bits_of(base), bits_of(eps), rotary, adjacent};
    return qk_forward(q, k, q_weight, k_weight, positions, {base, eps, rotary, adjacent});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once(kQk);
    const auto saved = ctx->get_saved_variables();
    const Tensor &gq = grads[0], &gk = grads[1];   // (zeros for an output that nothing used)
    const c10::OptionalDeviceGuard guard(gq.device());
    const auto settings = ctx->saved_data[kSettings].toIntVector();
    const QkSettings s{double_of(settings[0]), double_of(settings[1]), settings[2], settings[3] != 0};
    const Tensor &q = saved[0], &k = saved[1];
    const Tensor q_weight = packed(saved[2]), k_weight = packed(saved[3]);
    const Tensor positions = saved[4].defined() ? saved[4].contiguous() : Tensor();
    TORCH_CHECK(q.sizes() == gq.sizes() && k.sizes() == gk.sizes() && q.scalar_type() == gq.scalar_type() &&
                    q.device() == gq.device(),
                "qk_norm_rope: the saved q or k came back as another tensor");
    qk_check(q, k, q_weight, k_weight, positions, s);
    // (numbered among the tensors that were given)
    Tensor dq, dk, dwq, dwk, ws;
    if (q_weight.defined() && ctx->needs_input_grad(2)) dwq = at::empty_like(q_weight);
    if (k_weight.defined() && ctx->needs_input_grad(q_weight.defined() ? 3 : 2)) dwk = at::empty_like(k_weight);
    // what is frozen has no heads: no row of it is read or written
    const bool with_q = ctx->needs_input_grad(0) || dwq.defined(), with_k = ctx->needs_input_grad(1) || dwk.defined();
    if (!with_q && !with_k) return variable_list(9);
    const Operand oq = with_q ? operand(q) : Operand{q, 0, 0}, ok = with_k ? operand(k) : Operand{k, 0, 0};
    concord_qk_args a = qk_args(oq, ok, q_weight, k_weight, positions, s);
    a.dq_weight = ptr(dwq), a.dk_weight = ptr(dwk);
    Operand og, oh;
    if (with_q) {
      og = operand(gq);
      dq = at::empty(q.sizes(), q.options());
      a.dq_out = ptr(og.t), a.dq_t = og.token, a.dq_h = og.head, a.dq = ptr(dq);
    } else {
      a.H = 0, a.q = a.q_weight = nullptr;
    }
    if (with_k) {
      oh = operand(gk);
      dk = at::empty(k.sizes(), k.options());
      a.dk_out = ptr(oh.t), a.dk_t = oh.token, a.dk_h = oh.head, a.dk = ptr(dk);
    } else {
      a.HK = 0, a.k = a.k_weight = nullptr;
    }
    size_t need = 0;
    if (dwq.defined() || dwk.defined()) {
      need = concord_qk_norm_rope_workspace_bytes(&a);
      ws = bytes(need, q);
    }
    check(concord_qk_norm_rope_bwd(&a, ptr(ws), need, stream_of(q)), "qk_norm_rope backward");
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::vector<Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const MaybeTensor& q_weight_, const MaybeTensor& k_weight_,
                                 const MaybeTensor& positions_, double base, std::optional<int64_t> rotary, bool adjacent,
                                 double eps) {
  Tensor q_weight = value(q_weight_), k_weight = value(k_weight_), positions = value(positions_);
  const QkSettings s{base, eps, rotary ? *rotary : q.dim() ? q.size(-1) : 0, adjacent};
  no_tangent(kQk, {&q, &k, &q_weight, &k_weight});
  qk_check(q, k, q_weight, k_weight, positions, s);
  const c10::OptionalDeviceGuard guard(q.device());
  if (q_weight.defined()) q_weight = q_weight.contiguous();
  if (k_weight.defined()) k_weight = k_weight.contiguous();
  if (positions.defined()) positions = positions.contiguous();
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(q_weight) || wants_grad(k_weight)))
    return QkNormRopeNode::apply(q, k, maybe(q_weight), maybe(k_weight), maybe(positions), base, eps, s.rotary, adjacent);
  return qk_forward(q, k, q_weight, k_weight, positions, s);
}

// ---- activations in 8 bits ----------------------------------------------------------
constexpr int64_t kBlock8 = 32;   // values that share an exponent

void act8_check(const Tensor& x, const char* op, bool gated) {
  TORCH_CHECK_TYPE(dtype_of(x) >= 0, op, ": x must be float32, bfloat16 or float16 (got ", x.scalar_type(), ")");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, op, ": x needs a last dimension of at least 1");
  TORCH_CHECK_VALUE(!gated || x.size(-1) % 2 == 0, op, ": the last dimension holds two halves (got ", x.size(-1), ")");
  need_gpu(x, op, "x");
}

// codes with x's shape, exponents [..., blocks] or [..., 2, blocks]
std::vector<Tensor> empty8(const Tensor& x, bool gated) {
  auto shape = x.sizes().vec();
  Tensor codes = at::empty(shape, x.options().dtype(at::kChar));
  const int64_t width = shape.back();
  shape.back() = gated ? 2 : (width + kBlock8 - 1) / kBlock8;
  if (gated) shape.push_back((width / 2 + kBlock8 - 1) / kBlock8);
  return {codes, at::empty(shape, x.options().dtype(at::kByte))};
}

int8_t* codes_of(const Tensor& t) { return (int8_t*)ptr(t); }
uint8_t* exponents_of(const Tensor& t) { return (uint8_t*)ptr(t); }

std::vector<Tensor> pack8(const Tensor& x) {
  no_tangent("pack8", {&x});
  act8_check(x, "pack8", false);
  const c10::OptionalDeviceGuard guard(x.device());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  const Rows r = rows_of(x, rows, width);
  const std::vector<Tensor> kept = empty8(x, false);
  check(concord_pack8(ptr(r.t), r.ld, dtype_of(x), rows, width, codes_of(kept[0]), exponents_of(kept[1]), stream_of(x)),
        "pack8");
  return kept;
}

Tensor unpack8(const Tensor& codes_, const Tensor& exponents_, at::ScalarType dtype) {
  TORCH_CHECK_TYPE(codes_.scalar_type() == at::kChar && exponents_.scalar_type() == at::kByte,
                   "unpack8: codes must be int8 and exponents uint8 (got ", codes_.scalar_type(), " and ",
                   exponents_.scalar_type(), ")");
  TORCH_CHECK_TYPE(dtype == at::kFloat || dtype == at::kBFloat16 || dtype == at::kHalf,
                   "unpack8: dtype must be float32, bfloat16 or float16 (got ", dtype, ")");
  TORCH_CHECK_VALUE(codes_.dim() >= 1 && codes_.size(-1) >= 1, "unpack8: codes need a last dimension of at least 1");
  const int64_t width = codes_.size(-1), rows = codes_.numel() / width;
  TORCH_CHECK_VALUE(exponents_.dim() == codes_.dim() &&
                        exponents_.sizes().slice(0, codes_.dim() - 1) == codes_.sizes().slice(0, codes_.dim() - 1) &&
                        exponents_.size(-1) == (width + kBlock8 - 1) / kBlock8,
                    "unpack8: codes ", codes_.sizes(), " and exponents ", exponents_.sizes(), " do not belong together");
  TORCH_CHECK_VALUE(codes_.device() == exponents_.device(), "unpack8: exponents are on ", exponents_.device(), ", codes on ",
                    codes_.device());
  need_gpu(codes_, "unpack8", "codes");
  const c10::OptionalDeviceGuard guard(codes_.device());
  const Tensor codes = codes_.contiguous(), exponents = exponents_.contiguous();
  Tensor x = at::empty(codes.sizes(), codes.options().dtype(dtype));
  check(concord_unpack8(codes_of(codes), exponents_of(exponents), rows, width, ptr(x), width, dtype_of(x), stream_of(x)),
        "unpack8");
  return x;
}

const char* gelu8_name(bool gated) { return gated ? "geglu8" : "gelu8"; }

// y, and x in 8 bits where `kept` has room for it
Tensor gelu8_forward(const Tensor& x, bool gated, bool tanh, const std::vector<Tensor>& kept) {
  const int64_t wide = x.size(-1), width = gated ? wide / 2 : wide, rows = x.numel() / wide;
  const Rows r = rows_of(x, rows, wide);
  auto shape = x.sizes().vec();
  shape.back() = width;
  Tensor y = at::empty(shape, x.options());
  check(concord_gelu8_fwd(ptr(r.t), r.ld, dtype_of(x), rows, width, gated, tanh, ptr(y), width,
                          kept.empty() ? nullptr : codes_of(kept[0]), kept.empty() ? nullptr : exponents_of(kept[1]),
                          stream_of(x)),
        gelu8_name(gated));
  return y;
}

struct Gelu8Node : torch::autograd::Function<Gelu8Node> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, bool gated, bool tanh) {
    const std::vector<Tensor> kept = empty8(x, gated);
    ctx->save_for_backward({kept[0], kept[1]});
    ctx->saved_data[kSettings] = (int64_t)gated | (int64_t)tanh << 1;
    return gelu8_forward(x, gated, tanh, kept);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t settings = ctx->saved_data[kSettings].toInt();
    const bool gated = settings & 1, tanh = settings >> 1;
    only_once(gelu8_name(gated));
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    const c10::OptionalDeviceGuard guard(dy.device());
    const int64_t width = dy.size(-1), rows = dy.numel() / width, half = gated ? 2 : 1;
    const Tensor codes = packed(saved[0]), exponents = packed(saved[1]);
    came_back(codes, at::kChar, rows * width * half, dy, gelu8_name(gated), "codes");
    came_back(exponents, at::kByte, rows * half * ((width + kBlock8 - 1) / kBlock8), dy, gelu8_name(gated), "exponents");
    const Rows g = rows_of(dy, rows, width);
    auto shape = dy.sizes().vec();
    shape.back() = width * half;
    Tensor dx = at::empty(shape, dy.options());
    check(concord_gelu8_bwd(ptr(g.t), g.ld, codes_of(codes), exponents_of(exponents), dtype_of(dy), rows, width, gated,
                            tanh, ptr(dx), width * half, stream_of(dy)),
          gated ? "geglu8 backward" : "gelu8 backward");
    return {dx, Tensor(), Tensor()};
  }
};

Tensor gelu8(const Tensor& x, const std::string& approximate, bool gated) {
  const char* op = gelu8_name(gated);
  no_tangent(op, {&x});
  TORCH_CHECK_VALUE(approximate == "none" || approximate == "tanh", op, ": approximate must be 'none' or 'tanh' (got '",
                    approximate, "')");
  act8_check(x, op, gated);
  const c10::OptionalDeviceGuard guard(x.device());
  const bool tanh = approximate == "tanh";
  if (at::GradMode::is_enabled() && wants_grad(x)) return Gelu8Node::apply(x, gated, tanh);
  return gelu8_forward(x, gated, tanh, {});
}

// an optional torch.dtype (no caster of the installed torch's takes one)
std::optional<at::ScalarType> dtype_arg(const pybind11::object& o, const char* op) {
  if (o.is_none()) return std::nullopt;
  TORCH_CHECK_TYPE(THPDtype_Check(o.ptr()), op, ": dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o.ptr())->scalar_type;
}

const concord_ops::Register add_block_ops([](pybind11::module_& m) {
  m.def("embedding", [](const Tensor& tokens, const Tensor& weight, double scale, const pybind11::object& dtype) {
    return embedding(tokens, weight, scale, dtype_arg(dtype, kEmbedding));
  });
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("gelu8", [](const Tensor& x, const std::string& approximate) { return gelu8(x, approximate, false); });
  m.def("geglu8", [](const Tensor& x, const std::string& approximate) { return gelu8(x, approximate, true); });
  m.def("pack8", &pack8);
  m.def("unpack8", [](const Tensor& codes, const Tensor& exponents, const pybind11::object& dtype) {
    return unpack8(codes, exponents, dtype_arg(dtype, "unpack8").value_or(at::kBFloat16));
  });
});

}  // namespace
