// Python bindings for the language-model training kernels (csrc/include/grace_lm.h): embedding,
// residual norms, the global gradient norm.
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPException.h>

#include <algorithm>
#include <array>
#include <tuple>

#include "grace_lm.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using DevGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
inline hipStream_t cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

grace::ElType el_type(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return grace::ElType::kF32;
    case at::kBFloat16: return grace::ElType::kBF16;
    case at::kHalf: return grace::ElType::kF16;
    default: TORCH_CHECK(false, what, " must be float32, bfloat16 or float16");
  }
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_on(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), what, " must be on ", like.device());
}

// ---------------------------------------------------------------- embedding
grace::EmbedIds embed_ids(const Tensor& ids, int64_t vocab, int64_t width, int64_t pad) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
              "embedding: ids must be a contiguous int64 or int32 GPU tensor");
  TORCH_CHECK(ids.numel() < INT32_MAX && vocab < INT32_MAX, "embedding: at most 2^31 - 2 tokens and rows");
  TORCH_CHECK(width <= grace::kEmbedMaxWidth, "embedding: rows of at most ", grace::kEmbedMaxWidth, " values");
  TORCH_CHECK(pad >= -1 && pad < vocab, "embedding: padding_idx out of range");
  return {ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), vocab, pad};
}

Tensor embed_fwd(const Tensor& ids, const Tensor& weight, double scale, at::ScalarType dtype) {
  TORCH_CHECK(weight.is_cuda() && weight.dim() == 2 && (weight.stride(1) == 1 || weight.size(1) <= 1),
              "embedding: the table must be a 2-D GPU tensor with contiguous rows");
  check_on(ids, weight, "embedding: ids");
  TORCH_CHECK(weight.size(0) > 0 || ids.numel() == 0, "embedding: the table has no rows");
  const grace::EmbedIds e = embed_ids(ids, weight.size(0), weight.size(1), -1);
  DevGuard guard(weight.device());
  auto shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor out = at::empty(shape, weight.options().dtype(dtype));
  grace::embed_forward(e, weight.data_ptr(), el_type(weight.scalar_type(), "embedding: the table"), weight.stride(0),
                       weight.size(1), (float)scale, out.data_ptr(), el_type(dtype, "embedding: the output"),
                       cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}

Tensor embed_bwd(const Tensor& ids, const Tensor& dy, int64_t vocab, int64_t pad, double scale, at::ScalarType dtype) {
  TORCH_CHECK(dy.is_cuda() && dy.is_contiguous() && dy.dim() >= 1, "embedding: the gradient must be contiguous on a GPU");
  const int64_t d = dy.size(-1);
  TORCH_CHECK(dy.numel() == ids.numel() * d, "embedding: the gradient must be [tokens, width]");
  check_on(ids, dy, "embedding: ids");
  const grace::EmbedIds e = embed_ids(ids, vocab, d, pad);
  DevGuard guard(dy.device());
  const auto tdw = el_type(dtype, "embedding: the table"), tdy = el_type(dy.scalar_type(), "embedding: the gradient");
  if (e.n == 0 || vocab == 0 || d == 0) return at::zeros({vocab, d}, dy.options().dtype(dtype));
  Tensor dw = at::empty({vocab, d}, dy.options().dtype(dtype));
  const int64_t bytes = grace::embed_backward_ws(e.n, vocab, d);
  const Tensor ws = bytes > 0 ? at::empty({bytes}, dy.options().dtype(at::kByte)) : Tensor();
  grace::embed_backward(e, dy.data_ptr(), tdy, d, (float)scale, dw.data_ptr(), tdw,
                        bytes > 0 ? ws.data_ptr() : nullptr, cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dw;
}

// The differentiable calls are C++ autograd functions: a training call costs a few microseconds of host
// time, where a Python function costs some fifty.  They are differentiable once.
void once_only(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: no create_graph");
}

// A backward that is captured into a graph reaches its leaves on the stream where autograd met them first; an
// eager graph that is still alive keeps that.  If it is the default stream, which no capture can join, the
// process would end: refused while nothing is recorded for the leaf.
void no_foreign_leaf(const char* what) {
  const hipStream_t stream = cur_stream();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) != hipSuccess) {
    (void)hipGetLastError();
    return;
  }
  const auto node = torch::autograd::get_current_node();
  if (status == hipStreamCaptureStatusNone || node == nullptr) return;
  for (const auto& edge : node->next_edges()) {
    const auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get());
    if (leaf == nullptr) continue;
    const auto of = edge.function->stream();
    TORCH_CHECK(!of.has_value() || of->id() != 0, what, ": a captured backward reaches a leaf that an eager graph on "
                "the default stream still holds; let go of that graph's outputs first, or run it on another stream");
  }
}

// A call that autograd does not follow would lose forward-mode tangents without a word.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, " has no forward-mode derivative");
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale,
                        int64_t pad, at::ScalarType dtype) {
    ctx->save_for_backward({ids});
    ctx->saved_data["args"] = std::vector<int64_t>{weight.size(0), pad, (int64_t)weight.scalar_type()};
    ctx->saved_data["scale"] = scale;
    return embed_fwd(ids, weight, scale, dtype);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    once_only("embedding");
    no_foreign_leaf("embedding");
    const Tensor ids = ctx->get_saved_variables()[0];
    const auto args = ctx->saved_data["args"].toIntVector();
    return {embed_bwd(ids, grads[0].contiguous(), args[0], args[1], ctx->saved_data["scale"].toDouble(),
                      (at::ScalarType)args[2]),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, const c10::optional<int64_t>& padding_idx,
                 const c10::optional<at::ScalarType>& out) {
  auto refuse = [](const std::string& what) { return "embedding: " + what; };
  const auto tw = weight.scalar_type(), dtype = out.value_or(tw);
  if (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt)
    throw py::type_error(refuse(c10::str("ids must be int64 or int32, got ", ids.scalar_type())));
  if (weight.dim() != 2) throw py::value_error(refuse(c10::str("the table must be [rows, width], got ", weight.sizes())));
  if (ids.device() != weight.device())
    throw py::value_error(refuse(c10::str("ids on ", ids.device(), ", table on ", weight.device())));
  const int64_t rows = weight.size(0);
  if (rows == 0 && ids.numel() > 0) throw py::value_error(refuse("the table has no rows"));
  int64_t pad = -1;
  if (padding_idx.has_value()) {
    pad = *padding_idx < 0 ? *padding_idx + rows : *padding_idx;
    if (pad < 0 || pad >= rows)
      throw py::value_error(refuse(c10::str("padding_idx ", *padding_idx, " outside a table of ", rows, " rows")));
  }
  for (const auto t : {tw, dtype})
    if (t != at::kFloat && t != at::kBFloat16 && t != at::kHalf)
      throw py::type_error(refuse(c10::str("float32, bfloat16 or float16 on a GPU, got ", tw, " -> ", dtype)));
  if (ids.numel() >= INT32_MAX || rows >= INT32_MAX) throw py::value_error(refuse("at most 2^31 - 2 tokens and rows"));
  if (weight.size(1) > grace::kEmbedMaxWidth)
    throw py::value_error(refuse(c10::str("rows of ", weight.size(1), " values: at most ", grace::kEmbedMaxWidth)));
  no_tangent(weight, "embedding");
  const Tensor i = ids.contiguous();
  const Tensor w = weight.stride(1) != 1 && weight.size(1) > 1 ? weight.contiguous() : weight;
  if (at::GradMode::is_enabled() && w.requires_grad()) return EmbeddingFn::apply(w, i, scale, pad, dtype);
  return embed_fwd(i, w, scale, dtype);
}

// ---------------------------------------------------------------- residual norm
grace::NormParam norm_param(const Tensor& t, int64_t n, const Tensor& y, const char* what) {
  if (!t.defined()) return {nullptr, false};
  check_on(t, y, what);
  TORCH_CHECK(t.is_contiguous() && t.numel() == n, what, ": contiguous, ", n, " values");
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == y.scalar_type(), what,
              " must be float32 or of the block's type");
  return {t.data_ptr(), t.scalar_type() == at::kFloat};
}

grace::NormShape norm_shape(const Tensor& y, at::ScalarType tx, int64_t gate_rows, double alpha, double eps, bool rms,
                            bool post) {
  TORCH_CHECK(y.is_cuda() && y.dim() >= 1 && y.is_contiguous(), "residual norm: the block must be contiguous on a GPU");
  const int64_t d = y.size(-1);
  TORCH_CHECK(d >= 1 && d <= grace::kNormMaxWidth, "residual norm: widths 1 to ", grace::kNormMaxWidth);
  const int64_t rows = y.numel() / d;
  TORCH_CHECK(rows < INT32_MAX, "residual norm: at most 2^31 - 2 rows");
  TORCH_CHECK(rows == 0 || (gate_rows >= 1 && rows % gate_rows == 0), "residual norm: rows per gate row");
  grace::NormShape n{rows, gate_rows, (int)d, (float)alpha, (float)eps, rms, post,
                     el_type(tx, "residual norm: the residual"), el_type(y.scalar_type(), "residual norm: the block")};
  TORCH_CHECK(n.tx == n.ty || n.tx == grace::ElType::kF32, "residual norm: the residual must be float32 or of the block's type");
  return n;
}

int64_t gate_size(const grace::NormShape& n) { return n.rows / n.gate_rows * n.d; }  // of rows > 0

struct NormTensors {
  Tensor y, x, gate, weight, bias, post_weight, post_bias;  // undefined: not there
};
struct NormOptions {
  int64_t gate_rows;
  bool post, rms;
  double alpha, eps;
};

// Without a residual, a gate and a post norm the sum is the block itself.
bool is_plain(const NormTensors& t, const NormOptions& o) { return !t.x.defined() && !t.gate.defined() && !o.post; }

// (h, s, stats); s and stats are undefined where they are not wanted
std::tuple<Tensor, Tensor, Tensor> resnorm_fwd(const NormTensors& t, const NormOptions& o, bool want_sum,
                                               bool want_stats) {
  const Tensor& y = t.y;
  const auto tx = t.x.defined() ? t.x.scalar_type() : y.scalar_type();
  const grace::NormShape n = norm_shape(y, tx, o.gate_rows, o.alpha, o.eps, o.rms, o.post);
  if (t.x.defined()) {
    check_on(t.x, y, "residual norm: the residual");
    TORCH_CHECK(t.x.sizes() == y.sizes() && t.x.is_contiguous(), "residual norm: the residual must be like the block");
  }
  DevGuard guard(y.device());
  Tensor h = at::empty_like(y);
  Tensor s = want_sum ? at::empty(y.sizes(), y.options().dtype(tx)) : Tensor();
  Tensor stats = want_stats ? at::empty({o.post ? 4 : 2, n.rows}, y.options().dtype(at::kFloat)) : Tensor();
  if (n.rows > 0) {
    grace::resnorm_forward(n, t.x.defined() ? t.x.data_ptr() : nullptr, y.data_ptr(),
                           norm_param(t.gate, gate_size(n), y, "residual norm: the gate"),
                           norm_param(t.weight, n.d, y, "residual norm: weight"),
                           norm_param(t.bias, n.d, y, "residual norm: bias"),
                           norm_param(t.post_weight, n.d, y, "residual norm: post_weight"),
                           norm_param(t.post_bias, n.d, y, "residual norm: post_bias"), h.data_ptr(),
                           want_sum ? s.data_ptr() : nullptr, want_stats ? stats.data_ptr<float>() : nullptr,
                           cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {h, s, stats};
}

// The gradients of y, x, gate, weight, bias, post_weight, post_bias, undefined where want is not set; one
// tensor for y and x where they are equal.  s: the stored sum, or undefined: made again from x and y.
std::vector<Tensor> resnorm_bwd(const Tensor& dh, const Tensor& ds, const NormTensors& t, const NormOptions& o,
                                const Tensor& s, const Tensor& stats, const std::array<bool, 7>& want,
                                at::ScalarType tx, at::ScalarType ty) {
  const Tensor& like = dh.defined() ? dh : ds;
  const Tensor shape = like.scalar_type() == ty ? like : at::empty(like.sizes(), like.options().dtype(ty));
  const grace::NormShape n = norm_shape(shape, tx, o.gate_rows, o.alpha, o.eps, o.rms, o.post);
  auto check = [&](const Tensor& u, at::ScalarType type, const char* what) {
    if (!u.defined()) return;
    check_on(u, like, what);
    TORCH_CHECK(u.sizes() == like.sizes() && u.is_contiguous() && u.scalar_type() == type, what,
                " must be like the forward's");
  };
  check(s, tx, "residual norm: the saved sum");
  check(t.x, tx, "residual norm: the residual");
  check(t.y, ty, "residual norm: the block");
  check(dh, ty, "residual norm: the norm's gradient");
  check(ds, tx, "residual norm: the sum's gradient");
  TORCH_CHECK(s.defined() || t.y.defined(), "residual norm: neither the sum nor its parts were saved");
  TORCH_CHECK(t.y.defined() || !(t.gate.defined() || o.post), "residual norm: the block was not saved");
  TORCH_CHECK(stats.is_cuda() && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                  stats.numel() == (o.post ? 4 : 2) * n.rows, "residual norm: the saved statistics");
  DevGuard guard(like.device());
  auto made = [&](int k, const Tensor& p) {
    if (!want[k] || !p.defined()) return Tensor();
    return n.rows > 0 ? at::empty_like(p) : at::zeros_like(p);
  };
  Tensor dy = at::empty_like(shape);
  const bool one = !t.gate.defined() && !o.post && n.alpha == 1.f && n.tx == n.ty;
  Tensor dx = !want[1] ? Tensor() : one ? dy : at::empty(like.sizes(), like.options().dtype(tx));
  Tensor dgate = made(2, t.gate), dw = made(3, t.weight), db = made(4, t.bias), dpw = made(5, t.post_weight),
         dpb = made(6, t.post_bias);
  if (n.rows > 0) {
    const grace::NormParam gp = norm_param(t.gate, gate_size(n), shape, "residual norm: the gate");
    const grace::NormParam wp = norm_param(t.weight, n.d, shape, "residual norm: weight");
    const grace::NormParam bp = norm_param(t.bias, n.d, shape, "residual norm: bias");
    const grace::NormParam pwp = norm_param(t.post_weight, n.d, shape, "residual norm: post_weight");
    const grace::NormParam pbp = norm_param(t.post_bias, n.d, shape, "residual norm: post_bias");
    auto ptr = [](const Tensor& u) { return u.defined() ? u.data_ptr() : nullptr; };
    const grace::NormGrads g{ptr(dx), dy.data_ptr(), ptr(dgate), ptr(dw), ptr(db), ptr(dpw), ptr(dpb), bp.f32, pbp.f32};
    Tensor ws = at::empty({grace::resnorm_backward_ws(n)}, like.options().dtype(at::kByte));
    grace::resnorm_backward(n, ptr(s), ptr(t.x), ptr(t.y), stats.data_ptr<float>(), gp, wp, pwp, pbp, ptr(dh), ptr(ds),
                            g, ws.data_ptr(), cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {want[0] ? dy : Tensor(), dx, dgate, dw, db, dpw, dpb};
}

struct ResidualNormFn : torch::autograd::Function<ResidualNormFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& y,
                                                const OptTensor& ox, const OptTensor& ogate, const OptTensor& oweight,
                                                const OptTensor& obias, const OptTensor& opost_weight,
                                                const OptTensor& opost_bias, const NormOptions& o, bool return_sum) {
    auto get = [](const OptTensor& t) { return has(t) ? *t : Tensor(); };
    const Tensor x = get(ox), gate = get(ogate), weight = get(oweight), bias = get(obias),
                 post_weight = get(opost_weight), post_bias = get(opost_bias);
    const NormTensors t{y, x, gate, weight, bias, post_weight, post_bias};
    const auto tx = x.defined() ? x.scalar_type() : y.scalar_type();
    const bool plain = is_plain(t, o), stored = !plain && tx == at::kFloat;
    auto [h, s, stats] = resnorm_fwd(t, o, !plain && (return_sum || stored), true);
    const bool keeps_y = gate.defined() || o.post || !(plain || stored);
    ctx->save_for_backward({plain ? y : stored ? s : Tensor(), plain || stored ? Tensor() : x, keeps_y ? y : Tensor(),
                            gate, weight, bias, post_weight, post_bias, stats});
    ctx->saved_data["ints"] = std::vector<int64_t>{o.gate_rows, o.post, o.rms, (int64_t)tx, (int64_t)y.scalar_type(),
                                                  x.defined()};
    ctx->saved_data["alpha"] = o.alpha;
    ctx->saved_data["eps"] = o.eps;
    ctx->set_materialize_grads(false);
    if (!return_sum) return {h};
    // the plain sum is an output of its own: its gradient joins the norm's before the one rounding
    return {h, plain ? y.detach() : s};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    once_only("residual norm");
    no_foreign_leaf("residual norm");
    torch::autograd::variable_list out(9);
    const Tensor dh = grads[0].defined() ? grads[0].contiguous() : Tensor();
    const Tensor ds = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
    if (!dh.defined() && !ds.defined()) return out;
    const auto v = ctx->get_saved_variables();
    const auto i = ctx->saved_data["ints"].toIntVector();
    const NormOptions o{i[0], i[1] != 0, i[2] != 0, ctx->saved_data["alpha"].toDouble(), ctx->saved_data["eps"].toDouble()};
    // only the tensors that are there have an edge
    const std::array<bool, 7> there{true,           i[5] != 0,      v[3].defined(), v[4].defined(),
                                    v[5].defined(), v[6].defined(), v[7].defined()};
    std::array<bool, 7> want;
    for (size_t k = 0, edge = 0; k < want.size(); ++k) want[k] = there[k] && ctx->needs_input_grad(edge++);
    const auto g = resnorm_bwd(dh, ds, {v[2], v[1], v[3], v[4], v[5], v[6], v[7]}, o, v[0], v[8], want,
                               (at::ScalarType)i[3], (at::ScalarType)i[4]);
    std::copy(g.begin(), g.end(), out.begin());
    return out;
  }
};

// Consecutive rows of y that share one row of the gate, or -1: the gate is [width], or of y's shape with 1 in
// place of trailing dimensions before the last.
int64_t gate_rows_of(const Tensor& gate, const Tensor& y) {
  const int64_t lead = y.dim() - 1;
  if (gate.size(-1) != y.size(-1) || (gate.dim() != 1 && gate.dim() != y.dim())) return -1;
  auto size = [&](int64_t k) { return gate.dim() == y.dim() ? gate.size(k) : 1; };
  int64_t k = 0, rows = 1;
  while (k < lead && size(k) == y.size(k)) ++k;
  for (; k < lead; ++k) {
    if (size(k) != 1) return -1;
    rows *= y.size(k);
  }
  return rows;
}

// The same refusals, by value and by type, as the Python form of the operator makes for CPU tensors.
template <typename Error, typename... A>
void refuse_if(bool bad, const A&... what) {
  if (C10_UNLIKELY(bad)) throw Error(c10::str("residual_norm: ", what...));
}

// h, and s with return_sum
std::vector<Tensor> residual_norm(const Tensor& y, const OptTensor& x, const OptTensor& weight, const OptTensor& bias,
                                  const std::string& kind, double eps, const OptTensor& gate, double alpha, bool post,
                                  const OptTensor& post_weight, const OptTensor& post_bias, bool return_sum) {
  const bool rms = kind == "rms";
  using Value = py::value_error;
  using Type = py::type_error;
  refuse_if<Value>(!rms && kind != "layer", "kind '", kind, "': 'layer' or 'rms'");
  refuse_if<Value>(y.dim() < 1 || y.size(-1) < 1, "a block of shape ", y.sizes());
  refuse_if<Value>(!post && (has(post_weight) || has(post_bias)), "post_weight and post_bias need post=True");
  const auto ty = y.scalar_type();
  refuse_if<Type>(ty != at::kFloat && ty != at::kBFloat16 && ty != at::kHalf, "a block of ", ty);
  const int64_t width = y.size(-1);
  if (has(x)) {
    refuse_if<Value>(x->sizes() != y.sizes() || x->device() != y.device(), "a residual of ", x->sizes(), " on ",
                     x->device(), " for a block of ", y.sizes(), " on ", y.device());
    refuse_if<Type>(x->scalar_type() != ty && x->scalar_type() != at::kFloat, "a residual of ", x->scalar_type(),
                    " for a block of ", ty);
  } else {
    refuse_if<Value>(alpha != 1.0, "alpha scales a residual, and there is none");
  }
  auto param = [&](const OptTensor& p, const char* name, bool shaped) {
    if (!has(p)) return Tensor();
    refuse_if<Value>(p->device() != y.device(), name, " on ", p->device(), ", the block on ", y.device());
    refuse_if<Type>(p->scalar_type() != ty && p->scalar_type() != at::kFloat, name, " of ", p->scalar_type(),
                    " for a block of ", ty);
    refuse_if<Value>(shaped && (p->dim() != 1 || p->size(0) != width), name, " of shape ", p->sizes(), " for a width of ",
                     width);
    return p->contiguous();
  };
  const NormTensors t{y.contiguous(),
                      has(x) ? x->contiguous() : Tensor(),
                      param(gate, "gate", false),
                      param(weight, "weight", true),
                      param(bias, "bias", true),
                      param(post_weight, "post_weight", true),
                      param(post_bias, "post_bias", true)};
  const int64_t rows = y.numel() / width;
  int64_t gate_rows = rows;
  if (t.gate.defined()) {
    gate_rows = t.gate.dim() < 1 ? -1 : gate_rows_of(t.gate, y);
    refuse_if<Value>(gate_rows < 0, "a gate of shape ", t.gate.sizes(), " for a block of ", y.sizes(),
                     ": it is [width], or the block's shape with 1 in place of trailing dimensions before the last");
  }
  refuse_if<Value>(width > grace::kNormMaxWidth, "a width of ", width, ": at most ", grace::kNormMaxWidth, " on a GPU");
  refuse_if<Value>(rows >= INT32_MAX, "at most 2^31 - 2 rows");
  const NormOptions o{gate_rows, post, rms, alpha, eps};
  const bool follow = at::GradMode::is_enabled();
  bool grad = false;
  for (const Tensor* p : {&t.y, &t.x, &t.gate, &t.weight, &t.bias, &t.post_weight, &t.post_bias}) {
    if (!p->defined()) continue;
    no_tangent(*p, "residual norm");
    grad |= follow && p->requires_grad();
  }
  if (grad) {
    auto opt = [](const Tensor& u) { return u.defined() ? OptTensor(u) : OptTensor(); };
    return ResidualNormFn::apply(t.y, opt(t.x), opt(t.gate), opt(t.weight), opt(t.bias), opt(t.post_weight),
                                 opt(t.post_bias), o, return_sum);
  }
  const bool plain = is_plain(t, o);
  auto [h, s, stats] = resnorm_fwd(t, o, return_sum && !plain, false);
  if (!return_sum) return {h};
  return {h, plain ? t.y : s};
}

// ---------------------------------------------------------------- global gradient norm
// The tensors as memory, each once: an exact repetition counts once, other overlaps are refused.
std::vector<grace::GradTensor> grad_list(const std::vector<Tensor>& grads) {
  std::vector<grace::GradTensor> g;
  g.reserve(grads.size());
  for (const Tensor& t : grads) {
    TORCH_CHECK(t.is_cuda() && t.device() == grads[0].device(), "gradient norm: every tensor on one GPU");
    TORCH_CHECK(t.is_non_overlapping_and_dense(), "gradient norm: tensors must be dense");
    if (t.numel() > 0) g.push_back({t.data_ptr(), t.numel(), el_type(t.scalar_type(), "gradient norm: tensors")});
  }
  std::vector<int> order(g.size());
  for (size_t i = 0; i < g.size(); ++i) order[i] = (int)i;
  std::sort(order.begin(), order.end(), [&](int a, int b) { return g[a].p != g[b].p ? g[a].p < g[b].p : a < b; });
  std::vector<char> twice(g.size(), 0);
  bool any = false;
  for (size_t i = 1, last = 0; i < g.size(); ++i) {
    const auto &a = g[order[last]], &b = g[order[i]];
    if (a.p == b.p && a.len == b.len && a.type == b.type) {
      twice[order[i]] = 1;
      any = true;
      continue;
    }
    TORCH_CHECK(static_cast<char*>(a.p) + a.len * grace::el_bytes(a.type) <= static_cast<char*>(b.p),
                "gradient norm: two tensors overlap");
    last = i;
  }
  if (any) {
    size_t k = 0;
    for (size_t i = 0; i < g.size(); ++i)
      if (!twice[i]) g[k++] = g[i];
    g.resize(k);
  }
  return g;
}

grace::NormKind norm_kind(int64_t kind) {
  TORCH_CHECK(kind >= 0 && kind <= 2, "gradient norm: kind 0 (max), 1 or 2");
  return (grace::NormKind)kind;
}

Tensor parts_of(const std::vector<grace::GradTensor>& g, grace::NormKind kind, const Tensor& like) {
  Tensor part = at::empty({grace::gradnorm_parts(g.data(), (int64_t)g.size())}, like.options().dtype(at::kDouble));
  grace::gradnorm_partial(g.data(), (int64_t)g.size(), kind, part.data_ptr<double>(), cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return part;
}

// fp64 partial values of |g|^p over tensors of one GPU
Tensor grad_norm_parts(const std::vector<Tensor>& grads, int64_t kind) {
  TORCH_CHECK(!grads.empty(), "gradient norm: no tensors");
  DevGuard guard(grads[0].device());
  return parts_of(grad_list(grads), norm_kind(kind), grads[0]);
}

// [norm, factor] fp32 from partial values
Tensor grad_norm_finish(const Tensor& part, int64_t kind, double max_norm) {
  TORCH_CHECK(part.is_cuda() && part.scalar_type() == at::kDouble && part.is_contiguous(), "gradient norm: fp64 parts");
  DevGuard guard(part.device());
  Tensor out = at::empty({2}, part.options().dtype(at::kFloat));
  grace::gradnorm_finish(part.data_ptr<double>(), part.numel(), norm_kind(kind), (float)max_norm,
                         out.data_ptr<float>(), cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}

// grads *= factor (fp32, one device value)
void grad_scale(const std::vector<Tensor>& grads, const Tensor& factor) {
  if (grads.empty()) return;
  check_on(factor, grads[0], "gradient norm: the factor");
  TORCH_CHECK(factor.scalar_type() == at::kFloat && factor.numel() == 1, "gradient norm: one fp32 factor");
  DevGuard guard(grads[0].device());
  const auto g = grad_list(grads);
  grace::grad_scale(g.data(), (int64_t)g.size(), factor.data_ptr<float>(), cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  for (const Tensor& t : grads) t.unsafeGetTensorImpl()->bump_version();
}

// [norm, factor] fp32 of the parameters' gradients, which are scaled in place with `scale`; none where they
// are not all dense gradients of a kernel's type on one GPU, or not there
OptTensor grad_clip(const std::vector<Tensor>& params, int64_t kind, double max_norm, bool scale) {
  std::vector<Tensor> grads;
  grads.reserve(params.size());
  for (const Tensor& p : params) {
    const Tensor& g = p.grad();
    if (!g.defined()) continue;
    const auto t = g.scalar_type();
    if (!g.is_cuda() || g.layout() != at::kStrided || (t != at::kFloat && t != at::kBFloat16 && t != at::kHalf) ||
        (!grads.empty() && g.device() != grads[0].device()) || !g.is_non_overlapping_and_dense())
      return c10::nullopt;
    grads.push_back(g);
  }
  if (grads.empty()) return c10::nullopt;
  DevGuard guard(grads[0].device());
  const auto g = grad_list(grads);
  const Tensor part = parts_of(g, norm_kind(kind), grads[0]);
  if (!scale || g.empty()) return grad_norm_finish(part, kind, max_norm);
  Tensor out = at::empty({2}, grads[0].options().dtype(at::kFloat));
  grace::grad_clip(g.data(), (int64_t)g.size(), part.data_ptr<double>(), part.numel(), norm_kind(kind),
                   (float)max_norm, out.data_ptr<float>(), cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  for (const Tensor& t : grads) t.unsafeGetTensorImpl()->bump_version();
  return out;
}

at::ScalarType scalar_type(const py::object& dtype) {
  if (!THPDtype_Check(dtype.ptr())) throw py::type_error("dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
}

}  // namespace

void grace_bind_lm(py::module& m) {
  m.def("embedding", [](const Tensor& ids, const Tensor& weight, double scale, const c10::optional<int64_t>& padding_idx,
                        const py::object& dtype) {
    return embedding(ids, weight, scale, padding_idx,
                     dtype.is_none() ? c10::optional<at::ScalarType>() : scalar_type(dtype));
  });
  m.def("residual_norm", &residual_norm);
  m.def("grad_norm_parts", &grad_norm_parts);
  m.def("grad_norm_finish", &grad_norm_finish);
  m.def("grad_scale", &grad_scale);
  m.def("grad_clip", &grad_clip);
}
