// Python bindings for the language-model training kernels (csrc/include/grace_lm.h): embedding,
// residual norms, the global gradient norm.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPException.h>

#include <algorithm>

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
grace::EmbedIds embed_ids(const Tensor& ids, int64_t vocab, int64_t pad) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
              "embedding: ids must be a contiguous int64 or int32 GPU tensor");
  TORCH_CHECK(ids.numel() < INT32_MAX && vocab < INT32_MAX, "embedding: at most 2^31 - 2 tokens and rows");
  TORCH_CHECK(pad >= -1 && pad < vocab, "embedding: padding_idx out of range");
  return {ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), vocab, pad};
}

Tensor embed_fwd(const Tensor& ids, const Tensor& weight, double scale, at::ScalarType dtype) {
  TORCH_CHECK(weight.is_cuda() && weight.dim() == 2 && (weight.stride(1) == 1 || weight.size(1) <= 1),
              "embedding: the table must be a 2-D GPU tensor with contiguous rows");
  check_on(ids, weight, "embedding: ids");
  TORCH_CHECK(weight.size(0) > 0 || ids.numel() == 0, "embedding: the table has no rows");
  const grace::EmbedIds e = embed_ids(ids, weight.size(0), -1);
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
  const grace::EmbedIds e = embed_ids(ids, vocab, pad);
  DevGuard guard(dy.device());
  const auto tdw = el_type(dtype, "embedding: the table"), tdy = el_type(dy.scalar_type(), "embedding: the gradient");
  Tensor dw = at::zeros({vocab, d}, dy.options().dtype(dtype));
  Tensor ws = at::empty({grace::embed_backward_ws(e.n, vocab, d)}, dy.options().dtype(at::kByte));
  grace::embed_backward(e, dy.data_ptr(), tdy, d, (float)scale, dw.data_ptr(), tdw, ws.data_ptr(), cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dw;
}

// ---------------------------------------------------------------- residual norm
grace::NormParam norm_param(const OptTensor& t, int64_t n, const Tensor& y, const char* what) {
  if (!has(t)) return {nullptr, false};
  check_on(*t, y, what);
  TORCH_CHECK(t->is_contiguous() && t->numel() == n, what, ": contiguous, ", n, " values");
  TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == y.scalar_type(), what,
              " must be float32 or of the block's type");
  return {t->data_ptr(), t->scalar_type() == at::kFloat};
}

grace::NormShape norm_shape(const Tensor& y, at::ScalarType tx, int64_t gate_rows, double alpha, double eps, bool rms,
                            bool post) {
  TORCH_CHECK(y.is_cuda() && y.dim() >= 1 && y.is_contiguous(), "residual norm: the block must be contiguous on a GPU");
  const int64_t d = y.size(-1);
  TORCH_CHECK(d >= 1 && d <= grace::kNormMaxWidth, "residual norm: widths 1 to ", grace::kNormMaxWidth);
  const int64_t rows = y.numel() / d;
  TORCH_CHECK(rows == 0 || (gate_rows >= 1 && rows % gate_rows == 0), "residual norm: rows per gate row");
  grace::NormShape n{rows, gate_rows, (int)d, (float)alpha, (float)eps, rms, post,
                     el_type(tx, "residual norm: the residual"), el_type(y.scalar_type(), "residual norm: the block")};
  TORCH_CHECK(n.tx == n.ty || n.tx == grace::ElType::kF32, "residual norm: the residual must be float32 or of the block's type");
  return n;
}

int64_t gate_size(const grace::NormShape& n) { return n.rows == 0 ? -1 : n.rows / n.gate_rows * n.d; }

// returns (h, s, stats); s and stats are undefined where they are not wanted
std::vector<Tensor> resnorm_fwd(const Tensor& y, const OptTensor& x, const OptTensor& gate, int64_t gate_rows,
                                const OptTensor& weight, const OptTensor& bias, const OptTensor& post_weight,
                                const OptTensor& post_bias, bool post, bool rms, double alpha, double eps,
                                bool want_sum, bool want_stats) {
  const auto tx = has(x) ? x->scalar_type() : y.scalar_type();
  const grace::NormShape n = norm_shape(y, tx, gate_rows, alpha, eps, rms, post);
  if (has(x)) {
    check_on(*x, y, "residual norm: the residual");
    TORCH_CHECK(x->sizes() == y.sizes() && x->is_contiguous(), "residual norm: the residual must be like the block");
  }
  DevGuard guard(y.device());
  Tensor h = at::empty_like(y);
  Tensor s = want_sum ? at::empty(y.sizes(), y.options().dtype(tx)) : Tensor();
  Tensor stats = want_stats ? at::empty({post ? 4 : 2, n.rows}, y.options().dtype(at::kFloat)) : Tensor();
  if (n.rows > 0) {
    grace::resnorm_forward(n, has(x) ? x->data_ptr() : nullptr, y.data_ptr(),
                           norm_param(gate, gate_size(n), y, "residual norm: the gate"),
                           norm_param(weight, n.d, y, "residual norm: weight"),
                           norm_param(bias, n.d, y, "residual norm: bias"),
                           norm_param(post_weight, n.d, y, "residual norm: post_weight"),
                           norm_param(post_bias, n.d, y, "residual norm: post_bias"), h.data_ptr(),
                           want_sum ? s.data_ptr() : nullptr, want_stats ? stats.data_ptr<float>() : nullptr,
                           cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {h, s, stats};
}

// want: dx, dy (always made), dgate, dweight, dbias, dpost_weight, dpost_bias.
// returns those in that order, undefined where not wanted; one tensor for dx and dy where they are equal
std::vector<Tensor> resnorm_bwd(const OptTensor& dh, const OptTensor& ds, const Tensor& s, const Tensor& y,
                                const Tensor& stats, const OptTensor& gate, int64_t gate_rows, const OptTensor& weight,
                                const OptTensor& bias, const OptTensor& post_weight, const OptTensor& post_bias,
                                bool post, bool rms, double alpha, double eps, std::vector<bool> want) {
  const grace::NormShape n = norm_shape(y, s.scalar_type(), gate_rows, alpha, eps, rms, post);
  TORCH_CHECK(want.size() == 7, "residual norm: seven flags");
  auto like = [&](const Tensor& t, at::ScalarType type, const char* what) {
    check_on(t, y, what);
    TORCH_CHECK(t.sizes() == y.sizes() && t.is_contiguous() && t.scalar_type() == type, what, " must be like the forward's");
  };
  like(s, s.scalar_type(), "residual norm: the saved sum");
  if (has(dh)) like(*dh, y.scalar_type(), "residual norm: the norm's gradient");
  if (has(ds)) like(*ds, s.scalar_type(), "residual norm: the sum's gradient");
  TORCH_CHECK(stats.is_cuda() && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                  stats.numel() == (post ? 4 : 2) * n.rows, "residual norm: the saved statistics");
  DevGuard guard(y.device());
  const grace::NormParam gp = norm_param(gate, gate_size(n), y, "residual norm: the gate");
  const grace::NormParam wp = norm_param(weight, n.d, y, "residual norm: weight");
  const grace::NormParam bp = norm_param(bias, n.d, y, "residual norm: bias");
  const grace::NormParam pwp = norm_param(post_weight, n.d, y, "residual norm: post_weight");
  const grace::NormParam pbp = norm_param(post_bias, n.d, y, "residual norm: post_bias");
  auto made = [&](int k, const OptTensor& p) {
    if (!want[k] || !has(p)) return Tensor();
    return n.rows > 0 ? at::empty_like(*p) : at::zeros_like(*p);
  };
  Tensor dy = at::empty_like(y);
  const bool one = !gp.p && !post && (float)alpha == 1.f && n.tx == n.ty;
  Tensor dx = !want[0] ? Tensor() : one ? dy : at::empty_like(s);
  Tensor dgate = made(2, gate), dw = made(3, weight), db = made(4, bias), dpw = made(5, post_weight),
         dpb = made(6, post_bias);
  if (n.rows > 0) {
    auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    const grace::NormGrads g{ptr(dx), dy.data_ptr(), ptr(dgate), ptr(dw), ptr(db), ptr(dpw), ptr(dpb), bp.f32, pbp.f32};
    Tensor ws = at::empty({grace::resnorm_backward_ws(n)}, y.options().dtype(at::kByte));
    grace::resnorm_backward(n, s.data_ptr(), y.data_ptr(), stats.data_ptr<float>(), gp, wp, pwp, pbp,
                            has(dh) ? dh->data_ptr() : nullptr, has(ds) ? ds->data_ptr() : nullptr, g, ws.data_ptr(),
                            cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {dx, dy, dgate, dw, db, dpw, dpb};
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
}

// norm, factor and scaling of tensors of one GPU; returns [norm, factor]
Tensor grad_clip(const std::vector<Tensor>& grads, int64_t kind, double max_norm) {
  TORCH_CHECK(!grads.empty(), "gradient norm: no tensors");
  DevGuard guard(grads[0].device());
  const auto g = grad_list(grads);
  Tensor part = parts_of(g, norm_kind(kind), grads[0]);
  Tensor out = grad_norm_finish(part, kind, max_norm);
  grace::grad_scale(g.data(), (int64_t)g.size(), out.data_ptr<float>() + 1, cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}

at::ScalarType scalar_type(const py::object& dtype) {
  return reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
}

}  // namespace

void grace_bind_lm(py::module& m) {
  m.def("embed_fwd", [](const Tensor& ids, const Tensor& weight, double scale, const py::object& dtype) {
    return embed_fwd(ids, weight, scale, scalar_type(dtype));
  });
  m.def("embed_bwd", [](const Tensor& ids, const Tensor& dy, int64_t vocab, int64_t pad, double scale,
                        const py::object& dtype) { return embed_bwd(ids, dy, vocab, pad, scale, scalar_type(dtype)); });
  m.attr("resnorm_max_width") = (int64_t)grace::kNormMaxWidth;
  m.def("resnorm_fwd", &resnorm_fwd);
  m.def("resnorm_bwd", &resnorm_bwd);
  m.def("grad_norm_parts", &grad_norm_parts);
  m.def("grad_norm_finish", &grad_norm_finish);
  m.def("grad_scale", &grad_scale);
  m.def("grad_clip", &grad_clip);
}
