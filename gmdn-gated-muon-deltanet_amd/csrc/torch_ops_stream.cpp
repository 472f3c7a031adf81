// torch.ops.gmdn.* along an LM's residual stream (include/gmdn_lm.h): token
// embedding, a branch's residual with its norms, and log probabilities from
// hidden states and the head's weight, with autograd on the forward operators.
// gmdn_amd/ops.py documents them.
#include "../../include/gmdn_lm.h"
#include "torch_ops_rows.h"

namespace {

using namespace gmdn_ops;

// A (vocab, d) table's rows.
Rows table_of(const Tensor& weight) {
  check_rank(weight, 2, "weight");
  TORCH_CHECK(weight.size(0) > 0, "weight has at least one row, got shape ", weight.sizes());
  return rows_of(weight, "weight");
}
Tensor none_like(const Tensor& x, ScalarType dtype) { return fresh(x, {0}, dtype); }

// ----------------------------------------------------------- token embedding
Tensor embed_fwd(const Tensor& weight, const Tensor& tokens, double scale, int64_t /*padding_idx*/) {
  const c10::DeviceGuard guard(weight.device());
  const int32_t code = type_code(weight.scalar_type(), "weight");
  const Rows w = table_of(weight);
  const Tensor tk = tokens_of(tokens, weight, tokens.sizes());
  Tensor y = fresh(weight, with_last(tokens.sizes().vec(), w.d), weight.scalar_type());
  if (tk.numel())
    check(gmdn_embed_fwd(w.ptr(), tk.data_ptr<int64_t>(), y.data_ptr(), tk.numel(), w.rows, w.d, w.stride, (float)scale,
                         code, stream_of(weight)),
          "gmdn_embed_fwd");
  return y;
}
Tensor embed_bwd(const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale, int64_t padding_idx) {
  const c10::DeviceGuard guard(dy.device());
  const int32_t code = type_code(dy.scalar_type(), "dy");
  TORCH_CHECK(vocab > 0, "a table has at least one row, got vocab ", vocab);
  TORCH_CHECK(dy.dim() >= 1, "dy has rows in its last dimension, got shape ", dy.sizes());
  const Tensor tk = tokens_of(tokens, dy, lead(dy));
  const Rows g = rows_of(dy, "dy");
  Tensor dw = fresh(dy, {vocab, g.d}, dy.scalar_type());
  const size_t need = gmdn_embed_bwd_workspace_bytes(g.rows, vocab, g.d);
  const Tensor ws = need ? fresh(dy, {(int64_t)need}, at::kByte) : Tensor();
  check(gmdn_embed_bwd(g.ptr(), tk.data_ptr<int64_t>(), dw.data_ptr(), need ? ws.data_ptr() : nullptr, need, g.rows,
                       vocab, g.d, g.stride, (float)scale, padding_idx, code, stream_of(dy)),
        "gmdn_embed_bwd");
  return dw;
}

// -------------------------------------------------- residual with its norms
// The vectors of a call, contiguous, of one type; absent ones stay so.
struct Vectors {
  OptTensor w, p, s;
  int32_t code = GMDN_DTYPE_F32;
};
Vectors vectors_of(const OptTensor& weight, const OptTensor& post_weight, const OptTensor& scale, const Tensor& x,
                   int64_t d) {
  Vectors v;
  std::optional<ScalarType> type;
  auto take = [&](const OptTensor& t, const char* what) -> OptTensor {
    if (!t) return t;
    check_like(*t, x, {d}, what);
    TORCH_CHECK(!type || *type == t->scalar_type(), "weight, post_weight and scale are of one type, got ", *type, " and ",
                t->scalar_type());
    type = t->scalar_type();
    v.code = type_code(*type, what);
    return t->contiguous();
  };
  v.w = take(weight, "weight");
  v.p = take(post_weight, "post_weight");
  v.s = take(scale, "scale");
  return v;
}
// A branch's output and gate beside the stream, or an absent one.
Rows branch_of(const Tensor& t, const Tensor& x, ScalarType dtype, const char* what) {
  check_like(t, x, x.sizes(), what);
  TORCH_CHECK(t.scalar_type() == dtype, what, " is ", dtype, ", got ", t.scalar_type());
  return rows_of(t, what);
}
Rows branch_of(const OptTensor& t, const Tensor& x, ScalarType dtype, const char* what) {
  return t ? branch_of(*t, x, dtype, what) : Rows{};
}
const void* ptr(const Rows& r) { return r.t.defined() ? r.t.data_ptr() : nullptr; }
using gmdn_ops::ptr;

using Residual = std::tuple<Tensor, Tensor, Tensor, Tensor>;
Residual residual_norm_fwd(const Tensor& x, const Tensor& y, const OptTensor& weight, const OptTensor& post_weight,
                           const OptTensor& gate, const OptTensor& scale, double eps) {
  const c10::DeviceGuard guard(x.device());
  const int32_t xc = type_code(x.scalar_type(), "x"), yc = type_code(y.scalar_type(), "y");
  const Rows r = rows_of(x, "x"), b = branch_of(y, x, y.scalar_type(), "y"),
             g = branch_of(gate, x, y.scalar_type(), "gate");
  const Vectors v = vectors_of(weight, post_weight, scale, x, r.d);
  Tensor out = fresh(x, x.sizes(), x.scalar_type()), z = fresh(x, x.sizes(), y.scalar_type()), rstd = fresh(x, lead(x));
  Tensor post_rstd = v.p ? fresh(x, lead(x)) : fresh(x, {0});
  if (r.rows)
    check(gmdn_residual_norm_fwd(r.ptr(), b.ptr(), ptr(v.w), ptr(v.p), ptr(g), ptr(v.s), out.data_ptr(), z.data_ptr(),
                                 fp(rstd), v.p ? fp(post_rstd) : nullptr, r.rows, r.d, r.stride, b.stride, g.stride,
                                 (float)eps, xc, yc, v.code, stream_of(x)),
          "gmdn_residual_norm_fwd");
  return {out, z, rstd, post_rstd};
}

// Whether the backward reads the stream that the forward returned, r, and not y:
// a float32 one with nothing but the sum.
bool from_r(const Tensor& x, bool plain) { return plain && x.scalar_type() == at::kFloat; }

using Grads6 = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
Grads6 residual_norm_bwd(const OptTensor& dr, const OptTensor& dz, const Tensor& r_or_x, const OptTensor& y,
                         const OptTensor& weight, const OptTensor& post_weight, const OptTensor& gate,
                         const OptTensor& scale, const Tensor& rstd_, const Tensor& post_rstd_,
                         std::optional<ScalarType> y_dtype) {
  const c10::DeviceGuard guard(r_or_x.device());
  const Tensor& x = r_or_x;
  const ScalarType xt = x.scalar_type(), yt = y ? y->scalar_type() : y_dtype.value_or(xt);
  const int32_t xc = type_code(xt, "the stream"), yc = type_code(yt, "y");
  TORCH_CHECK(y || from_r(x, !post_weight && !gate && !scale),
              "y is given but for a float32 stream without post norm, gate and scale");
  const Rows r = rows_of(x, "the stream"), a = branch_of(dr, x, xt, "dr"), z = branch_of(dz, x, yt, "dz"),
             b = branch_of(y, x, yt, "y"), g = branch_of(gate, x, yt, "gate");
  const Vectors v = vectors_of(weight, post_weight, scale, x, r.d);
  const Tensor rstd = stat(rstd_, x, lead(x), "rstd"), post = v.p ? stat(post_rstd_, x, lead(x), "post_rstd") : Tensor();
  const bool same = !v.p && !v.s && !gate && xt == yt;  // dy is dx
  Tensor dx = fresh(x, x.sizes(), xt), dy = same ? none_like(x, yt) : fresh(x, x.sizes(), yt);
  Tensor dg = gate ? fresh(x, x.sizes(), yt) : none_like(x, yt);
  auto grad = [&](const OptTensor& t) { return t ? at::empty_like(*t) : fresh(x, {0}); };
  Tensor dw = grad(v.w), dp = grad(v.p), ds = grad(v.s);
  const bool vectors = v.w || v.p || v.s;
  const size_t need = vectors ? gmdn_residual_norm_bwd_workspace_floats(r.rows, r.d) : 0;
  const Tensor ws = need ? fresh(x, {(int64_t)need}) : Tensor();
  if (r.rows || vectors)
    check(gmdn_residual_norm_bwd(ptr(a), ptr(z), r.ptr(), ptr(b), ptr(v.w), ptr(v.p), ptr(g), ptr(v.s), fp(rstd),
                                 v.p ? fp(post) : nullptr, dx.data_ptr(), same ? nullptr : dy.data_ptr(),
                                 gate ? dg.data_ptr() : nullptr, v.w ? dw.data_ptr() : nullptr,
                                 v.p ? dp.data_ptr() : nullptr, v.s ? ds.data_ptr() : nullptr, need ? fp(ws) : nullptr,
                                 need, r.rows, r.d, a.stride, z.stride, r.stride, b.stride, g.stride, xc, yc, v.code,
                                 stream_of(x)),
          "gmdn_residual_norm_bwd");
  return {dx, dy, dw, dp, dg, ds};
}

// ----------------------------- log probabilities from hidden states and a head
Rows head_of(const Tensor& weight, const Tensor& x, const Rows& r) {
  const Rows w = table_of(weight);
  TORCH_CHECK(weight.device() == x.device(), "weight is on ", weight.device(), ", x on ", x.device());
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "x and weight are of one type, got ", x.scalar_type(), " and ",
              weight.scalar_type());
  TORCH_CHECK(w.d == r.d, "weight has rows of ", w.d, " values where x has ", r.d);
  return w;
}
// The operands' type code; `precision` is of float32 ones.
int32_t operands_code(const Tensor& x, int64_t precision) {
  const int32_t code = type_code(x.scalar_type(), "x");
  TORCH_CHECK(precision == GMDN_PREC_TF32 || precision == GMDN_PREC_IEEE, "precision is 0 ('tf32') or 1 ('ieee'), got ",
              precision);
  return code == GMDN_DTYPE_F32 && precision == GMDN_PREC_IEEE ? GMDN_DTYPE_F32_IEEE : code;
}
std::tuple<Tensor, Tensor, Tensor> linear_logprobs_fwd(const Tensor& x, const Tensor& weight, const Tensor& tokens,
                                                       int64_t ignore_index, int64_t precision) {
  const c10::DeviceGuard guard(x.device());
  const int32_t code = operands_code(x, precision);
  const Rows r = rows_of(x, "x"), w = head_of(weight, x, r);
  const Tensor tk = tokens_of(tokens, x, lead(x));
  Tensor lp = fresh(x, lead(x)), entropy = fresh(x, lead(x)), stats = fresh(x, with_last(lead(x), 2));
  const size_t need =
      gmdn_linear_logprobs_fwd_workspace_bytes(r.ptr(), w.ptr(), r.rows, w.rows, r.d, r.stride, w.stride, code);
  const Tensor ws = need ? fresh(x, {(int64_t)need}, at::kByte) : Tensor();
  if (r.rows)
    check(gmdn_linear_logprobs_fwd(r.ptr(), w.ptr(), tk.data_ptr<int64_t>(), fp(lp), fp(entropy), fp(stats),
                                   need ? ws.data_ptr() : nullptr, need, r.rows, w.rows, r.d, r.stride, w.stride,
                                   ignore_index, code, stream_of(x)),
          "gmdn_linear_logprobs_fwd");
  return {lp, entropy, stats};
}
std::tuple<Tensor, Tensor> linear_logprobs_bwd(const Tensor& x, const Tensor& weight, const Tensor& tokens,
                                               const Tensor& stats_, const Tensor& entropy_, const OptTensor& dlogprob,
                                               const OptTensor& dentropy, int64_t ignore_index, bool need_x,
                                               bool need_weight, int64_t precision) {
  const c10::DeviceGuard guard(x.device());
  const int32_t code = operands_code(x, precision);
  const Rows r = rows_of(x, "x"), w = head_of(weight, x, r);
  const auto shape = lead(x);
  const Tensor tk = tokens_of(tokens, x, shape);
  const Tensor stats = stat(stats_, x, with_last(shape, 2), "stats"), entropy = stat(entropy_, x, shape, "entropy");
  const OptTensor dl = stat(dlogprob, x, shape, "dlogprob"), dh = stat(dentropy, x, shape, "dentropy");
  Tensor dx = need_x ? fresh(x, x.sizes(), x.scalar_type()) : none_like(x, x.scalar_type());
  Tensor dw = need_weight ? fresh(x, weight.sizes(), x.scalar_type()) : none_like(x, x.scalar_type());
  if (!need_x && !need_weight) return {dx, dw};
  if (r.rows == 0) return {dx, dw.zero_()};
  const size_t need =
      gmdn_linear_logprobs_bwd_workspace_bytes(r.ptr(), w.ptr(), r.rows, w.rows, r.d, r.stride, w.stride, code);
  const Tensor ws = need ? fresh(x, {(int64_t)need}, at::kByte) : Tensor();
  check(gmdn_linear_logprobs_bwd(r.ptr(), w.ptr(), tk.data_ptr<int64_t>(), fp(stats), fp(entropy), fp(dl), fp(dh),
                                 need_x ? dx.data_ptr() : nullptr, need_weight ? dw.data_ptr() : nullptr,
                                 need ? ws.data_ptr() : nullptr, need, r.rows, w.rows, r.d, r.stride, w.stride,
                                 ignore_index, code, stream_of(x)),
        "gmdn_linear_logprobs_bwd");
  return {dx, dw};
}

// ------------------------------------------------------------------ autograd
struct EmbedFwd : torch::autograd::Function<EmbedFwd> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, double scale,
                        c10::SymInt padding_idx) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.sym_size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
    return GMDN_OP(embed_fwd).call(weight, tokens, scale, padding_idx);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const Tensor none;
    if (!g[0].defined()) return {none, none, none, none};
    return {GMDN_OP(embed_bwd).call(g[0], ctx->get_saved_variables()[0], ctx->saved_data["vocab"].toSymInt(),
                                    ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding_idx"].toSymInt()),
            none, none, none};
  }
};
Tensor embed_fwd_ad(const Tensor& weight, const Tensor& tokens, double scale, c10::SymInt padding_idx) {
  refuse_tangents("embed_fwd", {&weight});
  if (!wants_grad({&weight})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GMDN_OP(embed_fwd).call(weight, tokens, scale, padding_idx);
  }
  return EmbedFwd::apply(weight, tokens, scale, padding_idx);
}

struct ResidualNormFwd : torch::autograd::Function<ResidualNormFwd> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const OptTensor& weight,
                               const OptTensor& post_weight, const OptTensor& gate, const OptTensor& scale, double eps,
                               std::pair<Tensor, Tensor>* rest) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [r, z, rstd, post_rstd] =
        GMDN_OP(residual_norm_fwd).call(x, y, weight, post_weight, gate, scale, eps);
    *rest = {rstd, post_rstd};
    ctx->set_materialize_grads(false);
    const bool after = from_r(x, !post_weight && !gate && !scale);
    ctx->save_for_backward({after ? r : x, after ? Tensor() : y, opt(weight), opt(post_weight), opt(gate), opt(scale),
                            rstd, post_rstd});
    ctx->saved_data["y_dtype"] = y.scalar_type();
    return {r, z};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const Tensor none;
    variable_list out(8);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const ScalarType yt = ctx->saved_data["y_dtype"].toScalarType();
    auto [dx, dy, dw, dp, dg, ds] = GMDN_OP(residual_norm_bwd)
                                        .call(opt(g[0]), opt(g[1]), s[0], opt(s[1]), opt(s[2]), opt(s[3]), opt(s[4]),
                                              opt(s[5]), s[6], s[7], yt);
    const bool same = !s[3].defined() && !s[4].defined() && !s[5].defined() && s[0].scalar_type() == yt;
    out[0] = dx;
    out[1] = same ? dx : dy;
    if (s[2].defined()) out[2] = dw;
    if (s[3].defined()) out[3] = dp;
    if (s[4].defined()) out[4] = dg;
    if (s[5].defined()) out[5] = ds;
    return out;
  }
};
Residual residual_norm_fwd_ad(const Tensor& x, const Tensor& y, const OptTensor& weight, const OptTensor& post_weight,
                              const OptTensor& gate, const OptTensor& scale, double eps) {
  const Tensor w = opt(weight), p = opt(post_weight), g = opt(gate), s = opt(scale);
  refuse_tangents("residual_norm_fwd", {&x, &y, &w, &p, &g, &s});
  if (!wants_grad({&x, &y, &w, &p, &g, &s})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GMDN_OP(residual_norm_fwd).call(x, y, weight, post_weight, gate, scale, eps);
  }
  std::pair<Tensor, Tensor> rest;
  auto r = ResidualNormFwd::apply(x, y, weight, post_weight, gate, scale, eps, &rest);
  return {r[0], r[1], rest.first, rest.second};
}

struct LinearLogprobsFwd : torch::autograd::Function<LinearLogprobsFwd> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& tokens,
                               c10::SymInt ignore_index, c10::SymInt precision, Tensor* rest) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [lp, entropy, stats] = GMDN_OP(linear_logprobs_fwd).call(x, weight, tokens, ignore_index, precision);
    *rest = stats;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, tokens, stats, entropy});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["precision"] = precision;
    ctx->saved_data["need_x"] = x.requires_grad();
    ctx->saved_data["need_weight"] = weight.requires_grad();
    return {lp, entropy};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const Tensor none;
    if (!g[0].defined() && !g[1].defined()) return {none, none, none, none, none, none};
    const auto s = ctx->get_saved_variables();
    const bool need_x = ctx->saved_data["need_x"].toBool(), need_weight = ctx->saved_data["need_weight"].toBool();
    auto [dx, dw] = GMDN_OP(linear_logprobs_bwd)
                        .call(s[0], s[1], s[2], s[3], s[4], opt(g[0]), opt(g[1]),
                              ctx->saved_data["ignore_index"].toSymInt(), need_x, need_weight,
                              ctx->saved_data["precision"].toSymInt());
    return {need_x ? dx : none, need_weight ? dw : none, none, none, none, none};
  }
};
std::tuple<Tensor, Tensor, Tensor> linear_logprobs_fwd_ad(const Tensor& x, const Tensor& weight, const Tensor& tokens,
                                                          c10::SymInt ignore_index, c10::SymInt precision) {
  refuse_tangents("linear_logprobs_fwd", {&x, &weight});
  if (!wants_grad({&x, &weight})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GMDN_OP(linear_logprobs_fwd).call(x, weight, tokens, ignore_index, precision);
  }
  Tensor stats;
  auto r = LinearLogprobsFwd::apply(x, weight, tokens, ignore_index, precision, &stats);
  return {r[0], r[1], stats};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(gmdn, m) {
  const std::vector<at::Tag> PT2{at::Tag::pt2_compliant_tag};
  m.def("embed_fwd(Tensor weight, Tensor tokens, float scale=1.0, SymInt padding_idx=-1) -> Tensor", PT2);
  m.def("embed_bwd(Tensor dy, Tensor tokens, SymInt vocab, float scale, SymInt padding_idx) -> Tensor", PT2);
  m.def("residual_norm_fwd(Tensor x, Tensor y, Tensor? weight, Tensor? post_weight, Tensor? gate, Tensor? scale, "
        "float eps) -> (Tensor, Tensor, Tensor, Tensor)", PT2);
  m.def("residual_norm_bwd(Tensor? dr, Tensor? dz, Tensor r_or_x, Tensor? y, Tensor? weight, Tensor? post_weight, "
        "Tensor? gate, Tensor? scale, Tensor rstd, Tensor post_rstd, ScalarType? y_dtype=None) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", PT2);
  m.def("linear_logprobs_fwd(Tensor x, Tensor weight, Tensor tokens, SymInt ignore_index, SymInt precision=0) -> "
        "(Tensor, Tensor, Tensor)", PT2);
  m.def("linear_logprobs_bwd(Tensor x, Tensor weight, Tensor tokens, Tensor stats, Tensor entropy, Tensor? dlogprob, "
        "Tensor? dentropy, SymInt ignore_index, bool need_x, bool need_weight, SymInt precision=0) -> (Tensor, Tensor)",
        PT2);
}

TORCH_LIBRARY_IMPL(gmdn, CUDA, m) {
  m.impl("embed_fwd", embed_fwd);
  m.impl("embed_bwd", embed_bwd);
  m.impl("residual_norm_fwd", residual_norm_fwd);
  m.impl("residual_norm_bwd", residual_norm_bwd);
  m.impl("linear_logprobs_fwd", linear_logprobs_fwd);
  m.impl("linear_logprobs_bwd", linear_logprobs_bwd);
}

TORCH_LIBRARY_IMPL(gmdn, Autograd, m) {
  m.impl("embed_fwd", embed_fwd_ad);
  m.impl("residual_norm_fwd", residual_norm_fwd_ad);
  m.impl("linear_logprobs_fwd", linear_logprobs_fwd_ad);
  // No derivative of their own: differentiating through them raises.
  for (const char* name : {"embed_bwd", "residual_norm_bwd", "linear_logprobs_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
