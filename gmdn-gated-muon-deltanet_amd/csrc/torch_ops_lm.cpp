// torch.ops.gmdn.* of the LM around the mixer (include/gmdn_lm.h): layer norm,
// 8-bit activation checkpoints, log probabilities of given tokens, with
// autograd on the forward operators.  gmdn_amd/ops.py documents them.
//
// Inputs are (..., d) tensors read in place where their rows have unit stride
// and one stride between them (slices of wider tensors, padded vocabularies),
// else copied; outputs are contiguous.
#include "../../include/gmdn_lm.h"
#include "torch_ops.h"

#include <ATen/hip/EmptyTensor.h>

#include <array>

namespace {

using namespace gmdn_ops;
using at::ScalarType;

// A contiguous tensor beside x, straight from the allocator: five of them
// through the dispatcher are a sixth of a small call's host time.
Tensor fresh(const Tensor& x, at::IntArrayRef sizes, ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, x.device(), std::nullopt);
}
Tensor fresh(const Tensor& x, at::IntArrayRef sizes) { return fresh(x, sizes, at::kFloat); }

int32_t type_code(ScalarType t, const char* what) {
  TORCH_CHECK(t == at::kBFloat16 || t == at::kFloat, what, " is bfloat16 or float32, got ", t);
  return t == at::kFloat ? GMDN_DTYPE_F32 : GMDN_DTYPE_BF16;
}

// t as `rows` rows of d values.
struct Rows {
  Tensor t;
  int64_t rows, d, stride;
  const void* ptr() const { return t.data_ptr(); }
};
Rows rows_of(const Tensor& t, const char* what) {
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) > 0, what, " has rows of at least one value in its last dimension, got shape ",
              t.sizes());
  const int64_t d = t.size(-1), rows = t.numel() / d;
  bool fits = d == 1 || t.stride(-1) == 1;
  int64_t stride = d, extent = -1;  // extent: what the dimension outside has to stride by
  for (int64_t i = t.dim() - 2; fits && i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (extent < 0)
      stride = t.stride(i);
    else
      fits = t.stride(i) == extent;
    extent = t.stride(i) * t.size(i);
  }
  if (rows == 0) return {t, 0, d, d};
  return fits ? Rows{t, rows, d, stride} : Rows{t.contiguous(), rows, d, d};
}

std::vector<int64_t> lead(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1).vec(); }
std::vector<int64_t> with_last(std::vector<int64_t> s, int64_t n) {
  s.push_back(n);
  return s;
}

void check_like(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* what) {
  TORCH_CHECK(t.device() == x.device(), what, " is on ", t.device(), ", the operator's input on ", x.device());
  TORCH_CHECK(t.sizes() == shape, what, " has shape ", t.sizes(), " where ", shape, " is expected");
}
// A float32 vector of per-row (or per-group) values, contiguous.
Tensor stat(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* what) {
  check_like(t, x, shape, what);
  TORCH_CHECK(t.scalar_type() == at::kFloat, what, " is float32, got ", t.scalar_type());
  return t.contiguous();
}
OptTensor stat(const OptTensor& t, const Tensor& x, at::IntArrayRef shape, const char* what) {
  if (!t) return t;
  check_like(*t, x, shape, what);
  return t->to(at::kFloat).contiguous();
}
const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// Norm weights: both of one type, contiguous.
struct Weights {
  OptTensor w, b;
  int32_t code = GMDN_DTYPE_F32;
};
Weights weights_of(const OptTensor& w, const OptTensor& b, const Tensor& x, int64_t d) {
  TORCH_CHECK(w || !b, "a layer norm's bias comes with a weight");
  Weights r;
  if (!w) return r;
  check_like(*w, x, {d}, "weight");
  r.code = type_code(w->scalar_type(), "weight");
  r.w = w->contiguous();
  if (b) {
    check_like(*b, x, {d}, "bias");
    TORCH_CHECK(b->scalar_type() == w->scalar_type(), "bias is ", b->scalar_type(), " and weight ", w->scalar_type());
    r.b = b->contiguous();
  }
  return r;
}

// A checkpoint's two tensors, contiguous; rows and d from q.
struct Kept {
  Tensor q, scale;
  int64_t rows, d;
};
Kept kept_of(const Tensor& q, const Tensor& scale) {
  TORCH_CHECK(q.scalar_type() == at::kChar, "a checkpoint's values are int8, got ", q.scalar_type());
  TORCH_CHECK(q.dim() >= 1 && q.size(-1) > 0, "a checkpoint has rows of at least one value, got shape ", q.sizes());
  const int64_t d = q.size(-1);
  return {q.contiguous(), stat(scale, q, with_last(lead(q), gmdn_act8_groups(d)), "scale"), q.numel() / d, d};
}
std::pair<Tensor, Tensor> new_kept(const Tensor& x) {
  return {fresh(x, x.sizes(), at::kChar),
          fresh(x, with_last(lead(x), gmdn_act8_groups(x.size(-1))))};
}

std::pair<Tensor, Tensor> kept_or_none(const Tensor& x, bool pack) {
  if (pack) return new_kept(x);
  return {fresh(x, {0}, at::kChar), fresh(x, {0})};
}

// ---------------------------------------------------------------- layer norm
using Norm = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
Norm layer_norm_fwd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, ScalarType dtype,
                    bool pack) {
  const c10::DeviceGuard guard(x.device());
  const int32_t xc = type_code(x.scalar_type(), "x"), yc = type_code(dtype, "a layer norm's output");
  const Rows r = rows_of(x, "x");
  const Weights w = weights_of(weight, bias, x, r.d);
  Tensor y = fresh(x, x.sizes(), dtype), mean = fresh(x, lead(x)), rstd = fresh(x, lead(x));
  auto [q, scale] = kept_or_none(x, pack);
  if (r.rows)
    check(gmdn_layer_norm_fwd(r.ptr(), ptr(w.w), ptr(w.b), y.data_ptr(), fp(mean), fp(rstd),
                              pack ? q.data_ptr<int8_t>() : nullptr, pack ? fp(scale) : nullptr, r.rows, r.d, r.stride,
                              (float)eps, xc, yc, w.code, stream_of(x)),
          "gmdn_layer_norm_fwd");
  return {y, mean, rstd, q, scale};
}

using Grads3 = std::tuple<Tensor, Tensor, Tensor>;
Grads3 norm_bwd(const Tensor& dy, const Tensor* x, const Kept* k, const OptTensor& weight, const Tensor& mean_,
                const Tensor& rstd_, ScalarType x_dtype) {
  const c10::DeviceGuard guard(dy.device());
  const int32_t xc = type_code(x_dtype, "x"), yc = type_code(dy.scalar_type(), "dy");
  const Rows g = rows_of(dy, "dy");
  const Weights w = weights_of(weight, OptTensor(), dy, g.d);
  const Tensor mean = stat(mean_, dy, lead(dy), "mean"), rstd = stat(rstd_, dy, lead(dy), "rstd");
  Rows r{};
  if (x) {
    check_like(*x, dy, dy.sizes(), "x");
    r = rows_of(*x, "x");
  } else {
    check_like(k->q, dy, dy.sizes(), "the checkpoint");
  }
  Tensor dx = fresh(dy, dy.sizes(), x_dtype);
  Tensor dw = w.w ? at::empty_like(*w.w) : fresh(dy, {0}), db = w.w ? at::empty_like(*w.w) : fresh(dy, {0});
  const size_t need = w.w ? gmdn_layer_norm_bwd_workspace_floats(g.rows, g.d) : 0;
  const Tensor ws = need ? fresh(dy, {(int64_t)need}) : Tensor();
  if (g.rows || w.w)
    check(gmdn_layer_norm_bwd(g.ptr(), x ? r.ptr() : nullptr, x ? nullptr : k->q.data_ptr<int8_t>(),
                              x ? nullptr : fp(k->scale), ptr(w.w), fp(mean), fp(rstd), dx.data_ptr(),
                              w.w ? dw.data_ptr() : nullptr, w.w ? db.data_ptr() : nullptr, need ? fp(ws) : nullptr, need, g.rows,
                              g.d, g.stride, x ? r.stride : 0, xc, yc, w.code, stream_of(dy)),
          "gmdn_layer_norm_bwd");
  return {dx, dw, db};
}
Grads3 layer_norm_bwd(const Tensor& dy, const Tensor& x, const OptTensor& weight, const Tensor& mean,
                      const Tensor& rstd) {
  return norm_bwd(dy, &x, nullptr, weight, mean, rstd, x.scalar_type());
}
Grads3 layer_norm8_bwd(const Tensor& dy, const Tensor& q, const Tensor& scale, const OptTensor& weight,
                       const Tensor& mean, const Tensor& rstd, ScalarType dtype) {
  const Kept k = kept_of(q, scale);
  return norm_bwd(dy, nullptr, &k, weight, mean, rstd, dtype);
}

Tensor layer_norm8_rebuild(const Tensor& q, const Tensor& scale, const OptTensor& weight, const OptTensor& bias,
                           const Tensor& mean_, const Tensor& rstd_, ScalarType dtype) {
  const c10::DeviceGuard guard(q.device());
  const int32_t yc = type_code(dtype, "a layer norm's output");
  const Kept k = kept_of(q, scale);
  const Weights w = weights_of(weight, bias, q, k.d);
  const Tensor mean = stat(mean_, q, lead(q), "mean"), rstd = stat(rstd_, q, lead(q), "rstd");
  Tensor y = fresh(q, q.sizes(), dtype);
  if (k.rows)
    check(gmdn_layer_norm8_rebuild(k.q.data_ptr<int8_t>(), fp(k.scale), ptr(w.w), ptr(w.b), fp(mean), fp(rstd),
                                   y.data_ptr(), k.rows, k.d, yc, w.code, stream_of(q)),
          "gmdn_layer_norm8_rebuild");
  return y;
}

// ------------------------------------------------------- 8-bit checkpoints
std::tuple<Tensor, Tensor> act8_pack(const Tensor& x) {
  const c10::DeviceGuard guard(x.device());
  const int32_t code = type_code(x.scalar_type(), "x");
  const Rows r = rows_of(x, "x");
  auto [q, scale] = new_kept(x);
  if (r.rows)
    check(gmdn_act8_pack(r.ptr(), q.data_ptr<int8_t>(), fp(scale), r.rows, r.d, r.stride, code, stream_of(x)),
          "gmdn_act8_pack");
  return {q, scale};
}
Tensor act8_unpack(const Tensor& q, const Tensor& scale, ScalarType dtype) {
  const c10::DeviceGuard guard(q.device());
  const int32_t code = type_code(dtype, "an unpacked checkpoint");
  const Kept k = kept_of(q, scale);
  Tensor x = fresh(q, q.sizes(), dtype);
  if (k.rows)
    check(gmdn_act8_unpack(k.q.data_ptr<int8_t>(), fp(k.scale), x.data_ptr(), k.rows, k.d, code, stream_of(q)),
          "gmdn_act8_unpack");
  return x;
}
std::tuple<Tensor, Tensor, Tensor> gelu8_fwd(const Tensor& h, bool pack) {
  const c10::DeviceGuard guard(h.device());
  const int32_t code = type_code(h.scalar_type(), "h");
  const Rows r = rows_of(h, "h");
  Tensor a = fresh(h, h.sizes(), h.scalar_type());
  auto [q, scale] = kept_or_none(h, pack);
  if (r.rows)
    check(gmdn_gelu8_fwd(r.ptr(), a.data_ptr(), pack ? q.data_ptr<int8_t>() : nullptr, pack ? fp(scale) : nullptr,
                         r.rows, r.d, r.stride, code, stream_of(h)),
          "gmdn_gelu8_fwd");
  return {a, q, scale};
}
std::tuple<Tensor, Tensor> gelu8_bwd(const Tensor& da, const Tensor& q, const Tensor& scale, bool with_output) {
  const c10::DeviceGuard guard(da.device());
  const int32_t code = type_code(da.scalar_type(), "da");
  const Kept k = kept_of(q, scale);
  check_like(k.q, da, da.sizes(), "the checkpoint");
  const Rows g = rows_of(da, "da");
  Tensor dh = fresh(da, da.sizes(), da.scalar_type());
  Tensor a = with_output ? fresh(da, da.sizes(), da.scalar_type()) : fresh(da, {0}, da.scalar_type());
  if (g.rows)
    check(gmdn_gelu8_bwd(g.ptr(), k.q.data_ptr<int8_t>(), fp(k.scale), dh.data_ptr(),
                         with_output ? a.data_ptr() : nullptr, g.rows, g.d, g.stride, code, stream_of(da)),
          "gmdn_gelu8_bwd");
  return {dh, a};
}

// -------------------------------------------------------- log probabilities
Tensor tokens_of(const Tensor& tokens, const Tensor& logits) {
  check_like(tokens, logits, lead(logits), "tokens");
  TORCH_CHECK(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens are int64 or int32, got ",
              tokens.scalar_type());
  return tokens.to(at::kLong).contiguous();
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> logprobs_fwd(const Tensor& logits, const Tensor& tokens, int64_t top,
                                                                int64_t ignore_index) {
  const c10::DeviceGuard guard(logits.device());
  const int32_t code = type_code(logits.scalar_type(), "logits");
  const Rows r = rows_of(logits, "logits");
  TORCH_CHECK(top >= 0 && top <= 32 && top <= r.d, "top is between 0 and 32 and at most the vocabulary (", r.d,
              "), got ", top);
  const Tensor tk = tokens_of(tokens, logits);
  const auto shape = lead(logits);
  Tensor lp = fresh(logits, shape), entropy = fresh(logits, shape), stats = fresh(logits, with_last(shape, 2));
  Tensor top_lp = fresh(logits, with_last(shape, top));
  Tensor top_tokens = fresh(logits, with_last(shape, top), at::kLong);
  const size_t need = gmdn_logprobs_fwd_workspace_bytes(r.rows, r.d, (int32_t)top);
  const Tensor ws = need ? fresh(logits, {(int64_t)need}, at::kByte) : Tensor();
  if (r.rows)
    check(gmdn_logprobs_fwd(r.ptr(), tk.data_ptr<int64_t>(), fp(lp), fp(entropy), fp(top_lp),
                            top ? top_tokens.data_ptr<int64_t>() : nullptr, fp(stats),
                            need ? ws.data_ptr() : nullptr, need, r.rows, r.d, r.stride,
                            (int32_t)top, ignore_index, code, stream_of(logits)),
          "gmdn_logprobs_fwd");
  return {lp, entropy, top_lp, top_tokens, stats};
}
Tensor logprobs_bwd(const Tensor& logits, const Tensor& tokens, const Tensor& stats_, const Tensor& entropy_,
                    const Tensor& top_tokens, const OptTensor& dlogprob, const OptTensor& dentropy,
                    const OptTensor& dtop, int64_t ignore_index) {
  const c10::DeviceGuard guard(logits.device());
  const int32_t code = type_code(logits.scalar_type(), "logits");
  const Rows r = rows_of(logits, "logits");
  const Tensor tk = tokens_of(tokens, logits);
  const auto shape = lead(logits);
  const Tensor stats = stat(stats_, logits, with_last(shape, 2), "stats"),
               entropy = stat(entropy_, logits, shape, "entropy");
  const OptTensor dl = stat(dlogprob, logits, shape, "dlogprob"), dh = stat(dentropy, logits, shape, "dentropy");
  int64_t top = 0;
  OptTensor dt;
  Tensor at_tokens;
  if (dtop) {
    top = top_tokens.dim() ? top_tokens.size(-1) : 0;
    check_like(top_tokens, logits, with_last(shape, top), "top_tokens");
    TORCH_CHECK(top_tokens.scalar_type() == at::kLong, "top_tokens are int64, got ", top_tokens.scalar_type());
    TORCH_CHECK(top <= 32 && top <= r.d, "at most 32 alternatives, and no more than the vocabulary (", r.d, "), got ",
                top);
    dt = stat(dtop, logits, with_last(shape, top), "dtop");
    at_tokens = top_tokens.contiguous();
  }
  Tensor dx = fresh(logits, logits.sizes(), logits.scalar_type());
  if (r.rows)
    check(gmdn_logprobs_bwd(r.ptr(), tk.data_ptr<int64_t>(), fp(stats), fp(entropy),
                            top ? at_tokens.data_ptr<int64_t>() : nullptr, (const float*)ptr(dl), (const float*)ptr(dh),
                            top ? fp(*dt) : nullptr, dx.data_ptr(), r.rows, r.d, r.stride, (int32_t)top, ignore_index,
                            code, stream_of(logits)),
          "gmdn_logprobs_bwd");
  return dx;
}

// ------------------------------------------------------------------ autograd
struct LayerNormFwd : torch::autograd::Function<LayerNormFwd> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                        double eps, ScalarType dtype, bool pack, std::array<Tensor, 4>* rest) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, mean, rstd, q, scale] = GMDN_OP(layer_norm_fwd).call(x, weight, bias, eps, dtype, pack);
    *rest = {mean, rstd, q, scale};
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({pack ? Tensor() : x, opt(weight), mean, rstd, pack ? q : Tensor(), pack ? scale : Tensor()});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["pack"] = pack;
    ctx->saved_data["dtype"] = x.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const Tensor none;
    if (!g[0].defined()) return {none, none, none, none, none, none, none};
    const auto s = ctx->get_saved_variables();
    Grads3 d = ctx->saved_data["pack"].toBool()
                   ? GMDN_OP(layer_norm8_bwd).call(g[0], s[4], s[5], opt(s[1]), s[2], s[3],
                                                   ctx->saved_data["dtype"].toScalarType())
                   : GMDN_OP(layer_norm_bwd).call(g[0], s[0], opt(s[1]), s[2], s[3]);
    return {std::get<0>(d), s[1].defined() ? std::get<1>(d) : none,
            ctx->saved_data["bias"].toBool() ? std::get<2>(d) : none, none, none, none, none};
  }
};
Norm layer_norm_fwd_ad(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, ScalarType dtype,
                       bool pack) {
  const Tensor w = opt(weight), b = opt(bias);
  refuse_tangents("layer_norm_fwd", {&x, &w, &b});
  if (!wants_grad({&x, &w, &b})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GMDN_OP(layer_norm_fwd).call(x, weight, bias, eps, dtype, pack);
  }
  std::array<Tensor, 4> rest;
  Tensor y = LayerNormFwd::apply(x, weight, bias, eps, dtype, pack, &rest);
  return {y, rest[0], rest[1], rest[2], rest[3]};
}

struct Gelu8Fwd : torch::autograd::Function<Gelu8Fwd> {
  static constexpr bool is_traceable = true;
  static Tensor forward(AutogradContext* ctx, const Tensor& h, std::pair<Tensor, Tensor>* kept) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [a, q, scale] = GMDN_OP(gelu8_fwd).call(h, true);
    *kept = {q, scale};
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, scale});
    return a;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    if (!g[0].defined()) return {Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    return {std::get<0>(GMDN_OP(gelu8_bwd).call(g[0], s[0], s[1], false)), Tensor()};
  }
};
std::tuple<Tensor, Tensor, Tensor> gelu8_fwd_ad(const Tensor& h, bool pack) {
  refuse_tangents("gelu8_fwd", {&h});
  if (!wants_grad({&h})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GMDN_OP(gelu8_fwd).call(h, pack);
  }
  TORCH_CHECK(pack, "gelu8_fwd without its checkpoint has no backward");
  std::pair<Tensor, Tensor> kept;
  Tensor a = Gelu8Fwd::apply(h, &kept);
  return {a, kept.first, kept.second};
}

struct LogprobsFwd : torch::autograd::Function<LogprobsFwd> {
  static constexpr bool is_traceable = true;
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, c10::SymInt top,
                               c10::SymInt ignore_index, std::pair<Tensor, Tensor>* rest) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [lp, entropy, top_lp, top_tokens, stats] = GMDN_OP(logprobs_fwd).call(logits, tokens, top, ignore_index);
    *rest = {top_tokens, stats};
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, stats, entropy, top_tokens});
    ctx->saved_data["ignore_index"] = ignore_index;
    return {lp, entropy, top_lp};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const Tensor none;
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return {none, none, none, none, none};
    const auto s = ctx->get_saved_variables();
    return {GMDN_OP(logprobs_bwd)
                .call(s[0], s[1], s[2], s[3], s[4], opt(g[0]), opt(g[1]), opt(g[2]),
                      ctx->saved_data["ignore_index"].toSymInt()),
            none, none, none, none};
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> logprobs_fwd_ad(const Tensor& logits, const Tensor& tokens,
                                                                   c10::SymInt top, c10::SymInt ignore_index) {
  refuse_tangents("logprobs_fwd", {&logits});
  if (!wants_grad({&logits})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GMDN_OP(logprobs_fwd).call(logits, tokens, top, ignore_index);
  }
  std::pair<Tensor, Tensor> rest;
  auto r = LogprobsFwd::apply(logits, tokens, top, ignore_index, &rest);
  return {r[0], r[1], r[2], rest.first, rest.second};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(gmdn, m) {
  const std::vector<at::Tag> PT2{at::Tag::pt2_compliant_tag};
  m.def("layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps, ScalarType dtype, bool pack) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor)", PT2);
  m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor? weight, Tensor mean, Tensor rstd) -> (Tensor, Tensor, Tensor)",
        PT2);
  m.def("layer_norm8_bwd(Tensor dy, Tensor q, Tensor scale, Tensor? weight, Tensor mean, Tensor rstd, "
        "ScalarType dtype) -> (Tensor, Tensor, Tensor)", PT2);
  m.def("layer_norm8_rebuild(Tensor q, Tensor scale, Tensor? weight, Tensor? bias, Tensor mean, Tensor rstd, "
        "ScalarType dtype) -> Tensor", PT2);
  m.def("act8_pack(Tensor x) -> (Tensor, Tensor)", PT2);
  m.def("act8_unpack(Tensor q, Tensor scale, ScalarType dtype) -> Tensor", PT2);
  m.def("gelu8_fwd(Tensor h, bool pack=True) -> (Tensor, Tensor, Tensor)", PT2);
  m.def("gelu8_bwd(Tensor da, Tensor q, Tensor scale, bool with_output) -> (Tensor, Tensor)", PT2);
  m.def("logprobs_fwd(Tensor logits, Tensor tokens, SymInt top, SymInt ignore_index) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor)", PT2);
  m.def("logprobs_bwd(Tensor logits, Tensor tokens, Tensor stats, Tensor entropy, Tensor top_tokens, Tensor? dlogprob, "
        "Tensor? dentropy, Tensor? dtop, SymInt ignore_index) -> Tensor", PT2);
}

TORCH_LIBRARY_IMPL(gmdn, CUDA, m) {
  m.impl("layer_norm_fwd", layer_norm_fwd);
  m.impl("layer_norm_bwd", layer_norm_bwd);
  m.impl("layer_norm8_bwd", layer_norm8_bwd);
  m.impl("layer_norm8_rebuild", layer_norm8_rebuild);
  m.impl("act8_pack", act8_pack);
  m.impl("act8_unpack", act8_unpack);
  m.impl("gelu8_fwd", gelu8_fwd);
  m.impl("gelu8_bwd", gelu8_bwd);
  m.impl("logprobs_fwd", logprobs_fwd);
  m.impl("logprobs_bwd", logprobs_bwd);
}

TORCH_LIBRARY_IMPL(gmdn, Autograd, m) {
  m.impl("layer_norm_fwd", layer_norm_fwd_ad);
  m.impl("gelu8_fwd", gelu8_fwd_ad);
  m.impl("logprobs_fwd", logprobs_fwd_ad);
  // No derivative of their own: differentiating through them raises.
  for (const char* name : {"layer_norm_bwd", "layer_norm8_bwd", "layer_norm8_rebuild", "act8_pack", "act8_unpack",
                           "gelu8_bwd", "logprobs_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
