// Entry points of the operators on 8-bit kept activations, with their autograd
// nodes: argument checks, casts and the choice of what is kept happen here, in
// one call from Python and none from the backward pass (in Python the same
// steps take 40 us of a small layer's 80). CPU tensors never come here: their
// plain form is ops/norm_act.py and ops/functional.py.
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

namespace turboprune {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

at::Tensor mask_apply(const at::Tensor&, const at::Tensor&, at::ScalarType);
std::tuple<at::Tensor, at::Tensor, at::Tensor> gelu_keep8_fwd(
    const at::Tensor&);
at::Tensor gelu_keep8_bwd(const at::Tensor&, const at::Tensor&,
                          const at::Tensor&);
std::tuple<at::Tensor, OptTensor, OptTensor, OptTensor, OptTensor> rms_fwd(
    const at::Tensor&, const OptTensor&, const at::Tensor&, double,
    at::ScalarType, bool, bool);
std::tuple<at::Tensor, OptTensor, at::Tensor> rms_bwd(
    const at::Tensor&, const OptTensor&, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, at::ScalarType, bool);
std::tuple<at::Tensor, OptTensor, OptTensor, OptTensor, OptTensor>
linear_act_fwd(const at::Tensor&, const at::Tensor&, const OptTensor&,
               const OptTensor&, bool, int64_t, bool);
std::tuple<OptTensor, OptTensor, OptTensor> linear_act_bwd(
    const at::Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
    const OptTensor&, const at::Tensor&, const OptTensor&, bool,
    c10::optional<at::ScalarType>, c10::optional<at::ScalarType>);

namespace {

bool is_float(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf;
}

void check_float(const char* op, const char* name, const at::Tensor& t) {
  TORCH_CHECK_TYPE(is_float(t.scalar_type()), op, ": ", name, " is ",
                   t.scalar_type(),
                   ": float32, bfloat16 or float16 expected");
}

void check_device(const char* op, const char* name, const at::Tensor& t,
                  const at::Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), op, ": ", name, " on ",
                    t.device(), ", x on ", x.device());
}

// keep: None or "e4m3"
bool keeps(const c10::optional<std::string>& keep) {
  TORCH_CHECK_VALUE(!keep || *keep == "e4m3", "keep='", keep ? *keep : "",
                    "': None or 'e4m3'");
  return keep.has_value();
}

bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (auto* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A dual tensor of forward-mode differentiation need not ask for gradients, and
// the kernels would drop its tangent.
void no_tangents(const char* op, std::initializer_list<const at::Tensor*> ts) {
  for (auto* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(
        !t->defined() || !t->_fw_grad(0).defined(), op,
        ": forward-mode derivatives are not available on a GPU");
}

void only_once() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "gradients of gradients are not available for this operator "
              "(create_graph=True)");
}

at::Tensor or_none(const OptTensor& t) { return t ? *t : at::Tensor(); }
OptTensor as_opt(const at::Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}

// ------------------------------------------------------------------- GELU
struct GeluKeep8 : Function<GeluKeep8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x) {
    auto [y, codes, scales] = gelu_keep8_fwd(x);
    ctx->save_for_backward({codes, scales});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_once();
    auto s = ctx->get_saved_variables();
    return {gelu_keep8_bwd(s[0], s[1], g[0])};
  }
};

// ------------------------------------------------------------------- norm
struct RmsNorm : Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x,
                               const OptTensor& residual,
                               const at::Tensor& weight, double eps,
                               int64_t out_dtype, bool keep) {
    ctx->set_materialize_grads(false);
    auto [y, h, rstd, codes, scales] = rms_fwd(
        x, residual, weight, eps, (at::ScalarType)out_dtype, true, keep);
    ctx->save_for_backward({h ? *h : x, weight, *rstd});
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->saved_data["r"] = residual.has_value();
    variable_list out = {y};
    if (h) out.push_back(*h);
    if (codes) {
      ctx->mark_non_differentiable({*codes, *scales});
      out.push_back(*codes);
      out.push_back(*scales);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_once();
    auto s = ctx->get_saved_variables();
    auto xt = (at::ScalarType)ctx->saved_data["x"].toInt();
    bool r = ctx->saved_data["r"].toBool();
    auto dy = g[0];
    auto dh = r ? g[1] : at::Tensor();
    at::Tensor dx, dr, dw, none;
    if (dy.defined()) {
      auto d = rms_bwd(dy, as_opt(dh), s[0], s[1], s[2], xt, r);
      dx = std::get<0>(d);
      dr = or_none(std::get<1>(d));
      dw = std::get<2>(d).to(s[1].scalar_type());
    } else if (dh.defined()) {   // only the sum was used
      dr = dh;
      dx = dh.to(xt);
    }
    return {dx, dr, dw, none, none, none};
  }
};

// ----------------------------------------------------------------- linear
struct LinearAct : Function<LinearAct> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& w, const at::Tensor& weight,
                            const OptTensor& mask, const OptTensor& bias,
                            const OptTensor& residual, bool act, bool keep,
                            const OptTensor& codes_in,
                            const OptTensor& scales_in) {
    int64_t K = w.size(1), N = w.size(0);
    auto x2 = x.reshape({-1, K});
    bool need_x = weight.requires_grad();   // for dw alone
    bool need_b = bias && bias->requires_grad();
    bool need_z = x.requires_grad() || need_x || need_b;   // for the slope
    at::Tensor codes, scales;
    if (keep && need_x && codes_in) {
      codes = codes_in->reshape(x2.sizes());
      scales = scales_in->reshape({x2.size(0), -1});
    }
    OptTensor r2;
    if (residual) r2 = residual->reshape({-1, N});
    auto [y, z, zs, xc, xs] =
        linear_act_fwd(x2, w, bias, r2, act, !need_z ? 0 : keep ? 2 : 1,
                       keep && need_x && !codes_in);
    if (xc) {
      codes = *xc;
      scales = *xs;
    }
    ctx->save_for_backward(
        {w, or_none(z), or_none(zs),
         !need_x ? at::Tensor() : keep ? codes : x, scales,
         need_x ? or_none(mask) : at::Tensor()});
    auto& d = ctx->saved_data;
    d["need"] = (int64_t)(x.requires_grad() | need_x << 1 | need_b << 2 |
                          residual.has_value() << 3);
    d["wt"] = (int64_t)weight.scalar_type();
    if (bias) d["bt"] = (int64_t)bias->scalar_type();
    d["x"] = x.sizes();
    d["w"] = weight.sizes();
    auto sizes = x.sizes().vec();
    sizes.back() = N;
    // not view(): autograd forbids changing a view that a node hands out, and
    // nothing else holds y
    return at::_unsafe_view(y, sizes);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_once();
    auto s = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    int64_t need = d["need"].toInt();
    auto w = s[0];
    auto xs = d["x"].toIntVector();
    int64_t N = w.size(0), K = w.size(1);
    at::Tensor dx, dw, db, none;
    if (need & 7) {
      OptTensor xk;
      if (s[3].defined()) xk = s[3].reshape({-1, K});
      c10::optional<at::ScalarType> wt, bt;
      if (need & 2) wt = (at::ScalarType)d["wt"].toInt();
      if (need & 4) bt = (at::ScalarType)d["bt"].toInt();
      auto r = linear_act_bwd(g[0].reshape({-1, N}), as_opt(s[1]),
                              as_opt(s[2]), xk, as_opt(s[4]), w,
                              as_opt(s[5]), need & 1, wt, bt);
      if (need & 1) dx = std::get<0>(r)->view(xs);
      if (need & 2) dw = std::get<1>(r)->view(d["w"].toIntVector());
      db = or_none(std::get<2>(r));
    }
    // the residual's gradient is the output's (dropped where not wanted)
    return {dx,   none, dw,   none, db, need & 8 ? g[0] : none,
            none, none, none, none};
  }
};

}  // namespace

at::Tensor gelu_keep8(const at::Tensor& x) {
  check_float("gelu", "x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1,
                    "gelu(keep=...): a tensor of at least one dimension");
  no_tangents("gelu", {&x});
  c10::DeviceGuard guard(x.device());
  return GeluKeep8::apply(x);
}

std::tuple<at::Tensor, at::Tensor, OptTensor, OptTensor> add_rms_norm(
    const at::Tensor& x, const OptTensor& residual, const at::Tensor& weight,
    double eps, const c10::optional<std::string>& keep_arg,
    c10::optional<at::ScalarType> out_dtype) {
  const char* op = "add_rms_norm";
  c10::DeviceGuard guard(x.device());
  bool keep = keeps(keep_arg);
  check_float(op, "x", x);
  check_float(op, "weight", weight);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, op,
                    ": x needs rows of at least one value, not shape ",
                    x.sizes());
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), op,
                    ": weight of shape (", x.size(-1), ",) expected, not ",
                    weight.sizes());
  check_device(op, "weight", weight, x);
  auto xt = x.scalar_type(), ot = out_dtype.value_or(xt);
  at::Tensor r = or_none(residual);
  no_tangents(op, {&x, &r, &weight});
  if (residual) {
    TORCH_CHECK_VALUE(r.sizes() == x.sizes(), op, ": residual of shape ",
                      x.sizes(), " expected, not ", r.sizes());
    TORCH_CHECK_TYPE(r.scalar_type() == xt || r.scalar_type() == at::kFloat,
                     op, ": residual in ", xt, " or float32 expected, not ",
                     r.scalar_type());
    check_device(op, "residual", r, x);
  }
  TORCH_CHECK_TYPE(ot == xt || (xt == at::kFloat &&
                                (ot == at::kBFloat16 || ot == at::kHalf)),
                   op, ": out_dtype ", ot, " for x in ", xt);
  if (!wants_grad({&x, &r, &weight})) {
    auto o = rms_fwd(x, residual, weight, eps, ot, false, keep);
    return {std::get<0>(o), r.defined() ? *std::get<1>(o) : x,
            std::get<3>(o), std::get<4>(o)};
  }
  auto o = RmsNorm::apply(x, residual, weight, eps, (int64_t)ot, keep);
  size_t k = 1;
  at::Tensor h = r.defined() ? o[k++] : x;
  if (!keep) return {o[0], h, c10::nullopt, c10::nullopt};
  return {o[0], h, o[k], o[k + 1]};
}

at::Tensor masked_linear_act(
    const at::Tensor& x_in, const at::Tensor& weight, const OptTensor& mask,
    const OptTensor& bias_in, const OptTensor& residual,
    const c10::optional<std::string>& act_arg, const OptTensor& cache,
    c10::optional<at::ScalarType> compute_dtype,
    const c10::optional<std::string>& keep_arg, const OptTensor& codes,
    const OptTensor& scales) {
  const char* op = "masked_linear_act";
  c10::DeviceGuard guard(x_in.device());
  bool keep = keeps(keep_arg);
  TORCH_CHECK_VALUE(!act_arg || *act_arg == "gelu", "act='",
                    act_arg ? *act_arg : "", "': None or 'gelu'");
  TORCH_CHECK_VALUE(weight.dim() == 2 && x_in.dim() >= 1 &&
                        x_in.size(-1) == weight.size(1),
                    op, ": x (..., K) and weight (N, K) expected, not ",
                    x_in.sizes(), " and ", weight.sizes());
  int64_t N = weight.size(0), K = weight.size(1);
  auto shape = [&](const char* name, const OptTensor& t,
                   at::IntArrayRef want) {
    if (!t) return;
    TORCH_CHECK_VALUE(t->sizes() == want, op, ": ", name, " of shape ", want,
                      " expected, not ", t->sizes());
    check_device(op, name, *t, x_in);
  };
  check_device(op, "weight", weight, x_in);
  shape("mask", mask, {N, K});
  shape("bias", bias_in, {N});
  shape("cache", cache, {N, K});
  auto out_sizes = x_in.sizes().vec();
  out_sizes.back() = N;
  shape("residual", residual, out_sizes);
  check_float(op, "x", x_in);
  check_float(op, "weight", weight);
  if (bias_in) check_float(op, "bias", *bias_in);
  TORCH_CHECK_TYPE(!mask || mask->scalar_type() == at::kFloat, op,
                   ": mask is ", mask ? mask->scalar_type() : at::kFloat,
                   ": float32 expected");
  auto ct = cache ? cache->scalar_type()
                  : compute_dtype.value_or(
                        weight.scalar_type() != at::kFloat
                            ? weight.scalar_type()
                            : x_in.scalar_type());
  TORCH_CHECK_TYPE(ct == at::kBFloat16 || ct == at::kHalf, op,
                   " computes in bfloat16 or float16 on a GPU, not in ", ct,
                   ": give a cache or a compute_dtype of such a type");
  if (residual)
    TORCH_CHECK_TYPE(residual->scalar_type() == ct ||
                         residual->scalar_type() == at::kFloat,
                     op, ": residual in ", ct, " or float32 expected, not ",
                     residual->scalar_type());
  TORCH_CHECK_VALUE(codes.has_value() == scales.has_value(), op,
                    ": kept needs codes and scales");
  if (codes) {
    TORCH_CHECK_VALUE(keep, op, ": kept needs keep='e4m3'");
    TORCH_CHECK_TYPE(codes->scalar_type() == at::kFloat8_e4m3fn &&
                         scales->scalar_type() == at::kFloat8_e8m0fnu,
                     "kept: float8_e4m3fn codes and float8_e8m0fnu scales "
                     "expected, not ", codes->scalar_type(), " and ",
                     scales->scalar_type());
    auto want = x_in.sizes().vec();
    shape("kept codes", codes, want);
    want.back() = (K + 31) / 32;
    shape("kept scales", scales, want);
  }
  at::Tensor bias = or_none(bias_in), r = or_none(residual), w;
  no_tangents(op, {&x_in, &weight, &bias, &r});
  if (cache) {
    w = cache->detach();
  } else {
    at::NoGradGuard no_grad;
    if (!mask)
      w = weight.detach().to(ct);
    else if (weight.scalar_type() == at::kFloat && ct == at::kBFloat16)
      w = mask_apply(weight, *mask, ct);
    else
      w = at::where(mask->ne(0), weight, at::zeros({}, weight.options()))
              .to(ct);
  }
  auto x = x_in.scalar_type() == ct ? x_in : x_in.to(ct);
  if (bias.defined() && bias.scalar_type() != ct &&
      bias.scalar_type() != at::kFloat)
    bias = bias.to(ct);
  bool act = act_arg.has_value();
  if (x.numel() == 0 || N == 0) {
    // no rows: the sum is empty and no kernel runs; every input stays in the
    // graph, so that each gets a gradient of zeros
    auto y = at::empty(out_sizes, x.options());
    TORCH_CHECK_VALUE(y.numel() == 0, op, ": rows of at least one value");
    auto zero = x.sum() + weight.sum().to(ct);
    if (bias.defined()) zero = zero + bias.sum().to(ct);
    y = y + zero * 0;
    return r.defined() ? (y + r).to(r.scalar_type()) : y;
  }
  if (!wants_grad({&x, &weight, &bias, &r})) {
    auto o = linear_act_fwd(
        x.dim() == 2 ? x : x.reshape({-1, K}), w, as_opt(bias),
        r.defined() ? OptTensor(r.dim() == 2 ? r : r.reshape({-1, N}))
                    : OptTensor(),
        act, 0, false);
    return x.dim() == 2 ? std::get<0>(o)
                        : at::_unsafe_view(std::get<0>(o), out_sizes);
  }
  return LinearAct::apply(x, w, weight, mask, as_opt(bias), residual, act,
                          keep, codes, scales);
}

}  // namespace turboprune
