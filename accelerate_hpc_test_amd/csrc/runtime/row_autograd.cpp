// Autograd nodes of the row operators (layer norm, rotary positions, token log-probabilities, expert routing) in C++: forward
// and backward run without a Python frame and the backward without the interpreter lock. A training call of these
// operators is a few microseconds of kernel at small sizes, where Python's autograd.Function cost 77-137 us of host time.
// Shapes are taken as they come: rows are viewed where strides allow it, copied where not, outputs have the input's shape.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

std::vector<torch::Tensor> layer_norm_fwd(torch::Tensor x, c10::optional<torch::Tensor> residual, c10::optional<torch::Tensor> w,
                                          c10::optional<torch::Tensor> b, double eps, bool stats);
std::vector<torch::Tensor> layer_norm_bwd(torch::Tensor dy, torch::Tensor s, c10::optional<torch::Tensor> w, torch::Tensor mean,
                                          torch::Tensor rstd, c10::optional<torch::Tensor> dres, bool want_dw, bool want_db,
                                          bool wide_params);
torch::Tensor rope_any(torch::Tensor src, torch::Tensor cos, torch::Tensor sin, c10::optional<torch::Tensor> pos, int64_t n_rot,
                       bool interleaved, double sign);
torch::Tensor rope_out(torch::Tensor src, torch::Tensor cos, torch::Tensor sin, c10::optional<torch::Tensor> pos,
                       int64_t n_rot_heads, int64_t n_heads_total, int64_t head_dim, double sign);
std::vector<torch::Tensor> token_logprobs_fwd(torch::Tensor logits, torch::Tensor tokens, int64_t K, double inv_t, int64_t ignore,
                                              bool want_stats);
torch::Tensor token_logprobs_bwd(torch::Tensor logits, torch::Tensor tokens, torch::Tensor stats,
                                 c10::optional<torch::Tensor> top_id, c10::optional<torch::Tensor> g_lp,
                                 c10::optional<torch::Tensor> g_ent, c10::optional<torch::Tensor> g_top, double inv_t,
                                 int64_t ignore);
std::vector<torch::Tensor> route_experts_fwd(torch::Tensor logits, int64_t k, bool softmax, c10::optional<torch::Tensor> bias,
                                             int64_t groups, int64_t top_groups, bool renorm, double scale);
torch::Tensor route_experts_bwd(torch::Tensor logits, torch::Tensor weights, torch::Tensor experts, torch::Tensor dw, bool softmax,
                                bool renorm, double scale);

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

OptTensor some(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
bool needs_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
bool last_contiguous(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 || t.numel() == 0; }

// [rows, width] with contiguous rows at one stride
Tensor rows_of(const Tensor& t) {
  const int64_t width = t.size(-1);
  if (t.dim() == 2) return last_contiguous(t) ? t : t.contiguous();
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  Tensor r = t.reshape({rows, width});
  return last_contiguous(r) ? r : r.contiguous();
}
// `t`, which nothing else holds, in another shape. No view of it: outputs of a node with several must not be changed in place if
// they are views that were made inside of it.
Tensor shaped(const Tensor& t, at::IntArrayRef sizes) { return t.sizes() == sizes ? t : at::_unsafe_view(t, sizes); }

// Gradients of a backward that runs to be differentiated again: whoever does that gets an error, not a zero.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list there;
  for (auto& g : grads)
    if (g.defined()) there.push_back(g.detach().requires_grad_(true));
  if (there.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>("this operator's backward is not differentiable", (int64_t)there.size());
  there = (*error)(std::move(there));
  size_t at = 0;
  for (auto& g : grads)
    if (g.defined()) g = there[at++];
  return grads;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b,
                               const OptTensor& residual, double eps) {
    const Tensor x2 = rows_of(x);
    auto out = layer_norm_fwd(x2, residual.has_value() ? OptTensor(rows_of(*residual)) : c10::nullopt, w, b, eps, true);
    Tensor y = shaped(out[0], x.sizes());
    ctx->saved_data["has"] = (int64_t)((w.has_value() ? 1 : 0) | (b.has_value() ? 2 : 0) | (residual.has_value() ? 4 : 0) |
                                       (needs_grad(w) ? 8 : 0) | (needs_grad(b) ? 16 : 0) |
                                       ((w.has_value() ? *w : b.has_value() ? *b : x).scalar_type() == at::kFloat ? 32 : 0));
    ctx->set_materialize_grads(false);
    if (!residual.has_value()) {
      ctx->save_for_backward({x2, w.value_or(Tensor()), out[2], out[3]});
      return {y};
    }
    Tensor s = shaped(out[1], x.sizes());
    ctx->save_for_backward({s, w.value_or(Tensor()), out[2], out[3]});
    return {y, s};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const int64_t has = ctx->saved_data["has"].toInt();
    const Tensor dres = g.size() > 1 ? g[1] : Tensor();
    if (!g[0].defined())  // y unused: only the residual stream carries a gradient
      return {dres, Tensor(), Tensor(), dres, Tensor()};
    const auto saved = ctx->get_saved_variables();
    auto d = layer_norm_bwd(rows_of(g[0]), rows_of(saved[0]), some(saved[1]), saved[2], saved[3],
                            dres.defined() ? OptTensor(rows_of(dres)) : c10::nullopt, has & 8, has & 16, has & 32);
    const Tensor dx = shaped(d[0], g[0].sizes());  // d(x + residual) flows to both summands
    return once({dx, d[1], d[2], has & 4 ? dx : Tensor(), Tensor()});
  }
};

// `whole`: bf16 heads rotated whole in halves, by the kernel for these.
Tensor rope_by(const Tensor& x, const Tensor& cos, const Tensor& sin, const OptTensor& pos, int64_t n_rot, bool interleaved,
               bool whole, double sign) {
  if (x.numel() == 0) return at::empty(x.sizes(), x.options());
  if (!whole) return rope_any(last_contiguous(x) ? x : x.contiguous(), cos, sin, pos, n_rot, interleaved, sign);
  const c10::DeviceGuard guard(x.device());
  return rope_out(x, cos, sin, pos.has_value() ? OptTensor(pos->reshape({-1}).contiguous()) : c10::nullopt, n_rot, x.size(2),
                  x.size(3), sign);
}

// The gradient turns back (`sign`). It is a rotation itself, and heads that are rotated whole in halves, which torch operations
// rotated before there were kernels for them, can be differentiated again as those can; the other forms once.
struct Rope : public torch::autograd::Function<Rope> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& cos, const Tensor& sin, const OptTensor& pos,
                        int64_t n_rot, bool interleaved, bool whole, double sign) {
    ctx->save_for_backward({cos, sin, pos.value_or(Tensor())});
    ctx->saved_data["n_rot"] = n_rot;
    ctx->saved_data["form"] = (int64_t)((interleaved ? 1 : 0) | (whole ? 2 : 0));
    ctx->saved_data["sign"] = sign;
    return rope_by(qkv, cos, sin, pos, n_rot, interleaved, whole, sign);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const int64_t form = ctx->saved_data["form"].toInt();
    const int64_t n_rot = ctx->saved_data["n_rot"].toInt();
    const double sign = -ctx->saved_data["sign"].toDouble();
    const bool again = !(form & 1) && 2 * saved[0].size(1) == g[0].size(-1);
    if (again && at::GradMode::is_enabled() && g[0].requires_grad())
      return {Rope::apply(g[0], saved[0], saved[1], some(saved[2]), n_rot, false, (form & 2) != 0, sign), Tensor(), Tensor(), Tensor(),
              Tensor(), Tensor(), Tensor(), Tensor()};
    variable_list d = {rope_by(g[0], saved[0], saved[1], some(saved[2]), n_rot, form & 1, form & 2, sign), Tensor(), Tensor(), Tensor(),
                       Tensor(), Tensor(), Tensor(), Tensor()};
    return again ? d : once(std::move(d));
  }
};

// log-probabilities and entropies [...], alternatives' log-probabilities and tokens [..., K]
variable_list logprobs_shaped(const std::vector<Tensor>& out, const Tensor& logits, int64_t K) {
  auto lead = logits.sizes().slice(0, logits.dim() - 1);
  variable_list r = {shaped(out[0], lead), shaped(out[1], lead)};
  if (K > 0) {
    auto sizes = lead.vec();
    sizes.push_back(K);
    r.push_back(shaped(out[2], sizes));
    r.push_back(shaped(out[3], sizes));
  }
  return r;
}

struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t K, double inv_t,
                               int64_t ignore) {
    const Tensor l2 = rows_of(logits);
    const Tensor t1 = tokens.reshape({-1}).contiguous();
    auto out = token_logprobs_fwd(l2, t1, K, inv_t, ignore, true);
    auto r = logprobs_shaped(out, logits, K);
    ctx->save_for_backward({l2, t1, out[4], K > 0 ? r[3] : Tensor()});
    ctx->saved_data["inv_t"] = inv_t;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["sizes"] = logits.sizes().vec();
    ctx->set_materialize_grads(false);
    if (K > 0) ctx->mark_non_differentiable({r[3]});
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const bool top = g.size() > 2 && g[2].defined();
    if (!g[0].defined() && !g[1].defined() && !top) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    auto flat = [](const Tensor& t) { return t.defined() ? OptTensor(t.reshape({-1})) : c10::nullopt; };
    OptTensor g_top, top_id;
    if (top) {
      g_top = g[2].contiguous().view({-1, g[2].size(-1)});
      top_id = saved[3].view({-1, g[2].size(-1)});
    }
    const Tensor d = token_logprobs_bwd(saved[0], saved[1], saved[2], top_id, flat(g[0]), flat(g[1]), g_top,
                                        ctx->saved_data["inv_t"].toDouble(), ctx->saved_data["ignore"].toInt());
    return once({shaped(d, ctx->saved_data["sizes"].toIntVector()), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct RouteExperts : public torch::autograd::Function<RouteExperts> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, bool softmax, const OptTensor& bias,
                               int64_t groups, int64_t top_groups, bool renorm, double scale) {
    const Tensor l2 = rows_of(logits);
    auto r = route_experts_fwd(l2, k, softmax, bias, groups, top_groups, renorm, scale);
    ctx->save_for_backward({l2, r[0], r[1]});
    ctx->saved_data["form"] = (int64_t)((softmax ? 1 : 0) | (renorm ? 2 : 0));
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r[1]});
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return variable_list(8);
    const auto saved = ctx->get_saved_variables();
    const int64_t form = ctx->saved_data["form"].toInt();
    const Tensor d = route_experts_bwd(saved[0], saved[1], saved[2], g[0].contiguous(), form & 1, form & 2,
                                       ctx->saved_data["scale"].toDouble());
    return once({d, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// [y] or [y, x + residual]. The parameters have one type: x's, or fp32.
std::vector<Tensor> layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, const OptTensor& residual, double eps) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || needs_grad(w) || needs_grad(b) || needs_grad(residual)))
    return LayerNorm::apply(x, w, b, residual, eps);
  auto out = layer_norm_fwd(rows_of(x), residual.has_value() ? OptTensor(rows_of(*residual)) : c10::nullopt, w, b, eps, false);
  if (!residual.has_value()) return {shaped(out[0], x.sizes())};
  return {shaped(out[0], x.sizes()), shaped(out[1], x.sizes())};
}

Tensor rope(const Tensor& qkv, const Tensor& cos, const Tensor& sin, const OptTensor& pos, int64_t n_rot, bool interleaved,
            bool whole) {
  if (at::GradMode::is_enabled() && qkv.requires_grad()) return Rope::apply(qkv, cos, sin, pos, n_rot, interleaved, whole, 1.0);
  return rope_by(qkv, cos, sin, pos, n_rot, interleaved, whole, 1.0);
}

std::vector<Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t K, double inv_t, int64_t ignore) {
  if (at::GradMode::is_enabled() && logits.requires_grad()) return TokenLogprobs::apply(logits, tokens, K, inv_t, ignore);
  return logprobs_shaped(token_logprobs_fwd(rows_of(logits), tokens.reshape({-1}).contiguous(), K, inv_t, ignore, false), logits, K);
}

std::vector<Tensor> route_experts(const Tensor& logits, int64_t k, bool softmax, const OptTensor& bias, int64_t groups,
                                  int64_t top_groups, bool renorm, double scale) {
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return RouteExperts::apply(logits, k, softmax, bias, groups, top_groups, renorm, scale);
  return route_experts_fwd(rows_of(logits), k, softmax, bias, groups, top_groups, renorm, scale);
}

}  // namespace

void register_row_autograd(pybind11::module& m) {
  m.def("layer_norm", &layer_norm);
  m.def("rope", &rope);
  m.def("token_logprobs", &token_logprobs);
  m.def("route_experts", &route_experts);
}
