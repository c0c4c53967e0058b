// nn_ops.cpp -- PyTorch operator registrations of the transformer operators
// (torch_point_ops_norm, torch_point_ops_attention, torch_point_ops_gated),
// which the reference does not have.  Validation, allocation and autograd as
// torch_ops.cpp does them; the kernels are libtpo_hip.so's.
#include "nn_shim.hpp"

namespace torch_point_ops {
namespace {

// --------------------------------------------------------------- layer norm
int ln_weight_dtype(const Tensor& x, const Tensor& w, const char* name, const char* op) {
  TORCH_CHECK(w.device() == x.device(), op, ": x and ", name, " must be on the same device");
  TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(-1), op, ": ", name, " must have shape (",
              x.size(-1), "), the width of x, but got ", w.sizes());
  TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, op, ": ", name,
              " must be of x's type or float32");
  return nn_dtype(w, op);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_hip(const Tensor& x_in, const OptTensor& weight,
                                                  const OptTensor& bias, double eps, bool stats) {
  const char* op = "layer_norm";
  check_hip(x_in, "x");
  TORCH_CHECK(x_in.dim() >= 1, "layer_norm expects x with at least one dimension");
  TORCH_CHECK(x_in.size(-1) > 0, "layer_norm: the last dimension of x is empty");
  TORCH_CHECK(eps >= 0, "layer_norm: eps must not be negative, but got ", eps);
  c10::OptionalDeviceGuard guard(x_in.device());
  const Tensor x = x_in.contiguous();
  const int64_t width = x.size(-1), rows = x.numel() / width;
  const int dt = nn_dtype(x, op);
  Tensor w = get(weight), b = get(bias);
  int wdt = dt;
  if (w.defined()) wdt = ln_weight_dtype(x, w, "weight", op);
  if (b.defined()) {
    const int bdt = ln_weight_dtype(x, b, "bias", op);
    TORCH_CHECK(!w.defined() || bdt == wdt, "layer_norm: weight and bias must have one type");
    wdt = bdt;
  }
  if (w.defined()) w = w.contiguous();
  if (b.defined()) b = b.contiguous();
  Tensor y = at::empty_like(x), mean, rstd;
  if (stats) {
    mean = at::empty({rows}, x.options().dtype(at::kFloat));
    rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  }
  check_rc(tpo_layer_norm_fwd(dt, wdt, x.data_ptr(), data_or_null(w), data_or_null(b), rows, width,
                              eps, y.data_ptr(), (float*)data_or_null(mean),
                              (float*)data_or_null(rstd), stream_of(x)),
           op);
  return {y, mean, rstd};
}

Tensor layer_norm_only_hip(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  return std::get<0>(layer_norm_hip(x, w, b, eps, false));
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_forward_hip(const Tensor& x, const OptTensor& w,
                                                          const OptTensor& b, double eps) {
  return layer_norm_hip(x, w, b, eps, true);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_hip(
    const Tensor& grad_in, const Tensor& x_in, const OptTensor& weight, const OptTensor& bias,
    const Tensor& mean_in, const Tensor& rstd_in, double eps, std::array<bool, 3> mask) {
  const char* op = "layer_norm_backward";
  check_hip(x_in, "x");
  c10::OptionalDeviceGuard guard(x_in.device());
  TORCH_CHECK(x_in.dim() >= 1 && x_in.size(-1) > 0, "layer_norm_backward: x is empty");
  TORCH_CHECK(grad_in.sizes() == x_in.sizes() && grad_in.device() == x_in.device(),
              "layer_norm_backward: the gradient must have x's shape and device");
  const Tensor x = x_in.contiguous(), g = grad_in.to(x.scalar_type()).contiguous();
  const int64_t width = x.size(-1), rows = x.numel() / width;
  const int dt = nn_dtype(x, op);
  Tensor w = get(weight);
  const Tensor b = get(bias);
  int wdt = dt;
  if (b.defined()) wdt = ln_weight_dtype(x, b, "bias", op);
  if (w.defined()) {
    wdt = ln_weight_dtype(x, w, "weight", op);
    w = w.contiguous();
  }
  for (const Tensor& t : {mean_in, rstd_in})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == rows && t.device() == x.device(),
                "layer_norm_backward: mean and rstd must hold a float32 a row");
  const Tensor mean = mean_in.contiguous(), rstd = rstd_in.contiguous();
  const bool want_w = mask[1] && w.defined(), want_b = mask[2] && b.defined();
  Tensor gx, gw, gb, ws;
  if (mask[0]) gx = at::empty_like(x);
  if (want_w) gw = at::empty({width}, w.options());
  if (want_b) gb = at::empty({width}, b.options());
  int64_t wsb = 0;
  if (want_w || want_b) {
    wsb = tpo_layer_norm_bwd_workspace_size(rows, width);
    ws = workspace(wsb, x, op);
  }
  check_rc(tpo_layer_norm_bwd(dt, wdt, g.data_ptr(), x.data_ptr(), data_or_null(w),
                              mean.data_ptr<float>(), rstd.data_ptr<float>(), rows, width, eps,
                              data_or_null(gx), data_or_null(gw), data_or_null(gb),
                              data_or_null(ws), wsb, stream_of(x)),
           op);
  if (!gx.defined()) gx = nothing(x);
  if (!gw.defined()) gw = nothing(x);
  if (!gb.defined()) gb = nothing(x);
  return {gx, gw, gb};
}

auto layer_norm_op() {
  static auto op = typed_op<Tensor(const Tensor&, const OptTensor&, const OptTensor&, double)>(
      "torch_point_ops_norm::layer_norm");
  return op;
}

class LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w,
                        const OptTensor& b, double eps) {
    static auto op = typed_op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const OptTensor&,
                                                                 const OptTensor&, double)>(
        "torch_point_ops_norm::layer_norm_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, mean, rstd] = op.call(x, w, b, eps);
    ctx->save_for_backward({x, get(w), get(b), mean, rstd});
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = typed_op<std::tuple<Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&,
        const Tensor&, double, std::array<bool, 3>)>("torch_point_ops_norm::layer_norm_backward");
    const auto s = ctx->get_saved_variables();
    // edges are counted over the tensors that were given
    const bool w = s[1].defined(), b = s[2].defined();
    const std::array<bool, 3> mask = {ctx->needs_input_grad(0), w && ctx->needs_input_grad(1),
                                      b && ctx->needs_input_grad(w ? 2 : 1)};
    auto [gx, gw, gb] = op.call(grads[0], s[0], opt(s[1]), opt(s[2]), s[3], s[4],
                                ctx->saved_data["eps"].toDouble(), mask);
    return {mask[0] ? gx : Tensor(), mask[1] ? gw : Tensor(), mask[2] ? gb : Tensor(), Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  if (!followed(x) && !(w && followed(*w)) && !(b && followed(*b))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_op().call(x, w, b, eps);
  }
  return LayerNormFunction::apply(x, w, b, eps);
}

// --------------------------------------------------------- packed attention
struct Packed {  // checked arguments of an attention call
  Tensor q, k, v, oq, ok, lq, lk;
  int64_t B, Tq, Tk, Hq, Hk, D;  // D padded to 16 bytes
  int dt;
};

Packed packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& oq,
                   const Tensor& ok, const OptTensor& lq, const OptTensor& lk, const char* op) {
  check_hip(q, "q");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, op,
              " expects q (Tq, Hq, D) and k, v (Tk, Hk, D)");
  TORCH_CHECK(k.sizes() == v.sizes(), op, ": k and v must have the same shape, but got ", k.sizes(),
              " and ", v.sizes());
  TORCH_CHECK(q.size(2) == k.size(2), op, ": q and k must have the same head size, but got ",
              q.size(2), " and ", k.size(2));
  TORCH_CHECK(k.size(1) > 0 && q.size(1) > 0 && q.size(1) % k.size(1) == 0, op, ": the ", q.size(1),
              " heads of q must be a multiple of the ", k.size(1), " heads of k");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), op,
              ": q, k and v must have one type");
  Packed p;
  p.dt = nn_dtype(q, op);
  p.lq = get(lq);
  p.lk = get(lk);
  for (const Tensor& t : {k, v, oq, ok, p.lq, p.lk})
    TORCH_CHECK(!t.defined() || t.device() == q.device(), op,
                ": all tensors must be on the same device");
  for (const Tensor& t : {oq, ok})
    TORCH_CHECK(t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) >= 1, op,
                ": offsets must be int64 with one entry more than there are sequences");
  TORCH_CHECK(oq.size(0) == ok.size(0), op, ": offsets_q and offsets_k differ in length: ",
              oq.size(0), " and ", ok.size(0));
  p.B = oq.size(0) - 1;
  for (const Tensor& t : {p.lq, p.lk})
    TORCH_CHECK(!t.defined() ||
                    (t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) == p.B),
                op, ": lengths must be int64 with one entry a sequence");
  TORCH_CHECK(q.size(2) > 0, op, ": the heads of q are empty");
  const int64_t per = 16 / q.element_size();
  p.D = (q.size(2) + per - 1) / per * per;
  p.q = head_rows(q, p.D);
  p.k = head_rows(k, p.D);
  p.v = head_rows(v, p.D);
  p.oq = oq.contiguous();
  p.ok = ok.contiguous();
  if (p.lq.defined()) p.lq = p.lq.contiguous();
  if (p.lk.defined()) p.lk = p.lk.contiguous();
  p.Tq = q.size(0);
  p.Tk = k.size(0);
  p.Hq = q.size(1);
  p.Hk = k.size(1);
  return p;
}

std::tuple<Tensor, Tensor, Tensor> packed_attention_hip(const Tensor& q, const Tensor& k, const Tensor& v,
                                                const Tensor& oq, const Tensor& ok,
                                                const OptTensor& lq, const OptTensor& lk,
                                                bool causal, double scale, bool stats) {
  const char* op = "packed_attention";
  const Packed p = packed_args(q, k, v, oq, ok, lq, lk, op);
  c10::OptionalDeviceGuard guard(q.device());
  Tensor out = at::empty({p.Tq, p.Hq, p.D}, q.options()), lse, rest;
  if (stats) lse = at::empty({p.Hq, p.Tq}, q.options().dtype(at::kFloat));
  if (stats) rest = p.dt == TPO_F32 ? nothing(q) : at::empty_like(out);
  const int64_t wsb = tpo_attention_fwd_workspace_size(p.dt, p.B, p.Tq, p.Tk, p.Hq, p.Hk, p.D);
  const Tensor ws = workspace(wsb, q, op);
  check_rc(tpo_attention_fwd(p.dt, p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(),
                             p.oq.data_ptr<int64_t>(), p.ok.data_ptr<int64_t>(),
                             (const int64_t*)data_or_null(p.lq), (const int64_t*)data_or_null(p.lk),
                             p.B, p.Tq, p.Tk, p.Hq, p.Hk, p.D, row_stride(p.q), head_stride(p.q),
                             row_stride(p.k), head_stride(p.k), row_stride(p.v), head_stride(p.v),
                             causal, scale, out.data_ptr(), (float*)data_or_null(lse), data_or_null(rest),
                             data_or_null(ws), wsb, stream_of(q)),
           op);
  if (stats && rest.dim() == 3) rest = cut_heads(rest, q.size(2));
  return {cut_heads(out, q.size(2)), lse, rest};
}

Tensor packed_attention_only_hip(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& oq, const Tensor& ok, const OptTensor& lq,
                                 const OptTensor& lk, bool causal, double scale) {
  return std::get<0>(packed_attention_hip(q, k, v, oq, ok, lq, lk, causal, scale, false));
}
std::tuple<Tensor, Tensor, Tensor> packed_attention_forward_hip(const Tensor& q, const Tensor& k,
                                                        const Tensor& v, const Tensor& oq,
                                                        const Tensor& ok, const OptTensor& lq,
                                                        const OptTensor& lk, bool causal,
                                                        double scale) {
  return packed_attention_hip(q, k, v, oq, ok, lq, lk, causal, scale, true);
}

std::tuple<Tensor, Tensor, Tensor> packed_attention_backward_hip(
    const Tensor& grad_in, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out_in,
    const Tensor& lse_in, const Tensor& rest_in, const Tensor& oq, const Tensor& ok,
    const OptTensor& lq, const OptTensor& lk, bool causal, double scale,
    std::array<bool, 3> mask) {
  const char* op = "packed_attention_backward";
  const Packed p = packed_args(q, k, v, oq, ok, lq, lk, op);
  c10::OptionalDeviceGuard guard(q.device());
  TORCH_CHECK(grad_in.sizes() == q.sizes() && out_in.sizes() == q.sizes(),
              "packed_attention_backward: out and its gradient must have q's shape");
  TORCH_CHECK(out_in.scalar_type() == q.scalar_type() && lse_in.scalar_type() == at::kFloat &&
                  lse_in.numel() == p.Tq * p.Hq,
              "packed_attention_backward: out and lse must be the forward's");
  TORCH_CHECK(rest_in.numel() == 0 || (rest_in.sizes() == q.sizes() &&
                                       rest_in.scalar_type() == q.scalar_type()),
              "packed_attention_backward: rest must be the forward's");
  for (const Tensor& t : {grad_in, out_in, lse_in, rest_in})
    TORCH_CHECK(t.device() == q.device(), op, ": all tensors must be on the same device");
  const Tensor g = head_rows(grad_in.to(q.scalar_type()).contiguous(), p.D);
  const Tensor out = head_rows(out_in.contiguous(), p.D);
  const Tensor lse = lse_in.contiguous();
  Tensor rest;
  if (rest_in.numel() > 0) rest = head_rows(rest_in.contiguous(), p.D);
  // dK and dV come from one kernel
  const bool keys = mask[1] || mask[2];
  Tensor gq, gk, gv, ws;
  int64_t wsb = 0;
  if (mask[0]) gq = at::empty({p.Tq, p.Hq, p.D}, q.options());
  if (keys) {
    gk = at::empty({p.Tk, p.Hk, p.D}, q.options());
    gv = at::empty({p.Tk, p.Hk, p.D}, q.options());
    wsb = tpo_attention_bwd_workspace_size(p.dt, p.B, p.Tq, p.Tk, p.Hq, p.Hk, p.D);
    ws = workspace(wsb, q, op);
  }
  check_rc(tpo_attention_bwd(p.dt, g.data_ptr(), p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(),
                             out.data_ptr(), data_or_null(rest), lse.data_ptr<float>(),
                             p.oq.data_ptr<int64_t>(), p.ok.data_ptr<int64_t>(),
                             (const int64_t*)data_or_null(p.lq), (const int64_t*)data_or_null(p.lk),
                             p.B, p.Tq, p.Tk, p.Hq, p.Hk, p.D, row_stride(p.q), head_stride(p.q),
                             row_stride(p.k), head_stride(p.k), row_stride(p.v), head_stride(p.v),
                             causal, scale, data_or_null(gq), data_or_null(gk), data_or_null(gv),
                             data_or_null(ws), wsb, stream_of(q)),
           op);
  const int64_t D = q.size(2);
  return {mask[0] ? cut_heads(gq, D) : nothing(q), mask[1] ? cut_heads(gk, D) : nothing(q),
          mask[2] ? cut_heads(gv, D) : nothing(q)};
}

auto packed_attention_op() {
  static auto op =
      typed_op<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                      const OptTensor&, const OptTensor&, bool, double)>(
          "torch_point_ops_attention::packed_attention");
  return op;
}

class PackedAttentionFunction : public torch::autograd::Function<PackedAttentionFunction> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Tensor& oq, const Tensor& ok, const OptTensor& lq,
                        const OptTensor& lk, bool causal, double scale) {
    static auto op = typed_op<std::tuple<Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
        const OptTensor&, const OptTensor&, bool, double)>(
        "torch_point_ops_attention::packed_attention_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse, rest] = op.call(q, k, v, oq, ok, lq, lk, causal, scale);
    ctx->save_for_backward({q, k, v, out, lse, rest, oq, ok, get(lq), get(lk)});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = typed_op<std::tuple<Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
        const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, bool,
        double, std::array<bool, 3>)>("torch_point_ops_attention::packed_attention_backward");
    const auto s = ctx->get_saved_variables();
    const std::array<bool, 3> mask = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                      ctx->needs_input_grad(2)};
    auto [gq, gk, gv] = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], opt(s[8]),
                                opt(s[9]), ctx->saved_data["causal"].toBool(),
                                ctx->saved_data["scale"].toDouble(), mask);
    const Tensor none;
    return {mask[0] ? gq : none, mask[1] ? gk : none, mask[2] ? gv : none,
            none, none, none, none, none, none};
  }
};

Tensor packed_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& oq, const Tensor& ok, const OptTensor& lq,
                                 const OptTensor& lk, bool causal, double scale) {
  if (!followed(q) && !followed(k) && !followed(v)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return packed_attention_op().call(q, k, v, oq, ok, lq, lk, causal, scale);
  }
  return PackedAttentionFunction::apply(q, k, v, oq, ok, lq, lk, causal, scale);
}

// --------------------------------------------------------- gated projection
struct Gated {
  Tensor x, wg, wu;
  int64_t M, K, F;
  int dt;
};

Gated gated_args(const Tensor& x, const Tensor& wg, const Tensor& wu, const char* op) {
  check_hip(x, "x");
  TORCH_CHECK(x.dim() >= 1 && wg.dim() == 2, op, " expects x (..., K) and weights (F, K)");
  TORCH_CHECK(wg.sizes() == wu.sizes(), op, ": w_gate and w_up must have the same shape, but got ",
              wg.sizes(), " and ", wu.sizes());
  TORCH_CHECK(x.size(-1) == wg.size(1) && wg.size(1) > 0, op, ": x has ", x.size(-1),
              " features, the weights take ", wg.size(1));
  TORCH_CHECK(x.scalar_type() == wg.scalar_type() && x.scalar_type() == wu.scalar_type(), op,
              ": x, w_gate and w_up must have one type");
  TORCH_CHECK(x.device() == wg.device() && x.device() == wu.device(), op,
              ": all tensors must be on the same device");
  Gated a;
  a.dt = nn_dtype(x, op);
  a.K = x.size(-1);
  a.M = x.numel() / a.K;
  a.F = wg.size(0);
  a.x = aligned16(x.contiguous());
  a.wg = aligned16(wg.contiguous());
  a.wu = aligned16(wu.contiguous());
  return a;
}

std::tuple<Tensor, Tensor> gated_projection_both(const Tensor& x, const Tensor& wg,
                                                 const Tensor& wu, int64_t act, bool keep) {
  const char* op = "gated_projection";
  const Gated a = gated_args(x, wg, wu, op);
  c10::OptionalDeviceGuard guard(x.device());
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = a.F;
  Tensor h = at::empty(shape, x.options()), kept;
  if (keep) kept = a.dt == TPO_F32 ? at::empty({a.M, 2 * a.F}, x.options()) : nothing(x);
  const int64_t wsb = tpo_gated_fwd_workspace_size(a.dt, a.M, a.K, a.F);
  const Tensor ws = workspace(wsb, x, op);
  check_rc(tpo_gated_fwd(a.dt, a.x.data_ptr(), a.wg.data_ptr(), a.wu.data_ptr(), a.M, a.K, a.F,
                         (int)act, h.data_ptr(), data_or_null(kept), data_or_null(ws), wsb,
                         stream_of(x)),
           op);
  return {h, kept};
}

Tensor gated_projection_hip(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
  return std::get<0>(gated_projection_both(x, wg, wu, act, false));
}
std::tuple<Tensor, Tensor> gated_projection_forward_hip(const Tensor& x, const Tensor& wg,
                                                        const Tensor& wu, int64_t act) {
  return gated_projection_both(x, wg, wu, act, true);
}

std::tuple<Tensor, Tensor, Tensor> gated_projection_backward_hip(const Tensor& grad_in,
                                                                 const Tensor& x, const Tensor& wg,
                                                                 const Tensor& wu,
                                                                 const Tensor& kept_in, int64_t act,
                                                                 std::array<bool, 2> mask) {
  const char* op = "gated_projection_backward";
  const Gated a = gated_args(x, wg, wu, op);
  c10::OptionalDeviceGuard guard(x.device());
  TORCH_CHECK(grad_in.dim() == x.dim() && grad_in.size(-1) == a.F &&
                  grad_in.numel() == a.M * a.F && grad_in.device() == x.device(),
              "gated_projection_backward: the gradient must have the output's shape and device");
  TORCH_CHECK(kept_in.numel() == 0 ||
                  (kept_in.scalar_type() == at::kFloat && x.scalar_type() == at::kFloat &&
                   kept_in.numel() == 2 * a.M * a.F && kept_in.device() == x.device()),
              "gated_projection_backward: kept must be the forward's");
  Tensor kept;
  if (kept_in.numel() > 0) kept = kept_in.contiguous();
  const Tensor g = grad_in.to(x.scalar_type()).contiguous();
  Tensor gx, gg, gu;
  if (mask[0]) gx = at::empty(x.sizes(), x.options());
  if (mask[1]) {
    gg = at::empty({a.F, a.K}, x.options());
    gu = at::empty({a.F, a.K}, x.options());
  }
  const int64_t wsb = tpo_gated_bwd_workspace_size(a.dt, a.M, a.K, a.F);
  const Tensor ws = workspace(wsb, x, op);
  check_rc(tpo_gated_bwd(a.dt, g.data_ptr(), a.x.data_ptr(), a.wg.data_ptr(), a.wu.data_ptr(),
                         data_or_null(kept), a.M, a.K, a.F, (int)act, data_or_null(gx), data_or_null(gg), data_or_null(gu),
                         data_or_null(ws), wsb, stream_of(x)),
           op);
  if (!gx.defined()) gx = nothing(x);
  if (!gg.defined()) gg = gu = nothing(x);
  return {gx, gg, gu};
}

auto gated_projection_op() {
  static auto op = typed_op<Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t)>(
      "torch_point_ops_gated::gated_projection");
  return op;
}

class GatedProjectionFunction : public torch::autograd::Function<GatedProjectionFunction> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        int64_t act) {
    static auto op =
        typed_op<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, int64_t)>(
            "torch_point_ops_gated::gated_projection_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [h, kept] = op.call(x, wg, wu, act);
    ctx->save_for_backward({x, wg, wu, kept});
    ctx->saved_data["act"] = act;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = typed_op<std::tuple<Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t,
        std::array<bool, 2>)>("torch_point_ops_gated::gated_projection_backward");
    const auto s = ctx->get_saved_variables();
    const bool gate = ctx->needs_input_grad(1), up = ctx->needs_input_grad(2);
    const std::array<bool, 2> mask = {ctx->needs_input_grad(0), gate || up};
    auto [gx, gg, gu] =
        op.call(grads[0], s[0], s[1], s[2], s[3], ctx->saved_data["act"].toInt(), mask);
    return {mask[0] ? gx : Tensor(), gate ? gg : Tensor(), up ? gu : Tensor(), Tensor()};
  }
};

Tensor gated_projection_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
  if (!followed(x) && !followed(wg) && !followed(wu)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return gated_projection_op().call(x, wg, wu, act);
  }
  return GatedProjectionFunction::apply(x, wg, wu, act);
}

// Under autocast the two operators that are products take its type, as torch's own
// products do; layer norm takes x and weights of different types as they are.
Tensor packed_attention_autocast(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& oq, const Tensor& ok, const OptTensor& lq,
                                 const OptTensor& lk, bool causal, double scale) {
  c10::impl::ExcludeDispatchKeyGuard below(c10::DispatchKey::AutocastCUDA);
  return packed_attention_op().call(autocast(q), autocast(k), autocast(v), oq, ok, lq, lk, causal,
                                    scale);
}
Tensor gated_projection_autocast(const Tensor& x, const Tensor& wg, const Tensor& wu,
                                 int64_t act) {
  c10::impl::ExcludeDispatchKeyGuard below(c10::DispatchKey::AutocastCUDA);
  return gated_projection_op().call(autocast(x), autocast(wg), autocast(wu), act);
}

// There are no CPU kernels: as Chamfer and EMD, a call says so.
Tensor layer_norm_cpu(const Tensor&, const OptTensor&, const OptTensor&, double) {
  TORCH_CHECK(false, "layer_norm is not implemented for CPU");
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_forward_cpu(const Tensor&, const OptTensor&,
                                                          const OptTensor&, double) {
  TORCH_CHECK(false, "layer_norm is not implemented for CPU");
}
Tensor packed_attention_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                            const Tensor&, const OptTensor&, const OptTensor&, bool, double) {
  TORCH_CHECK(false, "packed_attention is not implemented for CPU");
}
std::tuple<Tensor, Tensor, Tensor> packed_attention_forward_cpu(const Tensor&, const Tensor&,
                                                        const Tensor&, const Tensor&,
                                                        const Tensor&, const OptTensor&,
                                                        const OptTensor&, bool, double) {
  TORCH_CHECK(false, "packed_attention is not implemented for CPU");
}
std::tuple<Tensor, Tensor> gated_projection_forward_cpu(const Tensor&, const Tensor&,
                                                        const Tensor&, int64_t) {
  TORCH_CHECK(false, "gated_projection is not implemented for CPU");
}
Tensor gated_projection_cpu(const Tensor&, const Tensor&, const Tensor&, int64_t) {
  TORCH_CHECK(false, "gated_projection is not implemented for CPU");
}

}  // namespace

TORCH_LIBRARY(torch_point_ops_norm, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  // with the mean and the reciprocal deviation of each row
  m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor mean, "
        "Tensor rstd, float eps, bool[3] mask) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(torch_point_ops_norm, CPU, m) {
  m.impl("layer_norm", &layer_norm_cpu);
  m.impl("layer_norm_forward", &layer_norm_forward_cpu);
}
TORCH_LIBRARY_IMPL(torch_point_ops_norm, CUDA, m) {
  m.impl("layer_norm", &layer_norm_only_hip);
  m.impl("layer_norm_forward", &layer_norm_forward_hip);
  m.impl("layer_norm_backward", &layer_norm_backward_hip);
}
TORCH_LIBRARY_IMPL(torch_point_ops_norm, Autograd, m) {
  m.impl("layer_norm", &layer_norm_autograd);
  m.impl("layer_norm_forward", no_formula());
  m.impl("layer_norm_backward", no_formula());
}

TORCH_LIBRARY(torch_point_ops_attention, m) {
  m.def("packed_attention(Tensor q, Tensor k, Tensor v, Tensor offsets_q, Tensor offsets_k, "
        "Tensor? lengths_q, Tensor? lengths_k, bool causal, float scale) -> Tensor");
  // with the logarithm of each row's sum of exponentials, and what rounding took
  // from the result (half types)
  m.def("packed_attention_forward(Tensor q, Tensor k, Tensor v, Tensor offsets_q, "
        "Tensor offsets_k, Tensor? lengths_q, Tensor? lengths_k, bool causal, float scale) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("packed_attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor out, "
        "Tensor lse, Tensor rest, Tensor offsets_q, Tensor offsets_k, Tensor? lengths_q, "
        "Tensor? lengths_k, bool causal, float scale, bool[3] mask=[True, True, True]) -> "
        "(Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(torch_point_ops_attention, CPU, m) {
  m.impl("packed_attention", &packed_attention_cpu);
  m.impl("packed_attention_forward", &packed_attention_forward_cpu);
}
TORCH_LIBRARY_IMPL(torch_point_ops_attention, CUDA, m) {
  m.impl("packed_attention", &packed_attention_only_hip);
  m.impl("packed_attention_forward", &packed_attention_forward_hip);
  m.impl("packed_attention_backward", &packed_attention_backward_hip);
}
TORCH_LIBRARY_IMPL(torch_point_ops_attention, AutocastCUDA, m) {
  m.impl("packed_attention", &packed_attention_autocast);
}
TORCH_LIBRARY_IMPL(torch_point_ops_attention, Autograd, m) {
  m.impl("packed_attention", &packed_attention_autograd);
  m.impl("packed_attention_forward", no_formula());
  m.impl("packed_attention_backward", no_formula());
}

TORCH_LIBRARY(torch_point_ops_gated, m) {
  m.def("gated_projection(Tensor x, Tensor w_gate, Tensor w_up, int activation) -> Tensor");
  // with the projections themselves (float; empty for the half types)
  m.def("gated_projection_forward(Tensor x, Tensor w_gate, Tensor w_up, int activation) -> "
        "(Tensor, Tensor)");
  m.def("gated_projection_backward(Tensor grad, Tensor x, Tensor w_gate, Tensor w_up, "
        "Tensor kept, int activation, bool[2] mask) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(torch_point_ops_gated, CPU, m) {
  m.impl("gated_projection", &gated_projection_cpu);
  m.impl("gated_projection_forward", &gated_projection_forward_cpu);
}
TORCH_LIBRARY_IMPL(torch_point_ops_gated, CUDA, m) {
  m.impl("gated_projection", &gated_projection_hip);
  m.impl("gated_projection_forward", &gated_projection_forward_hip);
  m.impl("gated_projection_backward", &gated_projection_backward_hip);
}
TORCH_LIBRARY_IMPL(torch_point_ops_gated, AutocastCUDA, m) {
  m.impl("gated_projection", &gated_projection_autocast);
}
TORCH_LIBRARY_IMPL(torch_point_ops_gated, Autograd, m) {
  m.impl("gated_projection", &gated_projection_autograd);
  m.impl("gated_projection_forward", no_formula());
  m.impl("gated_projection_backward", no_formula());
}

}  // namespace torch_point_ops
