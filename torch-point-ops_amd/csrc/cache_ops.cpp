// cache_ops.cpp -- PyTorch operator registrations of rotary positions and of the 8-bit cache
// (torch_point_ops_rotary, torch_point_ops_cache), which the reference does not have.
// Validation, allocation and autograd as nn_ops.cpp does them.
#include "nn_shim.hpp"

namespace torch_point_ops {
namespace {

// Whether the values of a head lie together, as the kernels take rows of any distance.
Tensor with_heads_together(const Tensor& t) {
  return t.size(2) <= 1 || t.stride(2) == 1 ? t : t.contiguous();
}

// --------------------------------------------------------- rotary positions
struct Angles {  // checked places and frequencies
  Tensor at, f;
  int64_t axes = 1, pairs = 0;
  int dtype = TPO_I64;
};

Angles angles_of(const Tensor& x, const OptTensor& positions, const OptTensor& frequencies,
                 const char* op) {
  Angles a;
  if (frequencies.has_value()) {
    const Tensor& f = *frequencies;
    TORCH_CHECK(f.scalar_type() == at::kDouble && f.dim() == 1, op,
                ": frequencies must be float64 with one entry a pair");
    TORCH_CHECK(f.device() == x.device(), op, ": all tensors must be on the same device");
    TORCH_CHECK(2 * f.size(0) <= x.size(2), op, ": ", f.size(0), " pairs need heads of ",
                2 * f.size(0), " values, but got ", x.size(2));
    a.f = f.contiguous();
    a.pairs = f.size(0);
  }
  if (positions.has_value()) {
    const Tensor& p = *positions;
    TORCH_CHECK(p.scalar_type() == at::kLong || p.scalar_type() == at::kFloat, op,
                ": positions must be int64 or float32");
    TORCH_CHECK((p.dim() == 1 || p.dim() == 2) && p.size(0) == x.size(0), op,
                ": positions must have shape (", x.size(0), ") or (", x.size(0),
                ", axes), but got ", p.sizes());
    TORCH_CHECK(p.device() == x.device(), op, ": all tensors must be on the same device");
    a.axes = p.dim() == 2 ? p.size(1) : 1;
    TORCH_CHECK(a.axes >= 1 && a.pairs % a.axes == 0, op, ": ", a.pairs,
                " pairs do not share out among ", a.axes, " axes");
    a.at = p.contiguous();
    a.dtype = p.scalar_type() == at::kLong ? TPO_I64 : TPO_F32;
  }
  return a;
}

Tensor rotary_both(const Tensor& x_in, const Tensor& positions, const Tensor& frequencies,
                   bool interleaved, double amplitude, bool back, const char* op) {
  check_hip(x_in, "x");
  TORCH_CHECK(x_in.dim() == 3, op, " expects x (T, H, D), but got ", x_in.sizes());
  TORCH_CHECK(x_in.size(2) > 0, op, ": the heads of x are empty");
  c10::OptionalDeviceGuard guard(x_in.device());
  const int dt = nn_dtype(x_in, op);
  const Angles a = angles_of(x_in, positions, frequencies, op);
  const Tensor x = with_heads_together(x_in);
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  check_rc(tpo_rotary(dt, x.data_ptr(), x.size(0), x.size(1), x.size(2), x.stride(0), x.stride(1),
                      a.at.data_ptr(), a.dtype, a.axes, (const double*)a.f.data_ptr(), a.pairs,
                      interleaved, amplitude, back, y.data_ptr(), stream_of(x)),
           op);
  return y;
}

Tensor rotary_positions_hip(const Tensor& x, const Tensor& positions, const Tensor& frequencies,
                            bool interleaved, double amplitude) {
  return rotary_both(x, positions, frequencies, interleaved, amplitude, false, "rotary_positions");
}
Tensor rotary_positions_backward_hip(const Tensor& grad, const Tensor& positions,
                                     const Tensor& frequencies, bool interleaved,
                                     double amplitude) {
  return rotary_both(grad, positions, frequencies, interleaved, amplitude, true,
                     "rotary_positions_backward");
}

auto rotary_positions_op() {
  static auto op = typed_op<Tensor(const Tensor&, const Tensor&, const Tensor&, bool, double)>(
      "torch_point_ops_rotary::rotary_positions");
  return op;
}

class RotaryPositionsFunction : public torch::autograd::Function<RotaryPositionsFunction> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions,
                        const Tensor& frequencies, bool interleaved, double amplitude) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    return rotary_positions_op().call(x, positions, frequencies, interleaved, amplitude);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = typed_op<Tensor(const Tensor&, const Tensor&, const Tensor&, bool, double)>(
        "torch_point_ops_rotary::rotary_positions_backward");
    const auto s = ctx->get_saved_variables();
    const Tensor none;
    return {op.call(grads[0], s[0], s[1], ctx->saved_data["interleaved"].toBool(),
                    ctx->saved_data["amplitude"].toDouble()),
            none, none, none, none};
  }
};

Tensor rotary_positions_autograd(const Tensor& x, const Tensor& positions,
                                 const Tensor& frequencies, bool interleaved, double amplitude) {
  TORCH_CHECK(!followed(positions) && !followed(frequencies),
              "rotary_positions has no derivative in positions and frequencies");
  if (!followed(x)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return rotary_positions_op().call(x, positions, frequencies, interleaved, amplitude);
  }
  return RotaryPositionsFunction::apply(x, positions, frequencies, interleaved, amplitude);
}

// ------------------------------------------------------------- 8-bit cache
struct PagedCache {  // checked tensors of a cache
  int64_t pages, Hk, page, Dr, B, M;
};

PagedCache cache_of(const Tensor& like, const Tensor& keys, const Tensor& values,
                    const Tensor& key_scales, const Tensor& value_scales, const Tensor& table,
                    const Tensor& lengths, const char* op) {
  for (const Tensor& t : {keys, values, key_scales, value_scales, table, lengths})
    TORCH_CHECK(t.device() == like.device(), op, ": all tensors must be on the same device");
  for (const Tensor& t : {keys, values, key_scales, value_scales, table, lengths})
    TORCH_CHECK(t.is_contiguous(), op, ": the cache's tensors must be contiguous");
  TORCH_CHECK(keys.scalar_type() == at::kFloat8_e4m3fn && keys.dim() == 6 && keys.size(4) == 32 &&
                  keys.size(5) == 16,
              op, ": keys must be float8_e4m3fn (pages, Hk, page / 32, Dr / 16, 32, 16), but got ",
              keys.scalar_type(), " ", keys.sizes());
  PagedCache c;
  c.pages = keys.size(0);
  c.Hk = keys.size(1);
  c.page = keys.size(2) * 32;
  c.Dr = keys.size(3) * 16;
  TORCH_CHECK(values.scalar_type() == at::kFloat8_e4m3fn &&
                  values.sizes() == at::IntArrayRef({c.pages, c.Hk, keys.size(2), c.Dr, 32}),
              op,
              ": values must be float8_e4m3fn (pages, Hk, page / 32, Dr, 32) as keys are, but got ",
              values.scalar_type(), " ", values.sizes());
  for (const Tensor& t : {key_scales, value_scales})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == at::IntArrayRef({c.pages, c.Hk}), op,
                ": scales must be float32 (pages, Hk), but got ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2, op,
              ": the table must be int32 (B, pages of a sequence), but got ", table.scalar_type(),
              " ", table.sizes());
  c.B = table.size(0);
  c.M = table.size(1);
  TORCH_CHECK(lengths.scalar_type() == at::kLong && lengths.dim() == 1 && lengths.size(0) == c.B,
              op, ": lengths must be int64 with one entry a sequence");
  return c;
}

struct NewRows {  // offsets of a call's rows and how many are in use
  Tensor offsets, lengths;
};
NewRows new_rows(const Tensor& like, const PagedCache& c, const Tensor& offsets,
                 const OptTensor& lengths, const char* op) {
  NewRows r{offsets, get(lengths)};
  for (const Tensor& t : {r.offsets, r.lengths})
    TORCH_CHECK(!t.defined() || t.device() == like.device(), op,
                ": all tensors must be on the same device");
  TORCH_CHECK(offsets.scalar_type() == at::kLong && offsets.dim() == 1 &&
                  offsets.size(0) == c.B + 1,
              op, ": offsets must be int64 with one entry more than the table has sequences");
  TORCH_CHECK(!r.lengths.defined() || (r.lengths.scalar_type() == at::kLong &&
                                       r.lengths.dim() == 1 && r.lengths.size(0) == c.B),
              op, ": lengths must be int64 with one entry a sequence");
  r.offsets = r.offsets.contiguous();
  if (r.lengths.defined()) r.lengths = r.lengths.contiguous();
  return r;
}

Tensor cache_append_hip(const Tensor& k_in, const Tensor& v_in, Tensor keys, Tensor values,
                        Tensor key_scales, Tensor value_scales, const Tensor& table,
                        const Tensor& lengths, const Tensor& offsets, const OptTensor& lengths_new,
                        const OptTensor& q_in, const OptTensor& positions,
                        const OptTensor& frequencies, bool interleaved, double amplitude) {
  const char* op = "cache_append";
  check_hip(k_in, "k");
  TORCH_CHECK(k_in.dim() == 3 && v_in.dim() == 3, op, " expects k and v (T, Hk, D)");
  TORCH_CHECK(k_in.sizes() == v_in.sizes(), op, ": k and v must have the same shape, but got ",
              k_in.sizes(), " and ", v_in.sizes());
  TORCH_CHECK(k_in.scalar_type() == v_in.scalar_type() && k_in.device() == v_in.device(), op,
              ": k and v must have one type and device");
  c10::OptionalDeviceGuard guard(k_in.device());
  const int dt = nn_dtype(k_in, op);
  const PagedCache c =
      cache_of(k_in, keys, values, key_scales, value_scales, table, lengths, op);
  TORCH_CHECK(k_in.size(1) == c.Hk, op, ": k has ", k_in.size(1), " heads, the cache has ", c.Hk);
  const int64_t T = k_in.size(0), D = k_in.size(2);
  TORCH_CHECK(D > 0 && (D + 15) / 16 * 16 == c.Dr, op, ": heads of ", D,
              " values need a cache of ", (D + 15) / 16 * 16, ", but got ", c.Dr);
  const NewRows r = new_rows(k_in, c, offsets, lengths_new, op);
  const Angles a = angles_of(k_in, positions, frequencies, op);
  const Tensor k = with_heads_together(k_in), v = with_heads_together(v_in);
  Tensor q, q_out;
  if (q_in.has_value()) {
    TORCH_CHECK(frequencies.has_value(), op, ": q is turned: it needs frequencies");
    TORCH_CHECK(q_in->dim() == 3 && q_in->size(0) == T && q_in->size(2) == D, op,
                ": q must have shape (", T, ", Hq, ", D, "), but got ", q_in->sizes());
    TORCH_CHECK(q_in->scalar_type() == k.scalar_type() && q_in->device() == k.device(), op,
                ": q must have k's type and device");
    TORCH_CHECK(q_in->size(1) > 0, op, ": q has no heads");
    q = with_heads_together(*q_in);
    q_out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  }
  check_rc(tpo_cache_append(
               dt, k.data_ptr(), v.data_ptr(), data_or_null(q), r.offsets.data_ptr<int64_t>(),
               (const int64_t*)data_or_null(r.lengths), c.B, T, q.defined() ? q.size(1) : 0, D,
               k.stride(0), k.stride(1), v.stride(0), v.stride(1), q.defined() ? q.stride(0) : 0,
               q.defined() ? q.stride(1) : 0, data_or_null(a.at), a.dtype, a.axes,
               (const double*)data_or_null(a.f), a.pairs, interleaved, amplitude, keys.data_ptr(),
               values.data_ptr(), key_scales.data_ptr<float>(), value_scales.data_ptr<float>(),
               table.data_ptr<int32_t>(), lengths.data_ptr<int64_t>(), c.pages, c.Hk, c.page, c.Dr,
               c.M, data_or_null(q_out), stream_of(k)),
           op);
  return q_out.defined() ? q_out : nothing(k);
}

// New tokens change the cache in place: what autograd has kept of it is out of date then.
Tensor cache_append_autograd(const Tensor& k, const Tensor& v, Tensor keys, Tensor values,
                             Tensor key_scales, Tensor value_scales, const Tensor& table,
                             const Tensor& lengths, const Tensor& offsets,
                             const OptTensor& lengths_new, const OptTensor& q,
                             const OptTensor& positions, const OptTensor& frequencies,
                             bool interleaved, double amplitude) {
  static auto op = typed_op<Tensor(
      const Tensor&, const Tensor&, Tensor, Tensor, Tensor, Tensor, const Tensor&, const Tensor&,
      const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, bool,
      double)>("torch_point_ops_cache::append");
  bool any = followed(k) || followed(v) || (q && followed(*q)) ||
             (positions && followed(*positions)) || (frequencies && followed(*frequencies));
  for (const Tensor& t : {keys, values, key_scales, value_scales}) any = any || followed(t);
  TORCH_CHECK(!any, "cache_append has no derivative: call it under torch.no_grad()");
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(k, v, keys, values, key_scales, value_scales, table, lengths, offsets,
                  lengths_new, q, positions, frequencies, interleaved, amplitude);
  }
  for (const Tensor& t : {keys, values, key_scales, value_scales})
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
  return out;
}

Tensor cache_attention_hip(const Tensor& q_in, const Tensor& keys, const Tensor& values,
                           const Tensor& key_scales, const Tensor& value_scales,
                           const Tensor& table, const Tensor& lengths, const Tensor& offsets,
                           const OptTensor& lengths_q, bool causal, double scale) {
  const char* op = "cached_attention";
  check_hip(q_in, "q");
  TORCH_CHECK(q_in.dim() == 3, op, " expects q (T, Hq, D), but got ", q_in.sizes());
  c10::OptionalDeviceGuard guard(q_in.device());
  const int dt = nn_dtype(q_in, op);
  const PagedCache c = cache_of(q_in, keys, values, key_scales, value_scales, table, lengths, op);
  const int64_t T = q_in.size(0), Hq = q_in.size(1), D0 = q_in.size(2);
  TORCH_CHECK(c.Hk > 0 && Hq > 0 && Hq % c.Hk == 0, op, ": the ", Hq,
              " heads of q must be a multiple of the ", c.Hk, " heads of the cache");
  TORCH_CHECK(D0 > 0 && (D0 + 15) / 16 * 16 == c.Dr, op, ": heads of ", D0,
              " values need a cache of ", (D0 + 15) / 16 * 16, ", but got ", c.Dr);
  const NewRows r = new_rows(q_in, c, offsets, lengths_q, op);
  const int64_t per = 16 / q_in.element_size(), D = (D0 + per - 1) / per * per;
  const Tensor q = head_rows(q_in, D);
  Tensor out = at::empty({T, Hq, D}, q.options());
  const int64_t wsb =
      tpo_cache_attention_workspace_size(dt, c.B, T, Hq, c.Hk, D, c.page, c.M);
  const Tensor ws = workspace(wsb, q, op);
  check_rc(tpo_cache_attention(
               dt, q.data_ptr(), r.offsets.data_ptr<int64_t>(),
               (const int64_t*)data_or_null(r.lengths), c.B, T, Hq, D, row_stride(q),
               head_stride(q), keys.data_ptr(), values.data_ptr(), key_scales.data_ptr<float>(),
               value_scales.data_ptr<float>(), table.data_ptr<int32_t>(),
               lengths.data_ptr<int64_t>(), c.pages, c.Hk, c.page, c.Dr, c.M, causal, scale,
               out.data_ptr(), data_or_null(ws), wsb, stream_of(q)),
           op);
  return cut_heads(out, D0);
}

auto cache_attention_op() {
  static auto op =
      typed_op<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                      const Tensor&, const Tensor&, const Tensor&, const OptTensor&, bool, double)>(
          "torch_point_ops_cache::attention");
  return op;
}

Tensor cache_attention_autograd(const Tensor& q, const Tensor& keys, const Tensor& values,
                                const Tensor& key_scales, const Tensor& value_scales,
                                const Tensor& table, const Tensor& lengths, const Tensor& offsets,
                                const OptTensor& lengths_q, bool causal, double scale) {
  bool any = false;
  for (const Tensor& t : {q, keys, values, key_scales, value_scales}) any = any || followed(t);
  TORCH_CHECK(!any, "cached_attention has no derivative: call it under torch.no_grad()");
  at::AutoDispatchBelowADInplaceOrView below;
  return cache_attention_op().call(q, keys, values, key_scales, value_scales, table, lengths,
                                   offsets, lengths_q, causal, scale);
}

// Under autocast attention takes its type, as packed_attention does; the cache holds codes.
Tensor cache_attention_autocast(const Tensor& q, const Tensor& keys, const Tensor& values,
                                const Tensor& key_scales, const Tensor& value_scales,
                                const Tensor& table, const Tensor& lengths, const Tensor& offsets,
                                const OptTensor& lengths_q, bool causal, double scale) {
  c10::impl::ExcludeDispatchKeyGuard below(c10::DispatchKey::AutocastCUDA);
  return cache_attention_op().call(autocast(q), keys, values, key_scales, value_scales, table,
                                   lengths, offsets, lengths_q, causal, scale);
}

Tensor rotary_positions_cpu(const Tensor&, const Tensor&, const Tensor&, bool, double) {
  TORCH_CHECK(false, "rotary_positions is not implemented for CPU");
}
Tensor cache_append_cpu(const Tensor&, const Tensor&, Tensor, Tensor, Tensor, Tensor,
                        const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                        const OptTensor&, const OptTensor&, const OptTensor&, bool, double) {
  TORCH_CHECK(false, "cache_append is not implemented for CPU");
}
Tensor cache_attention_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                           const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                           const OptTensor&, bool, double) {
  TORCH_CHECK(false, "cached_attention is not implemented for CPU");
}

}  // namespace

TORCH_LIBRARY(torch_point_ops_rotary, m) {
  m.def("rotary_positions(Tensor x, Tensor positions, Tensor frequencies, bool interleaved, "
        "float amplitude) -> Tensor");
  m.def("rotary_positions_backward(Tensor grad, Tensor positions, Tensor frequencies, "
        "bool interleaved, float amplitude) -> Tensor");
}
TORCH_LIBRARY_IMPL(torch_point_ops_rotary, CPU, m) {
  m.impl("rotary_positions", &rotary_positions_cpu);
}
TORCH_LIBRARY_IMPL(torch_point_ops_rotary, CUDA, m) {
  m.impl("rotary_positions", &rotary_positions_hip);
  m.impl("rotary_positions_backward", &rotary_positions_backward_hip);
}
TORCH_LIBRARY_IMPL(torch_point_ops_rotary, Autograd, m) {
  m.impl("rotary_positions", &rotary_positions_autograd);
  m.impl("rotary_positions_backward", no_formula());
}

TORCH_LIBRARY(torch_point_ops_cache, m) {
  // q turned by its places, or nothing where none was given
  m.def("append(Tensor k, Tensor v, Tensor(a!) keys, Tensor(b!) values, Tensor(c!) key_scales, "
        "Tensor(d!) value_scales, Tensor table, Tensor lengths, Tensor offsets, "
        "Tensor? lengths_new, Tensor? q, Tensor? positions, Tensor? frequencies, "
        "bool interleaved, float amplitude) -> Tensor");
  m.def("attention(Tensor q, Tensor keys, Tensor values, Tensor key_scales, "
        "Tensor value_scales, Tensor table, Tensor lengths, Tensor offsets, Tensor? lengths_q, "
        "bool causal, float scale) -> Tensor");
}
TORCH_LIBRARY_IMPL(torch_point_ops_cache, CPU, m) {
  m.impl("append", &cache_append_cpu);
  m.impl("attention", &cache_attention_cpu);
}
TORCH_LIBRARY_IMPL(torch_point_ops_cache, CUDA, m) {
  m.impl("append", &cache_append_hip);
  m.impl("attention", &cache_attention_hip);
}
TORCH_LIBRARY_IMPL(torch_point_ops_cache, AutocastCUDA, m) {
  m.impl("attention", &cache_attention_autocast);
}
TORCH_LIBRARY_IMPL(torch_point_ops_cache, Autograd, m) {
  m.impl("append", &cache_append_autograd);
  m.impl("attention", &cache_attention_autograd);
}

}  // namespace torch_point_ops
