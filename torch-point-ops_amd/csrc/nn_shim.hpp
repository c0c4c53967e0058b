// nn_shim.hpp -- what the registrations of the transformer operators share: types, workspaces,
// rows of heads, what autocast and autograd ask for.
#pragma once

#include "shim_common.hpp"

#include <ATen/autocast_mode.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>

namespace torch_point_ops {
namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

[[maybe_unused]] int nn_dtype(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat: return TPO_F32;
    case at::kHalf: return TPO_F16;
    case at::kBFloat16: return TPO_BF16;
    default:
      TORCH_CHECK(false, op, " not implemented for '", t.scalar_type(), "'");
  }
  return -1;
}

[[maybe_unused]] Tensor workspace(int64_t bytes, const Tensor& like, const char* op) {
  TORCH_CHECK(bytes >= 0, op, ": ", tpo_last_error());
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
[[maybe_unused]] void* data_or_null(const Tensor& t) {
  return t.defined() ? t.data_ptr() : nullptr;
}
[[maybe_unused]] Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
[[maybe_unused]] OptTensor opt(const Tensor& t) {
  return t.defined() ? OptTensor(t) : std::nullopt;
}
// the place of a result that was not asked for
[[maybe_unused]] Tensor nothing(const Tensor& like) { return at::empty({0}, like.options()); }

// The distance of rows and of heads, also where there is one of them only.
[[maybe_unused]] int64_t row_stride(const Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}
[[maybe_unused]] int64_t head_stride(const Tensor& t) {
  return t.size(1) > 1 ? t.stride(1) : t.size(2);
}

// q, k and v may be slices (of one projection, say) or broadcast over heads: a
// head's values lie together, rows and heads at any distance that keeps 16-byte
// loads.  Others are copied, heads that are no multiple of 16 bytes padded.
[[maybe_unused]] Tensor head_rows(const Tensor& t, int64_t D) {
  const int64_t z = t.element_size();
  if (t.size(2) != D) return at::constant_pad_nd(t, {0, D - t.size(2)}).contiguous();
  const bool ok = (D == 1 || t.stride(2) == 1) && row_stride(t) > 0 &&
                  row_stride(t) * z % 16 == 0 && row_stride(t) * z < (1 << 25) &&
                  head_stride(t) * z % 16 == 0;
  return aligned16(ok ? t : t.contiguous());
}

// The first D values of each head of a result.
[[maybe_unused]] Tensor cut_heads(const Tensor& t, int64_t D) {
  return t.size(2) == D ? t : t.narrow(2, 0, D).contiguous();
}

// An input in autocast's type, as torch's own products take theirs.
[[maybe_unused]] Tensor autocast(const Tensor& t) {
  return at::autocast::cached_cast(at::autocast::get_autocast_dtype(at::kCUDA), t, at::kCUDA);
}
// The operators that autograd functions call have no formula of their own: a
// gradient of a gradient, or a tangent, is refused instead of left out.
[[maybe_unused]] torch::CppFunction no_formula() {
  return torch::autograd::autogradNotImplementedFallback();
}

}  // namespace
}  // namespace torch_point_ops
