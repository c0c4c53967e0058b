// shim_common.hpp -- what the operator registrations share: type codes, the
// current stream, error texts, the question whether autograd follows a call.
#pragma once

#include <torch/all.h>
#include <torch/library.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>

#include <tuple>

#include "tpo.h"

namespace torch_point_ops {
namespace {

[[maybe_unused]] int dtype_code(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat: return TPO_F32;
    case at::kDouble: return TPO_F64;
    case at::kHalf: return TPO_F16;
    default:
      TORCH_CHECK(false, op, " not implemented for '", t.scalar_type(), "'");
  }
  return -1;
}

// A tensor whose data starts on a 16-byte boundary (a copy if it does not).
[[maybe_unused]] at::Tensor aligned16(const at::Tensor& t) {
  return ((uintptr_t)t.data_ptr() & 15) ? t.clone(at::MemoryFormat::Contiguous) : t;
}

[[maybe_unused]] void* stream_of(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

[[maybe_unused]] void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == TPO_OK, op, " failed: ", tpo_last_error());
}

[[maybe_unused]] void check_hip(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
}

// Whether autograd has to follow the call.  Without it the operator runs as it
// is, also under transforms that a C++ autograd function refuses.  A tangent
// counts as well: forward mode has no formula here, and the function says so where
// the operator alone would return a result without one.
[[maybe_unused]] bool followed(const at::Tensor& a) {
  return (at::GradMode::is_enabled() && a.requires_grad()) ||
         (c10::AutogradState::get_tls_state().get_fw_grad_mode() && a._fw_grad(0).defined());
}

template <typename Op>
auto typed_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Op>();
}

}  // namespace
}  // namespace torch_point_ops
