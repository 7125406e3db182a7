// Shared by the sources of the compiled call path (_entry*.cpp).
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <type_traits>

#include "qrb200.h"

namespace qrb_entry {

inline void check_status(int status) {
  if (status != QRB_OK) {
    char buf[512];
    qrb_last_error(buf, sizeof buf);
    TORCH_CHECK(false, "libqrb200 error ", status, ": ", buf);
  }
}

// These calls have no forward-mode derivative: a result without a tangent would read as one of zero.
template <typename... T>
void check_no_tangent(const char* call, const T&... tensors) {
  auto has = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, at::Tensor>) return t._fw_grad(0).defined();
    else return t.has_value() && t->_fw_grad(0).defined();
  };
  if ((has(tensors) || ...)) TORCH_CHECK_NOT_IMPLEMENTED(false, call, " has no forward-mode derivative");
}

// Whether autograd would record a function of these tensors.
template <typename... T>
bool wants_grad(const T&... tensors) {
  auto one = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, at::Tensor>) return t.requires_grad();
    else return t.has_value() && t->requires_grad();
  };
  return at::GradMode::is_enabled() && (one(tensors) || ...);
}

// Tells autograd that a caller's tensor was written, so that a backward pass that kept it raises, as after
// torch's own in-place operations.  (A tensor of inference mode has no version to raise.)
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void bind_delta(pybind11::module_& m);
void bind_linear(pybind11::module_& m);

}  // namespace qrb_entry
