// Shared by the sources of the compiled call path (_entry*.cpp).
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "qrb200.h"

namespace qrb_entry {

inline void check_status(int status) {
  if (status != QRB_OK) {
    char buf[512];
    qrb_last_error(buf, sizeof buf);
    TORCH_CHECK(false, "libqrb200 error ", status, ": ", buf);
  }
}

// Tells autograd that a caller's tensor was written, so that a backward pass that kept it raises, as after
// torch's own in-place operations.  (A tensor of inference mode has no version to raise.)
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void bind_delta(pybind11::module_& m);
void bind_linear(pybind11::module_& m);

}  // namespace qrb_entry
