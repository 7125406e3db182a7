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

void bind_delta(pybind11::module_& m);
void bind_linear(pybind11::module_& m);

}  // namespace qrb_entry
