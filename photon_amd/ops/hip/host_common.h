// Host-side helpers shared by the .hip translation units.
#pragma once

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "common.h"

namespace photon_hip {

inline hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStream().stream();
}

// Before the kernels that write `t` in place: counting up its version, which
// they have to do, fails where this is not so.
inline void check_writable(const torch::Tensor& t, const char* name,
                           const char* what) {
  TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), name,
              ": ", what, " was made in inference mode and cannot be written "
              "outside of it");
}

// A kernel does not carry forward-mode tangents: without this they would be
// dropped in silence.
inline void check_no_tangent(const torch::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), name,
                              ": forward-mode derivatives are not supported");
}

#define DISPATCH_DTYPE(TENSOR, NAME, ...)                              \
  if ((TENSOR).scalar_type() == at::kBFloat16) {                       \
    using scalar_t = unsigned short;                                   \
    __VA_ARGS__;                                                       \
  } else if ((TENSOR).scalar_type() == at::kFloat) {                   \
    using scalar_t = float;                                            \
    __VA_ARGS__;                                                       \
  } else {                                                             \
    TORCH_CHECK(false, NAME ": unsupported dtype ", (TENSOR).dtype()); \
  }

}  // namespace photon_hip
