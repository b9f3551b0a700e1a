// torch_util.h -- what the torch operators' checks and launches share.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <utility>

#include "kda_abi.h"

namespace {

using NamedTensor = std::pair<const char *, const at::Tensor &>;

inline void check_same_device(const at::Tensor &x, const char *name, const at::Tensor &t, const char *x_name = "q") {
    TORCH_CHECK(t.device() == x.device(), name, " must be on the same device as ", x_name);
}

inline void check_ok(int status, const char *op) {
    TORCH_CHECK(status == KDA_OK, op, ": ", kda_status_string(status), " (status ", status, ")");
}

inline void *stream_of(const at::Tensor &t) {
    return static_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// The kernels run on a HIP device only; a host tensor is an error, never a
// fallback. Checked after the shape/layout rules so those are testable on a
// machine without a GPU.
inline void check_on_gpu(const char *name, const at::Tensor &t) {
    TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA (HIP) tensor");
}

}  // namespace
