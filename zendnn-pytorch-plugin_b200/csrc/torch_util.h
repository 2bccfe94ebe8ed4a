// What the translation units of the PyTorch boundary share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>

#include <optional>

#include "../../include/zentorch_b200.h"

namespace zentorch_b200 {

namespace {

#define ZT_TORCH_CALL(expr)                                         \
  do {                                                              \
    const int rc__ = (expr);                                        \
    TORCH_CHECK(rc__ == ZT_SUCCESS, zt_last_error());               \
  } while (0)

// Every tensor argument must live on the input's GPU: the kernels take raw pointers, and a host pointer or
// another device's pointer would fault on the GPU instead of raising here.
[[maybe_unused]] void check_on_device(const at::Tensor &t, const at::Tensor &input, const char *op, const char *name) {
  TORCH_CHECK(t.is_cuda() && t.device() == input.device(), op, ": ", name, " must be on the input's device (",
              input.device(), "), got ", t.device());
}
[[maybe_unused]] void check_on_device(const std::optional<at::Tensor> &t, const at::Tensor &input, const char *op, const char *name) {
  if (t.has_value() && t->defined()) check_on_device(*t, input, op, name);
}

}  // namespace

}  // namespace zentorch_b200
