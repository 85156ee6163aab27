// Checks that the torch extension's entry points share.
#pragma once

#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>

namespace ltc_torch {

// The entry points fill their outputs through raw pointers, where neither
// forward-mode differentiation nor a tracer looks: the one would take the tangent
// for zero, the other would record the outputs' allocation alone, and both without
// a word. So both are errors.
inline void check_tangent(const char* name, const torch::Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
                              " has no forward-mode derivative");
}

template <class... Tensors>
void check_modes(const char* name, const Tensors&... inputs) {
  (check_tangent(name, inputs), ...);
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() &&
          !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
      name, " cannot be traced");
}

}  // namespace ltc_torch
