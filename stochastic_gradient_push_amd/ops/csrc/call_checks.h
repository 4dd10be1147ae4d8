// What a kernel called past PyTorch's dispatcher cannot serve, refused.

#pragma once

#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>

// Wrapper, fake and functional tensors say that they are on the device but
// have no memory there: their address is null.
inline void check_memory(const char* op, const at::Tensor& t) {
  TORCH_CHECK(t.numel() == 0 || t.const_data_ptr() != nullptr, op,
              ": a tensor has no memory of its own (a wrapper, fake or "
              "functional tensor)");
}

// The kernels compute values only.  A dual tensor's tangent would be gone
// without a word: it does not show in requires_grad.
inline void check_tangent(const char* op, const at::Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), op,
              ": no forward-mode derivative on the device; detach() drops "
              "the tangent");
}

// A tracer records what goes through the dispatcher: the allocation of the
// result, but not the kernel that fills it.
inline void check_untraced(const char* op) {
  TORCH_CHECK(!torch::jit::tracer::isTracing()
              && !c10::impl::TorchDispatchModeTLS::get_mode(
                      c10::impl::TorchDispatchModeKey::PROXY).has_value(),
              op, " cannot be traced on the device: the trace would have its "
              "result's allocation without the kernel");
}
