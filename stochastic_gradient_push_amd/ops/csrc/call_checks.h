// What a kernel called past PyTorch's dispatcher cannot serve, refused.

#pragma once

#include <initializer_list>

#include <torch/extension.h>

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
