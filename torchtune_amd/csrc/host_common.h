// What the translation units of the host extension share: error codes to exceptions, checks, scratch memory.
#pragma once
#include <ATen/ATen.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/torchtune_amd.h"

namespace ttamd_host {

using at::Tensor;

inline void check(int rc, const char* what) {
  if (rc == TTAMD_OK) return;
  if (rc == TTAMD_EINVAL) TORCH_CHECK_VALUE(false, what, ": ", ttamd_last_error());
  TORCH_CHECK(false, what, " failed (code ", rc, "): ", ttamd_last_error());
}

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

inline void need_gpu(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, ": expected a tensor on an AMD GPU (device 'cuda'), got device '", t.device().str(),
              "'. torchtune_amd computes only through its HIP kernels.");
}

// a contiguous bf16 tensor on the GPU
inline Tensor bf16(const Tensor& t, const char* what) {
  need_gpu(t, what);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, what, ": expected a bfloat16 tensor, got ", t.scalar_type());
  return t.contiguous();
}

inline Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)(bytes > 16 ? bytes : 16)}, like.options().dtype(at::kByte));
}

inline size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// The gradient of a bias: the sum over the rows of gy [M, N], contiguous bf16 on the current device.  (torch's own sum clears
// counters by a memset where it cuts the rows, and a recorded one has given wrong sums on replays after the first.)
inline Tensor column_sum(const Tensor& gy) {
  const int64_t M = gy.size(0), N = gy.size(1);
  Tensor out = at::empty({N}, gy.options());
  const size_t bytes = ttamd_column_sum_workspace_bytes(M, N);
  const Tensor ws = bytes ? scratch(bytes, gy) : Tensor();
  check(ttamd_column_sum_bf16(gy.data_ptr(), out.data_ptr(), M, N, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(gy)), "column_sum");
  return out;
}

// The same for the nodes whose bias gradients are torch's sum to the bit: the own sum where the call is being recorded.
inline Tensor bias_gradient(const Tensor& gy) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return gy.sum(0);
  const Tensor c = gy.contiguous();
  return column_sum((reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone());
}

// True when the call has to be a node: something is differentiated backward, or carries a forward-mode tangent (the node
// then raises: none of them has a forward-mode rule, and a plain call would drop the tangent).
inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  const bool grad = at::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if (t->defined() && ((grad && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

}  // namespace ttamd_host
