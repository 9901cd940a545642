// Shared by the native host side of the layer operators (the `_host` module):
// argument checks that raise ValueError, type codes, the launch's device and
// stream.
#pragma once

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <initializer_list>
#include <string>

#include "rfm.h"

namespace rfm_host {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

#define RFM_REQUIRE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RFM_DTYPE_F32;
    case at::kBFloat16: return RFM_DTYPE_BF16;
    case at::kHalf: return RFM_DTYPE_F16;
    default: return -1;
  }
}

// The C ABI's return code as a RuntimeError that names the call.
inline void check_call(const char* func, int code) {
  TORCH_CHECK(code == RFM_OK, func, " failed: ", rfm_error_string(code), " (code ", code, ")");
}

inline void* current_stream(const at::Device& device) {
  return c10::cuda::getCurrentCUDAStream(device.index()).stream();
}

inline void* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline Tensor or_undefined(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

inline MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

inline bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Whether this thread's operators are being recorded, or run without data.  A
// recorder sees what goes through torch's dispatcher, and of the calls here that
// is the output's allocation alone: what it records would return memory that
// nobody wrote.
inline bool traced() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  return at::tracer::impl::is_dispatch_enabled() || Modes::get_mode(Key::PROXY).has_value() ||
         Modes::get_mode(Key::FAKE).has_value() || Modes::get_mode(Key::FUNCTIONAL).has_value();
}

// The same, or a function transform (torch.func's) that may have wrapped the
// tensors of a call: what a patched module asks before it leaves torch's path.
inline bool intercepted() {
  return traced() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

inline void refuse_traced(const char* op) {
  TORCH_CHECK(!traced(), op, " cannot be traced: its kernels are launched past torch's dispatcher");
}

// Forward-mode derivatives: an output made here has no tangent, which would read
// as one of zero.
inline void refuse_tangents(const char* op, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) {
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
  }
}

// `x` as [rows, last] with a unit stride along the rows' elements and rows that
// do not overlap: a view where the layout allows, else a copy.
inline Tensor rows_of(const Tensor& x) {
  const int64_t last = x.size(-1);
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
  Tensor y = x.dim() == 2 ? x : x.reshape({rows, last});
  if (y.numel() > 0 && ((last > 1 && y.stride(1) != 1) || (rows > 1 && y.stride(0) < last))) y = y.contiguous();
  return y;
}

// Elements between the rows of a rows_of result (any value does for one row).
inline int64_t row_stride(const Tensor& y) { return y.size(0) > 1 ? y.stride(0) : y.size(1); }

// Gradients as a backward returns them: where a graph of the backward itself is
// being recorded, a second derivative raises instead of reading as zero.
inline variable_list once(variable_list grads, const char* op) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list inputs;
  for (const Tensor& g : grads)
    if (g.defined()) inputs.push_back(g.detach().set_requires_grad(true));
  if (inputs.empty()) return grads;
  auto raise = std::make_shared<torch::autograd::DelayedError>(
      std::string(op) + " is differentiable once: its gradient has no derivative", static_cast<int64_t>(inputs.size()));
  variable_list out = (*raise)(std::move(inputs));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps);
Tensor linear(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, int64_t activation,
              const MaybeTensor& residual);

}  // namespace rfm_host
