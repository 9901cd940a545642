// The `_host` extension module: the layer operators' host side in native code.
//
// A call of these operators is a few microseconds of device work for small
// inputs, and a training step makes hundreds of them, each with a backward on
// autograd's own thread.  Checks, allocation and the autograd node are native
// here, so that the interpreter is entered once a call and never in a backward.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "host_adamw.h"
#include "host_common.h"

namespace {

namespace py = pybind11;
using rfm_host::MaybeTensor;
using rfm_host::TensorRefs;

// A Python list or tuple of tensors without taking references of its own; the
// caller keeps the interpreter's lock while it uses them.
TensorRefs refs(const py::handle& list, const char* name) {
  const bool is_list = PyList_Check(list.ptr());
  if (!is_list && !PyTuple_Check(list.ptr())) {
    throw py::value_error(std::string(name) + " must be a list or a tuple of tensors");
  }
  const Py_ssize_t n = is_list ? PyList_GET_SIZE(list.ptr()) : PyTuple_GET_SIZE(list.ptr());
  TensorRefs out(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = is_list ? PyList_GET_ITEM(list.ptr(), i) : PyTuple_GET_ITEM(list.ptr(), i);
    if (!THPVariable_Check(item)) throw py::value_error(std::string(name) + " must hold tensors");
    out[static_cast<size_t>(i)] = &THPVariable_Unpack(item);
  }
  return out;
}

std::optional<TensorRefs> maybe_refs(const py::handle& list, const char* name) {
  return list.is_none() ? std::optional<TensorRefs>() : refs(list, name);
}

void adamw_step(const py::handle& params, const py::handle& grads, const py::handle& exp_avg,
                const py::handle& exp_avg_sq, const py::handle& exp_avg_scale, const py::handle& exp_avg_sq_scale,
                int64_t step, const MaybeTensor& device_step, double lr, const MaybeTensor& device_lr, double beta1,
                double beta2, double eps, double weight_decay, const MaybeTensor& grad_scale) {
  rfm_host::adamw_step(refs(params, "params"), refs(grads, "grads"), refs(exp_avg, "exp_avg"),
                       refs(exp_avg_sq, "exp_avg_sq"), maybe_refs(exp_avg_scale, "scales"),
                       maybe_refs(exp_avg_sq_scale, "scales"), step, device_step, lr, device_lr, beta1, beta2, eps,
                       weight_decay, grad_scale);
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  const auto release = py::call_guard<py::gil_scoped_release>();
  m.def("layer_norm", &rfm_host::layer_norm, release);
  m.def("linear", &rfm_host::linear, release);
  m.def("adamw_step", &adamw_step);
  m.def("dequantize_moments", &rfm_host::dequantize_moments, release);
  m.def("intercepted", &rfm_host::intercepted);
}
