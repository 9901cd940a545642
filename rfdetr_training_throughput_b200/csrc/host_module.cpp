// The `_host` extension module: the layer operators' host side in native code.
//
// A call of these operators is a few microseconds of device work for small
// inputs, and a training step makes hundreds of them, each with a backward on
// autograd's own thread.  Checks, allocation and the autograd node are native
// here, so that the interpreter is entered once a call and never in a backward.
#include <torch/csrc/utils/pybind.h>

#include "host_adamw.h"
#include "host_common.h"

PYBIND11_MODULE(_host, m) {
  namespace py = pybind11;
  const auto release = py::call_guard<py::gil_scoped_release>();
  m.def("layer_norm", &rfm_host::layer_norm, release);
  m.def("linear", &rfm_host::linear, release);
  m.def("adamw_step", &rfm_host::adamw_step, release);
  m.def("dequantize_moments", &rfm_host::dequantize_moments, release);
}
