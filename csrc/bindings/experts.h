// Python bindings of the expert-parallel operators and 8-bit products
// (device pointers; gloo_amd/experts.py checks tensors and calls them).
#pragma once

#include <pybind11/pybind11.h>

namespace glooamd {

void bindExperts(pybind11::module_& m);

} // namespace glooamd
