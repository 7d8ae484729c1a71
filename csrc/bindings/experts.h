// Python bindings of the expert-parallel operators' and 8-bit products'
// launches, by device pointers, for callers without torch (gloo_amd/experts.py
// goes through csrc/torch/operators.cc), and the launches as one pointer.
#pragma once

#include <pybind11/pybind11.h>

namespace glooamd {

void bindExperts(pybind11::module_& m);

} // namespace glooamd
