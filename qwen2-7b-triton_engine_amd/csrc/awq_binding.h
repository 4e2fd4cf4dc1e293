// What the parts of the torch binding share (host code).
#pragma once

#include <torch/extension.h>

namespace awq_binding {

// AwqNativeError (kernels/_native.py) for a nonzero status of the C ABI.
void check_status(int st, const char* where);
// `t` when its data starts on a 16-byte boundary, else a copy (the kernels use
// 16-byte vector accesses; the reference's Triton path takes any view).
at::Tensor aligned16(const at::Tensor& t);
// The serving operators (awq_serving_binding.cpp).
void define_serving(py::module_& m);

}  // namespace awq_binding
