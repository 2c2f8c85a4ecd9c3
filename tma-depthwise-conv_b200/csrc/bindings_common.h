// bindings_common.h — helpers that the extension's source files share.
#pragma once

#include <torch/extension.h>

namespace tma_dwconv {

// Raises RuntimeError with the status code's text unless rc is TDC_OK.
void check_status(int rc, const char* what);

// torch's current stream of x's device, as the C ABI takes it.
void* stream_of(const torch::Tensor& x);

// Adds the sequence operators to the module (bindings_sequence.cpp).
void bind_sequence(pybind11::module_& m);

}  // namespace tma_dwconv
