// What the native host paths share: the C ABI's errors, element types, and tensors that they leave to general code.
#pragma once

#include <ATen/TensorSubclassLikeUtils.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "sa2.h"

namespace sa2_host {

using at::Tensor;

extern decltype(&sa2_strerror) err_fn;         // set by bind()

// A negative status of the C ABI; becomes simplical_attn_amd._lib.Sa2Error in Python
struct Status : std::runtime_error {
    int code;
    explicit Status(int c) : std::runtime_error("sa2 error " + std::to_string(c) + ": " + err_fn(c)), code(c) {}
};
inline void check(int rc) {
    if (rc != 0) throw Status(rc);
}

inline int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SA2_F32;
        case at::kBFloat16: return SA2_BF16;
        case at::kHalf: return SA2_F16;
        default: return -1;
    }
}

// no forward-mode tangent, no wrapper of a torch.func transform, no active dispatch mode
inline bool plain(const Tensor& t) { return !t._fw_grad(0).defined() && !at::isTensorSubclassLike(t); }

void define_layers(py::module_& m);            // sa2_torch_layers.cpp

}  // namespace sa2_host
