// What the files of the native torch binding share.
#pragma once

#include <ATen/ATen.h>

#include "enatten.h"

namespace {

inline int dtype_code(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return ENATTEN_F32;
        case at::kBFloat16: return ENATTEN_BF16;
        case at::kHalf: return ENATTEN_F16;
        case at::kDouble: return ENATTEN_F64;
        default: return -1;
    }
}

// The kernels take any strides on the leading axes but need unit stride on the
// channel axis.
inline at::Tensor kernel_layout(const at::Tensor &t) {
    return (t.stride(-1) != 1 && t.size(-1) != 1) ? t.contiguous() : t;
}

inline void check_rc(int rc) {
    if (rc == ENATTEN_OK) return;
    const char *msg = enatten_last_error();
    TORCH_CHECK_VALUE(rc != ENATTEN_EINVAL, msg);
    TORCH_CHECK(false, msg);
}

}  // namespace
