// What the files of the native torch binding share.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

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

inline void on_gpu(const char *what, const at::Tensor &t) {
    TORCH_CHECK(t.is_cuda() || t.is_meta(), what, ": tensors must be on the GPU; this build has no CPU path");
}
inline void *stream_now() { return c10::hip::getCurrentHIPStream().stream(); }
// A tangent of forward mode.  A tensor can have one without requires_grad and in every grad mode: calls that
// make no node look for it themselves.
inline bool has_tangent(const at::Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }
// Codes are rounded: the operators of a cache have no gradient, and a caller that would get none is told so.
inline void no_gradient(const char *what, std::initializer_list<const at::Tensor *> inputs) {
    const bool mode = at::GradMode::is_enabled();
    for (const at::Tensor *t : inputs)
        TORCH_CHECK(!(mode && t->requires_grad()) && !has_tangent(*t), what,
                    ": a cache of 8 bits has no gradient; call it under torch.no_grad() or on detached tensors, which "
                    "have no tangent");
}
inline int cache_code(const at::Tensor &t) {
    return t.scalar_type() == at::kChar ? ENATTEN_I8 : t.scalar_type() == at::kFloat8_e4m3fn ? ENATTEN_E4M3 : -1;
}

inline void check_rc(int rc) {
    if (rc == ENATTEN_OK) return;
    const char *msg = enatten_last_error();
    TORCH_CHECK_VALUE(rc != ENATTEN_EINVAL, msg);
    TORCH_CHECK(false, msg);
}

}  // namespace
