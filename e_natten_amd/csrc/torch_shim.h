// What the files of the native torch binding share.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <functional>
#include <utility>

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

// Whether two tensors of the same shape share an element.  Exact where both are dense, and where they have the
// same strides and these are nested (each longer than all that lies within it), as views of one pool have: the
// distance of the addresses is then a whole number of each stride, with two choices at most.  Other views whose
// ranges cross are let pass.
using Axis = std::pair<int64_t, int64_t>;  // stride, size
inline bool is_distance(int64_t distance, const Axis *axes, int n) {  // longest stride first
    if (n == 0) return distance == 0;
    int64_t inner = 0;
    for (int i = 1; i < n; i++) inner += axes[i].first * (axes[i].second - 1);
    const auto [stride, size] = axes[0];
    if (stride <= inner) return false;
    for (int64_t k = distance / stride - 1; k <= distance / stride + 1; k++)
        if (std::abs(k) < size && std::abs(distance - k * stride) <= inner &&
            is_distance(distance - k * stride, axes + 1, n - 1))
            return true;
    return false;
}
inline bool share_memory(const at::Tensor &a, const at::Tensor &b) {
    const int64_t size = a.element_size();
    const auto extent = [&](const at::Tensor &t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); i++) last += t.stride(i) * (t.size(i) - 1);
        return (last + 1) * size;
    };
    const int64_t distance = static_cast<const char *>(b.data_ptr()) - static_cast<const char *>(a.data_ptr());
    if (distance >= extent(a) || -distance >= extent(b)) return false;
    if (a.is_non_overlapping_and_dense() && b.is_non_overlapping_and_dense()) return true;
    Axis axes[5];
    int n = 0;
    for (int64_t i = 0; i < a.dim(); i++) {
        if (a.size(i) == 1) continue;
        if (a.stride(i) != b.stride(i)) return false;
        axes[n++] = {a.stride(i), a.size(i)};
    }
    std::sort(axes, axes + n, std::greater<Axis>());
    return distance % size == 0 && is_distance(distance / size, axes, n);
}

inline void check_rc(int rc) {
    if (rc == ENATTEN_OK) return;
    const char *msg = enatten_last_error();
    TORCH_CHECK_VALUE(rc != ENATTEN_EINVAL, msg);
    TORCH_CHECK(false, msg);
}

}  // namespace
