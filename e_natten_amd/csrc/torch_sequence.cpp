// Native torch binding of the operators of growing sequences: enatten::rotary (differentiable, any
// number of times), enatten::cache_append and enatten::cache_attention.  Host code only; the checks and
// error classes are those of the Python host side (sequence.py).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <functional>
#include <utility>

#include "torch_shim.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void on_gpu(const char *what, const Tensor &t) {
    TORCH_CHECK(t.is_cuda() || t.is_meta(), what, ": tensors must be on the GPU; this build has no CPU path");
}
void *stream_now() { return c10::hip::getCurrentHIPStream().stream(); }
// A tangent of forward mode.  A tensor can have one without requires_grad and in every grad mode: calls that
// make no node look for it themselves.
bool has_tangent(const Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }

// ---- rotary ----------------------------------------------------------------

void validate_rotary(const Tensor &q, const optional<Tensor> &k, const Tensor &positions, const Tensor &frequencies) {
    const char *what = "rotary";
    TORCH_CHECK_VALUE(q.dim() == 4, what, ": expected [B, heads, T, head_dim] tensors, got ", q.dim(), "-D q");
    TORCH_CHECK_VALUE(dtype_code(q) >= 0, what, ": dtype ", q.scalar_type(),
                      " is not supported (float32, bfloat16, float16, float64)");
    TORCH_CHECK_VALUE(q.numel() > 0, what, ": empty tensors are not supported");
    if (k.has_value()) {
        TORCH_CHECK_VALUE(k->dim() == 4 && k->size(0) == q.size(0) && k->size(2) == q.size(2) &&
                              k->size(3) == q.size(3) && k->size(1) > 0,
                          what, ": q and k must differ in their heads only, got ", q.sizes(), ", ", k->sizes());
        TORCH_CHECK_VALUE(k->scalar_type() == q.scalar_type(), what, ": q and k must share a dtype");
        TORCH_CHECK_VALUE(k->device() == q.device(), what, ": q and k must be on the same device");
    }
    TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, what,
                      ": positions must be int32 or int64, got ", positions.scalar_type());
    TORCH_CHECK_VALUE((positions.dim() == 1 || (positions.dim() == 2 && (positions.size(0) == q.size(0) || positions.size(0) == 1))) &&
                          positions.size(-1) == q.size(2),
                      what, ": positions must have shape [T] or [B, T], got ", positions.sizes());
    TORCH_CHECK_VALUE(frequencies.scalar_type() == at::kFloat || frequencies.scalar_type() == at::kDouble, what,
                      ": frequencies must be float32 or float64, got ", frequencies.scalar_type());
    TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.size(0) > 0 && 2 * frequencies.size(0) <= q.size(3), what,
                      ": frequencies must be one for every rotated pair, at most head_dim / 2, got ", frequencies.sizes());
    TORCH_CHECK_VALUE(q.size(0) <= 0x7fffffff && q.size(1) <= (1 << 20) && q.size(2) <= 0x7fffffff &&
                          (!k.has_value() || k->size(1) <= (1 << 20)),
                      what, ": tensor too large");
    TORCH_CHECK_VALUE(q.size(3) <= 1024, what, ": head_dim ", q.size(3), " exceeds the supported maximum of 1024");
    TORCH_CHECK(!at::GradMode::is_enabled() || !frequencies.requires_grad(), what,
                ": frequencies have no gradient; call it on detached ones");
    TORCH_CHECK_VALUE(positions.device() == q.device() && frequencies.device() == q.device(), what,
                      ": positions and frequencies must be on the device of q");
    on_gpu(what, q);
}

// like the attention operators' output, in the memory order of the input
Tensor empty_rows(const Tensor &x) { return kernel_layout(at::empty_like(x)); }

std::vector<Tensor> rotary_turn(const Tensor &q_, const optional<Tensor> &k_, const Tensor &positions_,
                                const Tensor &frequencies_, bool interleaved, double scale, bool inverse) {
    validate_rotary(q_, k_, positions_, frequencies_);
    const bool two = k_.has_value();
    std::vector<Tensor> out;
    if (q_.is_meta()) {
        out.push_back(empty_rows(kernel_layout(q_)));
        if (two) out.push_back(empty_rows(kernel_layout(*k_)));
        return out;
    }
    const c10::DeviceGuard guard(q_.device());
    const Tensor q = kernel_layout(q_), k = two ? kernel_layout(*k_) : Tensor();
    const Tensor positions = positions_.stride(-1) == 1 || positions_.size(-1) == 1 ? positions_ : positions_.contiguous();
    const Tensor frequencies = frequencies_.contiguous();
    out.push_back(empty_rows(q));
    if (two) out.push_back(empty_rows(k));
    check_rc(enatten_rotary(
        q.data_ptr(), two ? k.data_ptr() : nullptr, out[0].data_ptr(), two ? out[1].data_ptr() : nullptr,
        positions.data_ptr(), frequencies.data_ptr(), q.size(0), q.size(1), two ? k.size(1) : 0, q.size(2), q.size(3),
        2 * frequencies.size(0), dtype_code(q), positions.scalar_type() == at::kInt ? ENATTEN_I32 : ENATTEN_I64,
        frequencies.scalar_type() == at::kFloat ? ENATTEN_F32 : ENATTEN_F64, interleaved, inverse, q.strides().data(),
        two ? k.strides().data() : nullptr, out[0].strides().data(), two ? out[1].strides().data() : nullptr,
        positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0, scale, stream_now()));
    return out;
}

using RotarySig = std::vector<Tensor>(const Tensor &, const optional<Tensor> &, const Tensor &, const Tensor &, bool,
                                      double, bool);
// (through the dispatcher: tracers see one operator)
std::vector<Tensor> call_turn(const Tensor &q, const optional<Tensor> &k, const Tensor &positions,
                              const Tensor &frequencies, bool interleaved, double scale, bool inverse) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("enatten::rotary_turn", "").typed<RotarySig>();
    return op.call(q, k, positions, frequencies, interleaved, scale, inverse);
}
std::vector<Tensor> call_rotary(const Tensor &q, const optional<Tensor> &k, const Tensor &positions,
                                const Tensor &frequencies, bool interleaved, double scale, bool inverse) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("enatten::rotary", "").typed<RotarySig>();
    return op.call(q, k, positions, frequencies, interleaved, scale, inverse);
}

// The gradient is the turn the other way round of the upstream gradients: the same operator, so that it
// can be differentiated again.
struct RotaryFn : public torch::autograd::Function<RotaryFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const optional<Tensor> &k,
                                 const Tensor &positions, const Tensor &frequencies, bool interleaved, double scale,
                                 bool inverse) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        return call_turn(q, k, positions, frequencies, interleaved, scale, inverse);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
        const double scale = ctx->saved_data["scale"].toDouble();
        const bool two = grads.size() > 1 && grads[1].defined();
        Tensor dq, dk;
        if (grads[0].defined() || two) {
            const Tensor &first = grads[0].defined() ? grads[0] : grads[1];
            const optional<Tensor> second = grads[0].defined() && two ? optional<Tensor>(grads[1]) : c10::nullopt;
            const auto out = call_rotary(first, second, s[0], s[1], interleaved, scale, !inverse);
            (grads[0].defined() ? dq : dk) = out[0];
            if (second.has_value()) dk = out[1];
        }
        return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
std::vector<Tensor> rotary_autograd(const Tensor &q, const optional<Tensor> &k, const Tensor &positions,
                                    const Tensor &frequencies, bool interleaved, double scale, bool inverse) {
    TORCH_CHECK(!has_tangent(q) && !(k.has_value() && has_tangent(*k)) && !has_tangent(frequencies),
                "rotary: there is no forward-mode derivative; gradients come by the backward pass");
    if (!at::GradMode::is_enabled() || !(q.requires_grad() || (k.has_value() && k->requires_grad()))) {
        at::AutoDispatchBelowADInplaceOrView below;  // (no node: inference)
        return call_turn(q, k, positions, frequencies, interleaved, scale, inverse);
    }
    validate_rotary(q, k, positions, frequencies);
    return RotaryFn::apply(q, k, positions, frequencies, interleaved, scale, inverse);
}
std::vector<Tensor> rotary_plain(const Tensor &q, const optional<Tensor> &k, const Tensor &positions,
                                 const Tensor &frequencies, bool interleaved, double scale, bool inverse) {
    return call_turn(q, k, positions, frequencies, interleaved, scale, inverse);
}

// ---- cache -----------------------------------------------------------------

int cache_code(const Tensor &t) {
    return t.scalar_type() == at::kChar ? ENATTEN_I8 : t.scalar_type() == at::kFloat8_e4m3fn ? ENATTEN_E4M3 : -1;
}

// x: q, or k of new tokens
void validate_cache(const char *what, const char *name, const Tensor &x, const Tensor &kc, const Tensor &vc,
                    const Tensor &ks, const Tensor &vs, const Tensor &pages, const Tensor &lengths,
                    const optional<Tensor> &counts) {
    TORCH_CHECK_VALUE(x.dim() == 4, what, ": expected [B, heads, T, head_dim] tensors, got ", x.dim(), "-D ", name);
    const int code = dtype_code(x);
    TORCH_CHECK_VALUE(code >= 0 && code != ENATTEN_F64, what, ": dtype ", x.scalar_type(),
                      " is not supported (float32, bfloat16, float16)");
    TORCH_CHECK_VALUE(x.numel() > 0, what, ": empty tensors are not supported");
    TORCH_CHECK_VALUE(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.size(3) == x.size(3) && kc.numel() > 0, what,
                      ": k_cache and v_cache must be [pages, heads, tokens, ", x.size(3), "], got ", kc.sizes(), ", ",
                      vc.sizes());
    TORCH_CHECK_VALUE(cache_code(kc) >= 0 && vc.scalar_type() == kc.scalar_type(), what,
                      ": k_cache and v_cache must both be int8 or float8_e4m3fn, got ", kc.scalar_type(), ", ",
                      vc.scalar_type());
    for (const Tensor *t : {&kc, &vc})
        TORCH_CHECK_VALUE(t->stride(3) == 1, what, ": the cache needs unit stride on the channels");
    for (const Tensor *t : {&ks, &vs}) {
        TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == kc.size(0) && t->size(1) == kc.size(1), what,
                          ": k_scale and v_scale must be [pages, heads] = ", kc.sizes().slice(0, 2), ", got ", t->sizes());
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat, what, ": k_scale and v_scale must be float32");
    }
    TORCH_CHECK_VALUE(pages.dim() == 2 && pages.size(0) == x.size(0) && pages.size(1) > 0 && pages.scalar_type() == at::kInt,
                      what, ": pages must be int32 [B, columns], got ", pages.scalar_type(), " ", pages.sizes());
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == x.size(0) && lengths.scalar_type() == at::kInt, what,
                      ": lengths must be int32 [B], got ", lengths.scalar_type(), " ", lengths.sizes());
    if (counts.has_value())
        TORCH_CHECK_VALUE(counts->dim() == 1 && counts->size(0) == x.size(0) && counts->scalar_type() == at::kInt, what,
                          ": counts must be int32 [B], got ", counts->scalar_type(), " ", counts->sizes());
    for (const Tensor *t : {&kc, &vc, &ks, &vs, &pages, &lengths})
        TORCH_CHECK_VALUE(t->device() == x.device(), what, ": all tensors must be on the same device");
    TORCH_CHECK_VALUE(!counts.has_value() || counts->device() == x.device(), what,
                      ": all tensors must be on the same device");
    TORCH_CHECK_VALUE(pages.size(1) <= 0x7fffffff && kc.size(0) <= 0x7fffffff && kc.size(2) <= 1024, what,
                      ": too many pages, or more than 1024 tokens in one");
    TORCH_CHECK_VALUE(x.size(0) <= 0x7fffffff && x.size(1) <= (1 << 20) && x.size(2) <= 0x7fffffff && x.size(3) <= 256,
                      what, ": head_dim must be a multiple of 16 up to 256, got ", x.size(3));
}
// Whether two tensors of the same shape share an element.  Exact where both are dense, and where they have the
// same strides and these are nested (each longer than all that lies within it), as views of one pool have: the
// distance of the addresses is then a whole number of each stride, with two choices at most.  Other views whose
// ranges cross are let pass.
using Axis = std::pair<int64_t, int64_t>;  // stride, size
bool is_distance(int64_t distance, const Axis *axes, int n) {  // longest stride first
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
bool share_memory(const Tensor &a, const Tensor &b) {
    const int64_t size = a.element_size();
    const auto extent = [&](const Tensor &t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); i++) last += t.stride(i) * (t.size(i) - 1);
        return (last + 1) * size;
    };
    const int64_t distance = static_cast<const char *>(b.data_ptr()) - static_cast<const char *>(a.data_ptr());
    if (distance >= extent(a) || -distance >= extent(b)) return false;
    if (a.is_non_overlapping_and_dense() && b.is_non_overlapping_and_dense()) return true;
    Axis axes[4];
    int n = 0;
    for (int64_t i = 0; i < a.dim(); i++) {
        if (a.size(i) == 1) continue;
        if (a.stride(i) != b.stride(i)) return false;
        axes[n++] = {a.stride(i), a.size(i)};
    }
    std::sort(axes, axes + n, std::greater<Axis>());
    return distance % size == 0 && is_distance(distance / size, axes, n);
}
void validate_append(const Tensor &k, const Tensor &v, const Tensor &kc, const Tensor &vc, const Tensor &ks,
                     const Tensor &vs, const Tensor &pages, const Tensor &lengths, const optional<Tensor> &counts) {
    const char *what = "cache_append";
    validate_cache(what, "k", k, kc, vc, ks, vs, pages, lengths, counts);
    TORCH_CHECK_VALUE(v.sizes() == k.sizes(), what, ": k and v must have the same shape, got ", k.sizes(), ", ", v.sizes());
    TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type() && v.device() == k.device(), what,
                      ": k and v must share a dtype and a device");
    TORCH_CHECK_VALUE(kc.size(1) == k.size(1), what, ": k has ", k.size(1), " heads, the cache ", kc.size(1));
    for (const Tensor *t : {&kc, &vc, &ks, &vs}) at::assert_no_internal_overlap(*t);
    TORCH_CHECK_VALUE(!kc.is_same(vc) && !ks.is_same(vs) &&
                          (kc.is_meta() || !(share_memory(kc, vc) || share_memory(ks, vs))),
                      what, ": keys and values must not share a cache");
    on_gpu(what, k);
}
void validate_attention(const Tensor &q, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs,
                        const Tensor &pages, const Tensor &lengths, const optional<Tensor> &counts, int64_t kernel_size) {
    const char *what = "cache_attention";
    validate_cache(what, "q", q, kc, vc, ks, vs, pages, lengths, counts);
    TORCH_CHECK_VALUE(q.size(1) % kc.size(1) == 0, what, ": ", q.size(1), " heads are no multiple of the cache's ", kc.size(1));
    TORCH_CHECK_VALUE(kernel_size >= 0, what, ": kernel_size must be >= 1, or 0 for all tokens, got ", kernel_size);
    on_gpu(what, q);
}
// the columns of a row of pages are neighbours
Tensor page_rows(const Tensor &t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }

// rows at multiples of 16 bytes (head dims are multiples of 16): nearly always the tensor itself
Tensor aligned_rows(const Tensor &t) {
    const int64_t pack = 16 / t.element_size();
    const bool ok = t.stride(3) == 1 && (t.stride(0) | t.stride(1) | t.stride(2)) % pack == 0 &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

void cache_append(const Tensor &k_, const Tensor &v_, const Tensor &kc, const Tensor &vc, const Tensor &ks,
                  const Tensor &vs, const Tensor &pages_, const Tensor &lengths_, const optional<Tensor> &counts_) {
    validate_append(k_, v_, kc, vc, ks, vs, pages_, lengths_, counts_);
    if (k_.is_meta()) return;
    const c10::DeviceGuard guard(k_.device());
    const Tensor k = kernel_layout(k_), v = kernel_layout(v_), pages = page_rows(pages_);
    const Tensor lengths = lengths_.contiguous(), counts = counts_.has_value() ? counts_->contiguous() : Tensor();
    check_rc(enatten_cache_append(
        k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(),
        pages.data_ptr<int>(), lengths.data_ptr<int>(), counts.defined() ? counts.data_ptr<int>() : nullptr, k.size(0),
        k.size(1), k.size(2), k.size(3), kc.size(0), kc.size(2), pages.size(1), dtype_code(k), cache_code(kc),
        k.strides().data(), v.strides().data(), kc.strides().data(), vc.strides().data(), ks.strides().data(),
        vs.strides().data(), pages.stride(0), stream_now()));
}
Tensor cache_attention(const Tensor &q_, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs,
                       const Tensor &pages_, const Tensor &lengths_, const optional<Tensor> &counts_,
                       int64_t kernel_size, double scale) {
    validate_attention(q_, kc, vc, ks, vs, pages_, lengths_, counts_, kernel_size);
    if (q_.is_meta()) return empty_rows(kernel_layout(q_));
    const c10::DeviceGuard guard(q_.device());
    const Tensor rows = kernel_layout(q_), q = aligned_rows(rows), pages = page_rows(pages_);
    const Tensor lengths = lengths_.contiguous(), counts = counts_.has_value() ? counts_->contiguous() : Tensor();
    const Tensor o = aligned_rows(empty_rows(rows));
    const int window = (int)std::min<int64_t>(kernel_size, 0x7fffffff);
    const int B = q.size(0), N = q.size(1), Nk = kc.size(1), T = q.size(2), D = q.size(3);
    const int page = kc.size(2), columns = pages.size(1);
    const size_t need = enatten_cache_attention_workspace_bytes(B, N, Nk, T, D, page, columns, window, dtype_code(q));
    const Tensor ws = need ? at::empty({(int64_t)need}, q.options().dtype(at::kByte)) : Tensor();
    check_rc(enatten_cache_attention(
        q.data_ptr(), kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), pages.data_ptr<int>(),
        lengths.data_ptr<int>(), counts.defined() ? counts.data_ptr<int>() : nullptr, o.data_ptr(),
        need ? ws.data_ptr() : nullptr, B, N, Nk, T, D, kc.size(0), page, columns, window, dtype_code(q), cache_code(kc),
        q.strides().data(), o.strides().data(), kc.strides().data(), vc.strides().data(), ks.strides().data(),
        vs.strides().data(), pages.stride(0), (float)scale, stream_now()));
    return o;
}

// Codes are rounded: neither operator has a gradient, and a caller that would get none is told so.
void no_gradient(const char *what, std::initializer_list<const Tensor *> inputs) {
    const bool mode = at::GradMode::is_enabled();
    for (const Tensor *t : inputs)
        TORCH_CHECK(!(mode && t->requires_grad()) && !has_tangent(*t), what,
                    ": a cache of 8 bits has no gradient; call it under torch.no_grad() or on detached tensors, which "
                    "have no tangent");
}
using AppendSig = decltype(cache_append);
void call_append(const Tensor &k, const Tensor &v, const Tensor &kc, const Tensor &vc, const Tensor &ks,
                 const Tensor &vs, const Tensor &pages, const Tensor &lengths, const optional<Tensor> &counts) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("enatten::cache_append", "").typed<AppendSig>();
    op.call(k, v, kc, vc, ks, vs, pages, lengths, counts);
}
void cache_append_autograd(const Tensor &k, const Tensor &v, const Tensor &kc, const Tensor &vc, const Tensor &ks,
                           const Tensor &vs, const Tensor &pages, const Tensor &lengths, const optional<Tensor> &counts) {
    no_gradient("cache_append", {&k, &v, &kc, &vc, &ks, &vs});
    at::AutoDispatchBelowAutograd below;
    call_append(k, v, kc, vc, ks, vs, pages, lengths, counts);
}
// The version counters of what is written.  Ordinary tensors come here in inference mode too, where the
// autograd key is left out: a graph made before may have saved them.
void cache_append_in_place(const Tensor &k, const Tensor &v, const Tensor &kc, const Tensor &vc, const Tensor &ks,
                           const Tensor &vs, const Tensor &pages, const Tensor &lengths, const optional<Tensor> &counts) {
    {
        at::AutoDispatchBelowADInplaceOrView below;
        call_append(k, v, kc, vc, ks, vs, pages, lengths, counts);
    }
    for (const Tensor *t : {&kc, &vc, &ks, &vs})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
Tensor cache_attention_autograd(const Tensor &q, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs,
                                const Tensor &pages, const Tensor &lengths, const optional<Tensor> &counts,
                                int64_t kernel_size, double scale) {
    no_gradient("cache_attention", {&q, &kc, &vc, &ks, &vs});
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("enatten::cache_attention", "").typed<decltype(cache_attention)>();
    return op.call(q, kc, vc, ks, vs, pages, lengths, counts, kernel_size, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(enatten, m) {
    m.def("rotary_turn(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, bool interleaved, float scale, "
          "bool inverse) -> Tensor[]");
    m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, bool interleaved, float scale, "
          "bool inverse) -> Tensor[]");
    m.def("cache_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
          "Tensor(d!) v_scale, Tensor pages, Tensor lengths, Tensor? counts) -> ()");
    m.def("cache_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor pages, "
          "Tensor lengths, Tensor? counts, int kernel_size, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(enatten, CompositeExplicitAutograd, m) {
    m.impl("rotary_turn", &rotary_turn);
    m.impl("rotary", &rotary_plain);
    m.impl("cache_append", &cache_append);
    m.impl("cache_attention", &cache_attention);
}

TORCH_LIBRARY_IMPL(enatten, Autograd, m) {
    m.impl("rotary", &rotary_autograd);
    m.impl("cache_append", &cache_append_autograd);
    m.impl("cache_attention", &cache_attention_autograd);
}

TORCH_LIBRARY_IMPL(enatten, ADInplaceOrView, m) {
    m.impl("cache_append", &cache_append_in_place);
}
