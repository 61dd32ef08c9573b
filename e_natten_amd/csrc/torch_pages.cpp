// Native torch binding of the operators on pages of a cache: enatten::cache_fork, cache_reserve, cache_copy and
// cache_compact.  Host code only; the checks and error classes are those of the Python host side (pages.py).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include "torch_shim.h"

namespace {

using at::Tensor;
using c10::optional;

// int32 [n] without gaps, where the table is
void validate_numbers(const char *what, const char *name, const Tensor &t, int64_t n, const Tensor &pages) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.scalar_type() == at::kInt && (n < 0 ? t.size(0) > 0 : t.size(0) == n), what, ": ",
                      name, n < 0 ? " must be int32 [pages of the cache], got " : " must be int32 [B], got ",
                      t.scalar_type(), " ", t.sizes());
    TORCH_CHECK_VALUE(t.is_contiguous(), what, ": ", name, " must be contiguous");
    TORCH_CHECK_VALUE(t.device() == pages.device(), what, ": all tensors must be on the same device");
}
void validate_table(const char *what, const Tensor &pages, const Tensor &holders, int64_t page) {
    TORCH_CHECK_VALUE(pages.dim() == 2 && pages.scalar_type() == at::kInt && pages.numel() > 0, what,
                      ": pages must be int32 [B, columns], got ", pages.scalar_type(), " ", pages.sizes());
    TORCH_CHECK_VALUE(pages.size(1) == 1 || pages.stride(1) == 1, what, ": pages needs unit stride on the columns");
    TORCH_CHECK_VALUE(pages.size(0) == 1 || pages.stride(0) >= pages.size(1), what, ": the rows of pages must not overlap");
    TORCH_CHECK_VALUE(page >= 16 && page <= 1024 && page % 16 == 0, what,
                      ": pages must hold a multiple of 16 tokens up to 1024, got ", page);
    validate_numbers(what, "holders", holders, -1, pages);
    TORCH_CHECK_VALUE(pages.size(0) <= 0x7fffffff && pages.size(1) <= 0x7fffffff && holders.size(0) <= 1 << 30, what,
                      ": tensor too large");
}
Tensor workspace(size_t bytes, const Tensor &like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }

void cache_fork(const Tensor &pages, const Tensor &lengths, const Tensor &holders, const Tensor &parents_, int64_t page) {
    const char *what = "cache_fork";
    validate_table(what, pages, holders, page);
    validate_numbers(what, "lengths", lengths, pages.size(0), pages);
    const Tensor parents = parents_.contiguous();
    validate_numbers(what, "parents", parents, pages.size(0), pages);
    on_gpu(what, pages);
    if (pages.is_meta()) return;
    const c10::DeviceGuard guard(pages.device());
    check_rc(enatten_cache_fork(pages.data_ptr<int>(), lengths.data_ptr<int>(), holders.data_ptr<int>(),
                                parents.data_ptr<int>(), pages.size(0), pages.size(1), holders.size(0), page,
                                pages.stride(0), stream_now()));
}

Tensor cache_reserve(const Tensor &pages, const Tensor &lengths_, const Tensor &holders, int64_t page,
                     const optional<Tensor> &counts_, int64_t count) {
    const char *what = "cache_reserve";
    validate_table(what, pages, holders, page);
    const Tensor lengths = lengths_.contiguous(), counts = counts_.has_value() ? counts_->contiguous() : Tensor();
    validate_numbers(what, "lengths", lengths, pages.size(0), pages);
    if (counts.defined()) validate_numbers(what, "counts", counts, pages.size(0), pages);
    TORCH_CHECK_VALUE(count >= 0 && count <= 0x7fffffff, what, ": counts must not be negative, got ", count);
    on_gpu(what, pages);
    const Tensor copies = at::empty({pages.size(0), 3}, pages.options());
    if (pages.is_meta()) return copies;
    const c10::DeviceGuard guard(pages.device());
    const Tensor ws = workspace(enatten_cache_reserve_workspace_bytes(pages.size(0), pages.size(1), holders.size(0)), pages);
    check_rc(enatten_cache_reserve(pages.data_ptr<int>(), lengths.data_ptr<int>(),
                                   counts.defined() ? counts.data_ptr<int>() : nullptr, count, holders.data_ptr<int>(),
                                   copies.data_ptr<int>(), ws.data_ptr(), pages.size(0), pages.size(1), holders.size(0),
                                   page, pages.stride(0), stream_now()));
    return copies;
}

Tensor cache_compact(const Tensor &pages, const Tensor &holders, int64_t page) {
    const char *what = "cache_compact";
    validate_table(what, pages, holders, page);
    on_gpu(what, pages);
    const Tensor copies = at::empty({std::max<int64_t>(holders.size(0) / 2, 1), 3}, pages.options());
    if (pages.is_meta()) return copies;
    const c10::DeviceGuard guard(pages.device());
    const Tensor ws = workspace(enatten_cache_compact_workspace_bytes(holders.size(0)), pages);
    check_rc(enatten_cache_compact(pages.data_ptr<int>(), holders.data_ptr<int>(), copies.data_ptr<int>(), ws.data_ptr(),
                                   pages.size(0), pages.size(1), holders.size(0), page, pages.stride(0), stream_now()));
    return copies;
}

void cache_copy(const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &copies_) {
    const char *what = "cache_copy";
    TORCH_CHECK_VALUE((kc.dim() == 4 || kc.dim() == 5) && kc.sizes() == vc.sizes() && kc.numel() > 0, what,
                      ": k_cache and v_cache must be [pages, heads, tokens, head_dim], or that for some layers, got ",
                      kc.sizes(), ", ", vc.sizes());
    TORCH_CHECK_VALUE(cache_code(kc) >= 0 && vc.scalar_type() == kc.scalar_type(), what,
                      ": k_cache and v_cache must both be int8 or float8_e4m3fn, got ", kc.scalar_type(), ", ",
                      vc.scalar_type());
    const int64_t lead = kc.dim() - 4;
    for (const Tensor *t : {&kc, &vc})
        TORCH_CHECK_VALUE(t->stride(-1) == 1, what, ": the cache needs unit stride on the channels");
    for (const Tensor *t : {&ks, &vs}) {
        TORCH_CHECK_VALUE(t->sizes() == kc.sizes().slice(0, lead + 2), what, ": k_scale and v_scale must be [pages, heads] = ",
                          kc.sizes().slice(0, lead + 2), ", got ", t->sizes());
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat, what, ": k_scale and v_scale must be float32");
    }
    TORCH_CHECK_VALUE(copies_.dim() == 2 && copies_.size(1) == 3 && copies_.scalar_type() == at::kInt, what,
                      ": copies must be int32 [n, 3], got ", copies_.scalar_type(), " ", copies_.sizes());
    for (const Tensor *t : {&vc, &ks, &vs, &copies_})
        TORCH_CHECK_VALUE(t->device() == kc.device(), what, ": all tensors must be on the same device");
    for (const Tensor *t : {&kc, &vc, &ks, &vs}) at::assert_no_internal_overlap(*t);
    TORCH_CHECK_VALUE(!kc.is_same(vc) && !ks.is_same(vs) &&
                          (kc.is_meta() || !(share_memory(kc, vc) || share_memory(ks, vs))),
                      what, ": keys and values must not share a cache");
    TORCH_CHECK_VALUE(kc.size(lead) <= 0x7fffffff && kc.size(lead + 1) <= (1 << 20) && (lead == 0 || kc.size(0) <= (1 << 20)) &&
                          copies_.size(0) <= 0x7fffffff && kc.size(lead + 2) <= 1024 && kc.size(lead + 3) <= 256,
                      what, ": tensor too large, more than 1024 tokens in a page, or a head_dim above 256");
    on_gpu(what, kc);
    if (kc.is_meta()) return;
    const c10::DeviceGuard guard(kc.device());
    const Tensor copies = copies_.contiguous();
    int64_t strides[2][4], zstrides[2][3];
    const Tensor *codes[2] = {&kc, &vc}, *scales[2] = {&ks, &vs};
    for (int i = 0; i < 2; i++) {
        strides[i][0] = lead ? codes[i]->stride(0) : 0;
        zstrides[i][0] = lead ? scales[i]->stride(0) : 0;
        for (int j = 0; j < 3; j++) strides[i][j + 1] = codes[i]->stride(lead + j);
        for (int j = 0; j < 2; j++) zstrides[i][j + 1] = scales[i]->stride(lead + j);
    }
    check_rc(enatten_cache_copy(kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(),
                                copies.data_ptr<int>(), copies.size(0), lead ? kc.size(0) : 1, kc.size(lead + 1),
                                kc.size(lead + 3), kc.size(lead), kc.size(lead + 2), strides[0], strides[1], zstrides[0],
                                zstrides[1], stream_now()));
}

template <typename Sig>
const auto &op_named(const char *name) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
    return op;
}
void bump(std::initializer_list<const Tensor *> written) {
    for (const Tensor *t : written)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// The version counters of what is written.  Ordinary tensors come here in inference mode too, where the
// autograd key is left out: a graph made before may have saved them.
void cache_fork_in_place(const Tensor &pages, const Tensor &lengths, const Tensor &holders, const Tensor &parents, int64_t page) {
    {
        at::AutoDispatchBelowADInplaceOrView below;
        op_named<decltype(cache_fork)>("enatten::cache_fork").call(pages, lengths, holders, parents, page);
    }
    bump({&pages, &lengths, &holders});
}
Tensor cache_reserve_in_place(const Tensor &pages, const Tensor &lengths, const Tensor &holders, int64_t page,
                              const optional<Tensor> &counts, int64_t count) {
    Tensor copies;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        copies = op_named<decltype(cache_reserve)>("enatten::cache_reserve").call(pages, lengths, holders, page, counts, count);
    }
    bump({&pages, &holders});
    return copies;
}
Tensor cache_compact_in_place(const Tensor &pages, const Tensor &holders, int64_t page) {
    Tensor copies;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        copies = op_named<decltype(cache_compact)>("enatten::cache_compact").call(pages, holders, page);
    }
    bump({&pages, &holders});
    return copies;
}
void cache_copy_in_place(const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &copies) {
    {
        at::AutoDispatchBelowADInplaceOrView below;
        op_named<decltype(cache_copy)>("enatten::cache_copy").call(kc, vc, ks, vs, copies);
    }
    bump({&kc, &vc, &ks, &vs});
}
// (whole numbers have no gradient)
void cache_copy_autograd(const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &copies) {
    no_gradient("cache_copy", {&kc, &vc, &ks, &vs});
    at::AutoDispatchBelowAutograd below;
    op_named<decltype(cache_copy)>("enatten::cache_copy").call(kc, vc, ks, vs, copies);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(enatten, m) {
    m.def("cache_fork(Tensor(a!) pages, Tensor(b!) lengths, Tensor(c!) holders, Tensor parents, int page) -> ()");
    m.def("cache_reserve(Tensor(a!) pages, Tensor lengths, Tensor(b!) holders, int page, Tensor? counts, int count) -> Tensor");
    m.def("cache_copy(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor copies) -> ()");
    m.def("cache_compact(Tensor(a!) pages, Tensor(b!) holders, int page) -> Tensor");
}

TORCH_LIBRARY_IMPL(enatten, CompositeExplicitAutograd, m) {
    m.impl("cache_fork", &cache_fork);
    m.impl("cache_reserve", &cache_reserve);
    m.impl("cache_copy", &cache_copy);
    m.impl("cache_compact", &cache_compact);
}

TORCH_LIBRARY_IMPL(enatten, Autograd, m) { m.impl("cache_copy", &cache_copy_autograd); }

TORCH_LIBRARY_IMPL(enatten, ADInplaceOrView, m) {
    m.impl("cache_fork", &cache_fork_in_place);
    m.impl("cache_reserve", &cache_reserve_in_place);
    m.impl("cache_copy", &cache_copy_in_place);
    m.impl("cache_compact", &cache_compact_in_place);
}
