// cache_attention of sequences that continue one prompt (enatten_cache_attention_shared).
//
//   o = (f y + f' y') / (f l + f' l'),   f = exp(m - max(m, m')), f' likewise
//
// with maximum m, sum l and sums of values y over a sequence's own tokens, and m', l', y' over those that it
// shares with its run.  The latter are a product of their own with as many rows as the whole run has, so that
// the shared codes are read once for all of them and, from 49 rows on (65 of up to 64 channels), turned into
// float16 once.  Both are the kernels of cache_attention.hip over other rows and tokens: a first pass whose
// entries are runs leaves m', l' and y' in the workspace, a second one goes over the tokens behind and joins
// them in where it writes.
#include "cache_attention.h"

namespace enatten {
namespace {

// Both passes' plans, and where their workspaces lie: what the runs' rows come to, then what either pass needs.
struct SharedPlan {
    Plan first, second;
    int64_t canon;  // floats
    size_t bytes;
};
SharedPlan shared_plan(int B, int heads, int heads_kv, int T, int D, int page, int columns, int window, int dtype, int runs) {
    SharedPlan p;
    const int size = B / runs;
    p.first = plan_of(runs, heads, heads_kv, T * size, D, page, columns, window, dtype);
    p.second = plan_of(B, heads, heads_kv, T, D, page, columns, window, dtype);
    p.canon = ((int64_t)B * heads * T * (D + 2) + 3) / 4 * 4;
    const size_t a = workspace_bytes(p.first, runs, heads_kv, D), b = workspace_bytes(p.second, B, heads_kv, D);
    p.bytes = p.canon * sizeof(float) + (a > b ? a : b);
    return p;
}

}  // namespace
}  // namespace enatten

using namespace enatten;

extern "C" {
#pragma GCC visibility push(default)

size_t enatten_cache_attention_shared_workspace_bytes(int B, int heads, int heads_kv, int T, int D, int page, int columns,
                                                      int kernel_size, int dtype, int runs) {
    if (B < 1 || heads < 1 || heads_kv < 1 || heads % heads_kv || T < 1 || D < 1 || page < 1 || columns < 1 ||
        kernel_size < 0 || runs < 1 || B % runs || (int64_t)B * heads * T > (1 << 30))
        return 0;
    return shared_plan(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype, runs).bytes;
}

int enatten_cache_attention_shared(const void *q, const void *k_cache, const void *v_cache, const float *k_scale,
                                   const float *v_scale, const int *pages, const int *lengths, const int *counts,
                                   const int *shared, int runs, void *o, void *workspace, int B, int heads, int heads_kv,
                                   int T, int D, int num_pages, int page, int columns, int kernel_size, int dtype,
                                   int cache_dtype, const int64_t *q_strides, const int64_t *o_strides,
                                   const int64_t *k_cache_strides, const int64_t *v_cache_strides,
                                   const int64_t *k_scale_strides, const int64_t *v_scale_strides, int64_t pages_stride,
                                   float scale, void *stream) {
    const char *fn = "enatten_cache_attention_shared";
    SharedArgs a{};
    int rc = set_attention(fn, q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts, o, B, heads, heads_kv, T, D,
                           num_pages, page, columns, kernel_size, dtype, cache_dtype, q_strides, o_strides, k_cache_strides,
                           v_cache_strides, k_scale_strides, v_scale_strides, pages_stride, scale, &a);
    if (rc) return rc;
    if (!shared || runs < 1 || B % runs) {
        set_error("%s: shared must not be NULL, and its %d runs divide %d sequences", fn, runs, B);
        return ENATTEN_EINVAL;
    }
    const SharedPlan p = shared_plan(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype, runs);
    if (!workspace || (uintptr_t)workspace % 16) {
        set_error("%s: workspace is NULL or not 16-byte aligned", fn);
        return ENATTEN_EINVAL;
    }
    a.shared = shared;
    a.runs = runs;
    a.size = B / runs;
    a.canon = static_cast<float *>(workspace);
    a.ws = a.canon + p.canon;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool e = cache_dtype == ENATTEN_E4M3;
    a.row_tiles = p.first.row_tiles;
    a.parts = p.first.parts;
    if ((rc = launch_first(fn, a, p.first, e, st))) return rc;
    a.row_tiles = p.second.row_tiles;
    a.parts = p.second.parts;
    return launch_second(fn, a, p.second, e, st);
}

#pragma GCC visibility pop
}  // extern "C"
