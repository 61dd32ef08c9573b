// What the operators of growing sequences share: argument checks, views, 8-bit codes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "enatten.h"
#include "na2d_common.h"

namespace enatten {

// A [B, heads, T, D] tensor with unit stride on D; strides in elements.
struct Rows {
    const void *ptr;
    int64_t sb, sh, st;
};
// Codes [pages, heads, page, D] of one byte each, and the float32 scales [pages, heads].
struct Cache {
    void *codes;
    float *scales;
    int64_t sp, sh, st;  // page, head, token
    int64_t zp, zh;      // of the scales: page, head
};
// The pages of the sequences and how far these go.
struct Table {
    const int *pages, *lengths, *counts;  // counts: nullptr if all are T
    int64_t stride;
    int num_pages, page, columns, T;
};

// New tokens and total tokens of sequence b; false if the numbers do not fit together.
__device__ __forceinline__ bool sequence_of(const Table &tb, int b, int &len, int &count) {
    len = tb.lengths[b];
    count = tb.counts ? tb.counts[b] : tb.T;
    const bool ok = count >= 0 && count <= tb.T && len >= count && len <= (int64_t)tb.columns * tb.page;
    if (!ok) len = count = 0;
    return ok;
}

inline int set_rows(const char *fn, const char *name, const void *p, const int64_t *st, int heads, int T, int D,
                    Rows *out) {
    if (!p) {
        set_error("%s: %s is NULL", fn, name);
        return ENATTEN_EINVAL;
    }
    *out = st ? Rows{p, st[0], st[1], st[2]} : Rows{p, (int64_t)heads * T * D, (int64_t)T * D, D};
    if (out->sb < 0 || out->sh < 0 || out->st < 0) {
        set_error("%s: negative stride for %s", fn, name);
        return ENATTEN_EINVAL;
    }
    return ENATTEN_OK;
}

inline int set_cache(const char *fn, const char *name, void *codes, float *scales, const int64_t *st,
                     const int64_t *zst, int heads, int page, int D, int align, Cache *out) {
    if (!codes || !scales) {
        set_error("%s: %s_cache or %s_scale is NULL", fn, name, name);
        return ENATTEN_EINVAL;
    }
    out->codes = codes;
    out->scales = scales;
    out->sp = st ? st[0] : (int64_t)heads * page * D;
    out->sh = st ? st[1] : (int64_t)page * D;
    out->st = st ? st[2] : D;
    out->zp = zst ? zst[0] : heads;
    out->zh = zst ? zst[1] : 1;
    if (out->sp < 0 || out->sh < 0 || out->st < D || out->st > (1 << 20) || out->zp < 0 || out->zh < 0) {
        set_error("%s: strides of %s_cache and %s_scale must not be negative, and D to 2^20 between tokens", fn,
                  name, name);
        return ENATTEN_EINVAL;
    }
    if ((out->sp | out->sh | out->st | (int64_t)(uintptr_t)codes) % align) {
        set_error("%s: the address and the strides of %s_cache must be multiples of %d", fn, name, align);
        return ENATTEN_EINVAL;
    }
    return ENATTEN_OK;
}

// The sizes that both cache operators take.
inline int check_cache_sizes(const char *fn, int B, int heads, int T, int D, int num_pages, int page, int columns,
                             int dtype, int cache_dtype, int64_t pages_stride) {
    if (dtype != ENATTEN_F32 && dtype != ENATTEN_BF16 && dtype != ENATTEN_F16) {
        set_error("%s: dtype code %d is not ENATTEN_F32, BF16 or F16", fn, dtype);
        return ENATTEN_EINVAL;
    }
    if (cache_dtype != ENATTEN_I8 && cache_dtype != ENATTEN_E4M3) {
        set_error("%s: cache dtype code %d is not ENATTEN_I8 or ENATTEN_E4M3", fn, cache_dtype);
        return ENATTEN_EINVAL;
    }
    if (B < 1 || heads < 1 || T < 1 || num_pages < 1 || columns < 1) {
        set_error("%s: every dimension must be >= 1, got B=%d heads=%d T=%d num_pages=%d columns=%d", fn, B, heads, T,
                  num_pages, columns);
        return ENATTEN_EINVAL;
    }
    if (D < 16 || D > 256 || D % 16) {
        set_error("%s: head_dim must be a multiple of 16 up to 256, got %d", fn, D);
        return ENATTEN_EINVAL;
    }
    if (page < 16 || page > 1024 || page % 16) {
        set_error("%s: pages must hold a multiple of 16 tokens up to 1024, got %d", fn, page);
        return ENATTEN_EINVAL;
    }
    if (pages_stride < 0) {
        set_error("%s: negative stride for pages", fn);
        return ENATTEN_EINVAL;
    }
    // (counts of tokens, of rows, and of steps of 64 sequences stay within 31 bits)
    if ((int64_t)columns * page > (1 << 30) - 4096 || (int64_t)B * heads > (1 << 30) ||
        (int64_t)B * heads * T > (1 << 30)) {
        set_error("%s: more than 2^30 tokens in a sequence's pages, or rows in a call", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    return ENATTEN_OK;
}

inline int launched(const char *fn) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return ENATTEN_OK;
    set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return ENATTEN_ELAUNCH;
}

}  // namespace enatten
