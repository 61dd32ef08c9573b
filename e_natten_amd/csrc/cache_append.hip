// New tokens into a cache of 8 bits with one scale for each block (page, head).
//
//   scale' = max(scale, max |x| / M),  code = round(x / scale'),  M = 127 or 448
//
// and where a page holds older tokens and its scale grows, their codes are rounded anew.  A workgroup
// takes one block of k or v: it reads the block's new tokens, forms their maximum and writes the codes.
// The call reads each value once and writes one byte for it: bound by HBM, and for single tokens by the
// launch.  Nothing is shared between workgroups.
//
// Measured on MI355X: k and v of 16 heads of 128 channels, 2 x 8192 tokens, bfloat16: 43 us with pages of
// 64 tokens (201 MB, 4.6 TB/s; a plain copy reaches 5.0), 40 us in E4M3; one token each for 32 sequences of
// 8 heads: 3.8 us.  Where every page's scale grows, its older codes are read and written too: with pages of
// up to 256 tokens 16 us instead of 6, up to 64 level.
//
// The product with 1 / scale' instead of a division: a value next to the middle of two codes may go to
// either, which is half a step off in both cases.
#include "sequence_common.h"

namespace enatten {
namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
    Rows x[2];  // k and v
    Cache c[2];
    Table tb;
    int B, heads, D, touched;  // touched: pages that the new tokens of one sequence may lie on
};

constexpr float kTiny = 1.17549435e-38f;  // 2^-126

template <bool E4M3> constexpr float kTop = E4M3 ? 448.f : 127.f;

// 8 codes of x * f
template <bool E4M3> __device__ __forceinline__ u32x2 encode(f32x8 x, float f) {
    u32x2 r = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = fminf(fmaxf(x[j] * f, -kTop<E4M3>), kTop<E4M3>);
    if constexpr (E4M3) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j], x[4 * j + 1], 0, false);
            r[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2], x[4 * j + 3], w, true);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) r[j / 4] |= ((unsigned)(int)rintf(x[j]) & 0xffu) << (8 * (j % 4));
    }
    return r;
}
template <bool E4M3> __device__ __forceinline__ f32x8 decode(u32x2 r) {
    f32x8 x;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if constexpr (E4M3) {
            if (j % 2 == 0) {
                const auto p = j % 4 ? __builtin_amdgcn_cvt_pk_f32_fp8(r[j / 4], true)
                                     : __builtin_amdgcn_cvt_pk_f32_fp8(r[j / 4], false);
                x[j] = p[0];
                x[j + 1] = p[1];
            }
        } else {
            x[j] = (float)(int)(signed char)(r[j / 4] >> (8 * (j % 4)));
        }
    }
    return x;
}

// 8 values from p on, in float32; WIDE: by loads of 16 bytes
template <typename S, bool WIDE> __device__ __forceinline__ f32x8 load8(const S *p) {
    f32x8 r;
    if constexpr (WIDE) {
        constexpr int N = 16 / sizeof(S);
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            struct alignas(16) Pack { S v[N]; };
            const Pack k = *reinterpret_cast<const Pack *>(p + i);
#pragma unroll
            for (int j = 0; j < N; j++) r[i + j] = (float)k.v[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = (float)p[j];
    }
    return r;
}

// A unit is 8 channels of a token.  KEEP units per thread stay in registers between the maximum and
// the codes; what a block has beyond them is read again.
template <typename S, bool E4M3, bool WIDE, int THREADS, int KEEP>
__global__ __launch_bounds__(THREADS) void append_block(AppendArgs a) {
    int block = blockIdx.x;
    const int which = block & 1;
    block >>= 1;
    const int head = block % a.heads;
    block /= a.heads;
    const int n = block % a.touched, b = block / a.touched;
    const Rows &X = a.x[which];
    const Cache &c = a.c[which];
    const int page = a.tb.page;
    int len, count;
    if (!sequence_of(a.tb, b, len, count) || count == 0) return;
    const int start = len - count, column = start / page + n;
    const int lo = max(start, column * page), hi = min(len, (column + 1) * page);
    if (lo >= hi) return;
    const int at = a.tb.pages[b * a.tb.stride + column];
    const int older = lo - column * page;  // rows of the page that hold tokens already

    const S *x = static_cast<const S *>(X.ptr) + b * X.sb + head * X.sh + (lo - start) * X.st;
    const int wide = a.D / 8, units = (hi - lo) * wide;
    f32x8 kept[KEEP];
    unsigned most = 0;  // the largest magnitude as its bits: NaN counts as the largest of all
    auto take = [&](f32x8 v) {
#pragma unroll
        for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++) {
        const int u = threadIdx.x + i * THREADS;
        if (u < units) {
            const int row = u / wide;
            kept[i] = load8<S, WIDE>(x + row * X.st + (u - row * wide) * 8);
        } else {
            kept[i] = f32x8{};
        }
    }
    // (the page is asked for behind the loads of the tokens: they need not wait for it)
    if ((unsigned)at >= (unsigned)a.tb.num_pages) return;
    unsigned char *codes = static_cast<unsigned char *>(c.codes) + at * c.sp + head * c.sh;
    float *scale = c.scales + at * c.zp + head * c.zh;
    const float before = older ? *scale : 0.f;
#pragma unroll
    for (int i = 0; i < KEEP; i++) take(kept[i]);
    for (int u = threadIdx.x + KEEP * THREADS; u < units; u += THREADS) {
        const int row = u / wide;
        take(load8<S, WIDE>(x + row * X.st + (u - row * wide) * 8));
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = max(most, (unsigned)__shfl_xor((int)most, o, 64));
    if constexpr (THREADS > 64) {
        __shared__ unsigned part[THREADS / 64];
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / 64; i++) most = max(most, part[i]);
    }
    // (every thread has read the old scale: its load is before the reduction that all wait for)

    float after = fmaxf(before, __uint_as_float(most) / kTop<E4M3>), inverse = 0.f;
    if (most >= 0x7f800000u || !(fabsf(before) < INFINITY)) after = __uint_as_float(0x7fc00000u);
    else if (after < kTiny) after = 0.f;
    else inverse = 1.f / after;
    if (threadIdx.x == 0) *scale = after;

    if (after > before && older) {
        const float f = before * inverse;
        for (int u = threadIdx.x; u < older * wide; u += THREADS) {
            const int row = u / wide;
            u32x2 *p = reinterpret_cast<u32x2 *>(codes + row * c.st + (u - row * wide) * 8);
            *p = encode<E4M3>(decode<E4M3>(*p), f);
        }
    }
    codes += older * c.st;
    auto put = [&](int u, f32x8 v) {
        const int row = u / wide;
        const u32x2 r = inverse > 0.f ? encode<E4M3>(v, inverse) : u32x2{0u, 0u};
        *reinterpret_cast<u32x2 *>(codes + row * c.st + (u - row * wide) * 8) = r;
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++) {
        const int u = threadIdx.x + i * THREADS;
        if (u < units) put(u, kept[i]);
    }
    for (int u = threadIdx.x + KEEP * THREADS; u < units; u += THREADS) {
        const int row = u / wide;
        put(u, load8<S, WIDE>(x + row * X.st + (u - row * wide) * 8));
    }
}

template <typename S, bool E4M3, bool WIDE>
int launch_wide(const char *fn, const AppendArgs &a, hipStream_t st) {
    const int64_t blocks = (int64_t)2 * a.heads * a.touched * a.B;
    if (blocks > 0x7fffff) {  // (2^32 threads)
        set_error("%s: too many blocks of pages and heads", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    const int units = (a.tb.T < a.tb.page ? a.tb.T : a.tb.page) * (a.D / 8);
    ProfScope prof(ENATTEN_KERNEL_CACHE_APPEND, "append_block", st);
    // As few waves as hold the block's new tokens in registers, with up to 4 units each, since a small
    // workgroup's reduction is short and more of them are under way: pages of 16 tokens of 128 channels take
    // 43 us with one wave and 59 with four.  Blocks of more units than that have less to gain from it.
    if (units <= 64) append_block<S, E4M3, WIDE, 64, 1><<<(int)blocks, 64, 0, st>>>(a);
    else if (units <= 256) append_block<S, E4M3, WIDE, 64, 4><<<(int)blocks, 64, 0, st>>>(a);
    else if (units <= 512) append_block<S, E4M3, WIDE, 128, 4><<<(int)blocks, 128, 0, st>>>(a);
    else if (units <= 1024) append_block<S, E4M3, WIDE, 512, 2><<<(int)blocks, 512, 0, st>>>(a);
    else append_block<S, E4M3, WIDE, 256, 8><<<(int)blocks, 256, 0, st>>>(a);
    return launched(fn);
}

template <typename S>
int launch_type(const char *fn, const AppendArgs &a, int cache_dtype, hipStream_t st) {
    bool wide = true;
    for (const Rows &r : a.x)
        wide = wide && (uintptr_t)r.ptr % 16 == 0 && (r.sb | r.sh | r.st) % (16 / sizeof(S)) == 0;
    if (cache_dtype == ENATTEN_E4M3)
        return wide ? launch_wide<S, true, true>(fn, a, st) : launch_wide<S, true, false>(fn, a, st);
    return wide ? launch_wide<S, false, true>(fn, a, st) : launch_wide<S, false, false>(fn, a, st);
}

}  // namespace
}  // namespace enatten

using namespace enatten;

extern "C" {
#pragma GCC visibility push(default)

int enatten_cache_append(const void *k, const void *v, void *k_cache, void *v_cache, float *k_scale, float *v_scale,
                         const int *pages, const int *lengths, const int *counts, int B, int heads, int T, int D,
                         int num_pages, int page, int columns, int dtype, int cache_dtype, const int64_t *k_strides,
                         const int64_t *v_strides, const int64_t *k_cache_strides, const int64_t *v_cache_strides,
                         const int64_t *k_scale_strides, const int64_t *v_scale_strides, int64_t pages_stride,
                         void *stream) {
    const char *fn = "enatten_cache_append";
    int rc = check_cache_sizes(fn, B, heads, T, D, num_pages, page, columns, dtype, cache_dtype, pages_stride);
    if (rc) return rc;
    AppendArgs a{};
    if ((rc = set_rows(fn, "k", k, k_strides, heads, T, D, &a.x[0]))) return rc;
    if ((rc = set_rows(fn, "v", v, v_strides, heads, T, D, &a.x[1]))) return rc;
    if ((rc = set_cache(fn, "k", k_cache, k_scale, k_cache_strides, k_scale_strides, heads, page, D, 8, &a.c[0]))) return rc;
    if ((rc = set_cache(fn, "v", v_cache, v_scale, v_cache_strides, v_scale_strides, heads, page, D, 8, &a.c[1]))) return rc;
    if (!pages || !lengths) {
        set_error("%s: pages and lengths must not be NULL", fn);
        return ENATTEN_EINVAL;
    }
    a.tb = Table{pages, lengths, counts, pages_stride, num_pages, page, columns, T};
    a.B = B; a.heads = heads; a.D = D;
    a.touched = (T + page - 2) / page + 1;  // T tokens from any row of a page on
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case ENATTEN_F32: return launch_type<float>(fn, a, cache_dtype, st);
        case ENATTEN_BF16: return launch_type<__bf16>(fn, a, cache_dtype, st);
        default: return launch_type<_Float16>(fn, a, cache_dtype, st);
    }
}

#pragma GCC visibility pop
}  // extern "C"
