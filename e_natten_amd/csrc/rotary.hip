// Rotary positions for q and k: the first R channels of every row turn in pairs by the angle
// position * frequency, both tensors in one launch.
//
//   y1 = c x1 - s x2,  y2 = c x2 + s x1,  c = scale cos(p f), s = scale sin(p f)
//
// Every value is read and written once and takes three operations, so the kernel is bound by HBM.
// Sines and cosines depend on the token and the pair alone: a workgroup takes a few tokens, forms
// their R / 2 turns once into LDS and goes over the heads of both tensors with them.  Nothing is
// kept between calls, and no table bounds the positions.  With several axes (an image's rows and columns, a
// video's time besides) p is the pair's own of a token's positions; an axis that is not there gives NaN.
//
// Measured on MI355X: 8 + 8 heads of 64 channels, 4 x 16384 tokens, bfloat16: 56 us where rows lie
// [token, head] (4.8 TB/s, a plain copy of that size reaches 5.0), 46 us where they lie [head, token];
// 16 + 4 heads of 128, 64 of them turned, 2 x 8192 tokens, float16: 29 us; 64 single tokens: 3.5 us.
// 8 + 8 heads of 64 channels, 4 x 8192 tokens, by type: bfloat16 25 us, float32 48 (5.6 TB/s), float64 108 (5.0).
// Two axes, 4 + 4 heads of 128 channels, 4 images of 128 x 128 as a projection leaves them, bfloat16: 55 us (4.9 TB/s);
// three axes, 16 + 4 heads of 128, 96 of them turned, interleaved, 2 x 8192 tokens, float16: 30.9; 8 single tokens: 4.0.
// Stores past the caches take 47 us instead of 56, but the reader that follows pays: with one pass over
// both results behind it 114 us instead of 99.
#include "sequence_common.h"

namespace enatten {
namespace {

struct RotaryArgs {
    Rows x[2], y[2];  // q and k, in and out
    const void *positions, *frequencies;
    const int *axes;  // which of num_axes positions turns a pair; nullptr: there is one
    int64_t positions_stride, axis_stride;
    int num_axes;
    int heads[2];
    int B, T, D, R;
    bool wide_positions, wide_frequencies, head_first[2];
    float sign;  // -1: the other way round
    double scale;
    int tiles, slices, slice;  // token tiles per sequence; slices of `slice` heads of q and k together
    int batches;               // sequences of a workgroup, which have the same positions
};

template <typename S> struct Math { using type = float; };
template <> struct Math<double> { using type = double; };

template <typename S> __device__ __forceinline__ typename Math<S>::type widen(S x) { return (typename Math<S>::type)x; }

template <typename S, int VEC> struct alignas(VEC * sizeof(S)) Pack { S v[VEC]; };

// Far positions: the product with the frequency, and what it leaves over a whole turn, in double;
// 2^31 radians are then off by 2^-22.  What is left is at most half a turn, which float32 holds.
__device__ __forceinline__ void turn(double angle, float &c, float &s) {
    const double t = angle * 0.15915494309189535;
    sincospif((float)(2.0 * (t - rint(t))), &s, &c);
}
__device__ __forceinline__ void turn(double angle, double &c, double &s) { sincos(angle, &s, &c); }

// A unit of work is a pack of VEC channels: in the half layout one of the first channels of the pairs
// together with the one of the second channels, interleaved a pack of VEC / 2 pairs (with VEC 1 a single
// pair); behind the rotated channels a pack to copy.
// (AXES: whether there are several axes; asking for that in the kernel takes a single token 2.80 us instead of 2.68.
// SHARED: whether a workgroup has several sequences; with the loop over its only one 32 x 1024 tokens of 32 + 8 heads of
// 128 channels take 160 us instead of 142, and 65536 single tokens of one head with axes 87 instead of 72)
template <typename S, int VEC, bool INTERLEAVED, int TOKENS, bool AXES, bool SHARED>
__global__ __launch_bounds__(256) void rotary_turn(RotaryArgs a) {
    using C = typename Math<S>::type;
    struct alignas(2 * sizeof(C)) Turn { C c, s; };
    extern __shared__ __align__(16) char lds[];
    Turn *table = reinterpret_cast<Turn *>(lds);  // [TOKENS][R / 2]

    int block = blockIdx.x;
    const int slice = block % a.slices;
    block /= a.slices;
    const int tile = block % a.tiles, b0 = SHARED ? block / a.tiles * a.batches : block / a.tiles;
    const int t0 = tile * TOKENS, nt = min(TOKENS, a.T - t0), half = a.R / 2;
    auto position = [&](int64_t at) {
        return a.wide_positions ? (double)static_cast<const int64_t *>(a.positions)[at]
                                : (double)static_cast<const int *>(a.positions)[at];
    };
    auto frequency = [&](int f) {
        return a.wide_frequencies ? static_cast<const double *>(a.frequencies)[f]
                                  : (double)static_cast<const float *>(a.frequencies)[f];
    };
    if constexpr (AXES) {
        // The tokens' positions come into LDS at once: asked for pair by pair, behind its axis, they are waited for
        // in every round.
        constexpr int STAGED = 256;
        __shared__ double staged[STAGED];
        const bool few = a.num_axes <= STAGED / TOKENS;
        if (few) {
            for (int i = threadIdx.x; i < TOKENS * a.num_axes; i += 256)
                staged[i] = position(i / TOKENS * a.axis_stride + b0 * a.positions_stride + t0 + min(i % TOKENS, nt - 1));
            __syncthreads();
        }
        for (int i = threadIdx.x; i < nt * half; i += 256) {
            const int t = i / half, f = i - t * half, axis = a.axes[f];
            const bool there = (unsigned)axis < (unsigned)a.num_axes;
            const int at = there ? axis : 0;
            const double p =
                few ? staged[at * TOKENS + t] : position(at * a.axis_stride + b0 * a.positions_stride + t0 + t);
            C c, s;
            turn(p * frequency(f), c, s);
            if (!there) c = s = (C)NAN;
            table[i] = Turn{c * (C)a.scale, s * (C)a.scale * (C)a.sign};
        }
    } else {
        for (int i = threadIdx.x; i < nt * half; i += 256) {
            const int t = i / half, f = i - t * half;
            C c, s;
            turn(position(b0 * a.positions_stride + t0 + t) * frequency(f), c, s);
            table[i] = Turn{c * (C)a.scale, s * (C)a.scale * (C)a.sign};
        }
    }
    __syncthreads();

    constexpr bool IN_PACK = INTERLEAVED && VEC > 1;  // a pack holds whole pairs
    const int turned = IN_PACK ? a.R / VEC : half / VEC, units = turned + (a.D - a.R) / VEC;
    const int mate = INTERLEAVED ? 1 : half;          // where not: the second channel, so far behind the first
    const int h0 = slice * a.slice, h1 = min(h0 + a.slice, a.heads[0] + a.heads[1]);
    int b = b0;
    do {
#pragma unroll
    for (int which = 0; which < 2; which++) {
        const int lo = which ? max(h0 - a.heads[0], 0) : h0, hi = which ? h1 - a.heads[0] : min(h1, a.heads[0]);
        const int nh = hi - lo;
        if (nh <= 0) continue;
        const Rows &X = a.x[which], &Y = a.y[which];
        const S *x = static_cast<const S *>(X.ptr) + b * X.sb;
        S *y = static_cast<S *>(const_cast<void *>(Y.ptr)) + b * Y.sb;
        const bool head_first = a.head_first[which];
        const int total = nt * nh * units;
        // units whose loads are under way at a time: with 4 of them 50 us instead of 46 for the 4 x 16384
        // tokens above, and 109 instead of 108 with heads of 128
        constexpr int DEEP = 2;
        for (int i0 = threadIdx.x; i0 < total; i0 += 256 * DEEP) {
            Pack<S, VEC> u[DEEP], v[DEEP];
            int64_t to[DEEP];
            int ch[DEEP], tok[DEEP];
#pragma unroll
            for (int n = 0; n < DEEP; n++) {
                const int i = i0 + n * 256;
                ch[n] = -1;
                if (i < total) {
                    const int row = i / units, unit = i - row * units;
                    const int fast = head_first ? nh : nt, slow = row / fast, quick = row - slow * fast;
                    const int h = lo + (head_first ? quick : slow), t = head_first ? slow : quick;
                    const bool copy = unit >= turned;
                    const int c = copy ? a.R + (unit - turned) * VEC
                                       : INTERLEAVED && !IN_PACK ? 2 * unit : unit * VEC;
                    const S *p = x + h * X.sh + (t0 + t) * X.st + c;
                    ch[n] = c;
                    tok[n] = t;
                    to[n] = h * Y.sh + (t0 + t) * Y.st + c;
                    u[n] = *reinterpret_cast<const Pack<S, VEC> *>(p);
                    if (!IN_PACK && !copy) v[n] = *reinterpret_cast<const Pack<S, VEC> *>(p + mate);
                }
            }
#pragma unroll
            for (int n = 0; n < DEEP; n++) {
                if (ch[n] < 0) continue;
                if (ch[n] < a.R) {
                    if constexpr (IN_PACK) {
                        const Turn *w = table + tok[n] * half + ch[n] / 2;
#pragma unroll
                        for (int j = 0; j < VEC; j += 2) {
                            const C p = widen(u[n].v[j]), q = widen(u[n].v[j + 1]);
                            u[n].v[j] = (S)(p * w[j / 2].c - q * w[j / 2].s);
                            u[n].v[j + 1] = (S)(q * w[j / 2].c + p * w[j / 2].s);
                        }
                    } else {
                        const Turn *w = table + tok[n] * half + (INTERLEAVED ? ch[n] / 2 : ch[n]);
#pragma unroll
                        for (int j = 0; j < VEC; j++) {
                            const C p = widen(u[n].v[j]), q = widen(v[n].v[j]);
                            u[n].v[j] = (S)(p * w[j].c - q * w[j].s);
                            v[n].v[j] = (S)(q * w[j].c + p * w[j].s);
                        }
                        *reinterpret_cast<Pack<S, VEC> *>(y + to[n] + mate) = v[n];
                    }
                }
                *reinterpret_cast<Pack<S, VEC> *>(y + to[n]) = u[n];
            }
        }
    }
    } while (SHARED && ++b < min(b0 + a.batches, a.B));
}

template <typename S, int VEC, bool INTERLEAVED, bool AXES, bool SHARED>
void launch_turn(const RotaryArgs &a, int tokens, int blocks, size_t lds, hipStream_t st) {
    switch (tokens) {
        case 16: rotary_turn<S, VEC, INTERLEAVED, 16, AXES, SHARED><<<blocks, 256, lds, st>>>(a); break;
        case 8: rotary_turn<S, VEC, INTERLEAVED, 8, AXES, SHARED><<<blocks, 256, lds, st>>>(a); break;
        case 4: rotary_turn<S, VEC, INTERLEAVED, 4, AXES, SHARED><<<blocks, 256, lds, st>>>(a); break;
        case 2: rotary_turn<S, VEC, INTERLEAVED, 2, AXES, SHARED><<<blocks, 256, lds, st>>>(a); break;
        default: rotary_turn<S, VEC, INTERLEAVED, 1, AXES, SHARED><<<blocks, 256, lds, st>>>(a); break;
    }
}

template <typename S, int VEC, bool INTERLEAVED, bool AXES>
int launch_tokens(const char *fn, RotaryArgs &a, hipStream_t st) {
    const int heads = a.heads[0] + a.heads[1];
    // Tokens of a workgroup: its sines and cosines serve all heads of the slice.  With few tokens in
    // the call, fewer of them each, and then fewer heads, so that the chip has work.  With 8 at most the
    // single heads of 4 x 65536 tokens take 80 us instead of 38, since neighbours share fewer lines.
    int tokens = 16;
    while (tokens > 1 && ((int64_t)a.B * ((a.T + tokens - 1) / tokens) < 1024 ||
                          tokens * a.R * sizeof(typename Math<S>::type) > 32768))
        tokens /= 2;
    a.tiles = (a.T + tokens - 1) / tokens;
    a.slice = heads;
    a.slices = 1;
    while (a.slice > 4 && (int64_t)a.B * a.tiles * a.slices < 256) {
        a.slice = (a.slice + 1) / 2;
        a.slices = (heads + a.slice - 1) / a.slice;
    }
    // Up to four sequences with the same positions share a workgroup's sines and cosines where these count, with fewer
    // than 8 heads, and 2048 workgroups are left.  Both sides measured, us of each sequence by itself and together,
    // bfloat16 without axes: a head of 64 channels, 4 x 65536 tokens 30.5 and 19.1; 1 + 1 heads, 8 x 32768 tokens 37 and
    // 28; 2 + 2, 8 x 16384 28.2 and 25.1; 3 + 2, 16 x 4096, float16 18.5 and 17.2; 1 + 1 of 128, 8192 single tokens 14.3
    // and 13.8, but 27 with eight of them.  With more heads it does not pay: 4 + 4 of 128, 4 x 16384 tokens 46 and 48; 32 +
    // 8, 32 x 1024 141 and 149; 16 + 4, 16384 single tokens 31 and, 16 of them, 38.  With fewer workgroups neither: one
    // head of 128, 2048 single tokens 5.1 and 5.7.
    // With axes turns take longer, and it pays up to 8 heads and with 1024 workgroups left.  Two of them: the images of the
    // top 59.9 and 57.6 (55.9 and 55.2 in a graph), 4 + 4 heads of 64, 256 x 128 15.8 and 14.8, 8 x 8192 24.3 and 23.8, 3 +
    // 2, 16 x 4096, float16 20.0 and 17.7, but 4 + 4 of 128 that lie [token, head], 4 x 16384 46.3 and 48.6; 8 + 8 of
    // 64, 4 x 16384 45.4 and 47.6; 32 + 8 of 128, 32 x 1024 142 and 149.
    const auto blocks_of = [&](int64_t batches) { return (a.B + batches - 1) / batches * a.tiles * a.slices; };
    a.batches = 1;
    if (a.positions_stride == 0 && heads <= (AXES ? 8 : 7))
        while (a.batches < 4 && a.batches < a.B && blocks_of(2 * (int64_t)a.batches) >= (AXES ? 1024 : 2048)) a.batches *= 2;
    const int64_t blocks = blocks_of(a.batches);
    if (blocks > 0xffffff) {  // (2^32 threads)
        set_error("%s: too many tokens", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    const size_t lds = (size_t)tokens * a.R * sizeof(typename Math<S>::type);
    ProfScope prof(ENATTEN_KERNEL_ROTARY, "rotary_turn", st);
    if (a.batches > 1) launch_turn<S, VEC, INTERLEAVED, AXES, true>(a, tokens, (int)blocks, lds, st);
    else launch_turn<S, VEC, INTERLEAVED, AXES, false>(a, tokens, (int)blocks, lds, st);
    return launched(fn);
}

// Packs of 16 bytes where rows, pairs and copied channels are whole numbers of them, else single channels.
template <typename S, bool AXES>
int launch_type(const char *fn, RotaryArgs &a, bool interleaved, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(S);
    bool packed = (interleaved ? a.R : a.R / 2) % VEC == 0 && a.D % VEC == 0;
    for (int which = 0; which < (a.heads[1] ? 2 : 1); which++)
        for (const Rows *r : {&a.x[which], &a.y[which]})
            packed = packed && (uintptr_t)r->ptr % 16 == 0 && (r->sb | r->sh | r->st) % VEC == 0;
    if (interleaved)
        return packed ? launch_tokens<S, VEC, true, AXES>(fn, a, st) : launch_tokens<S, 1, true, AXES>(fn, a, st);
    return packed ? launch_tokens<S, VEC, false, AXES>(fn, a, st) : launch_tokens<S, 1, false, AXES>(fn, a, st);
}

template <typename S>
int launch_axes(const char *fn, RotaryArgs &a, bool interleaved, hipStream_t st) {
    return a.axes ? launch_type<S, true>(fn, a, interleaved, st) : launch_type<S, false>(fn, a, interleaved, st);
}

}  // namespace
}  // namespace enatten

using namespace enatten;

// axes: nullptr for one position per token
static int rotary_entry(const char *fn, const void *q, const void *k, void *q_out, void *k_out, const void *positions,
                        const void *frequencies, const int *axes, int num_axes, int B, int heads_q, int heads_k, int T,
                        int D, int R, int dtype, int positions_dtype, int frequencies_dtype, int interleaved,
                        int inverse, const int64_t *q_strides, const int64_t *k_strides,
                        const int64_t *q_out_strides, const int64_t *k_out_strides, int64_t positions_stride,
                        int64_t axis_stride, double scale, void *stream) {
    if (dtype != ENATTEN_F32 && dtype != ENATTEN_BF16 && dtype != ENATTEN_F16 && dtype != ENATTEN_F64) {
        set_error("%s: unknown dtype code %d (expected ENATTEN_F32/BF16/F16/F64)", fn, dtype);
        return ENATTEN_EINVAL;
    }
    if ((positions_dtype != ENATTEN_I32 && positions_dtype != ENATTEN_I64) ||
        (frequencies_dtype != ENATTEN_F32 && frequencies_dtype != ENATTEN_F64)) {
        set_error("%s: positions must be ENATTEN_I32 or I64, frequencies ENATTEN_F32 or F64", fn);
        return ENATTEN_EINVAL;
    }
    if (B < 1 || heads_q < 1 || heads_k < (k ? 1 : 0) || T < 1 || D < 1) {
        set_error("%s: every dimension must be >= 1, got B=%d heads=%d and %d T=%d D=%d", fn, B, heads_q, heads_k, T, D);
        return ENATTEN_EINVAL;
    }
    if (R < 2 || R % 2 || R > D || D > 1024) {
        set_error("%s: %d rotated channels must be even and at least 2, and fit a head_dim of %d (at most 1024)", fn,
                  R, D);
        return ENATTEN_EINVAL;
    }
    if (!positions || !frequencies || (k == nullptr) != (k_out == nullptr) || positions_stride < 0) {
        set_error("%s: positions and frequencies must not be NULL, k and k_out come together, strides are not negative", fn);
        return ENATTEN_EINVAL;
    }
    if ((int64_t)B * T * ((int64_t)heads_q + (k ? heads_k : 0)) > (int64_t)1 << 40 || heads_q > (1 << 20) ||
        heads_k > (1 << 20) || T > 0x7fffffff - 4096 || (int64_t)16 * ((int64_t)heads_q + heads_k) * D > 0x7fffffff) {
        set_error("%s: tensor too large", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    RotaryArgs a{};
    int rc;
    if ((rc = set_rows(fn, "q", q, q_strides, heads_q, T, D, &a.x[0]))) return rc;
    if ((rc = set_rows(fn, "q_out", q_out, q_out_strides, heads_q, T, D, &a.y[0]))) return rc;
    if (k) {
        if ((rc = set_rows(fn, "k", k, k_strides, heads_k, T, D, &a.x[1]))) return rc;
        if ((rc = set_rows(fn, "k_out", k_out, k_out_strides, heads_k, T, D, &a.y[1]))) return rc;
    }
    a.heads[0] = heads_q;
    a.heads[1] = k ? heads_k : 0;
    for (int which = 0; which < 2; which++) a.head_first[which] = a.x[which].sh < a.x[which].st;
    a.positions = positions;
    a.frequencies = frequencies;
    a.positions_stride = positions_stride;
    a.axes = axes;
    a.num_axes = num_axes;
    a.axis_stride = axis_stride;
    a.wide_positions = positions_dtype == ENATTEN_I64;
    a.wide_frequencies = frequencies_dtype == ENATTEN_F64;
    a.B = B; a.T = T; a.D = D; a.R = R;
    a.sign = inverse ? -1.f : 1.f;
    a.scale = scale;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case ENATTEN_F32: return launch_axes<float>(fn, a, interleaved, st);
        case ENATTEN_BF16: return launch_axes<__bf16>(fn, a, interleaved, st);
        case ENATTEN_F16: return launch_axes<_Float16>(fn, a, interleaved, st);
        default: return launch_axes<double>(fn, a, interleaved, st);
    }
}

extern "C" {
#pragma GCC visibility push(default)

int enatten_rotary(const void *q, const void *k, void *q_out, void *k_out, const void *positions,
                   const void *frequencies, int B, int heads_q, int heads_k, int T, int D, int R, int dtype,
                   int positions_dtype, int frequencies_dtype, int interleaved, int inverse,
                   const int64_t *q_strides, const int64_t *k_strides, const int64_t *q_out_strides,
                   const int64_t *k_out_strides, int64_t positions_stride, double scale, void *stream) {
    return rotary_entry("enatten_rotary", q, k, q_out, k_out, positions, frequencies, nullptr, 1, B, heads_q, heads_k, T,
                        D, R, dtype, positions_dtype, frequencies_dtype, interleaved, inverse, q_strides, k_strides,
                        q_out_strides, k_out_strides, positions_stride, 0, scale, stream);
}

int enatten_rotary_axes(const void *q, const void *k, void *q_out, void *k_out, const void *positions,
                        const void *frequencies, const int *axes, int num_axes, int B, int heads_q, int heads_k, int T,
                        int D, int R, int dtype, int positions_dtype, int frequencies_dtype, int interleaved,
                        int inverse, const int64_t *q_strides, const int64_t *k_strides,
                        const int64_t *q_out_strides, const int64_t *k_out_strides, int64_t positions_stride,
                        int64_t axis_stride, double scale, void *stream) {
    const char *fn = "enatten_rotary_axes";
    if (!axes || num_axes < 1 || axis_stride < 0) {
        set_error("%s: axes must not be NULL, there is one at least, and their stride is not negative", fn);
        return ENATTEN_EINVAL;
    }
    return rotary_entry(fn, q, k, q_out, k_out, positions, frequencies, axes, num_axes, B, heads_q, heads_k, T, D, R,
                        dtype, positions_dtype, frequencies_dtype, interleaved, inverse, q_strides, k_strides,
                        q_out_strides, k_out_strides, positions_stride, axis_stride, scale, stream);
}

#pragma GCC visibility pop
}  // extern "C"
