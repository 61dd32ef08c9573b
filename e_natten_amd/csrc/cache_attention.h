// What the kernels of cache_attention share: the split of a call's work, and codes to float16.
#pragma once

#include <type_traits>

#include "sequence_common.h"

namespace enatten {

struct AttnArgs {
    Rows q, o;
    Cache k, v;
    Table tb;
    int B, heads, group, heads_kv, T, D, window;  // group: query heads of a cache head
    int dtype;
    int row_tiles;   // per (sequence, cache head)
    int parts;       // workgroups per cache head that the split aims at; 0: one per row tile
    float scale;
    float *ws;       // (part_of)
};

// Sequences in runs that share their first tokens (cache_attention_shared.hip).  The first part of the work: an entry
// is a run, its rows are those of all its sequences, its tokens the shared ones; the second: an entry is a
// sequence with the tokens behind.  Types of their own, so that the other kernels' arguments stay what they are.
struct SharedArgs : AttnArgs {
    const int *shared;   // [runs], tokens
    int runs, size;      // sequences of a run
    // of the first part: what row_tiles, parts and ws are of the second; the items of a launch that are its own, which
    // come before the second part's; rows of a place of its workspace
    int first_tiles, first_parts, first_items, first_rows;
    float *first_ws;
};

// How a call is cut, from its sizes alone (the lengths are on the device).
struct Plan {
    int rows;       // of a tile
    int row_tiles;
    int parts;      // 0: one workgroup per row tile and cache head, no workspace
    int64_t items;  // workgroups per cache head
};

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFloor = -1e15f;  // the maximum of a row that has seen nothing: finite, below every logit
constexpr int kLeast = 256;       // tokens of a part at least: what a workgroup takes to get going pays from there
constexpr int kWideRows = 256;    // rows of those tiles
constexpr int kTop = 14;          // rows of q are brought to 2^kTop .. 2 * 2^kTop
constexpr int kPTop = 7;          // probabilities to 2^kPTop, and up to 2^kSlack times that where the
constexpr int kSlack = 8;         // running maximum is let lag behind

// The tokens that one row tile sees: [lo, hi), hi <= lo if none.
struct Span {
    int len, count, start, lo, hi;
    bool ok;
};
template <int ROWS>
__device__ __forceinline__ Span plain_span(const AttnArgs &a, int entry) {
    Span s;
    const int b = entry / a.row_tiles, tile = entry - b * a.row_tiles;
    s.ok = sequence_of(a.tb, b, s.len, s.count);
    s.start = s.len - s.count;
    const int first = tile * ROWS / a.group, last = min((tile * ROWS + ROWS - 1) / a.group, s.count - 1);
    s.lo = s.hi = 0;
    if (first < s.count) {
        s.lo = a.window ? max(s.start + first - a.window + 1, 0) : 0;
        s.hi = s.start + last + 1;
    }
    return s;
}
template <class Args> constexpr bool kShared = std::is_same_v<SharedArgs, Args>;
// (sequences or runs) x row tiles, and the rows that one of these has per cache head.  `first` wherever it stands: of
// the first part of a call with shared tokens.
template <class Args>
__device__ __forceinline__ int tiles_of(const Args &a, bool first) {
    if constexpr (kShared<Args>) return first ? a.first_tiles : a.row_tiles;
    else return a.row_tiles;
}
template <class Args>
__device__ __forceinline__ int entries_of(const Args &a, bool first) {
    if constexpr (kShared<Args>) return first ? a.runs * a.first_tiles : a.B * a.row_tiles;
    else return a.B * a.row_tiles;
}
template <class Args>
__device__ __forceinline__ int rows_of(const Args &a, bool first) {
    if constexpr (kShared<Args>) return a.T * a.group * (first ? a.size : 1);
    else return a.T * a.group;
}
template <class Args>
__device__ __forceinline__ int parts_of(const Args &a, bool first) {
    if constexpr (kShared<Args>) return first ? a.first_parts : a.parts;
    else return a.parts;
}
template <class Args>
__device__ __forceinline__ float *ws_of(const Args &a, bool first) {
    if constexpr (kShared<Args>) return first ? a.first_ws : a.ws;
    else return a.ws;
}
// How many tokens run r shares: whole pages.
__device__ __forceinline__ int shared_end(const SharedArgs &a, int r) {
    const int n = min(a.shared[r], a.tb.columns * a.tb.page);
    return n > 0 ? n / a.tb.page * a.tb.page : 0;
}
// ... and how many of them sequence b reads with its run: all, or none if its new tokens start before that end.
__device__ __forceinline__ int shared_by(const SharedArgs &a, int b, const Span &s) {
    const int end = shared_end(a, b / a.size);
    return s.ok && s.count > 0 && s.start >= end ? end : 0;
}
template <int ROWS, class Args>
__device__ __forceinline__ Span span_of(const Args &a, int entry, bool first) {
    if constexpr (kShared<Args>) {
        if (first) {
            const int r = entry / a.first_tiles;
            Span s{0, 0, 0, 0, shared_end(a, r), true};
            // (from the first token on that a row can see, as its own tokens are behind the shared ones: asking every
            // sequence of the run where it is took a run of 64 another 35 us)
            if (a.window) s.lo = max(s.hi + 1 - a.window, 0);
            return s;
        }
        Span s = plain_span<ROWS>(a, entry);
        if (s.hi > s.lo) s.lo = max(s.lo, shared_by(a, entry / a.row_tiles, s));
        return s;
    } else {
        return plain_span<ROWS>(a, entry);
    }
}
// steps of TOK tokens, from the group of 16 that holds the first one on
template <int TOK>
__device__ __forceinline__ int steps_of(const Span &s) { return s.hi > s.lo ? (s.hi - (s.lo & -16) + TOK - 1) / TOK : 0; }

// One workgroup's share: some steps of a row tile ("entry").  Entries are cut into items of at most
// `chunk` steps, about as many items as the call's `parts`; all items are equally long but the last of
// an entry.  Every wave finds its item from the lengths.
struct Share {
    int entry, first, items;  // entry < 0: nothing; the number of its first item, and how many it has
    int step0, step1, item;
};
// WAVES: how many waves share the steps of an item (each takes whole ones).
template <int ROWS, int TOK, int WAVES, class Args>
__device__ __forceinline__ Share share_of(const Args &a, int item, bool first) {
    Share w;
    w.item = item;
    const int entries = entries_of(a, first), lane = threadIdx.x & 63;
    auto steps_at = [&](int e) { return e < entries ? steps_of<TOK>(span_of<ROWS>(a, e, first)) : 0; };
    float total = 0.f;
    int steps = 0;
    for (int e0 = 0; e0 < entries; e0 += 64) {
        steps = steps_at(e0 + lane);
        total += (float)(unsigned)__builtin_amdgcn_readlane(running_sum(steps), 63);
    }
    // (a little more than the quotient: the items are at most `parts` and one for every entry)
    const int each = (int)(total * 1.00001f / parts_of(a, first)) + 1;
    int chunk = max(kLeast / TOK, each + WAVES - 1) / WAVES * WAVES;
    if constexpr (kShared<Args>) {
        if (first) {  // no more items than parts: all of them start at once
            if (entries > 64) chunk = (max(kLeast / TOK, (int)(total * 1.00001f / (parts_of(a, first) - entries)) + 1) + WAVES - 1) / WAVES * WAVES;
            else
                for (;;) {
                    const int n = lane < entries ? max(1, (steps + chunk - 1) / chunk) : 0;
                    const int all = __builtin_amdgcn_readlane(running_sum(n), 63);
                    if (all <= parts_of(a, first)) break;
                    chunk = max(chunk + WAVES, (int)((int64_t)chunk * all / parts_of(a, first)) / WAVES * WAVES);
                }
        }
    }
    int before = 0;
    for (int e0 = 0; e0 < entries; e0 += 64) {
        const int e = e0 + lane;
        if (entries > 64) steps = steps_at(e);
        const int n = e < entries ? max(1, (steps + chunk - 1) / chunk) : 0;
        const int upto = before + running_sum(n);
        const unsigned long long who = __ballot(item >= upto - n && item < upto);
        if (who) {
            const int l = __ffsll(who) - 1;
            w.entry = e0 + l;
            w.items = __builtin_amdgcn_readlane(n, l);
            w.first = __builtin_amdgcn_readlane(upto, l) - w.items;
            const int all = __builtin_amdgcn_readlane(steps, l);
            w.step0 = min((item - w.first) * chunk, all);
            w.step1 = min(w.step0 + chunk, all);
            return w;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    w.entry = -1;
    return w;
}

// Equal shares of a different kind, for tiles of many rows: the steps of all row tiles of all cache heads
// in one line (heads, then sequences, then row tiles; a tile without steps counts as one, so that its
// rows are written), cut into `parts` ranges.  A range takes what is left of a tile, whole tiles, and the
// beginning of one; only tiles that are cut have parts to join, and every workgroup has the same work.
constexpr int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
constexpr int64_t item_floats(int rows, int D) { return (int64_t)rows * (D + 2); }  // maxima, sums, sums of values
struct Ranges {
    int64_t line, each;  // steps of one cache head, of one range
    bool whole;          // no more tiles than ranges, and nearly as long as those: a tile each, none cut
};
template <int ROWS, int TOK, class Args>
__device__ __forceinline__ int counted_steps(const Args &a, int e, bool first) {
    return e < entries_of(a, first) ? max(1, steps_of<TOK>(span_of<ROWS>(a, e, first))) : 0;
}
template <int ROWS, int TOK, class Args>
__device__ __forceinline__ Ranges ranges_of(const Args &a, bool first) {
    const int entries = entries_of(a, first), lane = threadIdx.x & 63;
    Ranges r{0, 0, false};
    int most = 0;
    for (int e0 = 0; e0 < entries; e0 += 64) {
        const int n = counted_steps<ROWS, TOK>(a, e0 + lane, first);
        most = max(most, n);
        r.line += (unsigned)__builtin_amdgcn_readlane(running_sum(n), 63);
    }
    const int parts = parts_of(a, first);
    r.each = (r.line * a.heads_kv + parts - 1) / parts;
    if (first) {  // all tiles leave parts; ranges of 128 tokens at least
        r.each = max(r.each, (int64_t)(128 / TOK));
        return r;
    }
    // The parts of cut tiles are their rows' sums in float32, written and read, which takes as long as some
    // steps: at 128 channels about 2 for 64 tiles of 256 rows.  A tile for every workgroup pays where the
    // longest is hardly longer than that beyond the mean.  2048 tokens each of 16384 and 12288 (256 tiles
    // of 224 steps on average, 256 at most): 506 us cut, 570 whole; 256 tokens each of 8 sequences of 300
    // (128 tiles of 5): 37 us cut, 27 whole; half as many tiles: 21 us cut, 24 whole.
    const int64_t tiles = (int64_t)entries * a.heads_kv;
    const int64_t steps = tiles * min(ROWS, rows_of(a, first)) * padded(a.D) >> 20;
    r.whole = tiles <= a.parts && !__any(most > r.each + steps);
    return r;
}
// The row tile at step `y` of a head's line, and how far into it that is
template <int ROWS, int TOK, class Args>
__device__ __forceinline__ int tile_at(const Args &a, int64_t y, int &into, bool first) {
    const int entries = entries_of(a, first), lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < entries; e0 += 64) {
        const unsigned n = counted_steps<ROWS, TOK>(a, e0 + lane, first), upto = running_sum(n);
        const unsigned all = __builtin_amdgcn_readlane(upto, 63);
        if (y < all) {
            const unsigned long long who = __ballot((unsigned)y < upto);
            const int l = __ffsll(who) - 1;
            into = (int)((unsigned)y - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l)));
            return e0 + l;
        }
        y -= all;
    }
    into = 0;
    return -1;
}
// Workspace of the ranges: for each the number of the tile that it starts within, or -1; then two slots
// each, for the tile that it starts within and for the one that it ends within.
__device__ __forceinline__ float *slot_of(const AttnArgs &a, int slot) {
    return a.ws + (a.parts + 3) / 4 * 4 + slot * item_floats(kWideRows, padded(a.D));
}

// The workspace: first item and items of every entry, then for every (item, cache head) the maxima and
// sums of its rows and rows x D sums of values.
__host__ __device__ inline int64_t head_floats(int64_t entries) { return (2 * entries + 3) / 4 * 4; }
template <class Args>
__device__ __forceinline__ float *part_of(const Args &a, int rows, int item, int head, bool first) {
    return ws_of(a, first) + head_floats((int64_t)entries_of(a, first)) + ((int64_t)item * a.heads_kv + head) * item_floats(rows, a.D);
}
// (for the launch that joins the parts)
template <class Args>
__device__ __forceinline__ void note_share(const Args &a, const Share &w, int head, bool first) {
    if (w.item == w.first && head == 0 && threadIdx.x == 0) {
        int *note = reinterpret_cast<int *>(ws_of(a, first)) + 2 * w.entry;
        note[0] = w.first;
        note[1] = w.items;
    }
}

__device__ __forceinline__ f16x2 as_half(unsigned x) { return __builtin_bit_cast(f16x2, x); }

// Two codes side by side as float16: int8 in the lower byte of halves of 0x6400, offset by 128; E4M3 in
// the upper byte of each half: sign, 4 exponent and 3 mantissa bits move to the places of float16's,
// whose exponents are offset by 8 more, which gives the value times 2^-8.
__device__ __forceinline__ f16x2 from_int8(unsigned x) {
    return as_half(x) + f16x2{(_Float16)-1152.f, (_Float16)-1152.f};
}
__device__ __forceinline__ f16x2 from_e4m3(unsigned x) {
    const s16x2 s = __builtin_bit_cast(s16x2, x) >> 1;
    return as_half(__builtin_bit_cast(unsigned, s) & 0xbfffbfffu);
}
// The conversion instruction gives the same and takes half the operations, but NaN for the codes 0x7f
// and 0xff: only where every row sees the tokens (a weight of 0 would not hide a NaN).
template <bool HIGH>
__device__ __forceinline__ f16x2 from_e4m3_word(unsigned x) {
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 0x1p-8f, HIGH));
}
// 8 consecutive codes
template <bool E4M3, bool SEEN>
__device__ __forceinline__ f16x8 widen_row(unsigned x0, unsigned x1) {
    f16x2 h[4];
    if constexpr (E4M3 && SEEN) {
        h[0] = from_e4m3_word<false>(x0);
        h[1] = from_e4m3_word<true>(x0);
        h[2] = from_e4m3_word<false>(x1);
        h[3] = from_e4m3_word<true>(x1);
    } else if constexpr (E4M3) {
        h[0] = from_e4m3(__builtin_amdgcn_perm(x0, x0, 0x010c000cu));
        h[1] = from_e4m3(__builtin_amdgcn_perm(x0, x0, 0x030c020cu));
        h[2] = from_e4m3(__builtin_amdgcn_perm(x1, x1, 0x010c000cu));
        h[3] = from_e4m3(__builtin_amdgcn_perm(x1, x1, 0x030c020cu));
    } else {
        x0 ^= 0x80808080u;
        x1 ^= 0x80808080u;
        h[0] = from_int8(__builtin_amdgcn_perm(0x64646464u, x0, 0x04010400u));
        h[1] = from_int8(__builtin_amdgcn_perm(0x64646464u, x0, 0x04030402u));
        h[2] = from_int8(__builtin_amdgcn_perm(0x64646464u, x1, 0x04010400u));
        h[3] = from_int8(__builtin_amdgcn_perm(0x64646464u, x1, 0x04030402u));
    }
    return f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}
// 4 channels (one word) of 8 tokens, transposed: out[i] is channel i of the 8 tokens
template <bool E4M3, bool SEEN>
__device__ __forceinline__ void widen_columns(const unsigned (&t)[8], f16x8 (&out)[4]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f16x2 h[4];
        if constexpr (E4M3 && !SEEN) {
            h[0] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x040c000cu));
            h[1] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x050c010cu));
            h[2] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x060c020cu));
            h[3] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x070c030cu));
        } else {
            // channel by channel the two tokens' codes
            unsigned lo = __builtin_amdgcn_perm(t[j + 1], t[j], 0x05010400u);
            unsigned hi = __builtin_amdgcn_perm(t[j + 1], t[j], 0x07030602u);
            if constexpr (E4M3) {
                h[0] = from_e4m3_word<false>(lo);
                h[1] = from_e4m3_word<true>(lo);
                h[2] = from_e4m3_word<false>(hi);
                h[3] = from_e4m3_word<true>(hi);
            } else {
                lo ^= 0x80808080u;
                hi ^= 0x80808080u;
                h[0] = from_int8(__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u));
                h[1] = from_int8(__builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u));
                h[2] = from_int8(__builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u));
                h[3] = from_int8(__builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            out[i][j] = h[i][0];
            out[i][j + 1] = h[i][1];
        }
    }
}

// A value scale that is not finite counts as NaN.
__device__ __forceinline__ float finite_or_nan(float z) { return fabsf(z) < INFINITY ? z : __uint_as_float(0x7fc00000u); }

// The value scales z' of the groups go into the probabilities relative to the largest power of two of
// them so far, 2^ref, times 2^kPTop.  `grow` brings ref up to date and returns what the sums so far are
// multiplied by.  (ref is the same in all lanes; `top` is log2 of the step's largest z'.)
__device__ __forceinline__ float grow(float &ref, float top) {
    if (!(top > ref)) return 1.f;
    const float old = ref;
    ref = ceilf(top);
    return __builtin_amdgcn_exp2f(old - ref);
}
// log2 of a group's factor.  Scales of 0 and far below the largest go in with a weight that float16
// drops, whatever the codes; NaN stays.
__device__ __forceinline__ float log_weight(float log_z, float ref) {
    const float x = log_z + ((float)kPTop - ref);
    return x < -40.f ? -40.f : x;
}
// For float32, where the last bits of log2 and exp2 would show, the factor itself.
__device__ __forceinline__ float plain_weight(float z, float ref) {
    const float x = __builtin_ldexpf(z, kPTop - (int)ref);
    return x < 0x1p-40f ? 0x1p-40f : x;
}
// Two values as two float16 terms each.  The compiler may form the rounded value twice, once of the
// rounded product that x is and once fused with that product; what is left has to be that of the one
// that is used.
__device__ __forceinline__ void two_terms(float x, float y, f16x2 &high, f16x2 &low) {
    unsigned w = __builtin_bit_cast(unsigned, f16x2{(_Float16)x, (_Float16)y});
    asm("" : "+v"(w));
    high = as_half(w);
    low = f16x2{(_Float16)(x - (float)high[0]), (_Float16)(y - (float)high[1])};
}
// Whether the sum of probabilities may be formed of what the second product takes, rounded to float16:
// then a rounding moves a weight in both, and the result stays a mean of values.  A group far below the
// largest scale has weights that float16 drops; they count in the sum all the same.
__device__ __forceinline__ bool close(float lz) { return __builtin_amdgcn_readfirstlane(lz >= 0.f); }
// What divides the factor out of a sum; 0 for NaN, which the sum of a row that sees such a group has
// itself, and one that does not is 0.
__device__ __forceinline__ float inverse_weight(float lz) { return lz == lz ? __builtin_amdgcn_exp2f(-lz) : 0.f; }
// 2^e, also where that is a number under 2^-126 (for which exp2 gives 0): products with it are exact while the
// result is not under 2^-126 itself.
__device__ __forceinline__ float power_of_two(float e) { return __builtin_ldexpf(1.f, (int)e); }
// sum of four float16 values in float32
__device__ __forceinline__ float sum4(_Float16 a, _Float16 b, _Float16 c, _Float16 d, float more) {
    const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
    return __builtin_amdgcn_fdot2(f16x2{c, d}, one, __builtin_amdgcn_fdot2(f16x2{a, b}, one, more, false), false);
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// max / sum over the lanes l, l ^ 32
__device__ __forceinline__ float pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// ... over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float row_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float row_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// N channels of a row, N a multiple of 8; rows lie at multiples of 16 bytes.  DT: the type, a constant, as
// what is done once per workgroup is paid by its size: code that was not run before comes from memory.
template <int DT, int N>
__device__ __forceinline__ void load_channels(const Rows &r, int64_t at, float (&x)[N]) {
    if constexpr (DT == ENATTEN_F32) {
        const float *p = static_cast<const float *>(r.ptr) + at;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 y = *reinterpret_cast<const f32x4 *>(p + i);
#pragma unroll
            for (int j = 0; j < 4; j++) x[i + j] = y[j];
        }
    } else {
        const unsigned short *p = static_cast<const unsigned short *>(r.ptr) + at;
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(p + i);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (DT == ENATTEN_BF16) x[i + j] = __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
                else x[i + j] = (float)as_half(w[j / 2])[j % 2];
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ u32x2 narrow4(f32x4 x) {
    u32x2 y;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if constexpr (DT == ENATTEN_BF16) {
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            y[i] = __builtin_bit_cast(unsigned, bf16x2{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
        } else {
            y[i] = __builtin_bit_cast(unsigned, f16x2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
        }
    }
    return y;
}
// 4 channels of a row
template <int DT>
__device__ __forceinline__ void store_channels(const Rows &r, int64_t at, f32x4 x) {
    if constexpr (DT == ENATTEN_F32) *reinterpret_cast<f32x4 *>(static_cast<float *>(const_cast<void *>(r.ptr)) + at) = x;
    else *reinterpret_cast<u32x2 *>(static_cast<unsigned short *>(const_cast<void *>(r.ptr)) + at) = narrow4<DT>(x);
}

// A row of an entry: sequence, new token, query head.
struct Place {
    int b, t, head;
};
template <class Args>
__device__ __forceinline__ Place place_of(const Args &a, int which, int head, int row, bool first) {  // which: sequence or run
    Place p{which, row / a.group, 0};
    p.head = head * a.group + row - p.t * a.group;
    if constexpr (kShared<Args>) {
        if (first) {
            const int i = p.t / a.T;
            p.b = which * a.size + i;
            p.t -= i * a.T;
        }
    }
    return p;
}
__device__ __forceinline__ int64_t offset_of(const Rows &r, const Place &p) { return p.b * r.sb + p.head * r.sh + p.t * r.st; }

// Parts of the first part's tiles of many rows.  Tiles and ranges that have one in common follow each other like steps
// of a staircase, so that (range + tile) is a place of its own for each such pair.  Before the places for every tile
// its first and its last range; a place has the maxima of its rows, their sums, and the sums of values in the order of
// the registers.
__device__ __forceinline__ float *stair_of(const SharedArgs &a, int64_t place) {
    const int64_t tiles = (int64_t)a.runs * a.first_tiles * a.heads_kv;
    return a.first_ws + (2 * tiles + 3) / 4 * 4 + place * item_floats(a.first_rows, padded(a.D));
}

__device__ __forceinline__ float lane_float(float x, int l) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l));
}
__device__ __forceinline__ int64_t lane_offset(int64_t x, int l) {
    const unsigned lo = __builtin_amdgcn_readlane((int)x, l), hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

}  // namespace

// Tiles of kWideRows rows (cache_attention_rows.hip), a.parts ranges
int launch_attend_rows(const char *fn, const AttnArgs &a, bool e4m3, hipStream_t st);
// Tiles of many rows of the first part, and the join behind both (cache_attention_shared_rows.hip)
int launch_first_rows(const char *fn, const SharedArgs &a, int rows, bool e4m3, hipStream_t st);
int launch_last_join(const char *fn, const SharedArgs &a, int rows, int second_rows, hipStream_t st);
// A call without shared tokens, its arguments checked; plans without tiles of kWideRows rows are not `wide`
int launch_plain(const char *fn, AttnArgs a, const Plan &p, void *workspace, bool e4m3, hipStream_t st);
Plan plan_of(int B, int heads, int heads_kv, int T, int D, int page, int columns, int window, int dtype, bool wide = true);
size_t workspace_bytes(const Plan &p, int B, int heads_kv, int D);  // B: sequences, or runs
// The arguments that all calls have, checked, but for row_tiles, parts and ws
int set_attention(const char *fn, const void *q, const void *k_cache, const void *v_cache, const float *k_scale,
                  const float *v_scale, const int *pages, const int *lengths, const int *counts, void *o, int B, int heads,
                  int heads_kv, int T, int D, int num_pages, int page, int columns, int kernel_size, int dtype,
                  int cache_dtype, const int64_t *q_strides, const int64_t *o_strides, const int64_t *k_cache_strides,
                  const int64_t *v_cache_strides, const int64_t *k_scale_strides, const int64_t *v_scale_strides,
                  int64_t pages_stride, float scale, AttnArgs *a);

}  // namespace enatten
