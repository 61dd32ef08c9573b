// What the kernels of cache_attention share: the split of a call's work, and codes to float16.
#pragma once

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
    float *ws;       // [item][cache head]: row maxima, row sums, rows x D sums
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
constexpr float kFloor = -1e37f;  // the maximum of a row that has seen nothing: finite, below every logit
constexpr int kLeast = 256;       // tokens of a part at least: what a workgroup takes to get going pays from there
constexpr int kTop = 14;          // float16 operands are brought to 2^kTop

// The tokens that one row tile sees: [lo, hi), hi <= lo if none.
struct Span {
    int len, count, start, lo, hi;
    bool ok;
};
template <int ROWS>
__device__ __forceinline__ Span span_of(const AttnArgs &a, int entry) {
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
// steps of TOK tokens, from the group of 16 that holds the first one on
template <int TOK>
__device__ __forceinline__ int steps_of(const Span &s) { return s.hi > s.lo ? (s.hi - (s.lo & -16) + TOK - 1) / TOK : 0; }

// How the row tiles ("entries") are cut into items of at most `chunk` steps; the same in every wave.
__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}
template <int ROWS, int TOK>
__device__ __forceinline__ int chunk_of(const AttnArgs &a) {
    const int entries = a.B * a.row_tiles, lane = threadIdx.x & 63;
    long long total = 0;
    for (int e0 = 0; e0 < entries; e0 += 64) {
        const int e = e0 + lane;
        total += wave_sum(e < entries ? steps_of<TOK>(span_of<ROWS>(a, e)) : 0);
    }
    return max(kLeast / TOK, (int)((total + a.parts - 1) / a.parts));
}
__device__ __forceinline__ int items_of(int steps, int chunk) { return max(1, (steps + chunk - 1) / chunk); }
// The entry of item `item` and the number of its first item, or (by_entry) the first item of entry
// `item`; entry -1 if there is none.
template <int ROWS, int TOK>
__device__ __forceinline__ void find(const AttnArgs &a, int chunk, int item, bool by_entry, int &entry, int &first) {
    const int entries = a.B * a.row_tiles, lane = threadIdx.x & 63;
    int before = 0;
    entry = -1;
    first = 0;
    for (int e0 = 0; e0 < entries; e0 += 64) {
        const int e = e0 + lane;
        const int n = e < entries ? items_of(steps_of<TOK>(span_of<ROWS>(a, e)), chunk) : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o, 64);
            if (lane >= o) upto += x;
        }
        const bool mine = by_entry ? e == item : n > 0 && item >= before + upto - n && item < before + upto;
        const unsigned long long who = __ballot(mine);
        if (who) {
            const int l = __ffsll(who) - 1;
            entry = e0 + l;
            first = before + __shfl(upto - n, l, 64);
            return;
        }
        before += __shfl(upto, 63, 64);
    }
}

__device__ __forceinline__ f16x2 as_half(unsigned x) { return __builtin_bit_cast(f16x2, x); }

// Two codes side by side, each in the upper byte of a half (E4M3) or the lower byte of a half of
// 0x6400 (int8, offset 128), as float16.  E4M3: sign, 4 exponent and 3 mantissa bits move to the places
// of float16's, whose exponents are offset by 8 more: the value times 2^-8.
__device__ __forceinline__ f16x2 from_e4m3(unsigned x) {
    const s16x2 s = __builtin_bit_cast(s16x2, x) >> 1;
    return as_half(__builtin_bit_cast(unsigned, s) & 0xbfffbfffu);
}
__device__ __forceinline__ f16x2 from_int8(unsigned x) {
    return as_half(x) + f16x2{(_Float16)-1152.f, (_Float16)-1152.f};
}
// 8 consecutive codes
template <bool E4M3>
__device__ __forceinline__ f16x8 widen_row(unsigned x0, unsigned x1) {
    f16x2 h[4];
    if constexpr (E4M3) {
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
template <bool E4M3>
__device__ __forceinline__ void widen_columns(const unsigned (&t)[8], f16x8 (&out)[4]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f16x2 h[4];
        if constexpr (E4M3) {
            h[0] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x040c000cu));
            h[1] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x050c010cu));
            h[2] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x060c020cu));
            h[3] = from_e4m3(__builtin_amdgcn_perm(t[j + 1], t[j], 0x070c030cu));
        } else {
            const unsigned lo = __builtin_amdgcn_perm(t[j + 1], t[j], 0x05010400u) ^ 0x80808080u;
            const unsigned hi = __builtin_amdgcn_perm(t[j + 1], t[j], 0x07030602u) ^ 0x80808080u;
            h[0] = from_int8(__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u));
            h[1] = from_int8(__builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u));
            h[2] = from_int8(__builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u));
            h[3] = from_int8(__builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            out[i][j] = h[i][0];
            out[i][j + 1] = h[i][1];
        }
    }
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// max / sum over the four lanes of a row
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float row_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

__device__ __forceinline__ float load_row(const Rows &r, int dtype, int64_t at) {
    if (dtype == ENATTEN_F32) return static_cast<const float *>(r.ptr)[at];
    if (dtype == ENATTEN_BF16) return (float)static_cast<const __bf16 *>(r.ptr)[at];
    return (float)static_cast<const _Float16 *>(r.ptr)[at];
}
__device__ __forceinline__ void store_row(const Rows &r, int dtype, int64_t at, float x) {
    void *p = const_cast<void *>(r.ptr);
    if (dtype == ENATTEN_F32) static_cast<float *>(p)[at] = x;
    else if (dtype == ENATTEN_BF16) static_cast<__bf16 *>(p)[at] = (__bf16)x;
    else static_cast<_Float16 *>(p)[at] = (_Float16)x;
}

__device__ __forceinline__ int lane_int(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
__device__ __forceinline__ float lane_float(float x, int l) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l));
}
__device__ __forceinline__ int64_t lane_offset(int64_t x, int l) {
    const unsigned lo = __builtin_amdgcn_readlane((int)x, l), hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// Floats of one item's part of the workspace
constexpr int64_t item_floats(int rows, int D) { return (int64_t)rows * (D + 2); }

}  // namespace

// Tiles of kWideRows rows (cache_attention_rows.hip)
constexpr int kWideRows = 256;
int launch_attend_rows(const char *fn, const AttnArgs &a, bool e4m3, int64_t blocks, hipStream_t st);

}  // namespace enatten
