// The kernels of cache_attention.hip as functions, for calls of sequences by themselves and of runs that share
// their first tokens (cache_attention_shared.hip); the mathematics stands in the former.
#pragma once

#include "cache_attention.h"

namespace enatten {
namespace {

// The sequence of run r whose row of the table names the shared pages: the first that reads them; -1: none.
__device__ __forceinline__ int reader_of(const SharedArgs &a, int r, int end) {
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < a.size; i0 += 64) {
        int len, count;
        const bool reads = i0 + lane < a.size && sequence_of(a.tb, r * a.size + i0 + lane, len, count) && count > 0 &&
                           len - count >= end;
        const unsigned long long who = __ballot(reads);
        if (who) return r * a.size + i0 + __ffsll(who) - 1;
    }
    return -1;
}
// The first shared token that a row sees.
__device__ __forceinline__ int shared_lo(const SharedArgs &a, const Place &p, int end) {
    int len, count;
    if (!a.window || !sequence_of(a.tb, p.b, len, count) || p.t >= count || len - count < end) return 0;
    return min(max(len - count + p.t + 1 - a.window, 0), end);
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = max(x, __shfl_xor(x, o, 64));
    return __builtin_amdgcn_readfirstlane(x);
}

constexpr int kTile = 32;  // tokens of a step of a wave

// Waves per SIMD that the registers allow: the sums, q, logits and probabilities of every row tile, and
// two tiles of codes.
constexpr int waves_of(int DP, int R, int TERMS) {
    const int need = R * (DP / 4 + DP / 8 * TERMS + 8 + 4 * TERMS) + DP / 2 + 88;
    return need <= 168 ? 3 : need <= 256 ? 2 : 1;
}

// Whether steps that every row sees go the way of those that only some see.  With a form for either the
// widest tiles need more registers than there are (22 to 500 were spilled), and a spilled operand of a
// matrix instruction can come back incomplete: a part that the compiler keeps in an accumulation register
// is not restored into an operand that lies in such registers.  No kernel here may spill.
constexpr bool one_form(int DP, int R) { return DP * R > 256 || DP == 256; }

// DP: head_dim rounded up to 64, 128 or 256 (channels beyond D: zeros in q, any codes); R: row tiles of
// 16 per workgroup; TERMS: float16 terms of q and p.
template <int DP, int R, bool E4M3, int DT, class Args>
__device__ __forceinline__ void attend_body(const Args &a) {
    constexpr int TERMS = DT == ENATTEN_F32 ? 2 : 1, TOK = kTile, ROWS = 16 * R, KC = DP / 64, VW = DP / 64, CW = DP / 16;
    constexpr bool ONE_FORM = one_form(DP, R);
    const int lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (branches on it are the wave's)

    // which row tile, and which of its steps
    const int head = blockIdx.x % a.heads_kv;
    int item = blockIdx.x / a.heads_kv;
    bool first = false;
    if constexpr (kShared<Args> && R == 1) {
        first = item < a.first_items;
        if (!first) item -= a.first_items;
    }
    const int parts = parts_of(a, first);
    Share w;
    if (parts) {
        w = share_of<ROWS, TOK, 4>(a, item, first);
        if (w.entry < 0) return;
        note_share(a, w, head, first);
    } else {
        w.entry = w.item = item;
        w.items = 1;
    }
    const int entry = w.entry;
    const Span s = span_of<ROWS>(a, entry, first);
    if (!parts) {
        w.step0 = 0;
        w.step1 = steps_of<TOK>(s);
    }
    const int which = entry / tiles_of(a, first), row0 = (entry - which * tiles_of(a, first)) * ROWS;
    int b = which, joins = 0;  // joins: shared tokens, which are not the second part's
    const int all_rows = rows_of(a, first);
    int step0 = w.step0, step1 = w.step1;
    if constexpr (kShared<Args>) {
        if (first) {
            if (s.hi == 0) return;  // (a run that shares nothing leaves nothing)
            b = reader_of(a, which, s.hi);
            if (b < 0) b = which * a.size, step0 = step1 = 0;  // (nobody reads them)
        } else {
            joins = shared_by(a, which, s);
        }
    }
    const int base = s.lo & -16;

    // q: lane (row n16, g4) has channels 64 c + 16 g4 .. + 15
    f16x8 qf[R][KC][2][TERMS];
    float unit[R];           // what a product of codes is multiplied by, besides z: log2 units, not negative
    const float flip = a.scale < 0.f ? -1.f : 1.f;
    int lo_r[R], hi_r[R];    // tokens that the lane's row sees
    int most_lo = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = min(row0 + r * 16 + n16, all_rows - 1);
        const Place where = place_of(a, which, head, row, first);
        const int tv = min(where.t, max(s.count - 1, 0));
        hi_r[r] = s.start + tv + 1;
        lo_r[r] = a.window ? max(hi_r[r] - a.window, 0) : 0;
        if constexpr (kShared<Args>) {
            lo_r[r] = max(lo_r[r], joins);
            if (first) {
                hi_r[r] = s.hi;  // (rows of a sequence that does not share them come to what nobody reads)
                lo_r[r] = shared_lo(a, where, s.hi);
                if (a.window) most_lo = max(most_lo, lo_r[r]);
            }
        }
        const int64_t at = offset_of(a.q, where);
        float x[KC][16], top = 0.f, nan = a.scale * 0.f;
#pragma unroll
        for (int c = 0; c < KC; c++) {
#pragma unroll
            for (int j = 0; j < 16; j++) x[c][j] = 0.f;
            if (c * 64 + g4 * 16 < a.D) load_channels<DT>(a.q, at + c * 64 + g4 * 16, x[c]);
        }
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                top = fmaxf(top, fabsf(x[c][j]));
                nan += x[c][j] * 0.f;  // a value that is not finite makes its row NaN, the factor all rows
            }
        nan = row_sum(nan);
        top = row_max(top);
        const int e = top > 0.f ? __builtin_amdgcn_frexp_expf(top) : 0;
        const int up = kTop + 1 - e;  // the largest to 2^14 .. 2^15
        unit[r] = __builtin_ldexpf(fabsf(a.scale) * kLog2e, -up + (E4M3 ? 8 : 0)) + nan;
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float y0 = __builtin_ldexpf(x[c][j] * flip, up), y1 = __builtin_ldexpf(x[c][j + 1] * flip, up);
                f16x8 &w = qf[r][c][j / 8][0];
                if constexpr (TERMS == 2) {
                    f16x2 high, low;
                    two_terms(y0, y1, high, low);
                    w[j % 8] = high[0];
                    w[j % 8 + 1] = high[1];
                    qf[r][c][j / 8][1][j % 8] = low[0];
                    qf[r][c][j / 8][1][j % 8 + 1] = low[1];
                } else {
                    w[j % 8] = (_Float16)y0;
                    w[j % 8 + 1] = (_Float16)y1;
                }
            }
    }
    // between these all rows see every token
    int all_lo = a.window ? max(s.start + min((row0 + ROWS - 1) / a.group, s.count - 1) + 1 - a.window, 0) : 0;
    int all_hi = s.start + row0 / a.group + 1;
    if constexpr (kShared<Args>) {
        all_lo = max(all_lo, joins);
        if (first) {
            all_lo = a.window ? wave_max(most_lo) : 0;
            all_hi = s.hi;
        }
    }

    f32x4 acc[R][CW];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        m[r] = kFloor;
        l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < CW; i++) acc[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float ref = -126.f;  // the z' so far are at most 2^ref

    // the wave's steps, and the places of their two groups of 16 tokens: lane i holds group `filled` + i
    const int quarter = (step1 - step0 + 3) / 4;
    const int w0 = min(step0 + wave * quarter, step1), w1 = min(w0 + quarter, step1);
    int filled = -64;
    int64_t k_at = 0, v_at = 0;
    float k_z = 0.f, v_z = 0.f;
    auto fill = [&](int group) {
        filled = group;
        const int token = base + (group + lane) * 16;
        k_at = v_at = 0;
        k_z = 0.f;
        v_z = TERMS == 1 ? -INFINITY : 0.f;  // (its log2, but for float32)
        if (token < s.hi && token >= 0) {
            const int column = token / a.tb.page, within = token - column * a.tb.page;
            const int at = a.tb.pages[b * a.tb.stride + column];
            if ((unsigned)at < (unsigned)a.tb.num_pages) {
                k_at = at * a.k.sp + head * a.k.sh + within * a.k.st;
                v_at = at * a.v.sp + head * a.v.sh + within * a.v.st;
                k_z = a.k.scales[at * a.k.zp + head * a.k.zh];
                v_z = finite_or_nan(a.v.scales[at * a.v.zp + head * a.v.zh]);
                if (TERMS == 1) v_z = __builtin_amdgcn_logf(v_z);
            } else {
                k_z = __uint_as_float(0x7fc00000u);
            }
        }
    };
    struct Tile {
        u32x4 k[2][KC];
        unsigned v[8][VW];
        float kz[2], vz[2];
    };
    auto fetch = [&](int step, Tile &t) {
        const int group = 2 * step;
        if (group >= filled + 64) fill(group);
        const char *kc = static_cast<const char *>(a.k.codes), *vc = static_cast<const char *>(a.v.codes);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int at = group + h - filled;
            const char *kp = kc + lane_offset(k_at, at), *vp = vc + lane_offset(v_at, at);
            t.kz[h] = lane_float(k_z, at);
            t.vz[h] = lane_float(v_z, at);
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const unsigned off = n16 * (unsigned)a.k.st + min(c * 64 + g4 * 16, a.D - 16);
                t.k[h][c] = *reinterpret_cast<const u32x4 *>(kp + off);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned off = (g4 * 4 + j) * (unsigned)a.v.st + min(n16 * CW, a.D - CW);
                if constexpr (VW == 1) {
                    t.v[h * 4 + j][0] = *reinterpret_cast<const unsigned *>(vp + off);
                } else if constexpr (VW == 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(vp + off);
                    t.v[h * 4 + j][0] = x[0];
                    t.v[h * 4 + j][1] = x[1];
                } else {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(vp + off);
#pragma unroll
                    for (int c = 0; c < 4; c++) t.v[h * 4 + j][c] = x[c];
                }
            }
        }
    };
    // SEEN: every row sees every token of the step; else some may be `hidden`
    auto work = [&](auto seen, bool hidden, int step, const Tile &t) {
        constexpr bool SEEN = decltype(seen)::value;
        const float most_z = fmaxf(t.vz[0], t.vz[1]), shrink = grow(ref, TERMS == 1 ? most_z : __builtin_amdgcn_logf(most_z));
        float lz[2], inv_z[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            lz[h] = TERMS == 1 ? log_weight(t.vz[h], ref) : plain_weight(t.vz[h], ref);
            inv_z[h] = inverse_weight(lz[h]);
        }
        f32x4 st[R][2];
#pragma unroll
        for (int r = 0; r < R; r++) st[r][0] = st[r][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const f16x8 kf = widen_row<E4M3, SEEN>(t.k[h][c][2 * u], t.k[h][c][2 * u + 1]);
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int i = TERMS - 1; i >= 0; i--) st[r][h] = mfma(kf, qf[r][c][u][i], st[r][h]);
                }
        f16x8 pf[R][TERMS];
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (!SEEN && hidden) {
                const int token = base + step * kTile;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = token + h * 16 + g4 * 4 + i;
                        st[r][h][i] = j >= lo_r[r] && j < hi_r[r] ? st[r][h][i] : -INFINITY;
                    }
            }
            const float u[2] = {unit[r] * t.kz[0], unit[r] * t.kz[1]};
            float top = kFloor;
#pragma unroll
            for (int h = 0; h < 2; h++)
                top = fmaxf(top, u[h] * fmaxf(fmaxf(st[r][h][0], st[r][h][1]), fmaxf(st[r][h][2], st[r][h][3])));
            float scale = shrink;
            if (__any(top > m[r] + kSlack)) {
                // (row by row: what other rows see changes nothing here)
                top = row_max(top);
                top = top > m[r] + kSlack ? top : m[r];
                const float alpha = __builtin_amdgcn_exp2f(m[r] - top);
                m[r] = top;
                l[r] *= alpha;
                scale *= alpha;
            }
            if (__any(scale != 1.f)) {
#pragma unroll
                for (int i = 0; i < CW; i++) acc[r][i] *= scale;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float shift = (TERMS == 1 ? lz[h] : 0.f) - m[r];
                f32x4 p;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float y = fmaf(st[r][h][i], u[h], shift);
                    if (!SEEN) y = st[r][h][i] == -INFINITY ? -INFINITY : y;
                    p[i] = __builtin_amdgcn_exp2f(y);
                }
                if constexpr (TERMS == 1) {
#pragma unroll
                    for (int i = 0; i < 4; i++) pf[r][0][h * 4 + i] = (_Float16)p[i];
                    const f16x8 &w = pf[r][0];
                    const float part = close(lz[h]) ? sum4(w[h * 4], w[h * 4 + 1], w[h * 4 + 2], w[h * 4 + 3], 0.f)
                                                    : (p[0] + p[1]) + (p[2] + p[3]);
                    l[r] = fmaf(part, inv_z[h], l[r]);
                } else {
                    l[r] += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        p[i] *= lz[h];
                        if (!SEEN) p[i] = st[r][h][i] == -INFINITY ? 0.f : p[i];  // (the factor may be NaN)
                    }
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        f16x2 high, low;
                        two_terms(p[i], p[i + 1], high, low);
                        pf[r][0][h * 4 + i] = high[0];
                        pf[r][0][h * 4 + i + 1] = high[1];
                        pf[r][1][h * 4 + i] = low[0];
                        pf[r][1][h * 4 + i + 1] = low[1];
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < VW; c++) {
            unsigned x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = t.v[j][c];
            f16x8 vf[4];
            widen_columns<E4M3, SEEN>(x, vf);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int k = TERMS - 1; k >= 0; k--) acc[r][c * 4 + i] = mfma(vf[i], pf[r][k], acc[r][c * 4 + i]);
        }
    };
    auto go = [&](int step, const Tile &t) {
        const int token = base + step * kTile;
        const bool hidden = token < all_lo || token + kTile > all_hi;
        if constexpr (ONE_FORM) {
            work(std::false_type{}, hidden, step, t);
        } else {
            if (hidden) work(std::false_type{}, true, step, t);
            else work(std::true_type{}, false, step, t);
        }
    };
    if (w0 < w1) {
        Tile t0, t1;
        fetch(w0, t0);
        int step = w0;
        for (; step + 1 < w1; step += 2) {
            fetch(step + 1, t1);
            go(step, t0);
            if (step + 2 < w1) fetch(step + 2, t0);
            go(step + 1, t1);
        }
        if (step < w1) go(step, t0);
    }

    // the four waves' parts
    const int rows = min(ROWS, all_rows - row0);
    __shared__ __align__(16) float part_o[4][ROWS][DP + 4];
    __shared__ float part_m[4][ROWS], part_l[4][ROWS];
    const float back = power_of_two(ref - kPTop + (E4M3 ? 8 : 0));
#pragma unroll
    for (int r = 0; r < R; r++) {
        const float sum = row_sum(l[r]);
        const int row = r * 16 + n16;
        if (row >= rows) continue;
        if (g4 == 0) {
            part_m[wave][row] = m[r];
            part_l[wave][row] = sum;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < CW; c += 4)
                *reinterpret_cast<f32x4 *>(&part_o[wave][row][(g4 * 4 + i) * CW + c]) =
                    f32x4{acc[r][c][i], acc[r][c + 1][i], acc[r][c + 2][i], acc[r][c + 3][i]} * back;
    }
    __syncthreads();
    const float poison = s.ok ? 0.f : __uint_as_float(0x7fc00000u);
    const bool leaves = kShared<Args> || w.items > 1;  // its part, for another launch
    float *part = part_of(a, ROWS, w.item, head, first);
    const int mc = threadIdx.x & 15;  // of the channels, 4 in 64
    for (int r = threadIdx.x >> 4; r < rows; r += 16) {
        float top = part_m[0][r], f[4], all = 0.f;
#pragma unroll
        for (int v = 1; v < 4; v++) top = fmaxf(top, part_m[v][r]);
#pragma unroll
        for (int v = 0; v < 4; v++) {
            f[v] = __builtin_amdgcn_exp2f(part_m[v][r] - top);
            all += f[v] * part_l[v][r];
        }
        if (leaves && mc == 0) {
            part[r] = top;
            part[ROWS + r] = all;
        }
        const Place where = place_of(a, which, head, row0 + r, first);
        const int64_t at = offset_of(a.o, where);
        const bool live = where.t < s.count;
        const float norm = all == 0.f || !live ? 0.f : 1.f / all;
#pragma unroll
        for (int c = 0; c < DP; c += 64) {
            const int d = c + mc * 4;
            if (d >= a.D) break;
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < 4; v++) y += f[v] * *reinterpret_cast<const f32x4 *>(&part_o[v][r][d]);
            if (leaves) *reinterpret_cast<f32x4 *>(part + 2 * ROWS + r * a.D + d) = y;
            else store_channels<DT>(a.o, at + d, (live ? y * norm : f32x4{0.f, 0.f, 0.f, 0.f}) + poison);
        }
    }
}

// The parts of a row joined: one workgroup per (row tile, cache head, row).
template <int ROWS, int DT>
__device__ __forceinline__ void join_body(const AttnArgs &a) {
    const int all_rows = a.T * a.group, per = min(ROWS, all_rows);
    int block = blockIdx.x;
    const int r = block % per;
    block /= per;
    const int head = block % a.heads_kv, entry = block / a.heads_kv;
    const int *note = reinterpret_cast<const int *>(a.ws) + 2 * entry;
    const int first = note[0], items = note[1];
    const int which = entry / a.row_tiles, row = (entry - which * a.row_tiles) * ROWS + r;
    if (items == 1 || row >= all_rows) return;
    const float *ws = part_of(a, ROWS, first, head, false);
    const int64_t stride = a.heads_kv * item_floats(ROWS, a.D);

    // lanes over the channels, 4 each, and the remaining factor of 256 over the items, each with the
    // maximum of its own so far
    __shared__ __align__(16) float red[256][4];
    __shared__ float tops[256], sums[256];
    const int lanes = a.D / 4, groups = 256 / lanes, c = threadIdx.x % lanes, g = threadIdx.x / lanes;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f, top = kFloor;
    if (g < groups) {
        constexpr int DEEP = 4;  // items whose loads are under way at a time
        for (int i0 = g; i0 < items; i0 += groups * DEEP) {
            float m[DEEP], l[DEEP];
            f32x4 x[DEEP];
#pragma unroll
            for (int k = 0; k < DEEP; k++) {
                const int i = i0 + k * groups;
                const float *p = ws + min(i, items - 1) * stride;
                m[k] = i < items ? p[r] : kFloor;
                l[k] = i < items ? p[ROWS + r] : 0.f;
                x[k] = *reinterpret_cast<const f32x4 *>(p + 2 * ROWS + r * a.D + c * 4);
                if (i >= items) x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            float most = top;
#pragma unroll
            for (int k = 0; k < DEEP; k++) most = fmaxf(most, m[k]);
            const float old = __builtin_amdgcn_exp2f(top - most);
            sum *= old;
            y *= old;
            top = most;
#pragma unroll
            for (int k = 0; k < DEEP; k++) {
                const float f = __builtin_amdgcn_exp2f(m[k] - top);
                sum += f * l[k];
                y += f * x[k];
            }
        }
    }
    tops[threadIdx.x] = top;
    sums[threadIdx.x] = sum;
    *reinterpret_cast<f32x4 *>(red[threadIdx.x]) = y;
    __syncthreads();
    if (g == 0) {
        for (int i = 1; i < groups; i++) top = fmaxf(top, tops[i * lanes]);
        sum = 0.f;
        y = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < groups; i++) {
            const float f = __builtin_amdgcn_exp2f(tops[i * lanes] - top);
            sum += f * sums[i * lanes];
            y += f * *reinterpret_cast<const f32x4 *>(red[i * lanes + c]);
        }
        const Place where = place_of(a, which, head, row, false);
        const int count = a.tb.counts ? a.tb.counts[which] : a.T;
        const float norm = sum == 0.f ? 0.f : 1.f / sum;
        store_channels<DT>(a.o, offset_of(a.o, where) + c * 4, where.t < count ? y * norm : f32x4{0.f, 0.f, 0.f, 0.f});
    }
}

}  // namespace
}  // namespace enatten
