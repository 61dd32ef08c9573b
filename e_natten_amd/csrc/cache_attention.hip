// Attention of a sequence's last tokens over its cache of 8-bit codes (enatten_cache_attention).
//
//   o = sum_j p_j z'_j v_j / sum_j p_j,   p_j = exp(scale z_j q.k_j - m),   j over the visible tokens
//
// with codes k_j, v_j and the scales z_j, z'_j of their blocks (page, head).  All query heads that share
// a head of the cache, and all new tokens, are rows of one problem per (sequence, cache head): a row tile
// of up to 64 of them goes over the tokens once, with the running maximum and sum of the softmax (calls
// with more rows: cache_attention_rows.hip).
//
// Products.  Codes are numbers that float16 holds exactly (int8 as they are, E4M3 times 2^-8), so both
// products run on the float16 matrix instructions whatever the type of q: rows of q are multiplied by a
// power of two that brings their largest value to 2^14 .. 2^15, which leaves bfloat16 values exact down
// to 2^-28 of the largest; float32 rows are the sum of two such terms.  The logits come out in float32
// and take scale, z_j and the power of two there.
//
// The first product forms S^T = K Q^T: a lane then holds 4 tokens of one row, and the softmax's
// statistics are one value per lane.  The order of the tokens within the second product's sum is free,
// so O^T = V^T P^T takes the probabilities from the registers where the first product left them, and V
// with the same permutation: lane (m, g) reads channels m * D/16 .. of tokens 4g .. 4g+3 of both halves
// of a tile of 32.  Neither K, V nor P passes through LDS, and no wave waits for another one on the way.
//
// Probabilities go into the second product as float16, at 2^7 for the running maximum.  That maximum is
// let lag by up to 2^8, so that the sums are seldom rescaled; what is below 2^-21 of the largest (2^-29
// with the lag) has fewer than 11 bits.  float32 takes two terms, 22 bits but no step under 2^-24, so that a
// probability is off by up to 2^-32 of the largest however small it is.  z'_j goes into them too, as a summand
// of the exponent: log2 of z'_j relative to the largest power of two among the z' so far, and the sums
// are scaled down where that grows.  The sum of the probabilities is formed of the rounded ones, so that
// a result stays a mean of values, but for groups whose z' is far below the largest, which float16 drops.
// The sums are formed before their division, so that a value times 2^8 times the number of tokens has to stay
// within float32.
//
// What bounds it.  One token of a sequence: every code is read once, two products of 16 rows cost a few
// percent of the matrix cores: HBM.  Work is split along the tokens so that the chip is filled whatever
// the number of sequences and heads; the parts leave their sums, maximum and output in the workspace and
// a second launch joins them.  The split goes by the lengths of this call, which are on the device:
// every workgroup computes it for itself.  Short calls are bound by the two launches and one chain of
// loads (lengths, pages, codes), and several rows by what a workgroup takes to get going: five tokens each
// for 8 sequences of up to 512 tokens, 16 + 2 heads of 64 channels, take 14 us, of which the join is 4.4, and
// 22 us with 32 times as many codes.
//
// Measured on MI355X, heads of 128 channels: 64 sequences of 4160 .. 8192 tokens, 32 + 8 heads, E4M3: 146 us
// (809 MB, 5.5 TB/s; reads alone reach 6.4), 32 sequences of 8448 .. 16384: 175 us (4.7 TB/s); 32 + 4 heads, a
// sequence of 131072 tokens, int8: 33 us as a graph, 37 as calls; 16 + 16 heads, one sequence: a window of 128
// tokens 6 us, of 1024, which is split, 11 us.
#include "cache_attention.h"

#include <type_traits>

namespace enatten {
namespace {

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
template <int DP, int R, bool E4M3, int DT>
__global__ __launch_bounds__(256, waves_of(DP, R, DT == ENATTEN_F32 ? 2 : 1)) void attend(AttnArgs a) {
    constexpr int TERMS = DT == ENATTEN_F32 ? 2 : 1, TOK = kTile, ROWS = 16 * R, KC = DP / 64, VW = DP / 64, CW = DP / 16;
    constexpr bool ONE_FORM = one_form(DP, R);
    const int lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (branches on it are the wave's)

    // which row tile, and which of its steps
    const int head = blockIdx.x % a.heads_kv;
    Share w;
    if (a.parts) {
        w = share_of<ROWS, TOK, 4>(a, blockIdx.x / a.heads_kv);
        if (w.entry < 0) return;
        note_share(a, w, head);
    } else {
        w.entry = blockIdx.x / a.heads_kv;
        w.items = 1;
    }
    const int entry = w.entry;
    const Span s = span_of<ROWS>(a, entry);
    if (!a.parts) {
        w.step0 = 0;
        w.step1 = steps_of<TOK>(s);
    }
    const int b = entry / a.row_tiles, row0 = (entry - b * a.row_tiles) * ROWS;
    const int step0 = w.step0, step1 = w.step1;
    const int base = s.lo & -16;

    // q: lane (row n16, g4) has channels 64 c + 16 g4 .. + 15
    f16x8 qf[R][KC][2][TERMS];
    float unit[R];           // what a product of codes is multiplied by, besides z: log2 units, not negative
    const float flip = a.scale < 0.f ? -1.f : 1.f;
    int lo_r[R], hi_r[R];    // tokens that the lane's row sees
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = min(row0 + r * 16 + n16, a.T * a.group - 1), t = row / a.group;
        const int tv = min(t, max(s.count - 1, 0));
        hi_r[r] = s.start + tv + 1;
        lo_r[r] = a.window ? max(hi_r[r] - a.window, 0) : 0;
        const int64_t at = b * a.q.sb + (head * a.group + row - t * a.group) * a.q.sh + t * a.q.st;
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
    const int all_lo = a.window ? max(s.start + min((row0 + ROWS - 1) / a.group, s.count - 1) + 1 - a.window, 0) : 0;
    const int all_hi = s.start + row0 / a.group + 1;

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
    const int rows = min(ROWS, a.T * a.group - row0);
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
    float *part = part_of(a, ROWS, w.item, head);
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
        if (w.items > 1 && mc == 0) {
            part[r] = top;
            part[ROWS + r] = all;
        }
        const int row = row0 + r, t = row / a.group;
        const int64_t at = b * a.o.sb + (head * a.group + row - t * a.group) * a.o.sh + t * a.o.st;
        const bool live = t < s.count;
        const float norm = all == 0.f || !live ? 0.f : 1.f / all;
#pragma unroll
        for (int c = 0; c < DP; c += 64) {
            const int d = c + mc * 4;
            if (d >= a.D) break;
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < 4; v++) y += f[v] * *reinterpret_cast<const f32x4 *>(&part_o[v][r][d]);
            if (w.items > 1) *reinterpret_cast<f32x4 *>(part + 2 * ROWS + r * a.D + d) = y;
            else store_channels<DT>(a.o, at + d, (live ? y * norm : f32x4{0.f, 0.f, 0.f, 0.f}) + poison);
        }
    }
}

// The parts of a row joined: one workgroup per (row tile, cache head, row).
template <int ROWS, int DT>
__global__ __launch_bounds__(256) void attend_join(AttnArgs a) {
    const int per = min(ROWS, a.T * a.group);
    int block = blockIdx.x;
    const int r = block % per;
    block /= per;
    const int head = block % a.heads_kv, entry = block / a.heads_kv;
    const int *note = reinterpret_cast<const int *>(a.ws) + 2 * entry;
    const int first = note[0], items = note[1];
    const int b = entry / a.row_tiles, row = (entry - b * a.row_tiles) * ROWS + r;
    if (items == 1 || row >= a.T * a.group) return;
    const float *ws = part_of(a, ROWS, first, head);
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
        const int t = row / a.group;
        const int64_t at = b * a.o.sb + (head * a.group + row - t * a.group) * a.o.sh + t * a.o.st;
        const int count = a.tb.counts ? a.tb.counts[b] : a.T;
        const float norm = sum == 0.f ? 0.f : 1.f / sum;
        store_channels<DT>(a.o, at + c * 4, t < count ? y * norm : f32x4{0.f, 0.f, 0.f, 0.f});
    }
}

// How a call is cut, from its sizes alone (the lengths are on the device).
//
// Rows.  A wave holds q, the sums and the probabilities of all rows of its tile in registers, which
// leaves room for 64 rows of 64 channels, 48 of 128 and 16 of 256 with two tiles of codes under way.
// Beyond, tiles of 256 rows over codes that LDS holds as float16; 72 rows of 64 channels over 300 tokens
// (8 sequences, 2 heads of the cache) take 15 us there and took 33 in tiles of 32 here.  float32 rows of more than
// 128 channels have too many registers for that and stay here, where every 16 rows read the cache anew: 512
// tokens each of 16384 and 12288, 16 + 4 heads of 256 channels, take 783 us and 334 in bfloat16.
// Workgroups.  Two per CU where their registers leave room for two waves per SIMD, else one: with 48 rows
// of 128 channels a second one per CU only waits.
Plan plan_of(int B, int heads, int heads_kv, int T, int D, int page, int columns, int window, int dtype) {
    Plan p;
    const int64_t all = (int64_t)T * (heads / heads_kv);
    const int most = D > 128 ? 16 : D > 64 ? 48 : 64;
    p.rows = all <= most ? (int)(all + 15) / 16 * 16 : D > 128 && dtype == ENATTEN_F32 ? 16 : kWideRows;
    p.row_tiles = (int)((all + p.rows - 1) / p.rows);
    const int64_t entries = (int64_t)B * p.row_tiles;
    int64_t tokens = (int64_t)columns * page;
    if (window && window + (int64_t)p.rows < tokens) tokens = window + (int64_t)p.rows;
    p.parts = 0;
    p.items = entries;
    const int target = 256 * (waves_of(padded(D), p.rows / 16, dtype == ENATTEN_F32 ? 2 : 1) > 1 ? 2 : 1);
    if (p.rows == kWideRows) {
        p.parts = 256;  // ranges: one workgroup per CU
    } else if (entries * heads_kv < target && tokens > kLeast) {
        p.parts = (target + heads_kv - 1) / heads_kv;
        // no more than the longest possible sequences fill
        const int64_t useful = entries * ((tokens + 16 + kLeast - 1) / kLeast);
        if (useful < p.parts) p.parts = (int)useful;
        p.items = p.parts + entries;
    }
    return p;
}

template <int DP, int R, bool E4M3, int DT>
int launch(const char *fn, const AttnArgs &a, const Plan &p, hipStream_t st) {
    {
        ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "attend", st);
        attend<DP, R, E4M3, DT><<<(int)(p.items * a.heads_kv), 256, 0, st>>>(a);
    }
    const int rc = launched(fn);
    if (rc || !p.parts) return rc;
    const int64_t rows = a.T * (int64_t)a.group, blocks = (int64_t)a.B * p.row_tiles * a.heads_kv * (rows < 16 * R ? rows : 16 * R);
    if (blocks > 0x7fffffff) {
        set_error("%s: too many rows", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    ProfScope prof(ENATTEN_KERNEL_CACHE_JOIN, "attend_join", st);
    attend_join<16 * R, DT><<<(int)blocks, 256, 0, st>>>(a);
    return launched(fn);
}
template <int DP, int R, bool E4M3>
int launch_type(const char *fn, const AttnArgs &a, const Plan &p, hipStream_t st) {
    if (a.dtype == ENATTEN_BF16) return launch<DP, R, E4M3, ENATTEN_BF16>(fn, a, p, st);
    if (a.dtype == ENATTEN_F32) return launch<DP, R, E4M3, ENATTEN_F32>(fn, a, p, st);
    return launch<DP, R, E4M3, ENATTEN_F16>(fn, a, p, st);
}
template <int DP, bool E4M3>
int launch_rows(const char *fn, const AttnArgs &a, const Plan &p, hipStream_t st) {
    if (p.items * a.heads_kv > 0xffffff) {  // (2^32 threads)
        set_error("%s: too many row tiles", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    if (p.rows == kWideRows) return launch_attend_rows(fn, a, E4M3, st);
    if (p.rows == 16) return launch_type<DP, 1, E4M3>(fn, a, p, st);
    if constexpr (DP <= 128) {
        if (p.rows == 32) return launch_type<DP, 2, E4M3>(fn, a, p, st);
        if (p.rows == 48) return launch_type<DP, 3, E4M3>(fn, a, p, st);
    }
    if constexpr (DP == 64)
        if (p.rows == 64) return launch_type<DP, 4, E4M3>(fn, a, p, st);
    set_error("%s: no tile of %d rows of %d channels", fn, p.rows, a.D);
    return ENATTEN_EUNSUPPORTED;
}

}  // namespace
}  // namespace enatten

using namespace enatten;

extern "C" {
#pragma GCC visibility push(default)

size_t enatten_cache_attention_workspace_bytes(int B, int heads, int heads_kv, int T, int D, int page, int columns,
                                               int kernel_size, int dtype) {
    if (B < 1 || heads < 1 || heads_kv < 1 || heads % heads_kv || T < 1 || D < 1 || page < 1 || columns < 1 ||
        kernel_size < 0)
        return 0;
    const Plan p = plan_of(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype);
    if (!p.parts) return 0;
    if (p.rows == kWideRows) return ((size_t)(p.parts + 3) / 4 * 4 + 2 * p.parts * item_floats(kWideRows, padded(D))) * sizeof(float);
    return (size_t)(head_floats((int64_t)B * p.row_tiles) + p.items * heads_kv * item_floats(p.rows, D)) * sizeof(float);
}

int enatten_cache_attention(const void *q, const void *k_cache, const void *v_cache, const float *k_scale,
                            const float *v_scale, const int *pages, const int *lengths, const int *counts, void *o,
                            void *workspace, int B, int heads, int heads_kv, int T, int D, int num_pages, int page,
                            int columns, int kernel_size, int dtype, int cache_dtype, const int64_t *q_strides,
                            const int64_t *o_strides, const int64_t *k_cache_strides, const int64_t *v_cache_strides,
                            const int64_t *k_scale_strides, const int64_t *v_scale_strides, int64_t pages_stride,
                            float scale, void *stream) {
    const char *fn = "enatten_cache_attention";
    int rc = check_cache_sizes(fn, B, heads, T, D, num_pages, page, columns, dtype, cache_dtype, pages_stride);
    if (rc) return rc;
    if (heads_kv < 1 || heads % heads_kv) {
        set_error("%s: %d heads are no multiple of the cache's %d", fn, heads, heads_kv);
        return ENATTEN_EINVAL;
    }
    if (kernel_size < 0) {
        set_error("%s: kernel_size must be >= 1, or 0 for all tokens, got %d", fn, kernel_size);
        return ENATTEN_EINVAL;
    }
    AttnArgs a{};
    if ((rc = set_rows(fn, "q", q, q_strides, heads, T, D, &a.q))) return rc;
    if ((rc = set_rows(fn, "o", o, o_strides, heads, T, D, &a.o))) return rc;
    const int pack = dtype == ENATTEN_F32 ? 4 : 8;
    if (((uintptr_t)q | (uintptr_t)o) % 16 || (a.q.sb | a.q.sh | a.q.st | a.o.sb | a.o.sh | a.o.st) % pack) {
        set_error("%s: rows of q and o must lie at multiples of 16 bytes", fn);
        return ENATTEN_EINVAL;
    }
    if ((rc = set_cache(fn, "k", const_cast<void *>(k_cache), const_cast<float *>(k_scale), k_cache_strides,
                        k_scale_strides, heads_kv, page, D, 16, &a.k))) return rc;
    if ((rc = set_cache(fn, "v", const_cast<void *>(v_cache), const_cast<float *>(v_scale), v_cache_strides,
                        v_scale_strides, heads_kv, page, D, 16, &a.v))) return rc;
    if (!pages || !lengths) {
        set_error("%s: pages and lengths must not be NULL", fn);
        return ENATTEN_EINVAL;
    }
    const Plan p = plan_of(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype);
    if (p.parts && (!workspace || (uintptr_t)workspace % 16)) {
        set_error("%s: workspace is NULL or not 16-byte aligned", fn);
        return ENATTEN_EINVAL;
    }
    a.tb = Table{pages, lengths, counts, pages_stride, num_pages, page, columns, T};
    a.B = B; a.heads = heads; a.group = heads / heads_kv; a.heads_kv = heads_kv; a.T = T; a.D = D;
    a.window = kernel_size;
    a.dtype = dtype;
    a.row_tiles = p.row_tiles;
    a.parts = p.parts;
    a.scale = scale;
    a.ws = static_cast<float *>(workspace);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool e = cache_dtype == ENATTEN_E4M3;
    if (D <= 64) return e ? launch_rows<64, true>(fn, a, p, st) : launch_rows<64, false>(fn, a, p, st);
    if (D <= 128) return e ? launch_rows<128, true>(fn, a, p, st) : launch_rows<128, false>(fn, a, p, st);
    return e ? launch_rows<256, true>(fn, a, p, st) : launch_rows<256, false>(fn, a, p, st);
}

#pragma GCC visibility pop
}  // extern "C"
