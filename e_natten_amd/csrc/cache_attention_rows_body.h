// The kernels of cache_attention_rows.hip as functions, for calls of sequences by themselves and of runs that share
// their first tokens (cache_attention_shared.hip); what they do stands in the former.
#pragma once

#include "cache_attention_body.h"

namespace enatten {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// The kernel's arguments, read anew: what is used once per row tile or per 64 groups of tokens does not
// stay in scalar registers across the steps (held there, 124 of them were spilled, for 7% at head_dim 128).
template <class Args>
__device__ __forceinline__ const Args &args_again() {
    typedef const Args __attribute__((address_space(4))) *Kernarg;
    Kernarg p = (Kernarg)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Args *)p;
}

// DP: head_dim rounded up to 64, 128 or 256; DT: type of q and o, float32 in two float16 terms of q and p.
// TG: groups of the eight waves that share their rows and take some of a step's tokens each; their sums meet in LDS at
// the end of a tile (the first part of a call with shared tokens).  M: how many times as many tokens a step has.  With
// eight groups of 32 tokens a step's operands fill LDS and the next one's are put there when all have read them.
template <int DP, bool E4M3, int DT, int TG, int M, class Args>
__device__ __forceinline__ void rows_body(const Args &args) {
    constexpr bool FIRST = kShared<Args>;
    constexpr int RB = 8 / TG, ROWS = 32 * RB;  // blocks of 32 rows
    static_assert(TG == 1 || FIRST, "only parts are joined");
    constexpr int TERMS = DT == ENATTEN_F32 ? 2 : 1;
    constexpr int TOK = 8192 * M / DP;  // tokens of a step: 128, 64, 32, or twice as many
    constexpr int NB = TOK / 32;      // blocks of 32 of them
    constexpr int GR = TOK / 16;      // groups of 16, each within a page
    constexpr int NBW = NB / TG, GRW = GR / TG;  // those of a wave
    constexpr int BUFFERS = M == 4 ? 1 : 2;
    constexpr int SD = DP / 16;       // products along head_dim of S
    constexpr int OB = DP / 32;       // blocks of 32 channels of O
    constexpr int CH = DP / 16;       // loads of 16 codes per token
    constexpr int QUADS = DP / 4;     // words of 4 channels
    // operands of one step: K [NB][SD][64 lanes][8], V [OB][TOK / 16][64 lanes][8]; eight lanes that turn
    // one or two tokens write to as many operands of K, which therefore start 1 or 2 lanes apart in the banks
    constexpr int PART = 64 + (CH < 8 ? 8 / CH : 1);
    __shared__ f16x8 k_lds[BUFFERS][NB * SD * PART], v_lds[BUFFERS][TOK * DP / 8];
    __shared__ float z_lds[2][3][GR];  // of the step's groups: key scales, value scales (log2), their inverses
    __shared__ int z_bad[2][2];        // ... and which of either are not finite (0 in their place)
    // Rows of q stay in registers, at head dims above 128 all but the last operands, for which there are
    // none left: those a lane puts into LDS and reads again.
    constexpr int KEPT = DP == 256 ? 10 : SD;
    __shared__ f16x8 q_lds[8 * 64 * (SD - KEPT) + 1];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (branches on it are the wave's)
    const int rb = TG == 1 ? wave : wave % RB, tg = TG == 1 ? 0 : wave / RB;

    // The workgroup's range of steps.  Blocks 8 apart share an XCD and its L2: they get neighbouring ranges,
    // which read the same keys and values where they belong to the same head.
    const Args &a = args;
    const int range = blockIdx.x % 8 * (parts_of(a, FIRST) / 8) + blockIdx.x / 8;
    const Ranges line = ranges_of<ROWS, TOK>(a, FIRST);
    const int heads = a.heads_kv;
    int64_t end = min((range + 1) * line.each, line.line * heads);
    int64_t at_step = range * line.each;
    const int entries = entries_of(a, FIRST), all_rows = rows_of(a, FIRST);
    int *note = reinterpret_cast<int *>(ws_of(a, FIRST)) + range;
    int head, entry, into = 0;
    if (line.whole) {  // a tile each
        head = range / entries;
        entry = range - head * entries;
        at_step = head < heads ? 0 : end;
        end = min(end, (int64_t)1);
    } else {
        head = (int)(at_step / line.line);
        entry = at_step < end ? tile_at<ROWS, TOK>(a, at_step - head * line.line, into, FIRST) : 0;
    }
    if (!FIRST && threadIdx.x == 0) *note = into ? head * entries + entry : -1;

    for (; at_step < end; into = 0) {
    const Args &a = args_again<Args>();
    const Span s = span_of<ROWS>(a, entry, FIRST);
    if constexpr (FIRST) {
        if (s.hi == 0) {  // a run that shares nothing leaves nothing: its tile counts as one step
            at_step++;
            if (++entry == entries) {
                entry = 0;
                head++;
            }
            continue;
        }
    }
    const int total = steps_of<TOK>(s), counted = max(1, total), step0 = into;
    int step1 = line.whole ? total : min(total, (int)min((int64_t)counted, step0 + (end - at_step)));
    const bool parted = FIRST || (!line.whole && (into || step0 + (end - at_step) < counted));
    const int slot = into ? 2 * range : 2 * range + 1;
    if constexpr (FIRST) {
        if (into == 0 && threadIdx.x == 0) {  // (for the launch that joins the parts)
            int *ranges = reinterpret_cast<int *>(a.first_ws) + 2 * (head * entries + entry);
            ranges[0] = range;
            ranges[1] = (int)((at_step + counted - 1) / line.each);
        }
    }
    at_step += counted - into;
    const int which = entry / tiles_of(a, FIRST), row0 = (entry - which * tiles_of(a, FIRST)) * ROWS + rb * 32;
    const int base = s.lo & -16;
    int b = which;
    if constexpr (FIRST) {
        b = reader_of(a, which, s.hi);
        if (b < 0) b = which * a.size, step1 = step0;  // (nobody reads them)
    }

    // the lane's row; q: lane (n, h) has channels 16 c + 8 h .. + 7
    const Place where = place_of(a, which, head, min(row0 + n, all_rows - 1), FIRST);
    const bool live = row0 + n < all_rows && (FIRST || where.t < s.count);
    int hi_r = live ? s.start + where.t + 1 : 0, seen = a.window ? a.window : hi_r;  // tokens hi_r - seen .. hi_r - 1
    int most_lo = 0;
    if constexpr (FIRST) {  // (rows of a sequence that does not share them come to what nobody reads)
        const int first = shared_lo(a, where, s.hi);
        if (live) most_lo = first;
        hi_r = live ? s.hi : 0;
        seen = hi_r - first;
    }
    f16x8 qf[KEPT][TERMS], *q_rest = &q_lds[threadIdx.x];
    float unit, l;
    auto take_q = [&] {
        const int64_t at = offset_of(a.q, where);
        const float flip = a.scale < 0.f ? -1.f : 1.f;  // into q, so that units are not negative
        float x[SD][8], top = 0.f, nan = 0.f;
#pragma unroll
        for (int c = 0; c < SD; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[c][j] = 0.f;
            if (c * 16 < a.D) load_channels<DT>(a.q, at + c * 16 + h * 8, x[c]);
        }
#pragma unroll
        for (int c = 0; c < SD; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                top = fmaxf(top, fabsf(x[c][j]));
                nan += x[c][j] * 0.f;  // a value that is not finite makes its row NaN, the factor all rows
            }
        nan = pair_sum(nan);
        top = pair_max(top);
        const int up = kTop + 1 - (top > 0.f ? __builtin_amdgcn_frexp_expf(top) : 0);
        unit = __builtin_ldexpf(fabsf(a.scale) * kLog2e, -up + (E4M3 ? 8 : 0));
        l = nan + a.scale * 0.f;  // (and stays NaN for a row of q or a factor that is not finite)
#pragma unroll
        for (int c = 0; c < SD; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[c][j] = __builtin_ldexpf(x[c][j] * flip, up);
#pragma unroll
        for (int c = 0; c < SD; c++) {
            f16x8 w[TERMS];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                if constexpr (TERMS == 2) {
                    f16x2 high, low;
                    two_terms(x[c][j], x[c][j + 1], high, low);
                    w[0][j] = high[0];
                    w[0][j + 1] = high[1];
                    w[1][j] = low[0];
                    w[1][j + 1] = low[1];
                } else {
                    w[0][j] = (_Float16)x[c][j];
                    w[0][j + 1] = (_Float16)x[c][j + 1];
                }
            }
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                if (c < KEPT) qf[c][t] = w[t];
                else q_rest[(c - KEPT) * 512] = w[t];
            }
        }
    };
    if constexpr (!FIRST) take_q();
    // tokens that any, and that all rows of the wave see
    const int t_first = min(row0, all_rows - 1) / a.group, t_last = min(min(row0 + 31, all_rows - 1) / a.group, s.count - 1);
    const bool any_row = row0 < all_rows && t_first < s.count;
    int some_lo = any_row && a.window ? max(s.start + t_first + 1 - a.window, 0) : 0;
    int some_hi = any_row ? s.start + t_last + 1 : 0;
    int all_lo = a.window ? max(s.start + t_last + 1 - a.window, 0) : 0, all_hi = s.start + t_first + 1;
    if constexpr (FIRST) {
        some_lo = 0;
        some_hi = row0 < all_rows ? s.hi : 0;
        all_lo = a.window ? wave_max(most_lo) : 0;
        all_hi = s.hi;
    }

    f32x16 acc[OB];
#pragma unroll
    for (int i = 0; i < OB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
    float m = kFloor;
    float ref = -126.f;

    // places of the groups of 16 tokens: lane i holds group `filled` + i
    // Every wave brings keys and values, or, where a step has too few tokens for that, four waves keys and four values: the
    // latter are turned, which takes twice as long.  16 runs of 4 sequences (cache_attention_shared.hip): 53.5 us instead of 54.8.
    constexpr bool BOTH = M > 1;
    int filled = -64;
    const bool for_v = wave >= 4;
    int64_t at[BOTH ? 2 : 1] = {};    // of keys, of values
    float z_at[BOTH ? 2 : 1] = {};    // (of values log2, for float32 the scale itself)
    int64_t &k_at = at[0], &v_at = at[BOTH ? 1 : 0];
    float &k_z = z_at[0], &v_z = z_at[BOTH ? 1 : 0];
    auto fill = [&](int group) {
        const Args &a = args_again<Args>();
        filled = group;
        const int token = base + (group + lane) * 16;
        k_at = v_at = 0;
        if (BOTH || !for_v) k_z = 0.f;
        if (BOTH || for_v) v_z = TERMS == 1 ? -INFINITY : 0.f;
        if (token < s.hi && token >= 0) {
            const int column = token / a.tb.page, within = token - column * a.tb.page;
            const int p = a.tb.pages[b * a.tb.stride + column];
            const bool there = (unsigned)p < (unsigned)a.tb.num_pages;
            if (!there) k_z = v_z = __uint_as_float(0x7fc00000u);
            if (there && (BOTH || for_v)) {
                v_at = p * a.v.sp + head * a.v.sh + within * a.v.st;
                v_z = finite_or_nan(a.v.scales[p * a.v.zp + head * a.v.zh]);
                if (TERMS == 1) v_z = __builtin_amdgcn_logf(v_z);
            }
            if (there && (BOTH || !for_v)) {
                k_at = p * a.k.sp + head * a.k.sh + within * a.k.st;
                k_z = a.k.scales[p * a.k.zp + head * a.k.zh];
            }
        }
    };
    // What a thread brings: of keys runs of 16 codes, of values words of 4 channels of 8 tokens.
    constexpr int KR = BOTH ? M : 2, VR = BOTH ? M / 2 : 1;  // of either
    unsigned raw[M][8];  // BOTH: first the runs of keys, then the values; else one of the two
    float raw_z = 0.f;  // lanes 0 .. GR - 1 of wave 0: key scales of the step's groups, of wave 4: value scales
    // (offsets within a group of 16 tokens; a wave's 64 runs of keys lie in one group, its 64 words of
    // values too, but for DP 64, where each half of the wave has its own)
    const int kw = BOTH ? wave : wave & 3, vw = BOTH ? wave : wave & 3;
    const int run = vw * (64 * 4 / DP) * VR + lane / QUADS, quad = lane % QUADS;  // (the first) run of 8 tokens
    const unsigned k_within = (kw * (64 / CH) * KR + lane / CH) % 16 * (unsigned)a.k.st + min(lane % CH * 16, a.D - 16);
    const unsigned v_within = run % 2 * 4 * (unsigned)a.v.st + min(quad * 4, a.D - 4);
    auto fetch = [&](int step) {
        const int group = step * GR;
        if (group >= filled + 64) fill(group);
        const int here = group - filled;
        raw_z = __shfl(for_v ? v_z : k_z, here + (lane & (GR - 1)), 64);
        if (BOTH || !for_v) {
#pragma unroll
            for (int j = 0; j < KR; j++) {
                const char *from = static_cast<const char *>(a.k.codes) +
                                   lane_offset(k_at, here + (kw * (64 / CH) * KR + j * (64 / CH)) / 16);
                const u32x4 x = *reinterpret_cast<const u32x4 *>(from + (DP == 64 ? 0 : j % 2 * (64 / CH)) * a.k.st + k_within);
#pragma unroll
                for (int i = 0; i < 4; i++) raw[j / 2][j % 2 * 4 + i] = x[i];
            }
        }
        if (BOTH || for_v) {
#pragma unroll
            for (int k = 0; k < VR; k++) {
                const int first = (vw * VR + k) * (64 * 4 / DP) / 2;  // group
                int64_t off = lane_offset(v_at, here + first);
                if constexpr (DP == 64) off = lane < 32 ? off : lane_offset(v_at, here + first + 1);
                const char *from = static_cast<const char *>(a.v.codes) + off;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    raw[(BOTH ? KR / 2 : 0) + k][j] = *reinterpret_cast<const unsigned *>(from + (j % 4 + j / 4 * 8) * a.v.st + v_within);
            }
        }
    };
    if constexpr (FIRST) {
        if (step0 < step1) fetch(step0);  // (under way while the rows of q come)
        take_q();
    }
    auto put_as = [&](auto seen, int buffer) {
        constexpr bool SEEN = decltype(seen)::value;
        if (BOTH || !for_v) {
#pragma unroll
            for (int j = 0; j < KR; j++) {
                const int token = kw * (64 / CH) * KR + j * (64 / CH) + lane / CH, c = lane % CH;
                const unsigned *x = raw[j / 2] + j % 2 * 4;
                f16x8 *to = &k_lds[buffer][(token / 32 * SD + c) * PART + token % 32];
                to[0] = widen_row<E4M3, SEEN>(x[0], x[1]);
                to[32] = widen_row<E4M3, SEEN>(x[2], x[3]);
            }
        }
        if (BOTH || for_v) {
#pragma unroll
            for (int k = 0; k < VR; k++) {
                f16x8 v[4];
                widen_columns<E4M3, SEEN>(raw[(BOTH ? KR / 2 : 0) + k], v);
                const int r = run + k * (64 * 4 / DP);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int block = DP == 64 ? i / 2 : i + quad / 32 * 4, mm = DP == 64 ? (i & 1) * 16 + quad : quad & 31;
                    v_lds[buffer][(block * (TOK / 16) + r / 2) * 64 + r % 2 * 32 + mm] = v[i];
                }
            }
        }
        if ((wave & 3) == 0) {
            const bool finite = for_v && TERMS == 1 ? raw_z < INFINITY : fabsf(raw_z) < INFINITY;
            const float z = finite ? raw_z : for_v && TERMS == 1 ? -INFINITY : 0.f;
            if (lane < GR) {
                z_lds[buffer][for_v][lane] = z;
                if (for_v) z_lds[buffer][2][lane] = __builtin_amdgcn_exp2f(-z);
            }
            const int bad = (int)__ballot(!finite) & ((1 << GR) - 1);
            if (lane == 0) z_bad[buffer][for_v] = bad;
        }
    };
    // (the workgroup's first and last rows, for the shorter way of turning E4M3)
    const int wg_row = row0 - rb * 32, wg_last = min((wg_row + ROWS - 1) / a.group, s.count - 1);
    int wg_lo = a.window ? max(s.start + wg_last + 1 - a.window, 0) : 0, wg_hi = s.start + wg_row / a.group + 1;
    if constexpr (FIRST) {
        wg_lo = a.window ? s.hi : 0;
        wg_hi = s.hi;
    }
    auto put = [&](int buffer, int step) {
        const int token = base + step * TOK;
        if (E4M3 && token >= wg_lo && token + TOK <= wg_hi) put_as(std::true_type{}, buffer);
        else put_as(std::false_type{}, buffer);
    };

    // One step for the wave's rows.  Masked logits are a large negative number, not an infinity: units
    // are at least 1e-20, so that they end below -1e18 and their exponentials are 0 whatever the maximum
    // (kFloor at least), and a unit of 0 asks for nothing special.
    auto work = [&](bool whole, int token, int buffer) {
        float kz[GRW], lz[GRW], most_z = -INFINITY;
#pragma unroll
        for (int g = 0; g < GRW; g++) {
            kz[g] = z_lds[buffer][0][tg * GRW + g];
            lz[g] = z_lds[buffer][1][tg * GRW + g];
            most_z = fmaxf(most_z, lz[g]);
        }
        float scale = grow(ref, TERMS == 1 ? most_z : __builtin_amdgcn_logf(most_z));
#pragma unroll
        for (int g = 0; g < GRW; g++) lz[g] = TERMS == 1 ? log_weight(lz[g], ref) : plain_weight(lz[g], ref);

        f32x16 st[NBW];
#pragma unroll
        for (int i = 0; i < NBW; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) st[i][j] = 0.f;
        const f16x8 *kp = &k_lds[buffer][lane + tg * (NBW * SD * PART)];
#pragma unroll
        for (int c = 0; c < SD; c++) {
#pragma unroll
            for (int i = 0; i < NBW; i++) {
                const f16x8 kf = kp[(i * SD + c) * PART];
#pragma unroll
                for (int t = TERMS - 1; t >= 0; t--)
                    st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, c < KEPT ? qf[c][t] : q_rest[(c - KEPT) * 512], st[i], 0, 0, 0);
            }
        }

        // lane's tokens: 32 i + 16 g + 8 (j / 4) + 4 h + j % 4 for its 8 values j of a group
        if (!whole) {
#pragma unroll
            for (int i = 0; i < NBW; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int tk = token + i * 32 + j / 4 * 8 + h * 4 + j % 4;
                    st[i][j] = tk >= hi_r - seen && tk < hi_r ? st[i][j] : -3e38f;
                }
        }
        // scales that are not finite: NaN for the rows that see a token of the group
        const int bad = __builtin_amdgcn_readfirstlane(z_bad[buffer][0] | z_bad[buffer][1]);
        if (bad) {
#pragma unroll
            for (int g = 0; g < GRW; g++) {
                const int first = token + g * 16;
                if ((bad >> (tg * GRW + g) & 1) && first < hi_r && first + 16 > hi_r - seen) l = __uint_as_float(0x7fc00000u);
            }
        }
        const float unit_z = power_of_two(ref - kPTop);
        float u[GRW], top = kFloor;
#pragma unroll
        for (int g = 0; g < GRW; g++) {
            u[g] = fmaxf(unit * kz[g], 1e-20f);
            float most = -3e38f;  // (a constant to start from: else the compiler makes values canonical)
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, st[g / 2][g % 2 * 8 + j]);
            top = fmaxf(top, most * u[g]);
        }
        if (__any(top > m + kSlack)) {
            // (row by row: what other rows see changes nothing here)
            top = pair_max(top);
            top = top > m + kSlack ? top : m;
            const float alpha = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= alpha;
            scale *= alpha;
        }
        if (__any(scale != 1.f)) {
#pragma unroll
            for (int i = 0; i < OB; i++) acc[i] *= scale;
        }
        // group by group, so that the exponentials of one go beside the products of another
        const f16x8 *vp = &v_lds[buffer][lane + tg * (GRW * 64)];
#pragma unroll
        for (int g = 0; g < GRW; g++) {
            const float shift = (TERMS == 1 ? lz[g] : 0.f) - m;
            f16x8 pf[TERMS];
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(fmaf(st[g / 2][g % 2 * 8 + j], u[g], shift));
            }
            const float part = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            if constexpr (TERMS == 1) {
#pragma unroll
                for (int j = 0; j < 8; j++) pf[0][j] = (_Float16)p[j];
                // (at most 2^40, as the weight is at least 2^-40)
                l = fmaf(part, fminf(z_lds[buffer][2][tg * GRW + g] * unit_z, 0x1p40f), l);
            } else {
                l += part;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
#pragma unroll
                    for (int k = j; k < j + 2; k++) p[k] *= lz[g];
                    f16x2 high, low;
                    two_terms(p[j], p[j + 1], high, low);
                    pf[0][j] = high[0];
                    pf[0][j + 1] = high[1];
                    pf[1][j] = low[0];
                    pf[1][j + 1] = low[1];
                }
            }
#pragma unroll
            for (int i = 0; i < OB; i++) {
                const f16x8 vf = vp[(i * (TOK / 16) + g) * 64];
#pragma unroll
                for (int t = TERMS - 1; t >= 0; t--)
                    acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[t], acc[i], 0, 0, 0);
            }
        }
    };

    __syncthreads();  // (the last tile's operands are read)
    if (step0 < step1) {
        if constexpr (!FIRST) fetch(step0);
        put(0, step0);
        if (step0 + 1 < step1) fetch(step0 + 1);
    }
    for (int step = step0; step < step1; step++) {
        const int buffer = BUFFERS == 1 ? 0 : (step - step0) & 1;
        if (BUFFERS == 1 && step > step0) {
            __syncthreads();  // (the step before is read)
            put(0, step);
            if (step + 1 < step1) fetch(step + 1);
        }
        __syncthreads();
        if (BUFFERS == 2 && step + 1 < step1) {
            put(buffer ^ 1, step + 1);
            if (step + 2 < step1) fetch(step + 2);
        }
        const int token = base + step * TOK + tg * (NBW * 32);
        if (token >= some_hi || token + NBW * 32 <= some_lo) continue;
        work(token >= all_lo && token + NBW * 32 <= all_hi, token, buffer);
    }

    l = pair_sum(l);
    __syncthreads();  // (the last step's operands are read: their place is for the rows now)
    {
    const Args &a = args_again<Args>();
    const float back = power_of_two(ref - kPTop + (E4M3 ? 8 : 0));
    const float poison = s.ok ? 0.f : __uint_as_float(0x7fc00000u);
    const int row = row0 + n, all_rows = rows_of(a, FIRST);
    const bool here = row < all_rows, live = here && row / a.group < s.count;
    const float norm = l == 0.f ? 0.f : 1.f / l;
    // 4 neighbouring channels, 4 mm + 128 i: words of one value row, blocks i of O, or for DP 64 rows 16 apart too
    auto channels = [&](int i, int j) {
        if constexpr (DP == 64) return f32x4{acc[0][j], acc[0][j + 8], acc[1][j], acc[1][j + 8]};
        else return f32x4{acc[i * 4][j], acc[i * 4 + 1][j], acc[i * 4 + 2][j], acc[i * 4 + 3][j]};
    };
    constexpr int BIG = DP == 256 ? 2 : 1, JS = DP == 64 ? 8 : 16;
    if (parted) {
        // (lane by lane, as it lies in the registers)
        float *part;
        int rows = kWideRows;
        if constexpr (FIRST) {
            part = stair_of(a, (int64_t)range + head * entries_of(a, FIRST) + entry);
            rows = a.first_rows;
        } else {
            part = slot_of(a, slot);
        }
        f32x4 *to = reinterpret_cast<f32x4 *>(part + 2 * rows) + rb * (BIG * JS) * 64 + lane;
        if constexpr (TG > 1) {
            // the waves with the same rows: all sums into LDS, then each wave joins some of the words
            constexpr int WORDS = BIG * JS, MINE = WORDS / TG;
            static_assert(sizeof(k_lds) >= 4 * WORDS * 1024 && sizeof(v_lds) >= 4 * WORDS * 1024, "room for eight waves' sums");
            __shared__ float wave_m[8][32], wave_l[8][32];
            auto place = [&](int w) { return reinterpret_cast<f32x4 *>(w < 4 ? &k_lds[0][0] : &v_lds[0][0]) + (w & 3) * WORDS * 64 + lane; };
            f32x4 *out = place(wave);
#pragma unroll
            for (int i = 0; i < BIG; i++)
#pragma unroll
                for (int j = 0; j < JS; j++) out[(i * JS + j) * 64] = channels(i, j) * back;
            if (h == 0) {
                wave_m[wave][n] = m;
                wave_l[wave][n] = l;
            }
            __syncthreads();
            float f[TG], sum = 0.f, top = kFloor;
#pragma unroll
            for (int t = 0; t < TG; t++) top = fmaxf(top, wave_m[t * RB + rb][n]);
#pragma unroll
            for (int t = 0; t < TG; t++) {
                f[t] = __builtin_amdgcn_exp2f(wave_m[t * RB + rb][n] - top);
                sum += f[t] * wave_l[t * RB + rb][n];
            }
            if (tg == 0 && here && h == 0) {
                part[rb * 32 + n] = top;
                part[rows + rb * 32 + n] = sum;
            }
            if (row0 < all_rows) {
#pragma unroll
                for (int w = 0; w < MINE; w++) {
                    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < TG; t++) y += f[t] * place(t * RB + rb)[(tg * MINE + w) * 64];
                    to[(tg * MINE + w) * 64] = y;
                }
            }
        } else if (row0 < all_rows) {
            if (here && h == 0) {
                part[rb * 32 + n] = m;
                part[rows + rb * 32 + n] = l;
            }
#pragma unroll
            for (int i = 0; i < BIG; i++)
#pragma unroll
                for (int j = 0; j < JS; j++) to[(i * JS + j) * 64] = channels(i, j) * back;
        }
    } else if constexpr (DT == ENATTEN_F32) {
        const int t_row = row / a.group;
        const int64_t to = b * a.o.sb + (head * a.group + row - t_row * a.group) * a.o.sh + t_row * a.o.st;
#pragma unroll
        for (int i = 0; i < BIG; i++)
#pragma unroll
            for (int j = 0; j < JS; j++) {
                const int d = 4 * (j / 4 * 8 + h * 4 + j % 4) + i * 128;
                if (here && d < a.D) store_channels<DT>(a.o, to + d, (live ? channels(i, j) * norm * back : f32x4{0.f, 0.f, 0.f, 0.f}) + poison);
            }
    } else {
        // 64 channels at a time through LDS, so that a store takes whole lines of 8 rows and not pieces of
        // 8 bytes of 32: a wave's place is 32 rows of 128 bytes, their runs of 16 bytes swapped by row
        char *place = reinterpret_cast<char *>(&k_lds[0][0]) + wave * 4096;
        const int cols = lane % 8;
#pragma unroll
        for (int i = 0; i < BIG; i++)
#pragma unroll
            for (int q = 0; q < JS / 8; q++) {
                u32x2 y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const f32x4 x = (live ? channels(i, q * 8 + j) * norm * back : f32x4{0.f, 0.f, 0.f, 0.f}) + poison;
                    y[j] = narrow4<DT>(x);
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int mm = j / 4 * 8 + h * 4 + j % 4;
                    *reinterpret_cast<u32x2 *>(place + n * 128 + ((mm / 2) ^ (n / 2 & 7)) * 16 + mm % 2 * 8) = y[j];
                }
                __builtin_amdgcn_wave_barrier();
                const int d = i * 128 + q * 64 + cols * 8;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int r = k * 8 + lane / 8, to_row = row0 + r, t = to_row / a.group;
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(place + r * 128 + (cols ^ (r / 2 & 7)) * 16);
                    if (to_row < all_rows && d < a.D)
                        *reinterpret_cast<u32x4 *>(static_cast<unsigned short *>(const_cast<void *>(a.o.ptr)) + b * a.o.sb +
                                                   (head * a.group + to_row - t * a.group) * a.o.sh + t * a.o.st + d) = x;
                }
            }
    }
    }
    if (++entry == entries) {
        entry = 0;
        head++;
    }
    }
}

// Tiles that ranges cut, joined: one workgroup per (start of a range, 16 rows), the one of the first
// start within a tile for all its parts.  A wave takes every fourth part: 16 lanes over the rows, 4 over
// neighbouring words of 4 channels.
template <int DP, int DT>
__device__ __forceinline__ void join_rows_body(const AttnArgs &a) {
    constexpr int BLOCKS = kWideRows / 16, WORDS = DP / 16;
    const int range = blockIdx.x / BLOCKS, n = threadIdx.x % 16, c = threadIdx.x / 16 % 4, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int *note = reinterpret_cast<const int *>(a.ws);
    const int tile = note[range];
    if (tile < 0 || note[range - 1] == tile) return;  // (the first range starts with a tile)
    const int entries = entries_of(a, false), all_rows = rows_of(a, false), head = tile / entries, entry = tile - head * entries;
    const int which = entry / a.row_tiles, r = blockIdx.x % BLOCKS * 16 + n;
    const int row = (entry - which * a.row_tiles) * kWideRows + r;
    if (row - n >= all_rows) return;  // (none of the 16)
    const int count = a.tb.counts ? a.tb.counts[which] : a.T;
    // the parts: the end of the range before, then the beginnings of the ranges that start within the tile
    int parts = 1;
    for (;; parts += 64) {
        const int q = range + parts - 1 + lane;
        const unsigned long long others = __ballot(q >= a.parts || note[q] != tile);
        if (others) {
            parts += __ffsll(others) - 1;
            break;
        }
    }
    // rows behind the last one have no sums: they go along with its
    const int from = min(r, all_rows - 1 - (row - r));
    auto part_at = [&](int q) { return slot_of(a, q ? 2 * (range + q - 1) : 2 * range - 1); };
    float top = kFloor, sum = 0.f;
    for (int q = wave; q < parts; q += 4) top = fmaxf(top, part_at(q)[from]);
    f32x4 y[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; i++) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int q = wave; q < parts; q += 4) {
        const float *part = part_at(q);
        const float f = __builtin_amdgcn_exp2f(part[from] - top);
        sum += f * part[kWideRows + from];
        const f32x4 *x = reinterpret_cast<const f32x4 *>(part + 2 * kWideRows) + from / 32 * (DP / 8) * 64 + from % 32;
        // the word of channels 4 mm + 128 k .. lies at place 16 k + j of the lanes h
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            const int mm = i % 8 * 4 + c, place = i / 8 * 16 + mm / 8 * 4 + mm % 4, h = mm / 4 % 2;
            y[i] += f * x[place * 64 + h * 32];
        }
    }
    __shared__ __align__(16) f32x4 red[4][WORDS][64];
    __shared__ float tops[4][16], sums[4][16];
    if (c == 0) {
        tops[wave][n] = top;
        sums[wave][n] = sum;
    }
#pragma unroll
    for (int i = 0; i < WORDS; i++) red[wave][i][lane] = y[i];
    __syncthreads();
    top = kFloor;
#pragma unroll
    for (int v = 0; v < 4; v++) top = fmaxf(top, tops[v][n]);
    float f[4];
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < 4; v++) {
        f[v] = __builtin_amdgcn_exp2f(tops[v][n] - top);
        sum += f[v] * sums[v][n];
    }
    if (row >= all_rows) return;
    const Place where = place_of(a, which, head, row, false);
    const int64_t to = offset_of(a.o, where);
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < WORDS / 4; k++) {
        const int i = k * 4 + wave, d = i * 16 + c * 4;
        if (d >= a.D) break;
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < 4; v++) z += f[v] * red[v][i][lane];
        store_channels<DT>(a.o, to + d, where.t < count ? z * norm : f32x4{0.f, 0.f, 0.f, 0.f});
    }
}

}  // namespace
}  // namespace enatten
