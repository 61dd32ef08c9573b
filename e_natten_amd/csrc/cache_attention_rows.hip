// cache_attention with many rows per cache head (chunks of prompts): tiles of 256 rows.
//
// The mathematics is that of cache_attention.hip.  With this many rows the matrix cores bound the call,
// so the codes are turned into float16 once for all rows: eight waves take 32 rows each, and go
// together over steps of 8192 / DP tokens whose keys and values lie in LDS as the operands of
// v_mfma_f32_32x32x16_f16, in the order in which lanes read them.  Waves 0 to 3 turn keys, 4 to 7
// values; codes come two steps ahead into registers and are turned into the other half of LDS while the
// step's products run.
//
// S^T = K Q^T again leaves the probabilities in the registers that O^T = V^T P^T takes: lane (n, h) has
// the tokens 4h .. 4h+3 (+ 8, 16, ...) of row n, and V is laid out with the same tokens in a lane's eight.
//
// exp2 is a quarter-rate instruction on which as many cycles are spent as on the products, so the rest
// of the softmax is kept short: see cache_attention.hip.
#include "cache_attention.h"

#include <type_traits>

namespace enatten {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// DP: head_dim rounded up to 64, 128 or 256; TERMS: float16 terms of q and p.
template <int DP, bool E4M3, int TERMS>
__global__ __launch_bounds__(512, 2) void attend_rows(AttnArgs a) {
    constexpr int TOK = 8192 / DP;    // tokens of a step: 128, 64, 32
    constexpr int NB = TOK / 32;      // blocks of 32 of them
    constexpr int GR = TOK / 16;      // groups of 16, each within a page
    constexpr int SD = DP / 16;       // products along head_dim of S
    constexpr int OB = DP / 32;       // blocks of 32 channels of O
    constexpr int CH = DP / 16;       // loads of 16 codes per token
    constexpr int QUADS = DP / 4;     // words of 4 channels
    // operands of one step: K [NB][SD][64 lanes][8], V [OB][TOK / 16][64 lanes][8]; eight lanes that turn
    // one or two tokens write to as many operands of K, which therefore start 1 or 2 lanes apart in the banks
    constexpr int PART = 64 + (CH < 8 ? 8 / CH : 1);
    __shared__ f16x8 k_lds[2][NB * SD * PART], v_lds[2][1024];
    __shared__ float z_lds[2][3][GR];  // of the step's groups: key scales, value scales (log2), their inverses
    __shared__ int z_bad[2][2];        // ... and which of either are not finite (0 in their place)
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (branches on it are the wave's)

    // Which row tile, and which of its steps.  Blocks 8 apart share an XCD and its L2: neighbours in
    // the order of the cache heads go to different ones, the row tiles of a head to the same where
    // their number allows.  Later rows see more tokens: they come first.
    const int heads = a.heads_kv;
    int head;
    Share w;
    if (a.parts) {
        head = blockIdx.x % heads;
        w = share_of<kWideRows, TOK, 1>(a, blockIdx.x / heads);
        if (w.entry < 0) return;
        note_share(a, w, head);
    } else {
        const int pair = blockIdx.x % (heads * a.B);
        head = pair % heads;
        w.entry = pair / heads * a.row_tiles + a.row_tiles - 1 - blockIdx.x / (heads * a.B);
        w.items = 1;
    }
    const int entry = w.entry;
    const Span s = span_of<kWideRows>(a, entry);
    if (!a.parts) {
        w.step0 = 0;
        w.step1 = steps_of<TOK>(s);
    }
    const int b = entry / a.row_tiles, row0 = (entry - b * a.row_tiles) * kWideRows + wave * 32;
    const int step0 = w.step0, step1 = w.step1;
    const int base = s.lo & -16;
    const int all_rows = a.T * a.group;

    // the lane's row; q: lane (n, h) has channels 16 c + 8 h .. + 7
    const int row = min(row0 + n, all_rows - 1), t_row = row / a.group;
    const bool live = row0 + n < all_rows && t_row < s.count;
    const int hi_r = live ? s.start + t_row + 1 : 0, lo_r = live && a.window ? max(hi_r - a.window, 0) : 0;
    f16x8 qf[SD][TERMS];
    float unit, bad_q;
    {
        const int64_t at = b * a.q.sb + (head * a.group + row - t_row * a.group) * a.q.sh + t_row * a.q.st;
        const float flip = a.scale < 0.f ? -1.f : 1.f;  // into q, so that units are not negative
        float x[SD][8], top = 0.f, nan = 0.f;
#pragma unroll
        for (int c = 0; c < SD; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[c][j] = 0.f;
            if (c * 16 < a.D) load_channels<8>(a.q, a.dtype, a.wide_q, at + c * 16 + h * 8, x[c]);
        }
#pragma unroll
        for (int c = 0; c < SD; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                top = fmaxf(top, fabsf(x[c][j]));
                nan += x[c][j] * 0.f;  // a value that is not finite makes its row NaN
            }
        nan = pair_sum(nan);
        top = pair_max(top);
        const int up = kTop + 1 - (top > 0.f ? __builtin_amdgcn_frexp_expf(top) : 0);
        unit = __builtin_ldexpf(fabsf(a.scale) * kLog2e, -up + (E4M3 ? 8 : 0));
        bad_q = nan;
#pragma unroll
        for (int c = 0; c < SD; c++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float y0 = __builtin_ldexpf(x[c][j] * flip, up), y1 = __builtin_ldexpf(x[c][j + 1] * flip, up);
                if constexpr (TERMS == 2) {
                    f16x2 high, low;
                    two_terms(y0, y1, high, low);
                    qf[c][0][j] = high[0];
                    qf[c][0][j + 1] = high[1];
                    qf[c][1][j] = low[0];
                    qf[c][1][j + 1] = low[1];
                } else {
                    qf[c][0][j] = (_Float16)y0;
                    qf[c][0][j + 1] = (_Float16)y1;
                }
            }
    }
    // tokens that any, and that all rows of the wave see
    const int t_first = min(row0, all_rows - 1) / a.group, t_last = min(min(row0 + 31, all_rows - 1) / a.group, s.count - 1);
    const bool any_row = row0 < all_rows && t_first < s.count;
    const int some_lo = any_row && a.window ? max(s.start + t_first + 1 - a.window, 0) : 0;
    const int some_hi = any_row ? s.start + t_last + 1 : 0;
    const int all_lo = a.window ? max(s.start + t_last + 1 - a.window, 0) : 0, all_hi = s.start + t_first + 1;

    f32x16 acc[OB];
#pragma unroll
    for (int i = 0; i < OB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
    float m = kFloor, l = 0.f;
    float ref = -126.f;

    // places of the groups of 16 tokens: lane i holds group `filled` + i
    int filled = -64;
    int64_t at = 0;
    float z_k = 0.f, z_v = 0.f;
    const bool for_v = wave >= 4;
    auto fill = [&](int group) {
        filled = group;
        const int token = base + (group + lane) * 16;
        at = 0;
        z_k = 0.f;
        z_v = TERMS == 1 ? -INFINITY : 0.f;  // (its log2, but for float32)
        if (token < s.hi && token >= 0) {
            const int column = token / a.tb.page, within = token - column * a.tb.page;
            const int p = a.tb.pages[b * a.tb.stride + column];
            if ((unsigned)p < (unsigned)a.tb.num_pages) {
                at = for_v ? p * a.v.sp + head * a.v.sh + within * a.v.st : p * a.k.sp + head * a.k.sh + within * a.k.st;
                z_k = a.k.scales[p * a.k.zp + head * a.k.zh];
                z_v = finite_or_nan(a.v.scales[p * a.v.zp + head * a.v.zh]);
                if (TERMS == 1) z_v = __builtin_amdgcn_logf(z_v);
            } else {
                z_k = __uint_as_float(0x7fc00000u);
            }
        }
    };
    // What a thread brings: of keys two runs of 16 codes, of values a word of 4 channels of 8 tokens.
    unsigned raw[8];
    float raw_z = 0.f;  // lanes 0 .. GR - 1 of wave 0: key scales of the step's groups, of wave 4: value scales
    // (offsets within a group of 16 tokens; a wave's 64 runs of keys lie in one group, its 64 words of
    // values too, but for DP 64, where each half of the wave has its own)
    const int run = (wave & 3) * (64 * 4 / DP) + lane / QUADS, quad = lane % QUADS;  // runs of 8 tokens
    const unsigned within = for_v ? run % 2 * 4 * (unsigned)a.v.st + min(quad * 4, a.D - 4)
                                  : (wave * (128 / CH) + lane / CH) % 16 * (unsigned)a.k.st + min(lane % CH * 16, a.D - 16);
    auto fetch = [&](int step) {
        const int group = step * GR;
        if (group >= filled + 64) fill(group);
        const int here = group - filled;
        raw_z = __shfl(for_v ? z_v : z_k, here + (lane & (GR - 1)), 64);
        if (!for_v) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const char *from = static_cast<const char *>(a.k.codes) +
                                   lane_offset(at, here + (wave * (128 / CH) + j * (64 / CH)) / 16);
                const u32x4 x = *reinterpret_cast<const u32x4 *>(from + (DP == 64 ? 0 : j * (64 / CH)) * a.k.st + within);
#pragma unroll
                for (int i = 0; i < 4; i++) raw[j * 4 + i] = x[i];
            }
        } else {
            int64_t off = lane_offset(at, here + (wave & 3) * (64 * 4 / DP) / 2);
            if constexpr (DP == 64) off = lane < 32 ? off : lane_offset(at, here + (wave & 3) * 2 + 1);
            const char *from = static_cast<const char *>(a.v.codes) + off;
#pragma unroll
            for (int j = 0; j < 8; j++)
                raw[j] = *reinterpret_cast<const unsigned *>(from + (j % 4 + j / 4 * 8) * a.v.st + within);
        }
    };
    auto put_as = [&](auto seen, int buffer) {
        constexpr bool SEEN = decltype(seen)::value;
        if (!for_v) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int token = wave * (128 / CH) + j * (64 / CH) + lane / CH, c = lane % CH;
                f16x8 *to = &k_lds[buffer][(token / 32 * SD + c) * PART + token % 32];
                to[0] = widen_row<E4M3, SEEN>(raw[j * 4], raw[j * 4 + 1]);
                to[32] = widen_row<E4M3, SEEN>(raw[j * 4 + 2], raw[j * 4 + 3]);
            }
        } else {
            f16x8 v[4];
            widen_columns<E4M3, SEEN>(raw, v);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int block = DP == 64 ? i / 2 : i + quad / 32 * 4, mm = DP == 64 ? (i & 1) * 16 + quad : quad & 31;
                v_lds[buffer][(block * (TOK / 16) + run / 2) * 64 + run % 2 * 32 + mm] = v[i];
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
    const int wg_row = row0 - wave * 32, wg_last = min((wg_row + kWideRows - 1) / a.group, s.count - 1);
    const int wg_lo = a.window ? max(s.start + wg_last + 1 - a.window, 0) : 0, wg_hi = s.start + wg_row / a.group + 1;
    auto put = [&](int buffer, int step) {
        const int token = base + step * TOK;
        if (E4M3 && token >= wg_lo && token + TOK <= wg_hi) put_as(std::true_type{}, buffer);
        else put_as(std::false_type{}, buffer);
    };

    // One step for the wave's rows.  Masked logits are a large negative number, not an infinity: units
    // are at least 1e-20, so that they end below -1e18 and their exponentials are 0 whatever the maximum
    // (kFloor at least), and a unit of 0 asks for nothing special.
    auto work = [&](bool whole, int token, int buffer) {
        float kz[GR], lz[GR], most_z = -INFINITY;
#pragma unroll
        for (int g = 0; g < GR; g++) {
            kz[g] = z_lds[buffer][0][g];
            lz[g] = z_lds[buffer][1][g];
            most_z = fmaxf(most_z, lz[g]);
        }
        float scale = grow(ref, TERMS == 1 ? most_z : __builtin_amdgcn_logf(most_z));
#pragma unroll
        for (int g = 0; g < GR; g++) lz[g] = TERMS == 1 ? log_weight(lz[g], ref) : plain_weight(lz[g], ref);

        f32x16 st[NB];
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) st[i][j] = 0.f;
        const f16x8 *kp = &k_lds[buffer][lane];
#pragma unroll
        for (int c = 0; c < SD; c++) {
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const f16x8 kf = kp[(i * SD + c) * PART];
#pragma unroll
                for (int t = TERMS - 1; t >= 0; t--)
                    st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[c][t], st[i], 0, 0, 0);
            }
        }

        // lane's tokens: 32 i + 16 g + 8 (j / 4) + 4 h + j % 4 for its 8 values j of a group
        float cap = INFINITY;
        if (!whole) {
            if (token >= hi_r || token + TOK <= lo_r) cap = kFloor;  // the row sees none of them
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int tk = token + i * 32 + j / 4 * 8 + h * 4 + j % 4;
                    st[i][j] = tk >= lo_r && tk < hi_r ? st[i][j] : -3e38f;
                }
        }
        // scales that are not finite: NaN for the rows that see a token of the group
        const int bad = __builtin_amdgcn_readfirstlane(z_bad[buffer][0] | z_bad[buffer][1]);
        if (bad) {
#pragma unroll
            for (int g = 0; g < GR; g++) {
                const int first = token + g * 16;
                if ((bad >> g & 1) && first < hi_r && first + 16 > lo_r) l = __uint_as_float(0x7fc00000u);
            }
        }
        const float unit_z = __builtin_amdgcn_exp2f(ref - kPTop);
        float u[GR], top = kFloor;
#pragma unroll
        for (int g = 0; g < GR; g++) {
            u[g] = fmaxf(unit * kz[g], 1e-20f);
            float most = -3e38f;  // (a constant to start from: else the compiler makes values canonical)
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, st[g / 2][g % 2 * 8 + j]);
            top = fmaxf(top, most * u[g]);
        }
        top = fminf(top, cap);
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
        const f16x8 *vp = &v_lds[buffer][lane];
#pragma unroll
        for (int g = 0; g < GR; g++) {
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
                l = fmaf(part, fminf(z_lds[buffer][2][g] * unit_z, 0x1p40f), l);
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

    if (step0 < step1) {
        fetch(step0);
        put(0, step0);
        if (step0 + 1 < step1) fetch(step0 + 1);
    }
    for (int step = step0; step < step1; step++) {
        const int buffer = (step - step0) & 1;
        __syncthreads();
        if (step + 1 < step1) {
            put(buffer ^ 1, step + 1);
            if (step + 2 < step1) fetch(step + 2);
        }
        const int token = base + step * TOK;
        if (token >= some_hi || token + TOK <= some_lo) continue;
        work(token >= all_lo && token + TOK <= all_hi, token, buffer);
    }

    l += bad_q;
    l = pair_sum(l);
    if (row0 + n >= all_rows) return;
    const float back = __builtin_amdgcn_exp2f(ref - kPTop + (E4M3 ? 8 : 0));
    const float poison = s.ok ? 0.f : __uint_as_float(0x7fc00000u);
    const float norm = (l == 0.f ? 0.f : 1.f / l) * back;
    const int r = wave * 32 + n;
    float *part = part_of(a, kWideRows, w.item, head);
    if (w.items > 1 && h == 0) {
        part[r] = m;
        part[kWideRows + r] = l;
    }
    const int64_t to = b * a.o.sb + (head * a.group + row - t_row * a.group) * a.o.sh + t_row * a.o.st;
    const float f = w.items > 1 ? back : live ? norm : 0.f;
    // 4 neighbouring channels: words of one value row, blocks i of O, or for DP 64 rows 16 apart too
#pragma unroll
    for (int i = 0; i < OB; i += DP == 64 ? 2 : 4)
#pragma unroll
        for (int j = 0; j < (DP == 64 ? 8 : 16); j++) {
            const int mm = j / 4 * 8 + h * 4 + j % 4;
            f32x4 y;
            if constexpr (DP == 64) y = f32x4{acc[0][j], acc[0][j + 8], acc[1][j], acc[1][j + 8]};
            else y = f32x4{acc[i][j], acc[i + 1][j], acc[i + 2][j], acc[i + 3][j]};
            const int d = 4 * mm + i / 4 * 128;
            if (d >= a.D) continue;
            if (w.items > 1) *reinterpret_cast<f32x4 *>(part + 2 * kWideRows + r * a.D + d) = y * f;
            else store_channels(a.o, a.dtype, a.wide_o, to + d, (live ? y * f : f32x4{0.f, 0.f, 0.f, 0.f}) + poison);
        }
}

template <int DP, bool E4M3, int TERMS>
int launch(const char *fn, const AttnArgs &a, int64_t blocks, hipStream_t st) {
    ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "attend_rows", st);
    attend_rows<DP, E4M3, TERMS><<<(int)blocks, 512, 0, st>>>(a);
    return launched(fn);
}
template <int DP, bool E4M3>
int launch_terms(const char *fn, const AttnArgs &a, int64_t blocks, hipStream_t st) {
    if constexpr (DP <= 128)
        if (a.dtype == ENATTEN_F32) return launch<DP, E4M3, 2>(fn, a, blocks, st);
    return launch<DP, E4M3, 1>(fn, a, blocks, st);
}
template <bool E4M3>
int launch_dim(const char *fn, const AttnArgs &a, int64_t blocks, hipStream_t st) {
    if (a.D <= 64) return launch_terms<64, E4M3>(fn, a, blocks, st);
    if (a.D <= 128) return launch_terms<128, E4M3>(fn, a, blocks, st);
    return launch_terms<256, E4M3>(fn, a, blocks, st);
}

}  // namespace

int launch_attend_rows(const char *fn, const AttnArgs &a, bool e4m3, int64_t blocks, hipStream_t st) {
    return e4m3 ? launch_dim<true>(fn, a, blocks, st) : launch_dim<false>(fn, a, blocks, st);
}

}  // namespace enatten
