// cache_attention with many rows per cache head (chunks of prompts): tiles of 256 rows.
//
// The mathematics is that of cache_attention.hip, but that the sum of the probabilities is formed before
// they are rounded to float16: a result is a mean of values up to that rounding.  With this many rows the
// matrix cores bound the call, so the codes are turned into float16 once for all rows: eight waves take 32
// rows each, and go together over steps of 8192 / DP tokens whose keys and values lie in LDS as the operands of
// v_mfma_f32_32x32x16_f16, in the order in which lanes read them.  Waves 0 to 3 turn keys, 4 to 7
// values; codes come two steps ahead into registers and are turned into the other half of LDS while the
// step's products run.
//
// S^T = K Q^T again leaves the probabilities in the registers that O^T = V^T P^T takes: lane (n, h) has
// the tokens 4h .. 4h+3 (+ 8, 16, ...) of row n, and V is laid out with the same tokens in a lane's eight.
//
// What bounds it.  exp2 runs at a quarter of the rate: with 128 channels half as many cycles go into it as
// into the products, and about as many again into the other vector instructions, while the clock goes
// down under all of them (the matrix cores were busy for 41% of the time).  So the exponentials of a
// group of tokens are issued beside the products of another, and the rest of the softmax is kept short:
// the scales of values are a summand of the exponent, the maximum lags (by up to 2^8), masks are a
// constant and not a selection of exponents.
//
// Measured on MI355X, 2048 tokens each of sequences of 16384 and 12288, 16 heads of 128 channels over 4
// of an int8 cache, bfloat16: 490 to 510 us by the card, 880 to 910 TFLOP/s; a product of two 8192 x 8192 matrices
// reaches 1181 in float16.  64 channels: 327 us, where a logit takes as many vector instructions for half the
// products; 256 channels: 1135 us, with 50 registers spilled; float32, in two terms: 64 channels 472 us, 128:
// 825 us.  512 new tokens: 154 us, 128: 62 us; the first 8192 tokens of two prompts (8192 and 8192 long): 760 us.
#include "cache_attention.h"

#include <type_traits>

namespace enatten {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// The kernel's arguments, read anew: what is used once per row tile or per 64 groups of tokens does not
// stay in scalar registers across the steps (held there, 124 of them were spilled, for 7% at head_dim 128).
__device__ __forceinline__ const AttnArgs &args_again() {
    typedef const AttnArgs __attribute__((address_space(4))) *Kernarg;
    Kernarg p = (Kernarg)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const AttnArgs *)p;
}

// DP: head_dim rounded up to 64, 128 or 256; DT: type of q and o, float32 in two float16 terms of q and p.
template <int DP, bool E4M3, int DT>
__global__ __launch_bounds__(512, 2) void attend_rows(AttnArgs args) {
    constexpr int TERMS = DT == ENATTEN_F32 ? 2 : 1;
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
    // Rows of q stay in registers, at head dims above 128 all but the last operands, for which there are
    // none left: those a lane puts into LDS and reads again.
    constexpr int KEPT = DP == 256 ? 10 : SD;
    __shared__ f16x8 q_lds[8 * 64 * (SD - KEPT) + 1];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (branches on it are the wave's)

    // The workgroup's range of steps.  Blocks 8 apart share an XCD and its L2: they get neighbouring ranges,
    // which read the same keys and values where they belong to the same head.
    const AttnArgs &a = args;
    const int range = blockIdx.x % 8 * (a.parts / 8) + blockIdx.x / 8;
    const Ranges line = ranges_of<kWideRows, TOK>(a);
    const int heads = a.heads_kv;
    int64_t end = min((range + 1) * line.each, line.line * heads);
    int64_t at_step = range * line.each;
    const int entries = a.B * a.row_tiles, all_rows = a.T * a.group;
    int *note = reinterpret_cast<int *>(a.ws) + range;
    int head, entry, into = 0;
    if (line.whole) {  // a tile each
        head = range / entries;
        entry = range - head * entries;
        at_step = head < heads ? 0 : end;
        end = min(end, (int64_t)1);
    } else {
        head = (int)(at_step / line.line);
        entry = at_step < end ? tile_at<kWideRows, TOK>(a, at_step - head * line.line, into) : 0;
    }
    if (threadIdx.x == 0) *note = into ? head * entries + entry : -1;

    for (; at_step < end; into = 0) {
    const AttnArgs &a = args_again();
    const Span s = span_of<kWideRows>(a, entry);
    const int total = steps_of<TOK>(s), counted = max(1, total), step0 = into;
    const int step1 = line.whole ? total : min(total, (int)min((int64_t)counted, step0 + (end - at_step)));
    const bool parted = !line.whole && (into || step0 + (end - at_step) < counted);
    const int slot = into ? 2 * range : 2 * range + 1;
    at_step += counted - into;
    const int b = entry / a.row_tiles, row0 = (entry - b * a.row_tiles) * kWideRows + wave * 32;
    const int base = s.lo & -16;

    // the lane's row; q: lane (n, h) has channels 16 c + 8 h .. + 7
    const int row = min(row0 + n, all_rows - 1), t_row = row / a.group;
    const bool live = row0 + n < all_rows && t_row < s.count;
    const int hi_r = live ? s.start + t_row + 1 : 0, seen = a.window ? a.window : hi_r;  // tokens hi_r - seen .. hi_r - 1
    f16x8 qf[KEPT][TERMS], *q_rest = &q_lds[threadIdx.x];
    float unit, l;
    {
        const int64_t at = b * a.q.sb + (head * a.group + row - t_row * a.group) * a.q.sh + t_row * a.q.st;
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
    float m = kFloor;
    float ref = -126.f;

    // places of the groups of 16 tokens: lane i holds group `filled` + i
    int filled = -64;
    int64_t at = 0;
    float z_at = 0.f;  // of keys, or log2 of values (for float32 the scale itself)
    const bool for_v = wave >= 4;
    auto fill = [&](int group) {
        const AttnArgs &a = args_again();
        filled = group;
        const int token = base + (group + lane) * 16;
        at = 0;
        z_at = for_v && TERMS == 1 ? -INFINITY : 0.f;
        if (token < s.hi && token >= 0) {
            const int column = token / a.tb.page, within = token - column * a.tb.page;
            const int p = a.tb.pages[b * a.tb.stride + column];
            if ((unsigned)p >= (unsigned)a.tb.num_pages) {
                z_at = __uint_as_float(0x7fc00000u);
            } else if (for_v) {
                at = p * a.v.sp + head * a.v.sh + within * a.v.st;
                z_at = finite_or_nan(a.v.scales[p * a.v.zp + head * a.v.zh]);
                if (TERMS == 1) z_at = __builtin_amdgcn_logf(z_at);
            } else {
                at = p * a.k.sp + head * a.k.sh + within * a.k.st;
                z_at = a.k.scales[p * a.k.zp + head * a.k.zh];
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
        raw_z = __shfl(z_at, here + (lane & (GR - 1)), 64);
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
                    st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, c < KEPT ? qf[c][t] : q_rest[(c - KEPT) * 512], st[i], 0, 0, 0);
            }
        }

        // lane's tokens: 32 i + 16 g + 8 (j / 4) + 4 h + j % 4 for its 8 values j of a group
        if (!whole) {
#pragma unroll
            for (int i = 0; i < NB; i++)
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
            for (int g = 0; g < GR; g++) {
                const int first = token + g * 16;
                if ((bad >> g & 1) && first < hi_r && first + 16 > hi_r - seen) l = __uint_as_float(0x7fc00000u);
            }
        }
        const float unit_z = power_of_two(ref - kPTop);
        float u[GR], top = kFloor;
#pragma unroll
        for (int g = 0; g < GR; g++) {
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

    __syncthreads();  // (the last tile's operands are read)
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

    l = pair_sum(l);
    __syncthreads();  // (the last step's operands are read: their place is for the rows now)
    {
    const AttnArgs &a = args_again();
    const float back = power_of_two(ref - kPTop + (E4M3 ? 8 : 0));
    const float poison = s.ok ? 0.f : __uint_as_float(0x7fc00000u);
    const float norm = l == 0.f ? 0.f : 1.f / l;
    const int row = row0 + n;
    const bool here = row < a.T * a.group, live = here && row / a.group < s.count;
    // 4 neighbouring channels, 4 mm + 128 i: words of one value row, blocks i of O, or for DP 64 rows 16 apart too
    auto channels = [&](int i, int j) {
        if constexpr (DP == 64) return f32x4{acc[0][j], acc[0][j + 8], acc[1][j], acc[1][j + 8]};
        else return f32x4{acc[i * 4][j], acc[i * 4 + 1][j], acc[i * 4 + 2][j], acc[i * 4 + 3][j]};
    };
    constexpr int BIG = DP == 256 ? 2 : 1, JS = DP == 64 ? 8 : 16;
    if (parted) {
        // (lane by lane, as it lies in the registers)
        float *part = slot_of(a, slot);
        if (here && h == 0) {
            part[wave * 32 + n] = m;
            part[kWideRows + wave * 32 + n] = l;
        }
        f32x4 *to = reinterpret_cast<f32x4 *>(part + 2 * kWideRows) + wave * (BIG * JS) * 64 + lane;
        if (row0 < a.T * a.group) {
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
                    if (to_row < a.T * a.group && d < a.D)
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
__global__ __launch_bounds__(256) void join_rows(AttnArgs a) {
    constexpr int BLOCKS = kWideRows / 16, WORDS = DP / 16;
    const int range = blockIdx.x / BLOCKS, n = threadIdx.x % 16, c = threadIdx.x / 16 % 4, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int *note = reinterpret_cast<const int *>(a.ws);
    const int tile = note[range];
    if (tile < 0 || note[range - 1] == tile) return;  // (the first range starts with a tile)
    const int entries = a.B * a.row_tiles, head = tile / entries, entry = tile - head * entries;
    const int b = entry / a.row_tiles, r = blockIdx.x % BLOCKS * 16 + n;
    const int row = (entry - b * a.row_tiles) * kWideRows + r;
    if (row - n >= a.T * a.group) return;  // (none of the 16)
    const int count = a.tb.counts ? a.tb.counts[b] : a.T;
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
    const int from = min(r, a.T * a.group - 1 - (row - r));
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
    if (row >= a.T * a.group) return;
    const int t = row / a.group;
    const int64_t to = b * a.o.sb + (head * a.group + row - t * a.group) * a.o.sh + t * a.o.st;
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < WORDS / 4; k++) {
        const int i = k * 4 + wave, d = i * 16 + c * 4;
        if (d >= a.D) break;
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < 4; v++) z += f[v] * red[v][i][lane];
        store_channels<DT>(a.o, to + d, t < count ? z * norm : f32x4{0.f, 0.f, 0.f, 0.f});
    }
}

template <int DP, bool E4M3, int DT>
int launch(const char *fn, const AttnArgs &a, hipStream_t st) {
    {
        ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "attend_rows", st);
        attend_rows<DP, E4M3, DT><<<a.parts, 512, 0, st>>>(a);
    }
    const int rc = launched(fn);
    if (rc) return rc;
    ProfScope prof(ENATTEN_KERNEL_CACHE_JOIN, "join_rows", st);
    join_rows<DP, DT><<<a.parts * (kWideRows / 16), 256, 0, st>>>(a);
    return launched(fn);
}
template <int DP, bool E4M3>
int launch_type(const char *fn, const AttnArgs &a, hipStream_t st) {
    if (a.dtype == ENATTEN_BF16) return launch<DP, E4M3, ENATTEN_BF16>(fn, a, st);
    if constexpr (DP <= 128)
        if (a.dtype == ENATTEN_F32) return launch<DP, E4M3, ENATTEN_F32>(fn, a, st);
    return launch<DP, E4M3, ENATTEN_F16>(fn, a, st);
}
template <bool E4M3>
int launch_dim(const char *fn, const AttnArgs &a, hipStream_t st) {
    if (a.D <= 64) return launch_type<64, E4M3>(fn, a, st);
    if (a.D <= 128) return launch_type<128, E4M3>(fn, a, st);
    return launch_type<256, E4M3>(fn, a, st);
}

}  // namespace

int launch_attend_rows(const char *fn, const AttnArgs &a, bool e4m3, hipStream_t st) {
    return e4m3 ? launch_dim<true>(fn, a, st) : launch_dim<false>(fn, a, st);
}

}  // namespace enatten
