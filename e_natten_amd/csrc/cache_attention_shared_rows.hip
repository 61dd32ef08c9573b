// cache_attention of runs that share their first tokens (cache_attention_shared.hip): tiles of many rows, and
// the joins behind them.  The kernel is that of cache_attention_rows.hip.
#include "cache_attention_rows_body.h"

namespace enatten {
namespace {

// Tiles of 32, 64 or 128 rows, steps of 128 tokens (256 for 32 rows, and of up to 64 channels) that eight, four or two
// groups of waves share; above 128 channels, where LDS has no room for such steps, tiles of 256 rows.
//
// A workgroup takes 8.5 us to its first step (shares 1.4, who reads 1, pages and scales 1.3, rows of q 2.8, the first
// codes 2) and 2 to 3 to leave its part.  Steps of 128 rows by 128 tokens of 128 channels take 2.9 us, of which vector
// instructions (exponentials, the codes' widening) fill two thirds and the matrix cores one: a wave's widening takes 0.4
// to 0.7 us, the next loads' requests 0.3 to 0.6, products and exponentials 1.4.  Half of the waves one phase ahead of the
// others (products before widening) came to the same time, whichever half it was.  Steps of 32 rows by 256 tokens take 3.2
// us, 64 KB per CU, as fast as HBM brings them (5.2 TB/s).
template <int DP, bool E4M3, int DT, int TG>
__global__ __launch_bounds__(512, 2) void run_rows(SharedArgs args) {
    rows_body<DP, E4M3, DT, TG, TG == 1 ? 1 : TG == 8 && DP == 128 ? 4 : 2>(args);
}

// The parts of the first part's tiles joined, and with the second part's.  One workgroup per (tile, 16 rows, 32
// channels), as few tiles have many parts.  A wave takes every fourth part: 16 lanes over the rows, 4 over neighbouring
// words of 4 channels.
template <int DP, int DT>
__global__ __launch_bounds__(256) void run_join(SharedArgs a, int tile_rows, int second_rows) {
    constexpr int WORDS = 2, SPLIT = DP / 32;
    const int n = threadIdx.x % 16, c = threadIdx.x / 16 % 4, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int block = blockIdx.x;
    const int split = block % SPLIT;
    block /= SPLIT;
    const int groups = a.first_rows / 16, r = block % groups * 16 + n, tile = block / groups;
    const int entries = entries_of(a, true), all_rows = rows_of(a, true), head = tile / entries, entry = tile - head * entries;
    const int which = entry / a.first_tiles, row = (entry - which * a.first_tiles) * tile_rows + r;
    if (row - n >= all_rows || split * 32 >= a.D) return;
    const int *ranges = reinterpret_cast<const int *>(a.first_ws) + 2 * tile;
    const int end = shared_end(a, which);  // (0: the first part left nothing)
    const int first = end ? ranges[0] : 0, parts = end ? ranges[1] - first + 1 : 0;
    // rows behind the last one have no sums: they go along with its
    const int from = min(r, all_rows - 1 - (row - r));
    auto part_at = [&](int q) { return stair_of(a, (int64_t)first + q + tile); };
    float top = kFloor, sum = 0.f;
    for (int q = wave; q < parts; q += 4) top = fmaxf(top, part_at(q)[from]);
    f32x4 y[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; i++) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int q = wave; q < parts; q += 4) {
        const float *part = part_at(q);
        const float f = __builtin_amdgcn_exp2f(part[from] - top);
        sum += f * part[a.first_rows + from];
        const f32x4 *x = reinterpret_cast<const f32x4 *>(part + 2 * a.first_rows) + from / 32 * (DP / 8) * 64 + from % 32;
        // the word of channels 4 mm + 128 k.. lies at place 16 k + j of the lanes h
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            const int word = split * WORDS + i, mm = word % 8 * 4 + c, place = word / 8 * 16 + mm / 8 * 4 + mm % 4, h = mm / 4 % 2;
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
    const int d = (split * WORDS + wave) * 16 + c * 4;
    if (wave >= WORDS || row >= all_rows || d >= a.D) return;
    top = kFloor;
#pragma unroll
    for (int v = 0; v < 4; v++) top = fmaxf(top, tops[v][n]);
    sum = 0.f;
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; v++) {
        const float f = __builtin_amdgcn_exp2f(tops[v][n] - top);
        sum += f * sums[v][n];
        z += f * red[v][wave][lane];
    }
    const Place where = place_of(a, which, head, row, true);
    int len, count;
    const bool ok = sequence_of(a.tb, where.b, len, count);
    const bool shares = end && ok && count > 0 && len - count >= end;
    if (!shares) {
        top = kFloor;
        sum = 0.f;
        z = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int own = where.t * a.group + where.head - head * a.group, own_entry = where.b * a.row_tiles + own / second_rows;
    const int own_row = own % second_rows;
    const int *note = reinterpret_cast<const int *>(a.ws) + 2 * own_entry;
    const int own_first = a.parts ? note[0] : own_entry, items = a.parts ? note[1] : 1;
    for (int i = 0; i < items; i++) {
        const float *p = part_of(a, second_rows, own_first + i, head, false);
        const float m = p[own_row], most = fmaxf(top, m), f = __builtin_amdgcn_exp2f(top - most), g = __builtin_amdgcn_exp2f(m - most);
        z = f * z + g * *reinterpret_cast<const f32x4 *>(p + 2 * second_rows + own_row * a.D + d);
        sum = f * sum + g * p[second_rows + own_row];
        top = most;
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum, poison = ok ? 0.f : __uint_as_float(0x7fc00000u);
    store_channels<DT>(a.o, offset_of(a.o, where) + d, (where.t < count ? z * norm : f32x4{0.f, 0.f, 0.f, 0.f}) + poison);
}

template <int DP, bool E4M3, int DT>
int first_rows(const char *fn, const SharedArgs &a, int rows, hipStream_t st) {
    ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "run_rows", st);
    if constexpr (DP <= 128) {
        if (rows == 32) run_rows<DP, E4M3, DT, 8><<<a.first_parts, 512, 0, st>>>(a);
        else if (rows == 64) run_rows<DP, E4M3, DT, 4><<<a.first_parts, 512, 0, st>>>(a);
        else run_rows<DP, E4M3, DT, 2><<<a.first_parts, 512, 0, st>>>(a);
    } else {
        run_rows<DP, E4M3, DT, 1><<<a.first_parts, 512, 0, st>>>(a);
    }
    return launched(fn);
}
template <int DP, int DT>
int join(const char *fn, const SharedArgs &a, int rows, int second, hipStream_t st) {
    const int blocks = a.runs * a.first_tiles * a.heads_kv * (a.first_rows / 16) * (DP / 32);  // (fewer than 2^24)
    ProfScope prof(ENATTEN_KERNEL_CACHE_JOIN, "run_join", st);
    run_join<DP, DT><<<blocks, 256, 0, st>>>(a, rows, second);
    return launched(fn);
}

// f(head dim, whether E4M3, type) with constants; float32 above 128 channels has no such tiles
template <int V> using Const = std::integral_constant<int, V>;
template <int DP, class F>
int by_type(const SharedArgs &a, F f) {
    if (a.dtype == ENATTEN_BF16) return f(Const<DP>{}, Const<ENATTEN_BF16>{});
    if constexpr (DP <= 128)
        if (a.dtype == ENATTEN_F32) return f(Const<DP>{}, Const<ENATTEN_F32>{});
    return f(Const<DP>{}, Const<ENATTEN_F16>{});
}
template <class F>
int by_dim(const SharedArgs &a, F f) {
    return a.D <= 64 ? by_type<64>(a, f) : a.D <= 128 ? by_type<128>(a, f) : by_type<256>(a, f);
}

}  // namespace

int launch_first_rows(const char *fn, const SharedArgs &a, int rows, bool e4m3, hipStream_t st) {
    return by_dim(a, [&](auto dp, auto dt) {
        return e4m3 ? first_rows<dp.value, true, dt.value>(fn, a, rows, st) : first_rows<dp.value, false, dt.value>(fn, a, rows, st);
    });
}
int launch_last_join(const char *fn, const SharedArgs &a, int rows, int second, hipStream_t st) {
    return by_dim(a, [&](auto dp, auto dt) { return join<dp.value, dt.value>(fn, a, rows, second, st); });
}

}  // namespace enatten
