// cache_attention of sequences that continue one prompt (enatten_cache_attention_shared).
//
//   o = (f y + f' y') / (f l + f' l'),   f = exp(m - max(m, m')), f' likewise
//
// with maximum m, sum l and sums of values y over a sequence's own tokens, and m', l', y' over those that it
// shares with its run.  The latter are a product of their own with as many rows as the whole run has, so that
// the shared codes are read once for all of them.  Both parts of the work are the kernels of cache_attention.hip and
// cache_attention_rows.hip over other rows and tokens, and leave what they come to in the workspace; the last
// launch joins it.
//
// Up to 16 rows in a run both parts have tiles of 16 rows and are one launch, the first part cut so that all of its
// workgroups start at once.  Beyond, it has tiles of 32, 64 or 128 rows (256 above 128 channels) over codes that LDS
// holds as float16, and a launch of its own.
//
// Measured on MI355X, launches under the profiler, bfloat16, heads of 128 channels.  8 sequences, 16 + 16 heads, 480
// shared tokens and up to 40 of their own, int8: 8.8 us and 3.5 for the join.  64 sequences, 32 + 8
// heads, 16384 shared tokens and up to 500, E4M3: 35.6 us for the shared tokens (17.2 GFLOP, 480 TFLOP/s), 14.8 for the
// others, join 7.4.  16 runs of 4, 32 + 4 heads, up to 8192 shared tokens each and up to 300, int8: 41.5, 12.7 and 5.7.
// float32, 16 sequences of 8192 shared tokens, 8 + 8 heads: 15.5 in all (float16 14.8); 64 of them, 16 + 4 heads: 47.6;
// two runs of 14, 5 new tokens, 16 + 4 heads: float16 and bfloat16 52.7, with a window of 6000 tokens 51.8.
// Probabilities take 11 bits into the second product, as in cache_attention.hip; tiles of many rows sum them before that.
// Beside the first launches' steps, about 10 us each go to chains of loads (lengths, pages, codes, q) and the code's
// first run.
#include "cache_attention_body.h"

namespace enatten {
namespace {

template <int DP, int R, bool E4M3, int DT>
__global__ __launch_bounds__(256, waves_of(DP, R, DT == ENATTEN_F32 ? 2 : 1)) void run_attend(SharedArgs a) {
    attend_body<DP, R, E4M3, DT>(a);
}

// The parts of both halves of the work joined, where both have tiles of 16 rows: one workgroup per row.  Lanes over
// the channels, 4 each, and the remaining factor of 256 over the parts.
template <int DT>
__global__ __launch_bounds__(256) void run_join_tiles(SharedArgs a) {
    int block = blockIdx.x;
    const int head = block % a.heads, hk = head / a.group, g = head - hk * a.group;
    block /= a.heads;
    const int t = block % a.T, b = block / a.T, which = b / a.size;
    // (a part that is not cut is the item of its entry's number)
    const int row = ((b - which * a.size) * a.T + t) * a.group + g, own = t * a.group + g;
    const int entry = which * a.first_tiles + row / 16, own_entry = b * a.row_tiles + own / 16;
    const int *note = reinterpret_cast<const int *>(a.first_ws) + 2 * entry, *own_note = reinterpret_cast<const int *>(a.ws) + 2 * own_entry;
    int first = entry, items = 1, own_first = own_entry, own_items = 1;
    if (a.first_parts) first = note[0], items = note[1];
    if (a.parts) own_first = own_note[0], own_items = own_note[1];
    int len, count;
    const bool ok = sequence_of(a.tb, b, len, count);
    const int end = shared_end(a, which);
    if (!(end && ok && count > 0 && len - count >= end)) items = 0;  // (it does not share them)
    const int all = items + own_items;

    __shared__ __align__(16) float red[256][4];
    __shared__ float tops[256], sums[256];
    const int lanes = a.D / 4, groups = 256 / lanes, c = threadIdx.x % lanes, k = threadIdx.x / lanes;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f, top = kFloor;
    if (k < groups) {
#pragma unroll 4
        for (int i = k; i < all; i += groups) {
            const bool of_run = i < items;
            const int r = (of_run ? row : own) % 16;
            const float *p = part_of(a, 16, of_run ? first + i : own_first + i - items, hk, of_run);
            const float m = p[r], most = fmaxf(top, m), f = __builtin_amdgcn_exp2f(top - most), h = __builtin_amdgcn_exp2f(m - most);
            y = f * y + h * *reinterpret_cast<const f32x4 *>(p + 32 + r * a.D + c * 4);
            sum = f * sum + h * p[16 + r];
            top = most;
        }
    }
    tops[threadIdx.x] = top;
    sums[threadIdx.x] = sum;
    *reinterpret_cast<f32x4 *>(red[threadIdx.x]) = y;
    __syncthreads();
    if (k != 0) return;
    for (int i = 1; i < groups; i++) top = fmaxf(top, tops[i * lanes]);
    sum = 0.f;
    y = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < groups; i++) {
        const float f = __builtin_amdgcn_exp2f(tops[i * lanes] - top);
        sum += f * sums[i * lanes];
        y += f * *reinterpret_cast<const f32x4 *>(red[i * lanes + c]);
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum, poison = ok ? 0.f : __uint_as_float(0x7fc00000u);
    store_channels<DT>(a.o, b * a.o.sb + head * a.o.sh + t * a.o.st + c * 4, (t < count ? y * norm : f32x4{0.f, 0.f, 0.f, 0.f}) + poison);
}

// How a call is cut: both parts' plans, and where their workspaces lie (in floats).
struct SharedPlan {
    Plan first, second;
    bool shares;
    bool many;       // the first part has tiles of many rows
    bool fits;       // no launch has 2^32 threads
    int first_rows;  // of a place of its workspace
    int64_t second_at, floats;
};
// The codes are those of the table's columns.  Where these are many more than the sequences need a call is slower than a
// plain one; runs whose number of shared tokens is 0 leave nothing, which takes most of that back.  Tables of 32768 tokens,
// graph replays in us, plain, together, with zeros: 16 rows, 64 shared tokens and up to 40 others 7.8, 12.2 and 12.0; 512
// and 300 12.7, 13.4 and 15.5; 32 rows, 64 and 40 8.0, 22.6 and 13.2; 1024 and 300 25.3, 28.3 and 30.1; 256 rows, 512 and
// 500 17.1, 34.2 and 25.1; 256 channels, 256 and 100 11.6, 32.2 and 19.9.  (Parts of sequences that share nothing written at
// once as results: 1 us less of these, and 0.2 to 0.6 more in calls that share.)
// Whether a call is cut so at all: the codes that all sequences could have, read by each for itself, have to take longer
// than the further launches.  Both ways measured, graph replays in us, together and by themselves; bytes are of codes
// with head_dim rounded up to 64, 128 or 256, as the steps take their time by that (32 channels, 78 rows of 13
// sequences, 110 MB or 220 rounded up: 26 and 44; 192 channels, 138 MB rounded up: 39 and 26).
// One launch and the join, 16 rows: 7 MB 9.5 and 6.5, 13 MB 11.7 and 10.7, 17 MB 11.9 and 13.2, 38 MB 11.7 and 14.9, 139
// MB 13.7 and 24.1.
// Tiles of many rows, 32: 17 MB 25.5 and 13.1, 91 MB 31 and 28, 288 MB 41 and 55; 48: 69 MB 27 and 20, 221 MB 32 and 36;
// 64 of 64 channels: 46 MB 23.5 and 17.4, 145 MB 28 and 31; 256: 79 MB 26 and 12, 288 MB 29 and 30.
// Two sequences of up to 16 rows each have little to share: 270 MB 48 and 39 (three: 406 MB 47 and 67; two of 48 rows: 271
// MB 72 and 85).
// Sequences with too many rows for a tile of 16 to 64 have tiles of 256 by themselves, of which few rows are empty or
// many: 64 rows of 128 channels, 102 MB 57 and 61, 238 MB 78 and 110; 96: 98 and 112; 128: 122 and 114; 256: 212 and 160.
// Of 256 channels, 64 rows: 28 MB 57 and 54, 65 MB 69 and 77, 204 MB 96 and 137; 96: 125 and 139.
// Above 128 channels the first part has tiles of 256 rows too, and sequences of up to 16 rows have tiles of 16: 16 runs of 4
// 541 MB 107 and 64; 6 and more: 276 MB 54 and 34, 346 MB 60 and 65, 811 MB 109 and 169, 1352 MB 118 and 211.
constexpr int64_t kTilesFrom = 16 << 20, kRowsFrom = 160 << 20, kWideFrom = 320 << 20, kWideRowsFrom = 64 << 20;
bool pays(double bytes, bool many, int size, int64_t rows, int D) {  // rows: of a sequence, per cache head
    if (size == 1) return false;
    // (float32 rows above 128 channels are in tiles of 16 however many: fewer tiles, or nothing is gained)
    if (!many) return bytes >= kTilesFrom && (size * rows + 15) / 16 * 4 <= size * ((rows + 15) / 16) * 3;
    if (rows > 96) return false;
    if (D > 128) return rows > 16 ? bytes >= kWideRowsFrom : bytes >= kWideFrom && size >= 6;
    return bytes >= kRowsFrom && (size > 2 || rows > 16);
}
SharedPlan shared_plan(int B, int heads, int heads_kv, int T, int D, int page, int columns, int window, int dtype, int runs) {
    SharedPlan p;
    const int size = B / runs;
    const int64_t rows = (int64_t)T * size * (heads / heads_kv);
    p.second = plan_of(B, heads, heads_kv, T, D, page, columns, window, dtype, false);
    p.first = plan_of(runs, heads, heads_kv, T * size, D, page, columns, window, dtype);
    p.many = p.first.rows > 16;
    int64_t tokens = (int64_t)columns * page;
    if (window && window + (int64_t)T < tokens) tokens = window + (int64_t)T;
    p.shares = pays(2.0 * padded(D) * tokens * heads_kv * B, p.many, size, (int64_t)T * (heads / heads_kv), D);
    if (!p.shares) {
        p.second = plan_of(B, heads, heads_kv, T, D, page, columns, window, dtype);
        return p;
    }
    if (p.many) {
        p.first.rows = D > 128 ? kWideRows : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
        p.first.row_tiles = (int)((rows + p.first.rows - 1) / p.first.rows);
        p.first.parts = 256;  // ranges: one workgroup per CU
        p.first.items = 0;
        p.first_rows = rows < p.first.rows ? (int)(rows + 31) / 32 * 32 : p.first.rows;
        const int64_t tiles = (int64_t)runs * p.first.row_tiles * heads_kv;
        p.second_at = (2 * tiles + 3) / 4 * 4 + (tiles + p.first.parts) * item_floats(p.first_rows, padded(D));
    } else {
        const int64_t entries = (int64_t)runs * p.first.row_tiles;
        const int slots = 256 * (waves_of(padded(D), 1, dtype == ENATTEN_F32 ? 2 : 1) > 1 ? 2 : 1) / heads_kv;
        const int64_t useful = entries * (((int64_t)columns * page + 16 + kLeast - 1) / kLeast);
        p.first.parts = slots > entries && useful > entries ? (int)(slots < useful ? slots : useful) : 0;
        p.first.items = p.first.parts ? p.first.parts : entries;
        p.first_rows = 16;
        p.second_at = head_floats(entries) + p.first.items * heads_kv * item_floats(16, D);
    }
    const int64_t joins = p.many ? (int64_t)runs * p.first.row_tiles * heads_kv * (p.first_rows / 16) * (padded(D) / 32)
                                 : (int64_t)B * heads * T;
    p.fits = joins <= 0xffffff && (p.first.items + p.second.items) * heads_kv <= 0xffffff;
    p.floats = p.second_at + head_floats((int64_t)B * p.second.row_tiles) + p.second.items * heads_kv * item_floats(p.second.rows, D);
    return p;
}

template <int DP, int R, bool E4M3>
int launch_type(const char *fn, const SharedArgs &a, int64_t items, hipStream_t st) {
    const int blocks = (int)(items * a.heads_kv);
    ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "run_attend", st);
    if (a.dtype == ENATTEN_BF16) run_attend<DP, R, E4M3, ENATTEN_BF16><<<blocks, 256, 0, st>>>(a);
    else if (a.dtype == ENATTEN_F32) run_attend<DP, R, E4M3, ENATTEN_F32><<<blocks, 256, 0, st>>>(a);
    else run_attend<DP, R, E4M3, ENATTEN_F16><<<blocks, 256, 0, st>>>(a);
    return launched(fn);
}
template <int DP, bool E4M3>
int launch_tiles(const char *fn, const SharedArgs &a, int rows, int64_t items, hipStream_t st) {
    if (rows == 16) return launch_type<DP, 1, E4M3>(fn, a, items, st);
    if constexpr (DP <= 128) {
        if (rows == 32) return launch_type<DP, 2, E4M3>(fn, a, items, st);
        if (rows == 48) return launch_type<DP, 3, E4M3>(fn, a, items, st);
    }
    if constexpr (DP == 64)
        if (rows == 64) return launch_type<DP, 4, E4M3>(fn, a, items, st);
    set_error("%s: no tile of %d rows of %d channels", fn, rows, a.D);
    return ENATTEN_EUNSUPPORTED;
}
int launch_attend(const char *fn, const SharedArgs &a, int rows, int64_t items, bool e, hipStream_t st) {
    if (a.D <= 64) return e ? launch_tiles<64, true>(fn, a, rows, items, st) : launch_tiles<64, false>(fn, a, rows, items, st);
    if (a.D <= 128) return e ? launch_tiles<128, true>(fn, a, rows, items, st) : launch_tiles<128, false>(fn, a, rows, items, st);
    return e ? launch_tiles<256, true>(fn, a, rows, items, st) : launch_tiles<256, false>(fn, a, rows, items, st);
}

}  // namespace
}  // namespace enatten

using namespace enatten;

extern "C" {
#pragma GCC visibility push(default)

size_t enatten_cache_attention_shared_workspace_bytes(int B, int heads, int heads_kv, int T, int D, int page, int columns,
                                                      int kernel_size, int dtype, int runs) {
    if (B < 1 || heads < 1 || heads_kv < 1 || heads % heads_kv || T < 1 || D < 1 || page < 1 || columns < 1 ||
        kernel_size < 0 || runs < 1 || B % runs || (int64_t)B * heads * T > (1 << 30))
        return 0;
    const SharedPlan p = shared_plan(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype, runs);
    return !p.shares ? workspace_bytes(p.second, B, heads_kv, D) : p.fits ? p.floats * sizeof(float) : 0;
}

int enatten_cache_attention_shared(const void *q, const void *k_cache, const void *v_cache, const float *k_scale,
                                   const float *v_scale, const int *pages, const int *lengths, const int *counts,
                                   const int *shared, int runs, void *o, void *workspace, int B, int heads, int heads_kv,
                                   int T, int D, int num_pages, int page, int columns, int kernel_size, int dtype,
                                   int cache_dtype, const int64_t *q_strides, const int64_t *o_strides,
                                   const int64_t *k_cache_strides, const int64_t *v_cache_strides,
                                   const int64_t *k_scale_strides, const int64_t *v_scale_strides, int64_t pages_stride,
                                   float scale, void *stream) {
    const char *fn = "enatten_cache_attention_shared";
    SharedArgs a{};
    int rc = set_attention(fn, q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts, o, B, heads, heads_kv, T, D,
                           num_pages, page, columns, kernel_size, dtype, cache_dtype, q_strides, o_strides, k_cache_strides,
                           v_cache_strides, k_scale_strides, v_scale_strides, pages_stride, scale, &a);
    if (rc) return rc;
    if (!shared || runs < 1 || B % runs) {
        set_error("%s: shared must not be NULL, and its %d runs divide %d sequences", fn, runs, B);
        return ENATTEN_EINVAL;
    }
    const SharedPlan p = shared_plan(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype, runs);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool e = cache_dtype == ENATTEN_E4M3;
    if (!p.shares) return launch_plain(fn, a, p.second, workspace, e, st);
    if (!p.fits) {
        set_error("%s: too many rows for sequences that are read together", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    if (!workspace || (uintptr_t)workspace % 16) {
        set_error("%s: workspace is NULL or not 16-byte aligned", fn);
        return ENATTEN_EINVAL;
    }
    if (a.window >= (int64_t)columns * page) a.window = 0;  // (hides nothing: no row has to be asked where its begins)
    a.shared = shared;
    a.runs = runs;
    a.size = B / runs;
    a.first_ws = static_cast<float *>(workspace);
    a.ws = a.first_ws + p.second_at;
    a.first_tiles = p.first.row_tiles;
    a.first_parts = p.first.parts;
    a.first_rows = p.first_rows;
    a.row_tiles = p.second.row_tiles;
    a.parts = p.second.parts;
    if (p.many && (rc = launch_first_rows(fn, a, p.first.rows, e, st))) return rc;
    a.first_items = (int)p.first.items;
    if ((rc = launch_attend(fn, a, p.second.rows, a.first_items + p.second.items, e, st))) return rc;
    if (p.many) return launch_last_join(fn, a, p.first.rows, p.second.rows, st);
    ProfScope prof(ENATTEN_KERNEL_CACHE_JOIN, "run_join_tiles", st);
    const int blocks = B * heads * T;
    if (dtype == ENATTEN_BF16) run_join_tiles<ENATTEN_BF16><<<blocks, 256, 0, st>>>(a);
    else if (dtype == ENATTEN_F32) run_join_tiles<ENATTEN_F32><<<blocks, 256, 0, st>>>(a);
    else run_join_tiles<ENATTEN_F16><<<blocks, 256, 0, st>>>(a);
    return launched(fn);
}

#pragma GCC visibility pop
}  // extern "C"
