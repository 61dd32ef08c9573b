// Pages of a cache that sequences share, leave and get: rows of the page table that continue other rows,
// pages for new tokens, copies of pages, and held pages moved to the low end of the pool.
//
// All but the copy work on whole numbers: the table [B, columns], the tokens of each row, and for each page
// the number of entries that name it.  They read and write these once, some hundred kilobytes in a large
// server, so launches and chains of loads bound them, not memory; what they write goes by their arguments
// alone (sums by atomics of whole numbers, ranks by scans).  The copy moves codes: HBM.
//
// Measured on MI355X, single launches under the profiler.  4 beams, pages of 16: fork 2.4 us, reserve 5.1, copy 3.8.
// 128 samples of 32 prompts, pages of 64, 4 layers of 8 heads of 128: 3.1, 7.1 and 13.8 (50 MB, 3.6 TB/s).  64 rows of
// 1025 columns, half of which get prompts of up to 8192 tokens, pages of 16: 6.1 (two launches), 18.2 and 3.8.
// compact: 216 pages 6.0 us; 1594 pages 6.7, and 24.3 for the copy that it asks for (100 MB, 4.1 TB/s); in a graph 15.0 for
// 16384 pages and entries, and in three launches 10.2 for 3000 pages in a table of 64 x 1025, 12.4 for 65536, 34.8 for 10^6.
#include "sequence_common.h"

namespace enatten {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kMostRows = 4096;  // of the table: 64 KB of LDS hold four numbers of each

// Loads that some lanes do not need are made by all, of a place that is there: behind a branch each of them is waited
// for before the next one.
struct PageTable {
    int *pages;
    int64_t stride;
    int B, columns, num_pages, page;
    __device__ int &at(int b, int column) const { return pages[b * stride + column]; }
    __device__ bool is_page(int e) const { return (unsigned)e < (unsigned)num_pages; }
};

// 16 neighbouring numbers from p on; what lies behind the last one is any of them
__device__ __forceinline__ void load16(const int *from, int64_t p, int64_t total, int (&h)[16]) {
    if ((uintptr_t)from % 16 == 0 && p + 16 <= total) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const i32x4 x = *reinterpret_cast<const i32x4 *>(from + p + j);
#pragma unroll
            for (int k = 0; k < 4; k++) h[j + k] = x[k];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) h[j] = from[min(p + j, total - 1)];
    }
}

// Sum of x over the workgroup's threads up to and including each, and over all.  part: one number for every wave.
template <int THREADS>
__device__ __forceinline__ int block_sum(int x, int *part, int &total) {
    constexpr int WAVES = THREADS / 64;
    const int upto = running_sum(x), wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 63) part[wave] = upto;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        const int n = part[i];
        before += i < wave ? n : 0;
        total += n;
    }
    __syncthreads();  // (part may be written again)
    return before + upto;
}

// ---- rows that continue others ----------------------------------------------

struct ForkArgs {
    PageTable t;
    int *lengths, *holders;
    const int *parents;
    int width;         // columns of a workgroup
    bool with_lengths;  // one workgroup for the whole table: the lengths too
};
__device__ __forceinline__ bool moves(int parent, int b, int B) { return parent >= -1 && parent < B && parent != b; }

// Some columns of all rows: read as they are into LDS, written anew from there.  Parents and the lengths that they
// have are read once, beside the entries: 128 rows of 10 columns took 6.5 us with loads in front of every entry.
__global__ __launch_bounds__(1024) void fork_rows(ForkArgs a) {
    extern __shared__ int was[];  // [B][w]; per row its parent (-2: stays), its new tokens and their columns
    const int threads = blockDim.x;
    const int c0 = blockIdx.x * a.width, w = min(a.width, a.t.columns - c0), all = a.t.B * w;
    int *parent = was + a.t.B * a.width, *tokens = parent + a.t.B, *used = tokens + a.t.B;
    constexpr int DEEP = 4;
    for (int i0 = threadIdx.x; i0 < all; i0 += threads * DEEP) {
        int e[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; k++) {
            const int i = min(i0 + k * threads, all - 1), b = i / w;
            e[k] = a.t.at(b, c0 + i - b * w);
        }
#pragma unroll
        for (int k = 0; k < DEEP; k++) was[min(i0 + k * threads, all - 1)] = e[k];
    }
    for (int b = threadIdx.x; b < a.t.B; b += threads) {
        const int p = a.parents[b];
        const bool moved = moves(p, b, a.t.B);
        const int len = moved && p >= 0 ? a.lengths[p] : 0;
        parent[b] = moved ? p : -2;
        tokens[b] = len;
        used[b] = (int)(((int64_t)len + a.t.page - 1) / a.t.page);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += threads) {
        const int b = i / w, c = i - b * w, p = parent[b];
        if (p == -2) continue;
        const int old = was[i], e = p >= 0 && c0 + c < used[b] ? was[p * w + c] : -1;
        if (e == old) continue;
        a.t.at(b, c0 + c) = e;
        if (a.t.is_page(old)) atomicAdd(a.holders + old, -1);
        if (a.t.is_page(e)) atomicAdd(a.holders + e, 1);
    }
    if (!a.with_lengths) return;
    for (int b = threadIdx.x; b < a.t.B; b += threads)
        if (parent[b] != -2) a.lengths[b] = tokens[b];
}
// The lengths by a launch of their own, where several workgroups read them.
__global__ __launch_bounds__(1024) void fork_lengths(ForkArgs a) {
    extern __shared__ int tokens[];
    for (int b = threadIdx.x; b < a.t.B; b += 1024) {
        const int p = a.parents[b];
        tokens[b] = !moves(p, b, a.t.B) ? a.lengths[b] : p < 0 ? 0 : a.lengths[p];
    }
    __syncthreads();
    for (int b = threadIdx.x; b < a.t.B; b += 1024) a.lengths[b] = tokens[b];
}

// ---- pages for new tokens ----------------------------------------------------

struct ReserveArgs {
    PageTable t;
    const int *lengths, *counts;
    int *holders, *copies, *keeper, *dropped;  // the last two: workspace [num_pages] each
    int count;
};
// The columns that a row's new tokens go to.
struct Need {
    int first, columns, older;  // older: tokens in the first one already
};
__device__ __forceinline__ Need need_of(const ReserveArgs &a, int b) {
    const int len = a.lengths[b], count = a.counts ? a.counts[b] : a.count;
    Need n{0, 0, 0};
    if (count > 0 && count <= len && len <= (int64_t)a.t.columns * a.t.page) {
        const int start = len - count;
        n.first = start / a.t.page;
        n.older = start - n.first * a.t.page;
        n.columns = (len + a.t.page - 1) / a.t.page - n.first;
    }
    return n;
}
__device__ __forceinline__ void put_copy(const ReserveArgs &a, int b, int from, int to, int tokens) {
    a.copies[3 * b] = from;
    a.copies[3 * b + 1] = to;
    a.copies[3 * b + 2] = tokens;
}
// Stores and atomics of this wave are done: other waves see them in memory behind the next barrier.
__device__ __forceinline__ void settle() { __builtin_amdgcn_s_waitcnt(0x0f70); }
__device__ __forceinline__ int load_now(const int *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The first `wanted` free pages in order: put(rank, page).  Returns how many there are of them.
template <class F>
__device__ __forceinline__ int free_pages(const ReserveArgs &a, int wanted, int *part, F put) {
    constexpr int EACH = 16;  // pages of a thread
    auto look = [&](int64_t p0) {
        const int64_t p = p0 + threadIdx.x * EACH;
        unsigned free = 0;
        if (p < a.t.num_pages) {
            int h[EACH];
            load16(a.holders, p, a.t.num_pages, h);
#pragma unroll
            for (int j = 0; j < EACH; j++) free |= p + j < a.t.num_pages && h[j] == 0 ? 1u << j : 0u;
        }
        return free;
    };
    int given = 0;
    unsigned next = look(0);
    for (int64_t p0 = 0; p0 < a.t.num_pages && given < wanted; p0 += 1024 * EACH) {
        unsigned free = next;
        next = look(p0 + 1024 * EACH);  // (under way beside the sum)
        int total;
        int rank = given + block_sum<1024>(__popc(free), part, total) - __popc(free);
        if (free && rank < wanted) {
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                if ((free >> j & 1) && rank < wanted) put(rank, (int)p0 + (int)threadIdx.x * EACH + j);
                rank += free >> j & 1;
            }
        }
        given += total;
    }
    return min(given, wanted);
}

// New tokens may meet a page that others hold where no older token is: a row's length went back behind tokens that it
// shares.  Such entries become none, so that they get a page of their own; `dropped` counts them page by page, and the
// holders lose them when all pages are given out, as a page that a copy still has to read is not free in this call.
// Seldom, so that passes over the table and all pages do not matter.
__device__ __forceinline__ void drop_entries(const ReserveArgs &a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t p = threadIdx.x; p < a.t.num_pages; p += 1024) a.dropped[p] = 0;
    __threadfence();
    __syncthreads();
    for (int b = wave; b < a.t.B; b += 16) {
        const Need n = need_of(a, b);
        for (int c = lane + (n.older != 0); c < n.columns; c += 64) {
            int &e = a.t.at(b, n.first + c);
            const int page = load_now(&e);
            if (!a.t.is_page(page) || load_now(a.holders + page) <= 1) continue;
            atomicAdd(a.dropped + page, 1);
            e = -1;
        }
    }
    __threadfence();
    __syncthreads();
}
__device__ __forceinline__ void take_dropped(const ReserveArgs &a) {
    __threadfence();
    __syncthreads();
    for (int64_t p = threadIdx.x; p < a.t.num_pages; p += 1024) {
        const int n = load_now(a.dropped + p);
        if (n) a.holders[p] = load_now(a.holders + p) - n;
    }
}

constexpr int kShortRows = 1024, kShortColumns = 4;

// Up to 1024 rows, a thread each.  A row whose first page e holds older tokens and is held by others too (held > 1)
// leaves it to them; if all its holders would, the last of them keeps it.  page_of: a number for every row.
__device__ __forceinline__ bool leaves_page(const ReserveArgs &a, int e, int held, int *page_of) {
    const int b = threadIdx.x;
    const bool common = held > 1;
    page_of[b] = common ? e : -1;
    if (!__syncthreads_or(common) || !common) return false;
    int writers = 0, last = 0;
#pragma unroll 16
    for (int i = 0; i < a.t.B; i++) {
        const bool same = page_of[i] == e;
        writers += same;
        last = same ? i : last;
    }
    if (last == b) a.holders[e] = held - writers + (writers == held);
    return !(writers == held && last == b);
}

// Up to 1024 rows that need four columns each at most, as single tokens do.  False if they are not.
__device__ __forceinline__ bool reserve_short(const ReserveArgs &a, int *part, int *page_of, int *fresh) {
    const int b = threadIdx.x;
    Need n{0, 0, 0};
    if (a.t.B > kShortRows) return false;
    int e[kShortColumns];
    if (b < a.t.B) n = need_of(a, b);
#pragma unroll
    for (int i = 0; i < kShortColumns; i++) e[i] = a.t.at(min(b, a.t.B - 1), n.first + min(i, max(n.columns - 1, 0)));
    if (__syncthreads_or(n.columns > kShortColumns)) return false;
    bool met = false;  // (a page that others hold, with no older tokens: looked at again when all have left theirs)
#pragma unroll
    for (int i = 0; i < kShortColumns; i++)
        if (i < n.columns && !(i == 0 && n.older) && a.t.is_page(e[i])) met |= a.holders[e[i]] > 1;
    const bool leaves = leaves_page(a, e[0], n.older && a.t.is_page(e[0]) ? a.holders[e[0]] : 0, page_of);
    unsigned wants;
    int wanted, rank;
    auto count = [&] {
        wants = leaves ? 1u : 0u;
#pragma unroll
        for (int i = 0; i < kShortColumns; i++)
            if (i < n.columns && !(i == 0 && n.older) && !a.t.is_page(e[i])) wants |= 1u << i;
        const int mine = __popc(wants) + (met ? 1 << 16 : 0);  // (4096 pages at most)
        rank = (block_sum<1024>(mine, part, wanted) & 0xffff) - __popc(wants);
    };
    count();
    const bool drops = wanted >> 16;
    if (drops) {
        drop_entries(a);
        if (b < a.t.B)
            for (int i = 0; i < n.columns; i++) e[i] = load_now(&a.t.at(b, n.first + i));
        met = false;
        count();
    }
    int given = 0;
    if (wanted) {
        given = free_pages(a, wanted, part, [&](int r, int page) { fresh[r] = page; });
        __syncthreads();
    }
    if (b < a.t.B) {
        int to = -1;
#pragma unroll
        for (int i = 0; i < kShortColumns; i++) {
            if (!(wants >> i & 1)) continue;
            const int page = rank < given ? fresh[rank] : -1;
            rank++;
            a.t.at(b, n.first + i) = page;
            if (page >= 0) a.holders[page] = 1;
            if (i == 0 && leaves) to = page;
        }
        put_copy(a, b, to >= 0 ? e[0] : -1, to, to >= 0 ? n.older : 0);
    }
    if (drops) take_dropped(a);
    return true;
}

// Columns c0 .. c0 + 64 N - 1 of a row that a wave goes over, from n.first on: those that want a page, a bit per lane
// for each 64; `old` is what the lane's entries are.
template <int N>
__device__ __forceinline__ void wants_of(const ReserveArgs &a, int b, const Need &n, bool leaves, int c0, int (&old)[N],
                                         unsigned long long (&who)[N]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int c = c0 + j * 64 + lane;
        old[j] = a.t.at(b, n.first + min(c, n.columns - 1));
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int c = c0 + j * 64 + lane;
        who[j] = __ballot(c < n.columns && (c == 0 && n.older ? leaves : !a.t.is_page(old[j])));
    }
}

// One workgroup.  But for short calls: which rows leave a first page to others; how many pages each row wants, by a
// thread where it has up to four columns, else by a wave; the free pages in their order; and each to the entry of
// its rank.  (With a thread for every entry the one CU was bound by instructions: 8000 entries took 14 us.)
__global__ __launch_bounds__(1024) void reserve_pages(ReserveArgs a) {
    extern __shared__ int lds[];
    __shared__ int part[16], page_of[kShortRows], fresh_short[kShortRows * kShortColumns], long_rows, met;
    if (reserve_short(a, part, page_of, fresh_short)) return;
    int *count = lds, *row_of = lds + a.t.B;  // [B] each: pages that a row wants, then of the rows before; the long rows
    unsigned *left = reinterpret_cast<unsigned *>(lds + 2 * a.t.B), *common = left + (a.t.B + 31) / 32;  // a bit for each row
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto bit = [](const unsigned *set, int b) { return (set[b / 32] >> (b % 32) & 1u) != 0; };
    auto mark = [](unsigned *set, int b) { atomicOr(set + b / 32, 1u << (b % 32)); };
    for (int i = tid; i < 2 * ((a.t.B + 31) / 32); i += 1024) left[i] = 0;
    __syncthreads();

    // first pages that hold older tokens and that others hold
    auto first_page = [&](int b, const Need &n) {
        const int e = n.older ? a.t.at(b, n.first) : -1;
        return a.t.is_page(e) && a.holders[e] > 1 ? e : -1;
    };
    if (a.t.B <= kShortRows) {
        const int e = tid < a.t.B ? first_page(tid, need_of(a, tid)) : -1;
        if (leaves_page(a, e, e >= 0 ? a.holders[e] : 0, page_of)) mark(left, tid);
    } else {
        bool any = false;
        for (int b = tid; b < a.t.B; b += 1024) {
            const int e = first_page(b, need_of(a, b));
            if (e < 0) continue;
            any = true;
            a.keeper[e] = -1;
            mark(common, b);
        }
        settle();
        if (__syncthreads_or(any)) {
            for (int b = tid; b < a.t.B; b += 1024) {
                if (!bit(common, b)) continue;
                const int e = a.t.at(b, need_of(a, b).first);
                atomicMax(a.keeper + e, b);
                atomicAdd(a.holders + e, -1);
            }
            settle();
            __syncthreads();
            for (int b = tid; b < a.t.B; b += 1024) {
                if (!bit(common, b)) continue;
                const int e = a.t.at(b, need_of(a, b).first);
                if (load_now(a.holders + e) != 0 || load_now(a.keeper + e) != b) mark(left, b);
            }
            __syncthreads();
            for (int b = tid; b < a.t.B; b += 1024)
                if (bit(common, b) && !bit(left, b)) atomicAdd(a.holders + a.t.at(b, need_of(a, b).first), 1);
            settle();
        }
    }
    __syncthreads();

    constexpr int N = 8;  // (4: 1.5 us more in a call of 32 rows with 256 columns each)
    auto count_all = [&] {
        if (tid == 0) long_rows = met = 0;
        __syncthreads();
        for (int b = tid; b < a.t.B; b += 1024) {
            const Need n = need_of(a, b);
            if (n.columns > kShortColumns) {
                row_of[atomicAdd(&long_rows, 1)] = b;
                continue;
            }
            const bool leaves = bit(left, b);
            int wants = 0;
            for (int c = 0; c < n.columns; c++) {
                const int old = a.t.at(b, n.first + c);
                if (c == 0 && n.older) wants += leaves;
                else if (!a.t.is_page(old)) wants++;
                else if (a.holders[old] > 1) met = 1;
            }
            count[b] = wants;
            put_copy(a, b, -1, -1, 0);
        }
        __syncthreads();
        for (int i = wave; i < long_rows; i += 16) {
            const int b = __builtin_amdgcn_readfirstlane(row_of[i]);
            const Need n = need_of(a, b);
            const bool leaves = bit(left, b);
            int wants = 0;
            for (int c0 = 0; c0 < n.columns; c0 += 64 * N) {
                int old[N];
                unsigned long long who[N];
                wants_of(a, b, n, leaves, c0, old, who);
#pragma unroll
                for (int j = 0; j < N; j++) wants += __popcll(who[j]);
            }
            if (wants < n.columns - (n.older && !leaves)) {  // (some pages are there)
                for (int c = lane + (n.older != 0); c < n.columns; c += 64) {
                    const int e = a.t.at(b, n.first + c);
                    if (a.t.is_page(e) && a.holders[e] > 1) met = 1;
                }
            }
            if (lane == 0) {
                count[b] = wants;
                put_copy(a, b, -1, -1, 0);
            }
        }
        settle();
        __syncthreads();
    };
    count_all();
    const bool drops = met;
    if (drops) {
        drop_entries(a);
        count_all();
    }
    int wanted = 0;
    for (int b0 = 0; b0 < a.t.B; b0 += 1024) {
        const int b = b0 + tid, mine = b < a.t.B ? count[b] : 0;
        int total;
        const int sum = block_sum<1024>(mine, part, total);
        if (b < a.t.B) count[b] = wanted + sum - mine;
        wanted += total;
    }
    // (with drops some pages are wanted)
    if (wanted == 0) return;
    // (the places of `keeper` are free again: pages in the order in which they are given out)
    int *fresh = a.keeper;
    const int given = free_pages(a, wanted, part, [&](int r, int page) { fresh[r] = page; });
    settle();
    __syncthreads();

    auto fresh_at = [&](int rank) {
        const int page = fresh[min(rank, max(given - 1, 0))];
        return rank < given ? page : -1;
    };
    auto give = [&](int b, const Need &n, int c, int old, int page) {
        a.t.at(b, n.first + c) = page;
        if (page < 0) return;
        a.holders[page] = 1;
        if (c == 0 && n.older) put_copy(a, b, old, page, n.older);
    };
    for (int b = tid; b < a.t.B; b += 1024) {
        const Need n = need_of(a, b);
        if (n.columns > kShortColumns) continue;
        const bool leaves = bit(left, b);
        int rank = count[b];
        for (int c = 0; c < n.columns; c++) {
            const int old = a.t.at(b, n.first + c);
            if (c == 0 && n.older ? leaves : !a.t.is_page(old)) give(b, n, c, old, fresh_at(rank++));
        }
    }
    for (int i = wave; i < long_rows; i += 16) {
        const int b = __builtin_amdgcn_readfirstlane(row_of[i]);
        const Need n = need_of(a, b);
        const bool leaves = bit(left, b);
        int rank = count[b];
        for (int c0 = 0; c0 < n.columns; c0 += 64 * N) {
            int old[N];
            unsigned long long who[N];
            wants_of(a, b, n, leaves, c0, old, who);
            int page[N];
#pragma unroll
            for (int j = 0; j < N; j++) {
                page[j] = fresh_at(rank + __popcll(who[j] & ((1ull << lane) - 1)));
                rank += __popcll(who[j]);
            }
#pragma unroll
            for (int j = 0; j < N; j++)
                if (who[j] >> lane & 1) give(b, n, c0 + j * 64 + lane, old[j], page[j]);
        }
    }
    if (drops) take_dropped(a);
}

// ---- copies of pages ----------------------------------------------------------

struct PoolView {
    char *codes;
    float *scales;
    int64_t sl, sp, sh, st;  // layer, page, head, token
    int64_t zl, zp, zh;
};
struct CopyArgs {
    PoolView c[2];
    const int *copies;
    int n, layers, heads, D, num_pages, page, split;
};

// A workgroup takes pages `gridDim.x` apart, of each a share of its blocks (key or value, layer, head); 64 lines
// of the list are looked at together, as most may be empty.  A wave goes over its part of these block by block in
// chunks of 64 units of 16 codes, four of them under way; where that is comes by counting, since divisions for every
// unit took as long as the copy.
__global__ __launch_bounds__(256) void copy_pages(CopyArgs a) {
    constexpr int DEEP = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), blocks = 2 * a.layers * a.heads;
    const int per = (blocks + a.split - 1) / a.split, first = blockIdx.y * per, mine = min(per, blocks - first);
    if (mine <= 0) return;
    const int wide = a.D / 16;
    for (int64_t i0 = blockIdx.x; i0 < a.n; i0 += (int64_t)64 * gridDim.x) {
        const int64_t i = i0 + (int64_t)lane * gridDim.x;
        int source = -1, target = -1, tokens = 0;
        if (i < a.n) {
            source = a.copies[3 * i];
            target = a.copies[3 * i + 1];
            tokens = min(a.copies[3 * i + 2], a.page);
        }
        const bool there = (unsigned)source < (unsigned)a.num_pages && (unsigned)target < (unsigned)a.num_pages &&
                           source != target && tokens > 0;
        for (unsigned long long who = __ballot(there); who; who &= who - 1) {
            const int l = __ffsll(who) - 1;
            const int64_t from = __builtin_amdgcn_readlane(source, l), to = __builtin_amdgcn_readlane(target, l);
            const int units = __builtin_amdgcn_readlane(tokens, l) * wide, chunks = (units + 63) / 64;
            for (int k = threadIdx.x; k < mine; k += 256) {
                const int block = first + k, which = block & 1, head = block / 2 % a.heads, layer = block / 2 / a.heads;
                const PoolView &c = a.c[which];
                float *z = c.scales + layer * c.zl + head * c.zh;
                z[to * c.zp] = z[from * c.zp];
            }
            const int all = mine * chunks, share = (all + 3) / 4;  // (at most 2^16 blocks of 2^8 chunks)
            int at = wave * share;
            const int end = min(at + share, all);
            int block = first + at / chunks, chunk = at % chunks, head = block / 2 % a.heads, layer = block / 2 / a.heads;
            while (at < end) {
                u32x4 x[DEEP];
                char *put[DEEP];
#pragma unroll
                for (int k = 0; k < DEEP; k++) {
                    put[k] = nullptr;
                    if (at < end) {
                        const PoolView &c = a.c[block & 1];
                        const int unit = chunk * 64 + lane;
                        if (unit < units) {
                            char *p = c.codes + layer * c.sl + head * c.sh;
                            if (c.st == a.D) {
                                p += unit * 16;
                            } else {
                                const int row = (unsigned)unit / (unsigned)wide;
                                p += row * c.st + (unit - row * wide) * 16;
                            }
                            put[k] = p + to * c.sp;
                            x[k] = *reinterpret_cast<const u32x4 *>(p + from * c.sp);
                        }
                        at++;
                        if (++chunk == chunks) {
                            chunk = 0;
                            if (++block % 2 == 0 && ++head == a.heads) {
                                head = 0;
                                layer++;
                            }
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < DEEP; k++)
                    if (put[k]) *reinterpret_cast<u32x4 *>(put[k]) = x[k];
            }
        }
    }
}

// ---- held pages to the low end ---------------------------------------------------

constexpr int kSlab = 2048;  // pages of a workgroup

struct CompactArgs {
    PageTable t;
    int *holders, *copies, *counts, *place;  // workspace: held pages of each slab; for each page its move, or -1
    int slabs, most;                          // most: rows of copies
};
// 8 neighbouring pages of slab `slab`: a bit for each one that is held and lies below `end`.
__device__ __forceinline__ unsigned held_of(const CompactArgs &a, int slab, int64_t end) {
    unsigned held = 0;
    int h[8];
    const int64_t p = (int64_t)slab * kSlab + threadIdx.x * 8;
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = a.holders[min(p + j, (int64_t)a.t.num_pages - 1)];
#pragma unroll
    for (int j = 0; j < 8; j++) held |= p + j < end && h[j] != 0 ? 1u << j : 0u;
    return held;
}
__global__ __launch_bounds__(256) void count_held(CompactArgs a) {
    __shared__ int part[4];
    int total;
    block_sum<256>(__popc(held_of(a, blockIdx.x, a.t.num_pages)), part, total);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = total;
}
// With n held pages, the k-th held one from n on goes to the k-th free one below n.
__global__ __launch_bounds__(256) void match_pages(CompactArgs a) {
    __shared__ int part[4];
    int n, before, below, sum = 0, mine = 0;
    for (int i = threadIdx.x; i < a.slabs; i += 256) {
        const int c = a.counts[i];
        sum += c;
        mine += i < (int)blockIdx.x ? c : 0;
    }
    block_sum<256>(sum, part, n);
    block_sum<256>(mine, part, before);
    // held pages below n
    const int edge = n / kSlab;
    sum = 0;
    for (int i = threadIdx.x; i < edge; i += 256) sum += a.counts[i];
    sum += __popc(held_of(a, edge, n));
    block_sum<256>(sum, part, below);
    const int moved = n - below;

    const unsigned held = held_of(a, blockIdx.x, a.t.num_pages);
    int total;
    int rank = before + block_sum<256>(__popc(held), part, total) - __popc(held);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int64_t p = (int64_t)blockIdx.x * kSlab + threadIdx.x * 8 + j;
        if (p >= a.t.num_pages) break;
        const bool is_held = held >> j & 1;
        int place = -1;
        if (is_held && p >= n) {
            place = rank - below;
            a.copies[3 * place] = (int)p;
            a.copies[3 * place + 2] = a.t.page;
        } else if (!is_held && p < n) {
            a.copies[3 * ((int)p - rank) + 1] = (int)p;
        }
        a.place[p] = place;
        rank += is_held;
    }
    for (int64_t r = moved + (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.most; r += (int64_t)gridDim.x * 256) {
        a.copies[3 * r] = a.copies[3 * r + 1] = -1;
        a.copies[3 * r + 2] = 0;
    }
}
__global__ __launch_bounds__(256) void move_pages(CompactArgs a) {
    const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x, threads = (int64_t)gridDim.x * 256;
    for (int64_t i = tid; i < (int64_t)a.t.B * a.t.columns; i += threads) {
        const int b = (int)(i / a.t.columns);
        int &e = a.t.at(b, (int)(i - (int64_t)b * a.t.columns));
        if (!a.t.is_page(e)) continue;
        const int place = a.place[e];
        if (place >= 0) e = a.copies[3 * place + 1];
    }
    for (int64_t r = tid; r < a.most; r += threads) {
        const int source = a.copies[3 * r], target = a.copies[3 * r + 1];
        if (source < 0) continue;
        a.holders[target] = a.holders[source];
        a.holders[source] = 0;
    }
}

// Pools of up to kSmallPool pages and tables of about as many entries: all of it in one workgroup.
constexpr int kSmallPool = 16384;
__global__ __launch_bounds__(1024) void compact_small(CompactArgs a) {
    constexpr int EACH = kSmallPool / 1024;
    __shared__ int part[16];
    __shared__ unsigned short target[kSmallPool / 2], place[kSmallPool];  // of the k-th move; where a page goes
    const int p0 = threadIdx.x * EACH, total_pages = a.t.num_pages;
    int h[EACH];
    unsigned held = 0;
    load16(a.holders, p0, total_pages, h);
#pragma unroll
    for (int j = 0; j < EACH; j++) held |= p0 + j < total_pages && h[j] != 0 ? 1u << j : 0u;
    int n, below;
    int rank = block_sum<1024>(__popc(held), part, n) - __popc(held);
    // held pages below n
    const unsigned low = p0 >= n ? 0u : n - p0 >= EACH ? (1u << EACH) - 1 : (1u << (n - p0)) - 1;
    block_sum<1024>(__popc(held & low), part, below);
    const int moved = n - below;
    int before = rank;
#pragma unroll
    for (int j = 0; j < EACH; j++) {
        const int p = p0 + j;
        if (p < n && !(held >> j & 1)) target[p - before] = (unsigned short)p;
        before += held >> j & 1;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EACH; j++) {
        const int p = p0 + j;
        if (p >= total_pages) continue;
        int to = p;
        if ((held >> j & 1) && p >= n) {
            const int k = rank - below;
            to = target[k];
            a.holders[to] = h[j];
            a.holders[p] = 0;
            a.copies[3 * k] = p;
            a.copies[3 * k + 1] = to;
            a.copies[3 * k + 2] = a.t.page;
        }
        place[p] = (unsigned short)to;
        rank += held >> j & 1;
    }
    __syncthreads();
    for (int r = moved + threadIdx.x; r < a.most; r += 1024) {
        a.copies[3 * r] = a.copies[3 * r + 1] = -1;
        a.copies[3 * r + 2] = 0;
    }
    const int all = a.t.B * a.t.columns;
    constexpr int DEEP = 4;
    for (int i0 = threadIdx.x; i0 < all; i0 += 1024 * DEEP) {
        int *at[DEEP], was[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; k++) {
            const int i = min(i0 + k * 1024, all - 1), b = i / a.t.columns;
            at[k] = &a.t.at(b, i - b * a.t.columns);
            was[k] = *at[k];
        }
#pragma unroll
        for (int k = 0; k < DEEP; k++) {
            if (i0 + k * 1024 >= all || !a.t.is_page(was[k])) continue;
            const int to = place[was[k]];
            if (to != was[k]) *at[k] = to;
        }
    }
}

int set_table(const char *fn, int *pages, int B, int columns, int num_pages, int page, int64_t stride, PageTable *t) {
    if (!pages) {
        set_error("%s: pages is NULL", fn);
        return ENATTEN_EINVAL;
    }
    if (B < 1 || columns < 1 || num_pages < 1) {
        set_error("%s: every dimension must be >= 1, got B=%d columns=%d num_pages=%d", fn, B, columns, num_pages);
        return ENATTEN_EINVAL;
    }
    if (page < 16 || page > 1024 || page % 16) {
        set_error("%s: pages must hold a multiple of 16 tokens up to 1024, got %d", fn, page);
        return ENATTEN_EINVAL;
    }
    if (B > 1 && stride < columns) {
        set_error("%s: the rows of pages must not overlap", fn);
        return ENATTEN_EINVAL;
    }
    // (of 2^30 pages up to 2^29 move, whose lines of three numbers still have places of 32 bits; that many pages of
    // 16 tokens of 16 channels are 512 GB of keys and values)
    if (B > kMostRows || (int64_t)B * columns > 1 << 30 || num_pages > 1 << 30 || (int64_t)columns * page > (1 << 30) - 4096) {
        set_error("%s: more than 4096 rows, 2^30 entries, 2^30 pages, or 2^30 tokens in a row's pages", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    *t = PageTable{pages, B > 1 ? stride : 0, B, columns, num_pages, page};
    return ENATTEN_OK;
}
// What a call writes shares no memory with its other arguments.
struct Ints {
    const int *at;
    int64_t n;
};
bool meet(const Ints &x, const Ints &y) {
    const int64_t d = (const char *)y.at - (const char *)x.at;
    return x.at && y.at && d < x.n * (int64_t)sizeof(int) && -d < y.n * (int64_t)sizeof(int);
}
bool meet(const PageTable &t, const Ints &x) {  // (x may lie between the rows of a wider table)
    const int64_t unit = sizeof(int), row = t.columns * unit, stride = t.stride * unit, size = x.n * unit;
    const int64_t d = (const char *)x.at - (const char *)t.pages;
    if (!x.at || d >= (t.B - 1) * stride + row || -d >= size) return false;
    if (d <= 0) return true;
    const int64_t in_row = stride ? d % stride : d;
    return in_row < row || in_row + size > stride;
}
int apart(const char *fn, const PageTable &t, std::initializer_list<Ints> written, std::initializer_list<Ints> read) {
    bool met = false;
    for (const Ints &x : written) {
        met |= meet(t, x);
        for (const Ints &y : written) met |= &x < &y && meet(x, y);
        for (const Ints &y : read) met |= meet(x, y);
    }
    for (const Ints &y : read) met |= meet(t, y);
    if (!met) return ENATTEN_OK;
    set_error("%s: what is written must not share memory with other arguments", fn);
    return ENATTEN_EINVAL;
}
int missing(const char *fn) {
    set_error("%s: an argument is NULL", fn);
    return ENATTEN_EINVAL;
}
int bad_workspace(const char *fn) {
    set_error("%s: workspace is NULL or not 16-byte aligned", fn);
    return ENATTEN_EINVAL;
}

}  // namespace
}  // namespace enatten

using namespace enatten;

extern "C" {
#pragma GCC visibility push(default)

int enatten_cache_fork(int *pages, int *lengths, int *holders, const int *parents, int B, int columns, int num_pages,
                       int page, int64_t pages_stride, void *stream) {
    const char *fn = "enatten_cache_fork";
    ForkArgs a{};
    if (int rc = set_table(fn, pages, B, columns, num_pages, page, pages_stride, &a.t)) return rc;
    if (!lengths || !holders || !parents) return missing(fn);
    if (int rc = apart(fn, a.t, {{lengths, B}, {holders, num_pages}}, {{parents, B}})) return rc;
    a.lengths = lengths;
    a.holders = holders;
    a.parents = parents;
    // About 4 entries per thread, whole lines of the table where 64 KB of LDS hold that many of all rows
    int width = 4096 / B > 16 ? 4096 / B : 16;
    if (width > 4 * kMostRows / B - 3) width = 4 * kMostRows / B - 3;
    if (width > columns) width = columns;
    a.width = width;
    a.with_lengths = width == columns;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t lds = (size_t)B * (width + 3) * sizeof(int);
    {
        ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "fork_rows", st);
        fork_rows<<<(columns + width - 1) / width, (int64_t)B * width <= 512 ? 256 : 1024, lds, st>>>(a);
    }
    const int rc = launched(fn);
    if (rc || a.with_lengths) return rc;
    ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "fork_lengths", st);
    fork_lengths<<<1, 1024, (size_t)B * sizeof(int), st>>>(a);
    return launched(fn);
}

size_t enatten_cache_reserve_workspace_bytes(int B, int columns, int num_pages) {
    if (B < 1 || columns < 1 || num_pages < 1) return 0;
    return (size_t)2 * num_pages * sizeof(int);
}

int enatten_cache_reserve(int *pages, const int *lengths, const int *counts, int count, int *holders, int *copies,
                          void *workspace, int B, int columns, int num_pages, int page, int64_t pages_stride,
                          void *stream) {
    const char *fn = "enatten_cache_reserve";
    ReserveArgs a{};
    if (int rc = set_table(fn, pages, B, columns, num_pages, page, pages_stride, &a.t)) return rc;
    if (!lengths || !holders || !copies) return missing(fn);
    if (!workspace || (uintptr_t)workspace % 16) return bad_workspace(fn);
    if (int rc = apart(fn, a.t, {{holders, num_pages}, {copies, (int64_t)3 * B}, {static_cast<int *>(workspace), (int64_t)2 * num_pages}},
                       {{lengths, B}, {counts, counts ? B : 0}})) return rc;
    a.lengths = lengths;
    a.counts = counts;
    a.count = count;
    a.holders = holders;
    a.copies = copies;
    a.keeper = static_cast<int *>(workspace);
    a.dropped = a.keeper + num_pages;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "reserve_pages", st);
    reserve_pages<<<1, 1024, (2 * B + 2 * ((B + 31) / 32)) * sizeof(int), st>>>(a);
    return launched(fn);
}

int enatten_cache_copy(void *k_cache, void *v_cache, float *k_scale, float *v_scale, const int *copies, int n, int layers,
                       int heads, int D, int num_pages, int page, const int64_t *k_cache_strides,
                       const int64_t *v_cache_strides, const int64_t *k_scale_strides, const int64_t *v_scale_strides,
                       void *stream) {
    const char *fn = "enatten_cache_copy";
    if (n < 0 || layers < 1 || heads < 1 || num_pages < 1) {
        set_error("%s: every dimension must be >= 1, got layers=%d heads=%d num_pages=%d n=%d", fn, layers, heads, num_pages, n);
        return ENATTEN_EINVAL;
    }
    if (D < 16 || D > 256 || D % 16) {
        set_error("%s: head_dim must be a multiple of 16 up to 256, got %d", fn, D);
        return ENATTEN_EINVAL;
    }
    if (page < 16 || page > 1024 || page % 16) {
        set_error("%s: pages must hold a multiple of 16 tokens up to 1024, got %d", fn, page);
        return ENATTEN_EINVAL;
    }
    if ((int64_t)2 * layers * heads > 1 << 16) {  // (units of a page stay within 31 bits)
        set_error("%s: more than 2^15 heads of all layers", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    CopyArgs a{};
    void *const codes[2] = {k_cache, v_cache};
    float *const scales[2] = {k_scale, v_scale};
    const int64_t *const strides[2] = {k_cache_strides, v_cache_strides}, *const zstrides[2] = {k_scale_strides, v_scale_strides};
    for (int i = 0; i < 2; i++) {
        const int64_t *s = strides[i], *z = zstrides[i];
        if (!codes[i] || !scales[i]) return missing(fn);
        PoolView &c = a.c[i];
        c.codes = static_cast<char *>(codes[i]);
        c.scales = scales[i];
        c.st = s ? s[3] : D;
        c.sh = s ? s[2] : (int64_t)page * D;
        c.sp = s ? s[1] : (int64_t)heads * page * D;
        c.sl = s ? s[0] : (int64_t)num_pages * heads * page * D;
        c.zh = z ? z[2] : 1;
        c.zp = z ? z[1] : heads;
        c.zl = z ? z[0] : (int64_t)num_pages * heads;
        if (c.st < D || c.st > 1 << 20 || c.sh < 0 || c.sp < 0 || c.sl < 0 || c.zh < 0 || c.zp < 0 || c.zl < 0) {
            set_error("%s: strides must not be negative, and D to 2^20 between tokens", fn);
            return ENATTEN_EINVAL;
        }
        if ((c.st | c.sh | c.sp | c.sl | (int64_t)(uintptr_t)c.codes) % 16) {
            set_error("%s: the address and the strides of the cache must be multiples of 16", fn);
            return ENATTEN_EINVAL;
        }
    }
    if (n == 0) return ENATTEN_OK;
    if (!copies) return missing(fn);
    a.copies = copies;
    a.n = n; a.layers = layers; a.heads = heads; a.D = D; a.num_pages = num_pages; a.page = page;
    // About two thousand workgroups, which all start at once, of one share of a page's blocks each
    const int64_t blocks = (int64_t)2 * layers * heads;
    const int x = n < 1024 ? n : 1024;
    int64_t split = (2048 + x - 1) / x;
    if (split > blocks) split = blocks;
    a.split = (int)split;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    ProfScope prof(ENATTEN_KERNEL_CACHE_COPY, "copy_pages", st);
    copy_pages<<<dim3(x, a.split), 256, 0, st>>>(a);
    return launched(fn);
}

size_t enatten_cache_compact_workspace_bytes(int num_pages) {
    if (num_pages < 1) return 0;
    return ((size_t)(num_pages + (int64_t)kSlab - 1) / kSlab + num_pages) * sizeof(int);
}

int enatten_cache_compact(int *pages, int *holders, int *copies, void *workspace, int B, int columns, int num_pages,
                          int page, int64_t pages_stride, void *stream) {
    const char *fn = "enatten_cache_compact";
    CompactArgs a{};
    if (int rc = set_table(fn, pages, B, columns, num_pages, page, pages_stride, &a.t)) return rc;
    if (!holders || !copies) return missing(fn);
    if (!workspace || (uintptr_t)workspace % 16) return bad_workspace(fn);
    a.holders = holders;
    a.copies = copies;
    a.slabs = (int)(((int64_t)num_pages + kSlab - 1) / kSlab);
    a.most = num_pages > 1 ? num_pages / 2 : 1;
    a.place = static_cast<int *>(workspace);
    if (int rc = apart(fn, a.t, {{holders, num_pages}, {copies, (int64_t)3 * a.most}, {a.place, (int64_t)num_pages + a.slabs}}, {}))
        return rc;
    a.counts = a.place + num_pages;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (num_pages <= kSmallPool && (int64_t)B * columns <= kSmallPool) {
        ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "compact_small", st);
        compact_small<<<1, 1024, 0, st>>>(a);
        return launched(fn);
    }
    ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "compact_pages", st);
    count_held<<<a.slabs, 256, 0, st>>>(a);
    if (int rc = launched(fn)) return rc;
    match_pages<<<a.slabs, 256, 0, st>>>(a);
    if (int rc = launched(fn)) return rc;
    const int64_t work = (int64_t)B * columns > a.most ? (int64_t)B * columns : a.most;
    const int64_t groups = (work + 255) / 256;
    move_pages<<<(int)(groups < 1024 ? groups : 1024), 256, 0, st>>>(a);
    return launched(fn);
}

#pragma GCC visibility pop
}  // extern "C"
