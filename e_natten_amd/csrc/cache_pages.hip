// Pages of a cache that sequences share, leave and get: rows of the page table that continue other rows,
// pages for new tokens, copies of pages, and held pages moved to the low end of the pool.
//
// All but the copy work on whole numbers: the table [B, columns], the tokens of each row, and for each page
// the number of entries that name it.  They read and write these once, some hundred kilobytes in a large
// server, so launches and chains of loads bound them, not memory; what they write goes by their arguments
// alone (sums by atomics of whole numbers, ranks by scans).  The copy moves codes: HBM.
#include "sequence_common.h"

namespace enatten {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kMostRows = 8192;  // of the table: 64 KB of LDS hold two numbers of each

struct PageTable {
    int *pages;
    int64_t stride;
    int B, columns, num_pages, page;
    __device__ int &at(int b, int column) const { return pages[b * stride + column]; }
    __device__ bool is_page(int e) const { return (unsigned)e < (unsigned)num_pages; }
};

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
__device__ __forceinline__ int length_after(const ForkArgs &a, int b) {
    const int p = a.parents[b];
    return !moves(p, b, a.t.B) ? a.lengths[b] : p < 0 ? 0 : a.lengths[p];
}

// Some columns of all rows: read as they are into LDS, written anew from there.
__global__ __launch_bounds__(256) void fork_rows(ForkArgs a) {
    extern __shared__ int was[];  // [B][w], then the lengths
    const int c0 = blockIdx.x * a.width, w = min(a.width, a.t.columns - c0), all = a.t.B * w;
    for (int i = threadIdx.x; i < all; i += 256) {
        const int b = i / w;
        was[i] = a.t.at(b, c0 + i - b * w);
    }
    int *tokens = was + a.t.B * a.width;
    if (a.with_lengths)
        for (int b = threadIdx.x; b < a.t.B; b += 256) tokens[b] = length_after(a, b);
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += 256) {
        const int b = i / w, column = c0 + i - b * w, p = a.parents[b];
        if (!moves(p, b, a.t.B)) continue;
        int e = -1;
        if (p >= 0) {
            const int64_t used = ((int64_t)a.lengths[p] + a.t.page - 1) / a.t.page;
            if (column < used) e = was[p * w + column - c0];
        }
        const int old = was[i];
        if (e == old) continue;
        a.t.at(b, column) = e;
        if (a.t.is_page(old)) atomicAdd(a.holders + old, -1);
        if (a.t.is_page(e)) atomicAdd(a.holders + e, 1);
    }
    if (!a.with_lengths) return;
    __syncthreads();
    for (int b = threadIdx.x; b < a.t.B; b += 256) a.lengths[b] = tokens[b];
}
// The lengths by a launch of their own, where several workgroups read them.
__global__ __launch_bounds__(1024) void fork_lengths(ForkArgs a) {
    extern __shared__ int tokens[];
    for (int b = threadIdx.x; b < a.t.B; b += 1024) tokens[b] = length_after(a, b);
    __syncthreads();
    for (int b = threadIdx.x; b < a.t.B; b += 1024) a.lengths[b] = tokens[b];
}

// ---- pages for new tokens ----------------------------------------------------

struct ReserveArgs {
    PageTable t;
    const int *lengths, *counts;
    int *holders, *copies, *keeper, *list;  // workspace: [num_pages], [B * columns]
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
// Stores and atomics of this wave are done: other waves see them in memory behind the next barrier.
__device__ __forceinline__ void settle() { __builtin_amdgcn_s_waitcnt(0x0f70); }
__device__ __forceinline__ int load_now(const int *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// One workgroup.  Which rows leave a first page to others; the entries that want a page, in order; then the
// free pages in theirs, each to the entry of its rank.
__global__ __launch_bounds__(1024) void reserve_pages(ReserveArgs a) {
    extern __shared__ int lds[];
    __shared__ int part[16];
    int *offset = lds;                                                     // [B + 1]: columns of the rows before
    unsigned *common = reinterpret_cast<unsigned *>(lds + a.t.B + 1);      // a bit for each row: its first page
    const int words = (a.t.B + 31) / 32;                                   // holds older tokens, and others hold it
    unsigned *keeps = common + words;                                      // ... and it keeps it
    const int tid = threadIdx.x;
    auto bit = [](const unsigned *set, int b) { return (set[b / 32] >> (b % 32) & 1u) != 0; };
    for (int i = tid; i < 2 * words; i += 1024) common[i] = 0;
    __syncthreads();
    bool any = false;
    int upto = 0;
    for (int b0 = 0; b0 < a.t.B; b0 += 1024) {
        const int b = b0 + tid;
        Need n{0, 0, 0};
        if (b < a.t.B) {
            n = need_of(a, b);
            a.copies[3 * b] = a.copies[3 * b + 1] = -1;
            a.copies[3 * b + 2] = 0;
            if (n.columns && n.older) {
                const int e = a.t.at(b, n.first);
                if (a.t.is_page(e) && a.holders[e] > 1) {
                    any = true;
                    a.keeper[e] = -1;
                    atomicOr(common + b / 32, 1u << (b % 32));
                }
            }
        }
        int total;
        const int sum = block_sum<1024>(n.columns, part, total);
        if (b < a.t.B) offset[b] = upto + sum - n.columns;
        upto += total;
    }
    if (tid == 0) offset[a.t.B] = upto;
    // If all holders of a page write to it, the last of them keeps it.
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
            if (load_now(a.holders + e) == 0 && load_now(a.keeper + e) == b) atomicOr(keeps + b / 32, 1u << (b % 32));
        }
        __syncthreads();
        for (int b = tid; b < a.t.B; b += 1024)
            if (bit(keeps, b)) atomicAdd(a.holders + a.t.at(b, need_of(a, b).first), 1);
        settle();
        __syncthreads();
    }
    auto leaves = [&](int b) { return bit(common, b) && !bit(keeps, b); };

    int wanted = 0;
    for (int i0 = 0; i0 < upto; i0 += 1024) {
        const int i = i0 + tid;
        int entry = -1;
        if (i < upto) {
            int lo = 0, hi = a.t.B;  // offset[lo] <= i < offset[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (offset[mid] <= i) lo = mid;
                else hi = mid;
            }
            const Need n = need_of(a, lo);
            const int column = n.first + i - offset[lo];
            const bool begun = n.older && column == n.first;
            if (begun ? leaves(lo) : !a.t.is_page(a.t.at(lo, column))) entry = lo * a.t.columns + column;
        }
        int total;
        const int sum = block_sum<1024>(entry >= 0, part, total);
        if (entry >= 0) a.list[wanted + sum - 1] = entry;
        wanted += total;
    }
    settle();
    __syncthreads();  // (the list is read by other threads)
    if (wanted == 0) return;

    auto give = [&](int rank, int page) {
        const int entry = a.list[rank], b = entry / a.t.columns, column = entry - b * a.t.columns;
        int &at = a.t.at(b, column);
        if (page >= 0) {
            a.holders[page] = 1;
            const Need n = need_of(a, b);
            if (n.older && column == n.first) {
                a.copies[3 * b] = at;
                a.copies[3 * b + 1] = page;
                a.copies[3 * b + 2] = n.older;
            }
        }
        at = page;
    };
    constexpr int EACH = 16;  // pages of a thread
    const bool aligned = (uintptr_t)a.holders % 16 == 0;
    int given = 0;
    for (int64_t p0 = 0; p0 < a.t.num_pages && given < wanted; p0 += 1024 * EACH) {
        const int64_t p = p0 + tid * EACH;
        unsigned free = 0;
        if (aligned && p + EACH <= a.t.num_pages) {
#pragma unroll
            for (int j = 0; j < EACH; j += 4) {
                const i32x4 h = *reinterpret_cast<const i32x4 *>(a.holders + p + j);
#pragma unroll
                for (int k = 0; k < 4; k++) free |= h[k] == 0 ? 1u << (j + k) : 0u;
            }
        } else {
            for (int j = 0; j < EACH; j++)
                if (p + j < a.t.num_pages && a.holders[p + j] == 0) free |= 1u << j;
        }
        int total;
        int rank = given + block_sum<1024>(__popc(free), part, total) - __popc(free);
        while (free && rank < wanted) {
            const int j = __ffs(free) - 1;
            free &= free - 1;
            give(rank++, (int)p + j);
        }
        given += total;
    }
    for (int rank = given + tid; rank < wanted; rank += 1024) give(rank, -1);
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

// A unit is 16 codes of a token.  A workgroup takes pages `gridDim.x` apart, of each a share of its blocks
// (key or value, layer, head); 64 entries of the list are looked at together, as most may be empty.
__global__ __launch_bounds__(256) void copy_pages(CopyArgs a) {
    constexpr int DEEP = 4;  // units whose loads are under way at a time
    const int lane = threadIdx.x & 63, blocks = 2 * a.layers * a.heads;
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
            const unsigned units = __builtin_amdgcn_readlane(tokens, l) * wide;
            for (int k = threadIdx.x; k < mine; k += 256) {
                const int block = first + k, which = block & 1, head = block / 2 % a.heads, layer = block / 2 / a.heads;
                const PoolView &c = a.c[which];
                float *z = c.scales + layer * c.zl + head * c.zh;
                z[to * c.zp] = z[from * c.zp];
            }
            const int64_t all = (int64_t)mine * units;
            for (int64_t u0 = threadIdx.x; u0 < all; u0 += 256 * DEEP) {
                u32x4 x[DEEP];
                char *put[DEEP];
#pragma unroll
                for (int k = 0; k < DEEP; k++) {
                    const int64_t u = u0 + k * 256;
                    put[k] = nullptr;
                    if (u < all) {
                        const unsigned nth = (unsigned)u / units, unit = (unsigned)u - nth * units, row = unit / wide;
                        const int block = first + nth, which = block & 1, head = block / 2 % a.heads, layer = block / 2 / a.heads;
                        const PoolView &c = a.c[which];
                        char *at = c.codes + layer * c.sl + head * c.sh + row * c.st + (unit - row * wide) * 16;
                        put[k] = at + to * c.sp;
                        x[k] = *reinterpret_cast<const u32x4 *>(at + from * c.sp);
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
    const int64_t p = (int64_t)slab * kSlab + threadIdx.x * 8;
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (p + j < end && a.holders[p + j] != 0) held |= 1u << j;
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
    if (B > kMostRows || (int64_t)B * columns > 1 << 30 || (int64_t)columns * page > (1 << 30) - 4096) {
        set_error("%s: more than 8192 rows, 2^30 entries, or 2^30 tokens in a row's pages", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    *t = PageTable{pages, B > 1 ? stride : 0, B, columns, num_pages, page};
    return ENATTEN_OK;
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
    a.lengths = lengths;
    a.holders = holders;
    a.parents = parents;
    // About 8 entries per thread, whole lines of the table where 64 KB of LDS hold that many of all rows
    int width = 2048 / B > 16 ? 2048 / B : 16;
    if (width > 2 * kMostRows / B - 1) width = 2 * kMostRows / B - 1;
    if (width > columns) width = columns;
    a.width = width;
    a.with_lengths = width == columns;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t lds = ((size_t)B * width + (a.with_lengths ? B : 0)) * sizeof(int);
    {
        ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "fork_rows", st);
        fork_rows<<<(columns + width - 1) / width, 256, lds, st>>>(a);
    }
    const int rc = launched(fn);
    if (rc || a.with_lengths) return rc;
    ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "fork_lengths", st);
    fork_lengths<<<1, 1024, (size_t)B * sizeof(int), st>>>(a);
    return launched(fn);
}

size_t enatten_cache_reserve_workspace_bytes(int B, int columns, int num_pages) {
    if (B < 1 || columns < 1 || num_pages < 1) return 0;
    return ((size_t)num_pages + (size_t)B * columns) * sizeof(int);
}

int enatten_cache_reserve(int *pages, const int *lengths, const int *counts, int count, int *holders, int *copies,
                          void *workspace, int B, int columns, int num_pages, int page, int64_t pages_stride,
                          void *stream) {
    const char *fn = "enatten_cache_reserve";
    ReserveArgs a{};
    if (int rc = set_table(fn, pages, B, columns, num_pages, page, pages_stride, &a.t)) return rc;
    if (!lengths || !holders || !copies) return missing(fn);
    if (!workspace || (uintptr_t)workspace % 16) return bad_workspace(fn);
    a.lengths = lengths;
    a.counts = counts;
    a.count = count;
    a.holders = holders;
    a.copies = copies;
    a.keeper = static_cast<int *>(workspace);
    a.list = a.keeper + num_pages;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    ProfScope prof(ENATTEN_KERNEL_CACHE_PAGES, "reserve_pages", st);
    reserve_pages<<<1, 1024, (B + 1 + 2 * ((B + 31) / 32)) * sizeof(int), st>>>(a);
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
    // Shares of a page of 16 KB or so, up to some thousand workgroups in all
    const int64_t blocks = (int64_t)2 * layers * heads, bytes = blocks * page * D;
    const int x = n < 1024 ? n : 1024;
    int64_t split = (bytes + 16383) / 16384;
    if (split > blocks) split = blocks;
    if (split > 8192 / x) split = 8192 / x;
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
    a.counts = a.place + num_pages;
    const hipStream_t st = static_cast<hipStream_t>(stream);
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
