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
#include "cache_attention_body.h"

namespace enatten {
namespace {

template <int DP, int R, bool E4M3, int DT>
__global__ __launch_bounds__(256, waves_of(DP, R, DT == ENATTEN_F32 ? 2 : 1)) void attend(AttnArgs a) {
    attend_body<DP, R, E4M3, DT>(a);
}
template <int ROWS, int DT>
__global__ __launch_bounds__(256) void attend_join(AttnArgs a) {
    join_body<ROWS, DT>(a);
}

}  // namespace

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
Plan plan_of(int B, int heads, int heads_kv, int T, int D, int page, int columns, int window, int dtype, bool wide) {
    Plan p;
    const int64_t all = (int64_t)T * (heads / heads_kv);
    const int most = D > 128 ? 16 : D > 64 ? 48 : 64;
    p.rows = all <= most ? (int)(all + 15) / 16 * 16 : !wide || (D > 128 && dtype == ENATTEN_F32) ? most : kWideRows;
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

int set_attention(const char *fn, const void *q, const void *k_cache, const void *v_cache, const float *k_scale,
                  const float *v_scale, const int *pages, const int *lengths, const int *counts, void *o, int B, int heads,
                  int heads_kv, int T, int D, int num_pages, int page, int columns, int kernel_size, int dtype,
                  int cache_dtype, const int64_t *q_strides, const int64_t *o_strides, const int64_t *k_cache_strides,
                  const int64_t *v_cache_strides, const int64_t *k_scale_strides, const int64_t *v_scale_strides,
                  int64_t pages_stride, float scale, AttnArgs *a) {
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
    if ((rc = set_rows(fn, "q", q, q_strides, heads, T, D, &a->q))) return rc;
    if ((rc = set_rows(fn, "o", o, o_strides, heads, T, D, &a->o))) return rc;
    const int pack = dtype == ENATTEN_F32 ? 4 : 8;
    if (((uintptr_t)q | (uintptr_t)o) % 16 || (a->q.sb | a->q.sh | a->q.st | a->o.sb | a->o.sh | a->o.st) % pack) {
        set_error("%s: rows of q and o must lie at multiples of 16 bytes", fn);
        return ENATTEN_EINVAL;
    }
    if ((rc = set_cache(fn, "k", const_cast<void *>(k_cache), const_cast<float *>(k_scale), k_cache_strides,
                        k_scale_strides, heads_kv, page, D, 16, &a->k))) return rc;
    if ((rc = set_cache(fn, "v", const_cast<void *>(v_cache), const_cast<float *>(v_scale), v_cache_strides,
                        v_scale_strides, heads_kv, page, D, 16, &a->v))) return rc;
    if (!pages || !lengths) {
        set_error("%s: pages and lengths must not be NULL", fn);
        return ENATTEN_EINVAL;
    }
    a->tb = Table{pages, lengths, counts, pages_stride, num_pages, page, columns, T};
    a->B = B; a->heads = heads; a->group = heads / heads_kv; a->heads_kv = heads_kv; a->T = T; a->D = D;
    a->window = kernel_size;
    a->dtype = dtype;
    a->scale = scale;
    return ENATTEN_OK;
}
size_t workspace_bytes(const Plan &p, int B, int heads_kv, int D) {
    if (!p.parts) return 0;
    if (p.rows == kWideRows) return ((size_t)(p.parts + 3) / 4 * 4 + 2 * p.parts * item_floats(kWideRows, padded(D))) * sizeof(float);
    return (size_t)(head_floats((int64_t)B * p.row_tiles) + p.items * heads_kv * item_floats(p.rows, D)) * sizeof(float);
}

namespace {

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

int launch_plain(const char *fn, AttnArgs a, const Plan &p, void *workspace, bool e, hipStream_t st) {
    if (p.parts && (!workspace || (uintptr_t)workspace % 16)) {
        set_error("%s: workspace is NULL or not 16-byte aligned", fn);
        return ENATTEN_EINVAL;
    }
    a.row_tiles = p.row_tiles;
    a.parts = p.parts;
    a.ws = static_cast<float *>(workspace);
    if (a.D <= 64) return e ? launch_rows<64, true>(fn, a, p, st) : launch_rows<64, false>(fn, a, p, st);
    if (a.D <= 128) return e ? launch_rows<128, true>(fn, a, p, st) : launch_rows<128, false>(fn, a, p, st);
    return e ? launch_rows<256, true>(fn, a, p, st) : launch_rows<256, false>(fn, a, p, st);
}

}  // namespace enatten

using namespace enatten;

extern "C" {
#pragma GCC visibility push(default)

size_t enatten_cache_attention_workspace_bytes(int B, int heads, int heads_kv, int T, int D, int page, int columns,
                                               int kernel_size, int dtype) {
    if (B < 1 || heads < 1 || heads_kv < 1 || heads % heads_kv || T < 1 || D < 1 || page < 1 || columns < 1 ||
        kernel_size < 0)
        return 0;
    return workspace_bytes(plan_of(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype), B, heads_kv, D);
}

int enatten_cache_attention(const void *q, const void *k_cache, const void *v_cache, const float *k_scale,
                            const float *v_scale, const int *pages, const int *lengths, const int *counts, void *o,
                            void *workspace, int B, int heads, int heads_kv, int T, int D, int num_pages, int page,
                            int columns, int kernel_size, int dtype, int cache_dtype, const int64_t *q_strides,
                            const int64_t *o_strides, const int64_t *k_cache_strides, const int64_t *v_cache_strides,
                            const int64_t *k_scale_strides, const int64_t *v_scale_strides, int64_t pages_stride,
                            float scale, void *stream) {
    const char *fn = "enatten_cache_attention";
    AttnArgs a{};
    const int rc = set_attention(fn, q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts, o, B, heads, heads_kv, T,
                                 D, num_pages, page, columns, kernel_size, dtype, cache_dtype, q_strides, o_strides,
                                 k_cache_strides, v_cache_strides, k_scale_strides, v_scale_strides, pages_stride, scale, &a);
    if (rc) return rc;
    return launch_plain(fn, a, plan_of(B, heads, heads_kv, T, D, page, columns, kernel_size, dtype), workspace,
                        cache_dtype == ENATTEN_E4M3, static_cast<hipStream_t>(stream));
}

#pragma GCC visibility pop
}  // extern "C"
