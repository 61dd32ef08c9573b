// The kernels of cache_attention.hip in the two passes over runs of sequences that share their first tokens
// (cache_attention_shared.hip).
#pragma once

#include "cache_attention_body.h"

namespace enatten {
namespace {

template <int PASS, int DP, int R, bool E4M3, int DT>
__global__ __launch_bounds__(256, waves_of(DP, R, DT == ENATTEN_F32 ? 2 : 1)) void run_attend(PassArgs<PASS> a) {
    attend_body<DP, R, E4M3, DT>(a);
}
template <int PASS, int ROWS, int DT>
__global__ __launch_bounds__(256) void run_join(PassArgs<PASS> a) {
    join_body<ROWS, DT>(a);
}

template <int PASS, int DP, int R, bool E4M3, int DT>
int launch(const char *fn, const PassArgs<PASS> &a, const Plan &p, hipStream_t st) {
    const int64_t entries = (int64_t)(PASS == 1 ? a.runs : a.B) * p.row_tiles;
    const int64_t all = (int64_t)a.T * a.group * (PASS == 1 ? a.size : 1), blocks = entries * a.heads_kv * (all < 16 * R ? all : 16 * R);
    if (p.parts && blocks > 0x7fffffff) {
        set_error("%s: too many rows", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    {
        ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "run_attend", st);
        run_attend<PASS, DP, R, E4M3, DT><<<(int)(p.items * a.heads_kv), 256, 0, st>>>(a);
    }
    const int rc = launched(fn);
    if (rc || !p.parts) return rc;
    ProfScope prof(ENATTEN_KERNEL_CACHE_JOIN, "run_join", st);
    run_join<PASS, 16 * R, DT><<<(int)blocks, 256, 0, st>>>(a);
    return launched(fn);
}
template <int PASS, int DP, int R, bool E4M3>
int launch_type(const char *fn, const PassArgs<PASS> &a, const Plan &p, hipStream_t st) {
    if (a.dtype == ENATTEN_BF16) return launch<PASS, DP, R, E4M3, ENATTEN_BF16>(fn, a, p, st);
    if (a.dtype == ENATTEN_F32) return launch<PASS, DP, R, E4M3, ENATTEN_F32>(fn, a, p, st);
    return launch<PASS, DP, R, E4M3, ENATTEN_F16>(fn, a, p, st);
}
template <int PASS, int DP, bool E4M3>
int launch_rows(const char *fn, const PassArgs<PASS> &a, const Plan &p, hipStream_t st) {
    if (p.items * a.heads_kv > 0xffffff) {  // (2^32 threads)
        set_error("%s: too many row tiles", fn);
        return ENATTEN_EUNSUPPORTED;
    }
    if (p.rows == kWideRows) return PASS == 1 ? launch_rows_first(fn, a, E4M3, st) : launch_rows_second(fn, a, E4M3, st);
    if (p.rows == 16) return launch_type<PASS, DP, 1, E4M3>(fn, a, p, st);
    if constexpr (DP <= 128) {
        if (p.rows == 32) return launch_type<PASS, DP, 2, E4M3>(fn, a, p, st);
        if (p.rows == 48) return launch_type<PASS, DP, 3, E4M3>(fn, a, p, st);
    }
    if constexpr (DP == 64)
        if (p.rows == 64) return launch_type<PASS, DP, 4, E4M3>(fn, a, p, st);
    set_error("%s: no tile of %d rows of %d channels", fn, p.rows, a.D);
    return ENATTEN_EUNSUPPORTED;
}

template <int PASS>
int launch_pass(const char *fn, const SharedArgs &s, const Plan &p, bool e, hipStream_t st) {
    PassArgs<PASS> a;
    static_cast<SharedArgs &>(a) = s;
    if (a.D <= 64) return e ? launch_rows<PASS, 64, true>(fn, a, p, st) : launch_rows<PASS, 64, false>(fn, a, p, st);
    if (a.D <= 128) return e ? launch_rows<PASS, 128, true>(fn, a, p, st) : launch_rows<PASS, 128, false>(fn, a, p, st);
    return e ? launch_rows<PASS, 256, true>(fn, a, p, st) : launch_rows<PASS, 256, false>(fn, a, p, st);
}

}  // namespace
}  // namespace enatten
