// The tiles of 256 rows of cache_attention_rows.hip for runs that share their first tokens
// (cache_attention_shared.hip).
#include "cache_attention_rows_body.h"

namespace enatten {
namespace {

template <int PASS, int DP, bool E4M3, int DT>
__global__ __launch_bounds__(512, 2) void run_rows(PassArgs<PASS> args) {
    rows_body<DP, E4M3, DT>(args);
}
template <int PASS, int DP, int DT>
__global__ __launch_bounds__(256) void run_join_rows(PassArgs<PASS> a) {
    join_rows_body<DP, DT>(a);
}

template <int PASS, int DP, bool E4M3, int DT>
int launch(const char *fn, const PassArgs<PASS> &a, hipStream_t st) {
    {
        ProfScope prof(ENATTEN_KERNEL_CACHE_ATTENTION, "run_rows", st);
        run_rows<PASS, DP, E4M3, DT><<<a.parts, 512, 0, st>>>(a);
    }
    const int rc = launched(fn);
    if (rc) return rc;
    ProfScope prof(ENATTEN_KERNEL_CACHE_JOIN, "run_join_rows", st);
    run_join_rows<PASS, DP, DT><<<a.parts * (kWideRows / 16), 256, 0, st>>>(a);
    return launched(fn);
}
template <int PASS, int DP, bool E4M3>
int launch_type(const char *fn, const PassArgs<PASS> &a, hipStream_t st) {
    if (a.dtype == ENATTEN_BF16) return launch<PASS, DP, E4M3, ENATTEN_BF16>(fn, a, st);
    if constexpr (DP <= 128)
        if (a.dtype == ENATTEN_F32) return launch<PASS, DP, E4M3, ENATTEN_F32>(fn, a, st);
    return launch<PASS, DP, E4M3, ENATTEN_F16>(fn, a, st);
}
template <int PASS, bool E4M3>
int launch_dim(const char *fn, const PassArgs<PASS> &a, hipStream_t st) {
    if (a.D <= 64) return launch_type<PASS, 64, E4M3>(fn, a, st);
    if (a.D <= 128) return launch_type<PASS, 128, E4M3>(fn, a, st);
    return launch_type<PASS, 256, E4M3>(fn, a, st);
}

template <int PASS>
int launch_pass(const char *fn, const SharedArgs &s, bool e4m3, hipStream_t st) {
    PassArgs<PASS> a;
    static_cast<SharedArgs &>(a) = s;
    return e4m3 ? launch_dim<PASS, true>(fn, a, st) : launch_dim<PASS, false>(fn, a, st);
}

}  // namespace

int launch_rows_first(const char *fn, const SharedArgs &a, bool e4m3, hipStream_t st) { return launch_pass<1>(fn, a, e4m3, st); }
int launch_rows_second(const char *fn, const SharedArgs &a, bool e4m3, hipStream_t st) { return launch_pass<2>(fn, a, e4m3, st); }

}  // namespace enatten
