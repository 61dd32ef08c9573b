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
#include "cache_attention_rows_body.h"

namespace enatten {
namespace {

template <int DP, bool E4M3, int DT>
__global__ __launch_bounds__(512, 2) void attend_rows(AttnArgs args) {
    rows_body<DP, E4M3, DT, 1, 1>(args);
}
template <int DP, int DT>
__global__ __launch_bounds__(256) void join_rows(AttnArgs a) {
    join_rows_body<DP, DT>(a);
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
