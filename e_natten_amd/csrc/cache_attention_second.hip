// The second pass of cache_attention over runs of sequences that share their first tokens: up to 64 rows.
#include "cache_attention_passes.h"

namespace enatten {

int launch_second(const char *fn, const SharedArgs &a, const Plan &p, bool e4m3, hipStream_t st) {
    return launch_pass<2>(fn, a, p, e4m3, st);
}

}  // namespace enatten
