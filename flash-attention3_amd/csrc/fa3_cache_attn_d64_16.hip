// Attention to a cache of head dim up to 64 held in 16 bits (fa3_cache_attn_kernel.h).
#include "fa3_cache_attn_launch.h"

namespace fa3 {
void launch_cache_d64_16(const CacheAttnArgs& x, const CacheProblem& p, const CachePlan& f,
                    hipStream_t stream) {
    p.bf16 ? launch_cache<64, true, false>(x, p, f, stream)
           : launch_cache<64, false, false>(x, p, f, stream);
}
}  // namespace fa3
