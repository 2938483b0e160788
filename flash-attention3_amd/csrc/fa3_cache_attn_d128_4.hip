// Attention to a cache of head dim 65 to 128 held in 4 bits (fa3_cache_attn_kernel.h).
#include "fa3_cache_attn_launch.h"

namespace fa3 {
void launch_cache_d128_4(const CacheAttnArgs& x, const CacheProblem& p, const CachePlan& f,
                    hipStream_t stream) {
    p.bf16 ? launch_cache<128, true, true>(x, p, f, stream)
           : launch_cache<128, false, true>(x, p, f, stream);
}
}  // namespace fa3
