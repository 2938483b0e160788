// The attention backward's kernels for head dims up to 128 in bf16 (a file of
// their own, so that the build runs in parallel).
#include "fa3_attn_bwd_kernel.h"

namespace fa3 {
void launch_attn_bwd_d128_bf16(const AttnBwdArgs& a, const AttnBwdPlan& f, int cap, bool bias,
                              hipStream_t stream) {
    launch_bwd<128, true>(a, f, cap, bias, stream);
}
}  // namespace fa3
