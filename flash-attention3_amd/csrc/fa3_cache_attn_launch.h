// Launches of the cache's attention kernels for one head dim and one width of
// rows (fa3_cache_attn_d*_*.hip).
#pragma once

#include "fa3_cache_few_kernel.h"

namespace fa3 {
namespace {

template <int D, bool kBf16, bool kFour>
void launch_cache(const CacheAttnArgs& x, const CacheProblem& p, const CachePlan& f,
                  hipStream_t stream) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(f.jobs), dim3(kRegThreads), 0, stream, x);
    };
    auto kinds = [&](auto cz, auto bi) {
        constexpr bool kC = decltype(cz)::value, kBi = decltype(bi)::value;
        if (f.token) {
            auto few = [&](auto dealt) {
                constexpr bool kDealt = decltype(dealt)::value;
                f.row_tile == 16 ? go(cache_few_kernel<D, kBf16, kC, kBi, kFour, 1, kDealt>)
                                 : go(cache_few_kernel<D, kBf16, kC, kBi, kFour, 2, kDealt>);
            };
            f.slots > 0 ? few(std::true_type{}) : few(std::false_type{});
        } else if (f.split == 2) {
            go(cache_tile_kernel<D, kBf16, kC, kBi, kFour, 2>);
        } else {
            go(cache_tile_kernel<D, kBf16, kC, kBi, kFour, 1>);
        }
    };
    using T = std::true_type;
    using F = std::false_type;
    if (p.softcap > 0.f) p.bias ? kinds(T{}, T{}) : kinds(T{}, F{});
    else p.bias ? kinds(F{}, T{}) : kinds(F{}, F{});
    if (f.slots > 0) {
        hipLaunchKernelGGL((cache_join_kernel<D, kBf16>), dim3(ceil_div((int64_t)x.groups * x.rows, 4)),
                           dim3(256), 0, stream, x);
        return;
    }
    if (f.splits <= 1) return;
    auto join = [&](auto ways) {
        constexpr int kW = decltype(ways)::value;
        hipLaunchKernelGGL((attn_join_kernel<D, kBf16, kW>),
                           dim3(ceil_div((int64_t)x.groups * x.rows, 2048 / (D * kW))), dim3(256), 0,
                           stream, x);
    };
    f.splits >= 8 ? join(std::integral_constant<int, 512 / D>{})
                  : join(std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace fa3
