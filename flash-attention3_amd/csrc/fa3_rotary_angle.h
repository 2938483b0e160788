// The angles of rotary positions.
#pragma once

#include <hip/hip_runtime.h>

#include "shaobo_fa3_attn.h"

namespace fa3 {
namespace {

__device__ __forceinline__ double position(const void* p, int type, int64_t i) {
    if (type == SHAOBO_FA3_POSITIONS_INT32) return (double)((const int32_t*)p)[i];
    if (type == SHAOBO_FA3_POSITIONS_INT64) return (double)((const int64_t*)p)[i];
    return (double)((const float*)p)[i];
}

// x f / (2 pi) less a whole number of turns, for |x f| up to 2^53 within 2^-50
// of a turn.  g + gl is f / (2 pi), gl what g's rounding left off (an fma gives
// a product's exactly) with the constant's second half; t + tl likewise is its
// product with x.  Whole turns come off t exactly.
__device__ __forceinline__ double axis_turns(double x, double f) {
#pragma clang fp contract(off)
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLow = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
    const double g = f * kTurn, gl = __builtin_fma(f, kTurn, -g) + f * kTurnLow;
    const double t = x * g, tl = __builtin_fma(x, g, -t) + x * gl;
    return (t - rint(t)) + (tl - rint(tl));
}

}  // namespace
}  // namespace fa3
