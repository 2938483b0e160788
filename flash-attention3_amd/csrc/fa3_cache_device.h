// What the paged cache's kernels share: sequences, their pages, and the levels
// of 4-bit rows.
#pragma once

#include "fa3_attn_device.h"
#include "fa3_cache_internal.h"

namespace fa3 {
namespace {

// Tokens of sequence b with the call's, and how many rows of the call are tokens.
template <typename C>
__device__ __forceinline__ int cache_kv(const C& c, int b) {
    return cache_length(scalar_load(c.kv_lens + b), c.width << c.shift);
}
template <typename C>
__device__ __forceinline__ int cache_new(const C& c, int b, int seqlen) {
    return c.new_lens == nullptr ? seqlen : cache_length(scalar_load(c.new_lens + b), seqlen);
}
// The page of positions [n << shift, (n + 1) << shift), 0 <= n < width; -1 for none.
template <typename C>
__device__ __forceinline__ int cache_page(const C& c, int b, int n) {
    return cache_page_of(c.table[b * c.table_s + n], c.pages);
}
// The same where b and n are one for all lanes.
template <typename C>
__device__ __forceinline__ int cache_page_scalar(const C& c, int b, int n) {
    return cache_page_of(scalar_load(c.table + b * c.table_s + n), c.pages);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Two levels, byte kSel of w: its low half's in the low 16 bits.  (The
// conversion's own scale, a power of two, is 1: levels are exact.)
template <bool kBf16, int kSel>
__device__ __forceinline__ uint32_t cache_levels(uint32_t w) {
    if constexpr (kBf16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, kSel));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, kSel));
}
template <bool kBf16>
__device__ __forceinline__ f16x8 cache_levels8(uint32_t w) {
    const u32x4 x = {cache_levels<kBf16, 0>(w), cache_levels<kBf16, 1>(w),
                     cache_levels<kBf16, 2>(w), cache_levels<kBf16, 3>(w)};
    return __builtin_bit_cast(f16x8, x);
}

}  // namespace
}  // namespace fa3
