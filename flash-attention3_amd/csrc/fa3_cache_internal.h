// Host-side interface between the paged cache's C entries (fa3_cache_api.cpp)
// and its kernels.  Nothing here is exported.
#pragma once

#include "fa3_attn_internal.h"
#include "shaobo_fa3_cache.h"

namespace fa3 {

// What a page table holds and what a caller's lengths say, made safe: a page's
// number or -1, a length within 0 .. most.
__host__ __device__ inline int cache_page_of(int entry, int pages) {
    return (unsigned)entry < (unsigned)pages ? entry : -1;
}
__host__ __device__ inline int cache_length(int n, int most) { return n < 0 ? 0 : n < most ? n : most; }

// A cache as the kernels take it; strides in bytes.
struct CacheView {
    char *k, *v;
    int64_t k_ps, k_hs, k_rs, v_ps, v_hs, v_rs;
    const int* table;
    int64_t table_s;
    const int* kv_lens;
    const int* new_lens;  // null: all
    int pages, width, shift;  // a page has 1 << shift rows
};

// A resolved attention problem.
struct CacheProblem {
    int batch, heads_q, heads_kv, group, sq, d;
    int sk;  // places of a sequence's pages
    int page, count;  // count 0: every page
    bool bf16, four, causal, bias;
    float scale, softcap;
};

struct CacheAttnExtra {
    CacheView cv;
    const int* selected;  // [batch * heads_kv][sq][count], or null
    int count, per_query;
    FastDiv div_per_query;
    // slots > 0: the kernel for few rows deals parts of all sequences to as many
    // slots of each KV head; deal[b]: the first of sequence b's, and how many
    int slots, batch;
    int2* deal;
};
constexpr int kDealBatch = 256;  // sequences at most, four a lane
// The least part, in fours of blocks, for which count(blocks a part), the parts
// that `batch` sequences of `total` blocks make (an empty one too), are no more
// than the slots.  With P slots, B sequences and n blocks in all, parts of
// n / (P - B) blocks are at most n / (n / (P - B)) + B.
template <typename F>
__host__ __device__ inline uint32_t deal_part(uint32_t total, uint32_t slots, uint32_t batch, uint32_t least,
                                              F count) {
    const uint32_t spare = slots - batch;
    uint32_t lo = (total + 4 * slots - 1) / (4 * slots), hi = (total + 4 * spare - 1) / (4 * spare);
    lo = lo < least ? least : lo;
    hi = hi < lo ? lo : hi;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (count(4 * mid) <= slots) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
struct CacheAttnArgs : AttnFwdArgs {
    static constexpr bool kPaged = true;
    CacheAttnExtra x;
};

struct CachePlan {
    bool token;   // a kernel for few rows
    int row_tile; // rows of its jobs: 16 or 32
    int split;    // otherwise: workgroups of 128 / split rows
    int tiles;    // row tiles of a KV head (selected pages: of all its queries)
    int per_query;  // selected pages: row tiles of one query's heads
    int splits;   // parts of the key axis
    int slots;    // or, where it is cut by the sequences' lengths: slots of a KV head
    int jobs;
    size_t po_off, pl_off, deal_off, total;
    bool ok;
};
CachePlan plan_cache_attn(const CacheProblem& p);

// Workgroups of the kernel for few rows that a CU holds (waves a SIMD), by the
// registers of two blocks of keys and of the rows' outputs.
constexpr int few_waves(int D, bool four, int blocks) {
    return (D == 64 ? 5 : four ? 4 : 3) - blocks;
}

struct CacheSelectPlan {
    int chunks;  // parts of a sequence's pages, scored by a workgroup each
    size_t total;
    bool ok;
};
CacheSelectPlan plan_cache_select(const ShaoboFa3CacheSelectParams& p);

// How an append's workgroups share the tokens and heads.
struct AppendGrid {
    int units, lanes, tokens, run, segments, run_k, segments_k, hq, hk, hv, parts_q, parts_k, parts_v;
    bool ok;
};
AppendGrid append_grid(const ShaoboFa3CacheAppendParams& p);

CacheView cache_view(const ShaoboFa3Cache& c);

hipError_t launch_cache_append(const ShaoboFa3CacheAppendParams& p, hipStream_t stream);
hipError_t launch_cache_read(const ShaoboFa3CacheReadParams& p, hipStream_t stream);
hipError_t launch_cache_select(const ShaoboFa3CacheSelectParams& p, hipStream_t stream);
// The attention kernels, compiled one file per head dim and bits.
void launch_cache_d64_16(const CacheAttnArgs&, const CacheProblem&, const CachePlan&, hipStream_t);
void launch_cache_d128_16(const CacheAttnArgs&, const CacheProblem&, const CachePlan&, hipStream_t);
void launch_cache_d64_4(const CacheAttnArgs&, const CacheProblem&, const CachePlan&, hipStream_t);
void launch_cache_d128_4(const CacheAttnArgs&, const CacheProblem&, const CachePlan&, hipStream_t);
hipError_t launch_cache_attn(const CacheProblem& p, const ShaoboFa3CacheAttnParams& a, AttnMask m,
                             hipStream_t stream);

}  // namespace fa3
