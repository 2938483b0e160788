// Attention to a paged cache: the kernels of fa3_attn_fwd.hip with a page
// looked up for every 32 or 64 keys.
//
// cache_tile_kernel walks 16-bit pages as attn_fwd_kernel does dense tensors.
// From 4-bit pages it makes its LDS tiles itself: a thread loads the codes of
// the next tile before this one's products and writes their levels, 16 bits
// each, behind them.  (Vector and matrix instructions bound it: 1531 tokens
// over 9211 of 4 bits, 32 heads to 8, D 128, 298 us, 711 TFLOP/s, 57 % and 30 %
// of the SIMDs' cycles; a part of the vector ones is the rows' own softmax, the
// rest levels and scales.  fp16, whose P goes as two terms: 397 us.)
#pragma once

#include "fa3_attn_fwd_kernel.h"
#include "fa3_cache_device.h"

namespace fa3 {

namespace {

// Whether row `row` of KV head hkv sees any key: lane g4 of its four looks at
// every fourth page, last first.
template <typename A>
__device__ __forceinline__ bool cache_sees(const A& z, int row, int b, int hkv, int g4) {
    const int kv = cache_kv(z.x.cv, b), n = cache_new(z.x.cv, b, z.sq);
    const AttnRow r = attn_row(row, n * z.group, hkv, z.group, z.div_group);
    const int lim = r.ok ? attn_limit(r.i, kv - n, kv, z.m.causal, attn_prefix(z.m, b)) : 0;
    bool any = false;
    if (z.x.selected != nullptr) {
        const int* list = z.x.selected + ((int64_t)(b * z.heads_kv + hkv) * z.sq + (r.ok ? r.i : 0)) * z.x.count;
#pragma unroll 1
        for (int k = z.x.count - 1 - g4; k >= 0 && lim > 0 && !any; k -= 4) {
            const int p = list[k];
            any = (unsigned)p < (unsigned)z.x.cv.width && p <= (lim - 1) >> z.x.cv.shift &&
                  cache_page(z.x.cv, b, p) >= 0;
        }
    } else {
#pragma unroll 1
        for (int p = ((lim - 1) >> z.x.cv.shift) - g4; p >= 0 && lim > 0 && !any; p -= 4)
            any = cache_page(z.x.cv, b, p) >= 0;
    }
    return max_groups(any ? 1.f : 0.f) > 0.f;
}

// A job's rows: [row0, end) are written, those at `rows` and behind are padding.
struct CacheJob {
    int b, hkv, grp, split, row0, rows, end, query;
    int kv, off, prefix, lim;  // lim: keys that any of its rows sees
};
template <typename A>
__device__ __forceinline__ CacheJob cache_job_of(const A& a, const FwdJob& f, int row_tile) {
    CacheJob j;
    j.b = f.b;
    j.hkv = f.hkv;
    j.grp = f.grp;
    j.split = f.split;
    const int n = cache_new(a.x.cv, j.b, a.sq);
    j.query = 0;
    j.row0 = f.tile * row_tile;
    j.end = a.rows;
    if (a.x.selected != nullptr) {
        j.query = fdiv(a.x.div_per_query, f.tile);
        j.row0 = j.query * a.group + (f.tile - j.query * a.x.per_query) * row_tile;
        j.end = (j.query + 1) * a.group;
    }
    j.rows = min(n * a.group, j.end);
    j.kv = cache_kv(a.x.cv, j.b);
    j.off = j.kv - n;
    j.prefix = attn_prefix(a.m, j.b);
    j.lim = 0;
    if (j.row0 < j.rows) {
        const int last = min(j.row0 + row_tile, j.rows) - 1;
        j.lim = attn_limit(fdiv(a.div_group, last), j.off, j.kv, a.m.causal, j.prefix);
    }
    return j;
}

template <typename A>
__device__ __forceinline__ CacheJob cache_job(const A& a, int id, int row_tile) {
    return cache_job_of(a, fwd_job(a, id), row_tile);
}

// Parts of the sequences dealt to the slots of a KV head: slot `slot` has part
// `split` of the `parts` of sequence b, which lie in the slots from first on;
// each is `part` blocks of 32 keys (deal_part).  b -1: nothing is left for the
// slot.  All lanes of all waves come to the same; a lane counts for every 64th
// sequence.
struct CacheDeal {
    int b, split, first, parts, part;
};
__device__ __forceinline__ uint32_t sum_lanes(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xF, 0xF, false);  // lane ^ 8
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, false);  // ^ 7
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, false);   // ^ 2
    x += (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, false);   // ^ 1
    auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = r[0] + r[1];
    r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(r[0] + r[1]);
}
template <typename A>
__device__ __forceinline__ CacheDeal cache_deal(const A& a, int slot) {
    constexpr int kChunks = kDealBatch / 64;
    const int lane = threadIdx.x & 63, B = a.x.batch;
    const auto& c = a.x.cv;
    uint32_t n[kChunks], mine[kChunks];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        const int b = 64 * k + lane;
        n[k] = mine[k] = 0;
        if (b < B) {
            const int kv = cache_length(c.kv_lens[b], c.width << c.shift);
            const int fresh = c.new_lens == nullptr ? a.sq : cache_length(c.new_lens[b], a.sq);
            n[k] = fresh > 0 ? (kv + 31) >> 5 : 0;
        }
    }
    uint32_t total = 0;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) total += n[k];
    total = sum_lanes(total);
    auto count = [&](uint32_t part) {
        uint32_t s = 0;
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
            if (64 * k < B) {
                mine[k] = 64 * k + lane < B ? max(1u, (n[k] + part - 1) / part) : 0u;
                s += mine[k];
            }
        return sum_lanes(s);
    };
    CacheDeal d{-1, 0, 0, 0, (int)(4 * deal_part(total, a.x.slots, B, a.part / 4, count))};
    count(d.part);
    int base = 0;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        if (64 * k >= B) continue;
        int upto = (int)mine[k];
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int x = __shfl_up(upto, o);
            if (lane >= o) upto += x;
        }
        const uint64_t past = __ballot(slot < base + upto);
        if (d.b < 0 && past != 0) {
            const int l = __builtin_ctzll(past);
            d.b = 64 * k + l;
            d.parts = __builtin_amdgcn_readlane((int)mine[k], l);
            d.first = base + __builtin_amdgcn_readlane(upto, l) - d.parts;
            d.split = slot - d.first;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
    }
    return d;
}

// Blocks of 32 keys that a job of few rows walks: [begin, end) of a sequence's
// (or of its selected pages'), in parts cut by what this sequence has.
struct CacheSpan {
    int begin, end;
};
template <typename A>
__device__ __forceinline__ CacheSpan cache_span(const A& a, const CacheJob& j) {
    int n = (j.lim + 31) >> 5;
    if (a.x.selected != nullptr) n = j.lim > 0 ? a.x.count << (a.x.cv.shift - 5) : 0;
    const int part = max((fdiv(a.div_splits, n + a.splits - 1) + 3) & ~3, a.part);
    const int64_t at = (int64_t)j.split * part;
    CacheSpan s;
    s.begin = at < n ? (int)at : n;
    s.end = n - s.begin > part ? s.begin + part : n;
    return s;
}
// Block `at`: its first place and its page (-1: none that is seen).
struct CacheBlock {
    int j0, page;
};
template <typename A>
__device__ __forceinline__ CacheBlock cache_block(const A& a, const CacheJob& j, int at, int end) {
    CacheBlock x{0, -1};
    if (at >= end) return x;
    const int shift = a.x.cv.shift;
    if (a.x.selected == nullptr) {
        x.j0 = at << 5;
        x.page = cache_page_scalar(a.x.cv, j.b, x.j0 >> shift);
        return x;
    }
    const int slot = at >> (shift - 5);
    const int p = scalar_load(a.x.selected + ((int64_t)j.grp * a.sq + j.query) * a.x.count + slot);
    if ((unsigned)p >= (unsigned)a.x.cv.width) return x;
    x.j0 = (p << shift) + ((at & ((1 << (shift - 5)) - 1)) << 5);
    if (x.j0 < j.lim) x.page = cache_page_scalar(a.x.cv, j.b, p);
    return x;
}

template <int D, bool kFour>
struct CacheTileCfg {
    static constexpr int kTileBytes = 64 * D * 2;
    static constexpr int kStageBytes = 2 * kTileBytes + (kFour ? 512 : 0);  // K, V, scales
    static constexpr int kBytes = 2 * kStageBytes;
    static constexpr int kDB = D / 16;
};

// A 64-key tile of 4-bit rows on its way: this lane's codes of row 16 w +
// lane / 4, 8-channel chunks lane % 4 + 4 i, and (lanes 0 .. 31) a scale.
template <int D>
struct FourTile {
    uint32_t k[D / 32], v[D / 32];
    float scale;
    // page: of the wave's 16 rows, which start at place j
    __device__ __forceinline__ void load(const char* kh, const char* vh, int64_t k_ps, int64_t v_ps,
                                         int page, int j, int kv, int shift, int lane) {
        const int mask = (1 << shift) - 1, row = (j & mask) + (lane >> 2);
        const bool ok = page >= 0 && j + (lane >> 2) < kv;
        const char* pk = kh + page * k_ps;
        const char* pv = vh + page * v_ps;
        const int at = row * (D / 2) + 4 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            k[i] = ok ? *(const uint32_t*)(pk + at + 16 * i) : 0u;
            v[i] = ok ? *(const uint32_t*)(pv + at + 16 * i) : 0u;
        }
        const int r = lane & 15;
        scale = 0.f;
        if (lane < 32 && page >= 0 && j + r < kv)
            scale = *(const float*)((lane < 16 ? pk : pv) + (D / 2 << shift) + ((j & mask) + r) * 4);
    }
    template <bool kBf16>
    __device__ __forceinline__ void store(FA3_LDS char* st, int w, int lane) const {
        const int row = 16 * w + (lane >> 2);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint32_t at = reg_tile_off<D>(row, (lane & 3) + 4 * i);
            lds_write_b128(st, at, cache_levels8<kBf16>(k[i]));
            lds_write_b128(st + 64 * D * 2, at, cache_levels8<true>(v[i]));
        }
        if (lane < 32)
            ((FA3_LDS float*)(st + 2 * 64 * D * 2))[(lane >> 4) * 64 + 16 * w + (lane & 15)] = scale;
    }
};

// 128 / kSplit rows a workgroup: attn_fwd_kernel with pages.
template <int D, bool kBf16, bool kCap, bool kBias, bool kFour, int kSplit>
__global__ __launch_bounds__(kRegThreads, D == 64 ? 3 : 2) void cache_tile_kernel(CacheAttnArgs) {
    typedef CacheAttnArgs Args;
    const auto& a = attn_args<Args>();
    using C = CacheTileCfg<D, kFour>;
    constexpr int kQb = kRegWaves / kSplit, kJob = 32 * kQb;
    __shared__ __attribute__((aligned(1024))) char smem_raw[C::kBytes];
    FA3_LDS char* smem = (FA3_LDS char*)smem_raw;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int qb = w & (kQb - 1), rs = w / kQb;
    const CacheJob job = cache_job(a, blockIdx.x, kJob);
    const int b = job.b, hkv = job.hkv, kv = job.kv;
    FwdRows<D, kBf16, kCap, kBias, Args, kFour> rows;
    rows.init(a, job.row0 + 32 * qb, job.rows, job.end, b, hkv, kv, job.prefix, job.off, lane);
    const int n_t = (job.lim + 63) >> 6;
    const int part = max(fdiv(a.div_splits, n_t + a.splits - 1), a.part);
    const int64_t at = (int64_t)job.split * part;
    const int begin = at < n_t ? (int)at : n_t;
    // (the rows' own place first, as in attn_fwd_kernel)
    const int own = fdiv(a.div_group, max(min(job.row0 + kJob, job.rows) - 1, 0)) + job.off;
    TileWalk walk(nullptr, begin, n_t - begin > part ? begin + part : n_t, DocSpan{0, 0, 0, 0, false},
                  own >> 6);
    const char* kh = a.x.cv.k + hkv * a.x.cv.k_hs;
    const char* vh = a.x.cv.v + hkv * a.x.cv.v_hs;
    const int shift = a.x.cv.shift;
    // the pages of a tile's halves; its second half behind the sequence: the first's
    struct Tile {
        int t, p0, p1;
    };
    auto look = [&]() {
        const auto& a = attn_args<Args>();
        Tile x;
        x.t = walk.next();
        x.p0 = x.p1 = -1;
        if (x.t >= 0) {
            const int n = (x.t * 64) >> shift;
            x.p0 = x.p1 = cache_page_scalar(a.x.cv, b, n);
            if (shift == 5 && x.t * 64 + 32 < kv) x.p1 = cache_page_scalar(a.x.cv, b, n + 1);
        }
        return x;
    };
    FourTile<D> four;
    auto issue = [&](FA3_LDS char* st, const Tile& x) {
        const auto& a = attn_args<Args>();
        const int lane = opaque_tid() & 63, j = x.t * 64 + 16 * w, page = w >> 1 ? x.p1 : x.p0;
        int64_t k_ps = a.x.cv.k_ps, v_ps = a.x.cv.v_ps;
        if constexpr (kFour) {
            four.load(kh, vh, k_ps, v_ps, page, j, kv, shift, lane);
        } else {
            constexpr int kLd = RegCfg<D>::kLd, kRows = 512 / D, kC = D / 8;
            const int row = lane / kC, at = j & ((1 << shift) - 1);
            const uint32_t c = ((uint32_t)(lane % kC) ^ reg_swz<D>(row)) & (kC - 1);
            const bool whole = page >= 0 && j + 16 <= kv && a.d == D;
            auto rows16 = [&](FA3_LDS char* tile, const char* head, int64_t ps, int64_t rs) {
                const char* p = head + page * ps + (at + row) * rs;
#pragma unroll
                for (int i = 0; i < kLd; ++i) {
                    const uint32_t ci = (c ^ reg_swz<D>(kRows * i)) & (kC - 1);
                    const char* y = p + (kRows * i) * rs + ci * 16;
                    if (!whole && !(page >= 0 && j + kRows * i + row < kv && (int)ci * 8 < a.d))
                        y = (const char*)attn_zeros;
                    __builtin_amdgcn_global_load_lds((const void*)y,
                                                     (FA3_LDS void*)(tile + (w * kLd + i) * 1024), 16, 0, 0);
                }
            };
            rows16(st, kh, k_ps, a.x.cv.k_rs);
            rows16(st + C::kTileBytes, vh, v_ps, a.x.cv.v_rs);
        }
    };
    auto settle4 = [&](FA3_LDS char* st) {
        if constexpr (kFour) four.template store<kBf16>(st, w, opaque_tid() & 63);
    };
    const RegReader<D> rd(lane, 0);
    const float c = a.m.c;
    FA3_LDS char* s0 = smem;
    FA3_LDS char* s1 = smem + C::kStageBytes;
    Tile cur = look();
    if (cur.t >= 0) issue(s0, cur);
    Tile next = look();
    rows.load(a, job.row0 + 32 * qb, job.rows, b, hkv, job.off, lane);
    if (cur.t >= 0) settle4(s0);
    auto stage = [&](FA3_LDS char* __restrict__ ld, const FA3_LDS char* __restrict__ st) {
        wait_vm_lgkm0<0>();
        barrier();
        if (next.t >= 0) issue(ld, next);
        const Tile far = look();
        const int j0 = cur.t * 64;
        const FA3_LDS char* sc = st + 2 * C::kTileBytes;
        if (kSplit == 2) {
            if ((rs ? cur.p1 : cur.p0) >= 0 && j0 + 32 * rs < rows.lim_max)
                rows.template step<2>(rd, st, st + C::kTileBytes, 2 * rs, j0 + 32 * rs, nullptr, c, sc + 128 * rs);
        } else if (cur.p0 >= 0 && cur.p1 >= 0) {
            if (j0 < rows.lim_max)
                rows.template step<4>(rd, st, st + C::kTileBytes, 0, j0, nullptr, c, sc);
        } else {
            const int h = cur.p0 >= 0 ? 0 : 1;  // (one half is none, or both)
            if ((cur.p0 & cur.p1) >= 0 && j0 + 32 * h < rows.lim_max)
                rows.template step<2>(rd, st + 32 * h * 2 * D, st + C::kTileBytes + 32 * h * 2 * D, 0,
                                      j0 + 32 * h, nullptr, c, sc + 128 * h);
        }
        if (next.t >= 0) settle4(ld);
        cur = next;
        next = far;
    };
    while (cur.t >= 0) {
        stage(s1, s0);
        if (cur.t < 0) break;
        stage(s0, s1);
    }
    wait_vm_lgkm0<0>();
    barrier();  // every wave is done with the stages: they take the outputs
    const CacheJob e = cache_job(attn_args<Args>(), blockIdx.x, kJob);
    const int ew = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6), eqb = ew & (kQb - 1);
    rows.template settle<true>(e.row0 + 32 * eqb, e.b, e.hkv);
    if constexpr (kSplit > 1) {
        rows.template meet<kSplit>((FA3_LDS float*)smem, smem + 2048, ew, eqb, ew / kQb);
        if (ew / kQb > 0) return;
    }
    rows.finish(e.row0 + 32 * eqb, e.end, e.b, e.hkv, e.grp, e.split,
                kSplit > 1 ? smem + 2048 + eqb * (C::kDB * 2048 + 512) : smem + ew * C::kDB * 1024);
}

}  // namespace
}  // namespace fa3
