// Forward attention with capped, biased and masked scores.
//
// One workgroup of four waves owns 128 rows of a KV head (a row is a query of
// one of its query heads) and walks the 64-key tiles that any of them sees,
// in one pass with the running maximum and sum of a softmax.  A wave owns 32
// rows: S^T = K Q^T with Q resident in registers as the B operand, the
// softmax down each lane's column, and O^T += V^T P^T, whose B operand is P
// as the score product left it, rounded (fa3_bwd_reg_kernel.h says why that
// needs no exchange).  K and V tiles go through two LDS stages, two (D 128)
// or three (D 64) workgroups share a CU.
//
// What bounds it.  The vector units as much as the matrix units: an element
// costs 16 cycles of exponential and about 16 more (a fma, a sum, half a
// maximum, half a conversion), a cap 40 on top, against 2 D / 8 cycles of
// products.  Measured, from box to box: B2 Hq32 Hkv8 S4096 D128 causal 280-299
// us (980-920 TFLOP/s), B2 H16 S8192 D64 full 627-662 us (877-830) and with a
// distance bias 555-600 (990-916 of the nominal work: tiles without weight are
// left), documents of ~1500 tokens at S4096 162-171 us (722-684 of the visible
// work).  Small launches are bound by one wave's chain, ~2 600 cycles a 32 x 32
// step of which 512 are products: making the next tile's scores behind this
// tile's exponentials (a pipeline within the wave) did not shorten it (S2011
// capped 48.9 -> 52.2 us), nor did sending the loads out later.
#include "fa3_attn_fwd_kernel.h"

namespace fa3 {
namespace {

// 128 / kSplit rows a workgroup.  kSplit 2: the two waves of a 32-row block
// take one 32-key half of every stage each.
template <int D, bool kBf16, bool kCap, bool kBias, int kSplit>
__global__ __launch_bounds__(kRegThreads, D == 64 ? 3 : 2) void attn_fwd_kernel(AttnFwdArgs) {
    typedef AttnFwdArgs Args;
    const auto& a = attn_args<Args>();
    using C = FwdCfg<D>;
    constexpr int kQb = kRegWaves / kSplit;  // 32-row blocks of the job
    __shared__ __attribute__((aligned(1024))) char smem_raw[C::kBytes];
    FA3_LDS char* smem = (FA3_LDS char*)smem_raw;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int qb = w & (kQb - 1), rs = w / kQb;
    const FwdJob job = fwd_job(a, blockIdx.x);
    const int b = job.b, hkv = job.hkv;
    const int kv = attn_kv(a.m, b, a.sk), prefix = attn_prefix(a.m, b), off = kv - a.sq;
    FwdRows<D, kBf16, kCap, kBias> rows;
    rows.init(a, (job.tile * kQb + qb) * 32, a.rows, a.rows, b, hkv, kv, prefix, off, lane);
    const int wg_last = min((job.tile + 1) * (32 * kQb), a.rows) - 1;
    const int wg_max = attn_limit(fdiv(a.div_group, wg_last), off, kv, a.m.causal, prefix);
    DocSpan doc{0, 0, 0, 0, false};
    if (a.m.doc_q != nullptr) doc = doc_span(rows.id, (FA3_LDS int*)(smem + C::kRangeOff), w, lane);

    const _Float16* kp = a.k.p + b * a.k.bs + hkv * a.k.hs;
    const _Float16* vp = a.v.p + b * a.v.bs + hkv * a.v.hs;
    const int* ids = a.m.doc_k == nullptr ? nullptr : a.m.doc_k + b * a.m.doc_k_bs;
    const int begin = job.split * a.part;
    // (the workgroup's own place among the keys: with a distance bias the
    // nearest tiles first, which leave little to rescale and much to skip)
    const int rows_at = fdiv(a.div_group, wg_last) + off;
    TileWalk walk(ids == nullptr ? nullptr : a.m.range_k + (int64_t)b * a.m.blocks_k, begin,
                  min(begin + a.part, (wg_max + 63) >> 6), doc, rows_at >> 6);
    // (held in scalar registers: read again per tile, as the arguments are
    // elsewhere, they are waited for before the tile's loads go out; opaque,
    // so that their multiples are not held too)
    const int64_t k_rs = a.k.rs, v_rs = a.v.rs;
    const bool wide = a.d == D;
    auto issue = [&](FA3_LDS char* st, int t) {
        const int j0 = t * 64, lane = opaque_tid() & 63;
        int64_t krs = k_rs, vrs = v_rs;
        __asm__ volatile("" : "+s"(krs), "+s"(vrs));
        if (j0 + 64 <= kv && wide && !(walk.cls & kTileHidden)) {
            attn_load_tile<D>(st, kp, krs, j0, w, lane);
            attn_load_tile<D>(st + C::kTileBytes, vp, vrs, j0, w, lane);
        } else {
            const auto& a = attn_args<Args>();
            auto seen = [&](int j) { return ids == nullptr || ids[j] >= 0; };
            attn_load_tile_edge<D>(st, kp, krs, j0, kv, a.d, w, lane, seen);
            attn_load_tile_edge<D>(st + C::kTileBytes, vp, vrs, j0, kv, a.d, w, lane, seen);
        }
        if (ids != nullptr && w == 0)
            attn_load_ids(st + 2 * C::kTileBytes, ids, j0, attn_args<Args>().sk, lane);
    };
    const RegReader<D> rd(lane, 0);
    const float c = a.m.c;
    FA3_LDS char* s0 = smem;
    FA3_LDS char* s1 = smem + C::kStageBytes;
    int t = walk.next();
    if (t >= 0) issue(s0, t);
    rows.load(a, (job.tile * kQb + qb) * 32, a.rows, b, hkv, off, lane);
    auto stage = [&](FA3_LDS char* __restrict__ ld, const FA3_LDS char* __restrict__ st) {
        const int cls = walk.cls, tn = walk.next();
        wait_vm_lgkm0<0>();
        barrier();
        if (tn >= 0) issue(ld, tn);
        if (cls & kTileMeets) {
            constexpr int kKeys = 64 / kSplit;
            const int j0 = t * 64 + kKeys * rs;
            if (j0 < rows.lim_max)
                rows.template step<4 / kSplit>(
                    rd, st, st + C::kTileBytes, kKeys / 16 * rs, j0,
                    cls & kTileSame ? nullptr : st + 2 * C::kTileBytes + 4 * kKeys * rs, c);
        }
        t = tn;
    };
    while (t >= 0) {
        stage(s1, s0);
        if (t < 0) break;
        stage(s0, s1);
    }
    wait_vm_lgkm0<0>();
    barrier();  // every wave is done with the stages: they take the outputs
    const FwdJob e = fwd_job(attn_args<Args>(), blockIdx.x);  // (decoded again: not held over the loop)
    const int ew = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6), eqb = ew & (kQb - 1);
    rows.template settle<true>((e.tile * kQb + eqb) * 32, e.b, e.hkv);
    if constexpr (kSplit > 1) {
        rows.template meet<kSplit>((FA3_LDS float*)smem, smem + 2048, ew, eqb, ew / kQb);
        if (ew / kQb > 0) return;
    }
    // (of the meeting, this wave reads only what it has read: its own block's slots)
    rows.finish((e.tile * kQb + eqb) * 32, attn_args<Args>().rows, e.b, e.hkv, e.grp, e.split,
                kSplit > 1 ? smem + 2048 + eqb * (C::kDB * 2048 + 512) : smem + ew * C::kDB * 1024);
}

// Few rows (32 at most of a KV head: single tokens), no documents: a
// workgroup's four waves all hold them and take every fourth 32-key block
// each, through two LDS stages of their own -- no barrier until they meet.
// Bound by reading the cache: 5.4 TB/s for 16 caches of 8192 keys (Hkv 8, D
// 128, 99 us, the rate of a large copy), 4.9 where they are filled to
// different lengths (64-69 us).
template <int D>
struct TokenCfg {
    static constexpr int kBlock = 32 * D * 2;   // 32 rows of K or V
    static constexpr int kStage = 2 * kBlock;
    static constexpr int kBytes = kRegWaves * 2 * kStage;
    static constexpr int kLd = kBlock / 1024;   // loads per wave, block and tensor
    static_assert(2048 + 3 * (D / 16 * 2048 + 512) <= kBytes, "the meeting fits the stages");
};

template <int D, bool kBf16, bool kCap, bool kBias>
__global__ __launch_bounds__(kRegThreads, D == 64 ? 2 : 1) void attn_token_kernel(AttnFwdArgs) {
    typedef AttnFwdArgs Args;
    const auto& a = attn_args<Args>();
    using C = TokenCfg<D>;
    __shared__ __attribute__((aligned(1024))) char smem_raw[C::kBytes];
    FA3_LDS char* smem = (FA3_LDS char*)smem_raw;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const FwdJob job = fwd_job(a, blockIdx.x);
    const int b = job.b, hkv = job.hkv;
    const int kv = attn_kv(a.m, b, a.sk), prefix = attn_prefix(a.m, b), off = kv - a.sq;
    const _Float16* kp = a.k.p + b * a.k.bs + hkv * a.k.hs;
    const _Float16* vp = a.v.p + b * a.v.bs + hkv * a.v.hs;
    // this wave's x-th block is keys 32 (first + 4 x) ..
    const int lim = attn_limit(a.sq - 1, off, kv, a.m.causal, prefix);
    const int first = 2 * job.split * a.part + w;
    const int end = min(2 * (job.split + 1) * a.part, (lim + 31) >> 5);
    const int n = end > first ? (end - first + 3) >> 2 : 0;
    auto load = [&](FA3_LDS char* st, const _Float16* src, int64_t rs, int j0, bool whole, int d) {
        constexpr int kRows = 512 / D, kC = D / 8;
        const int ln = opaque_tid() & 63, row = ln / kC;
        const uint32_t cc = ((uint32_t)(ln % kC) ^ reg_swz<D>(row)) & (kC - 1);
        const char* p = (const char*)(src + (int64_t)(j0 + row) * rs);
        auto put = [&](int j, const char* x) {
            __builtin_amdgcn_global_load_lds((const void*)x, (FA3_LDS void*)(st + j * 1024), 16, 0, 0);
        };
        auto chunk = [&](int j) { return (cc ^ reg_swz<D>(kRows * j)) & (kC - 1); };
        if (whole) {
#pragma unroll
            for (int j = 0; j < C::kLd; ++j) put(j, p + (int64_t)(kRows * j) * rs * 2 + chunk(j) * 16);
        } else {
#pragma unroll
            for (int j = 0; j < C::kLd; ++j) {
                const bool ok = j0 + kRows * j + row < kv && (int)chunk(j) * 8 < d;
                put(j, ok ? p + (int64_t)(kRows * j) * rs * 2 + chunk(j) * 16 : (const char*)attn_zeros);
            }
        }
    };
    // one stage: always 2 kLd loads, which the waits below count
    auto issue = [&](FA3_LDS char* st, int x) {
        const auto& a = attn_args<Args>();
        const int j0 = 32 * (first + 4 * x);
        const bool whole = j0 + 32 <= kv && a.d == D;
        load(st, kp, a.k.rs, j0, whole, a.d);
        load(st + C::kBlock, vp, a.v.rs, j0, whole, a.d);
    };
    FA3_LDS char* s0 = smem + w * 2 * C::kStage;
    FA3_LDS char* s1 = s0 + C::kStage;
    if (n > 0) issue(s0, 0);
    FwdRows<D, kBf16, kCap, kBias> rows;
    rows.init(a, 0, a.rows, a.rows, b, hkv, kv, prefix, off, lane);
    rows.load(a, 0, a.rows, b, hkv, off, lane);
    const RegReader<D> rd(lane, 0);
    const float c = a.m.c;
    int x = 0;
    auto stage = [&](FA3_LDS char* __restrict__ ld, const FA3_LDS char* __restrict__ st) {
        wait_vm_lgkm0<63>();  // (the block read from ld before is done with)
        wall();
        if (x + 1 < n) {
            issue(ld, x + 1);
            wall();
            wait_vm_lgkm0<2 * C::kLd>();
        } else {
            wait_vm_lgkm0<0>();
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        wall();
        const int j0 = 32 * (first + 4 * x);
        rows.template step<2>(rd, st, st + C::kBlock, 0, j0, nullptr, c);
        ++x;
    };
    while (x < n) {
        stage(s1, s0);
        if (x >= n) break;
        stage(s0, s1);
    }
    wait_vm_lgkm0<0>();
    barrier();
    const FwdJob e = fwd_job(attn_args<Args>(), blockIdx.x);
    const int ew = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6);
    rows.template settle<false>(0, e.b, e.hkv);
    rows.template meet<4>((FA3_LDS float*)smem, smem + 2048, ew, 0, ew);
    if (ew > 0) return;
    rows.finish(0, attn_args<Args>().rows, e.b, e.hkv, e.grp, e.split, smem + 2048);
}

// One wave per 64 positions.
__global__ __launch_bounds__(256) void attn_ranges_kernel(const int* ids, int64_t bs, int n,
                                                          int blocks, int total, AttnRange* out) {
    const int x = blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (x < total) attn_range(ids, bs, n, blocks, x, out, threadIdx.x & 63);
}

AttnView view(const ShaoboFa3AttnTensor& t) {
    return AttnView{(_Float16*)t.data, t.batch_stride, t.head_stride, t.row_stride};
}

}  // namespace

AttnFwdPlan plan_attn_fwd(const AttnProblem& p) {
    AttnFwdPlan f{};
    const int64_t rows = (int64_t)p.group * p.sq, groups = (int64_t)p.batch * p.heads_kv;
    const int D = p.d > 64 ? 128 : 64;
    const int n_t = ceil_div(p.sk, 64);
    // One 32-row block: every wave on the cache, not one of four (B1 Hq32 Hkv8
    // Sk16384 D128 19.4 us, 291 by row tiles with the key axis whole).
    f.token = rows <= 32 && !p.docs;
    // 64-row jobs until two of 128 rows a CU fill the chip: B1 Hq16 Hkv4 S2011
    // 45.0 us against 58.1, but B2 Hq32 Hkv8 S4096 398 against 302.
    f.split = !f.token && groups * ceil_div(rows, kAttnRows) < 512 ? 2 : 1;
    f.tiles = f.token ? 1 : ceil_div(rows, kAttnRows / f.split);
    f.splits = 1;
    f.part = n_t;
    const int64_t jobs = groups * f.tiles;
    // Jobs that leave the chip half empty cut the key axis, as long as a part
    // keeps a few tiles: B1 H7 S1923 32.6 us in two parts, 42.4 whole, but B1
    // Hq32 Hkv8 S512 23.3 in two and 16.2 whole.  (A CU holds one workgroup of
    // the kernel for few rows at D 128, two otherwise.)
    const int fill = f.token && D == 128 ? 256 : 512, least = f.token ? 4 : 8;
    if (jobs > 0 && 2 * jobs <= fill && n_t >= 2 * least) {
        const int want = (int)(fill / jobs), most = n_t / least;
        f.part = ceil_div(n_t, want < most ? want : most);
        f.splits = ceil_div(n_t, f.part);
    }
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t x = at;
        at += (n + 255) / 256 * 256;
        return x;
    };
    f.range_off = take(p.docs ? (size_t)p.batch * n_t * sizeof(AttnRange) : 0);
    if (f.splits > 1) {
        f.po_off = take((size_t)f.splits * groups * rows * D * 4);
        f.pl_off = take((size_t)f.splits * groups * rows * 4);
    }
    f.total = at;
    const int64_t all = groups * f.tiles * f.splits;
    f.ok = rows < (1ll << 30) && all < kMaxGrid && groups * rows / 4 < kMaxGrid &&
           (int64_t)p.batch * n_t < kMaxGrid;
    f.jobs = f.ok ? (int)all : 0;
    return f;
}

hipError_t launch_attn_fwd(const AttnProblem& p, const ShaoboFa3AttnParams& a, AttnMask m,
                           hipStream_t stream) {
    const AttnFwdPlan f = plan_attn_fwd(p);
    char* ws = (char*)a.workspace;
    AttnFwdArgs x{};
    x.q = view(a.q);
    x.k = view(a.k);
    x.v = view(a.v);
    x.out = view(a.out);
    x.lse = a.softmax_lse;
    x.heads_q = p.heads_q;
    x.heads_kv = p.heads_kv;
    x.group = p.group;
    x.sq = p.sq;
    x.sk = p.sk;
    x.d = p.d;
    x.rows = p.group * p.sq;
    x.tiles = f.tiles;
    x.splits = f.splits;
    x.part = f.part;
    x.groups = p.batch * p.heads_kv;
    x.div_hkv = make_fastdiv(p.heads_kv);
    x.div_group = make_fastdiv(p.group);
    x.div_groups = make_fastdiv(x.groups);
    x.div_gpart = make_fastdiv(x.groups / 8);
    x.div_splits = make_fastdiv(f.splits);
    x.levels = f.tiles * f.splits;
    x.div_levels = make_fastdiv(x.levels);
    // Causal jobs differ in length by their place: longest first (B4 H16 S2048
    // D128 88 us against 128 group after group).  Full ones do not, and with
    // documents the place says little: a group's keys in one L2 count for more
    // (B2 H16 S8192 D64 with bias 668 -> 551, B2 Hq32 Hkv8 S4096 with
    // documents 250 -> 199).
    x.by_group = !p.causal || p.docs;
    const bool cap = p.softcap > 0.f, bias = p.bias;
    // Maxima are taken over raw products: their scale must be positive.
    x.scored = 1;
    if (!cap) {
        if (m.c < 0.f) x.flip = 0x80008000u;
        x.scored = m.c != 0.f;
        m.c = m.c == 0.f ? 1.f : m.c < 0.f ? -m.c : m.c;
    }
    if (f.jobs == 0) return hipSuccess;
    if (p.docs && p.sk > 0) {
        AttnRange* r = (AttnRange*)(ws + f.range_off);
        const int blocks = ceil_div(p.sk, 64), total = p.batch * blocks;
        hipLaunchKernelGGL(attn_ranges_kernel, dim3(ceil_div(total, 4)), dim3(256), 0, stream,
                           m.doc_k, m.doc_k_bs, p.sk, blocks, total, r);
        m.range_k = r;
        m.blocks_k = ceil_div(p.sk, 64);
    }
    x.part_o = (float*)(ws + f.po_off);
    x.part_l = (float*)(ws + f.pl_off);
    x.m = m;
    auto pick = [&](auto d, auto bf) {
        constexpr int kD = decltype(d)::value;
        constexpr bool kB = decltype(bf)::value;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(f.jobs), dim3(kRegThreads), 0, stream, x);
        };
        auto join = [&](auto ways) {
            constexpr int kW = decltype(ways)::value;
            hipLaunchKernelGGL((attn_join_kernel<kD, kB, kW>),
                               dim3(ceil_div((int64_t)x.groups * x.rows, 2048 / (kD * kW))),
                               dim3(256), 0, stream, x);
        };
        auto kinds = [&](auto cz, auto bi) {
            constexpr bool kC = decltype(cz)::value, kBi = decltype(bi)::value;
            if (f.token) go(attn_token_kernel<kD, kB, kC, kBi>);
            else if (f.split == 2) go(attn_fwd_kernel<kD, kB, kC, kBi, 2>);
            else go(attn_fwd_kernel<kD, kB, kC, kBi, 1>);
        };
        using T = std::true_type;
        using F = std::false_type;
        if (cap) bias ? kinds(T{}, T{}) : kinds(T{}, F{});
        else bias ? kinds(F{}, T{}) : kinds(F{}, F{});
        if (f.splits > 1)
            f.splits >= 8 ? join(std::integral_constant<int, 512 / kD>{})
                          : join(std::integral_constant<int, 1>{});
    };
    using T = std::true_type;
    using F = std::false_type;
    if (p.d > 64) p.bf16 ? pick(std::integral_constant<int, 128>{}, T{}) : pick(std::integral_constant<int, 128>{}, F{});
    else p.bf16 ? pick(std::integral_constant<int, 64>{}, T{}) : pick(std::integral_constant<int, 64>{}, F{});
    return hipGetLastError();
}

}  // namespace fa3
