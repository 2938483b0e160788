// Backward of attention with capped, biased and masked scores.
//
// Two job roles in one launch, as in bwd_reg_kernel (fa3_bwd_reg_kernel.h):
// a dKV job owns 128 keys of a KV head and streams the 64-row query tiles of
// its query heads that see any of them; a dQ job owns 128 rows (query and
// query head) and streams the 64-key tiles.  Every output has one writer, so
// nothing is added atomically and results are reproducible.  P and dS stay
// in registers as the next product's operand.  A pass over dO and O before it
// leaves -lse log2 e and -delta per row, padded to whole tiles: a row that
// sees no key, or is not there, has -infinity in place of the first, which
// makes its P zero.
//
// What bounds it.  As bwd_reg_kernel, power and two waves' products, LDS reads
// and exponentials on one SIMD in large launches: B2 Hq32 Hkv8 S4096 D128
// causal 852-872 us (806-788 TFLOP/s of five products), documents of ~1500
// tokens 656-676 us (521-506 of the visible work; a document of 3391 tokens
// among them makes the longest job).  Small ones are bound by a job's chain,
// hence the cuts of plan_attn_bwd.  dQ recomputes S and dP (seven products
// instead of five): adding dS K across workgroups would need atomics or an
// S^2-sized workspace.
#pragma once

#include "fa3_attn_device.h"

namespace fa3 {
namespace {

template <int D>
struct BwdCfg {
    using R = RegCfg<D>;
    // two tiles, the rows' statistics, the documents of 64 rows or keys
    static constexpr int kStageBytes = R::kStageBytes + 256, kIdsOff = R::kStageBytes;
    static constexpr int kRangeOff = 2 * kStageBytes;
    static constexpr int kBytes = kRangeOff + 64;
    static constexpr int kKs = D / 32, kDB = D / 16;
};

// Workgroup id's job: level < kv_tiles * parts is a dKV job's key tile and
// part (first keys first: causal's longest), then come the dQ jobs, last rows
// first -- or, where the launch is no more than two jobs a CU, first rows
// first: the longest dKV job then has the shortest dQ job beside it.
struct BwdJob {
    int b, hkv, level;
};
template <typename Args>
__device__ __forceinline__ BwdJob bwd_job(const Args& a, int id) {
    BwdJob j;
    int grp;
    // (group after group leaves the last group's dKV jobs to the end: B2 Hq32
    // Hkv8 S4096 D128 causal 852 -> 1138 us, full 1613 -> 1743)
    attn_job(id, a.groups, false, a.div_groups, a.div_gpart, a.div_gpart, 0, j.level, grp);
    j.b = fdiv(a.div_hkv, grp);
    j.hkv = grp - j.b * a.heads_kv;
    return j;
}

template <typename Args>
__device__ __forceinline__ int dq_tile(const Args& a, int level) {
    const int x = level - a.kv_tiles * a.parts;
    return a.rising ? x : a.q_tiles - 1 - x;
}

// One workgroup per 64 rows of a query head; with documents, behind them, one
// per four 64-position blocks of the queries' and then the keys' documents
// (a launch of their own each took 2.5 us).
template <int D, bool kBf16>
__global__ __launch_bounds__(256) void attn_delta_kernel(AttnBwdArgs a) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes;
    if ((int)blockIdx.x >= a.delta_blocks) {
        const int lane = threadIdx.x & 63;
        int x = ((int)blockIdx.x - a.delta_blocks) * 4 + (int)(threadIdx.x >> 6);
        const int nq = (a.q_blocks + 3) / 4 * 4;
        if (x < a.q_blocks)
            attn_range(a.m.doc_q, a.m.doc_q_bs, a.sq, a.m.blocks_q, x, (AttnRange*)a.m.range_q, lane);
        x -= nq;
        if (x >= 0 && x < a.k_blocks)
            attn_range(a.m.doc_k, a.m.doc_k_bs, a.sk, a.m.blocks_k, x, (AttnRange*)a.m.range_k, lane);
        return;
    }
    const int blk = blockIdx.x, nb = a.sqp / 64;
    const int bh = fdiv(a.div_blocks, blk), t = blk - bh * nb;
    const int b = fdiv(a.div_hq, bh), h = bh - b * a.heads_q;
    const int c = threadIdx.x % kLanes;
    bool idle = false;
#pragma unroll
    for (int j = 0; j < 64 / kRows; ++j) {
        const int i = t * 64 + j * kRows + (int)(threadIdx.x / kLanes);
        const bool there = i < a.sq;
        const _Float16* x = a.dout.p + b * a.dout.bs + h * a.dout.hs + (there ? i * a.dout.rs : 0);
        const _Float16* y = a.out.p + b * a.out.bs + h * a.out.hs + (there ? i * a.out.rs : 0);
        const float l = there ? a.lse[(int64_t)bh * a.sq + i] : kNegInf;
        const f16x8 u = attn_row8(x, c, a.d, there), v = attn_row8(y, c, a.d, there);
        float acc = dot8<kBf16>(u, v, 0.f);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) acc += __shfl_xor(acc, o, kLanes);
        const bool none = l == kNegInf;
        idle |= none;
        if (none) acc = 0.f;
        if (c == 0) {
            a.nlse2[(int64_t)bh * a.sqp + i] = none ? kNegInf : -l * kLog2e;
            a.ndelta[(int64_t)bh * a.sqp + i] = -acc;
            if (there && a.softmax_d != nullptr) a.softmax_d[(int64_t)bh * a.sq + i] = acc;
        }
    }
    const int any = __syncthreads_or(idle);
    if (threadIdx.x == 0) a.flags[blk] = any;
}

// Bit x of the result as all ones or zeros.
__device__ __forceinline__ uint32_t bit_mask(uint32_t v, int x) {
    return (uint32_t)((int32_t)(v << (31 - x)) >> 31);
}
// P and dS of one element.  s: raw product, dp: dP - delta, nl: -lse log2 e,
// far: distance (bias), vis: all ones, or zeros where the element is masked.
template <bool kCap, bool kBias>
__device__ __forceinline__ void attn_pds(float s, float dp, float nl, float c, float k1,
                                         float cap2, bool fine, float slope, float far,
                                         uint32_t vis, float& p, float& ds) {
    float x, t = 0.f;
    if constexpr (kCap) {
        if (fine) wall();  // (one element at a time, for the registers)
        t = fine ? attn_tanh_fine(s, k1) : attn_tanh(s, k1);
        x = __builtin_fmaf(t, cap2, nl);
    } else {
        x = __builtin_fmaf(s, c, nl);
    }
    if constexpr (kBias) x = __builtin_fmaf(-slope, __builtin_fabsf(far), x);
    p = fast_exp2(x);
    p = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, p) & vis);
    ds = p * dp;
    if constexpr (kCap) ds *= __builtin_fmaf(-t, t, 1.f);
}

// Key tile `tile` (128 / kSplit keys).  kSplit 2: the two waves of a 32-key
// block take one 32-row half of every stage each, and add up at the end.
template <int D, bool kBf16, bool kCap, bool kBias, bool kFine, int kSplit>
__device__ __forceinline__ void attn_dkv(int b, int hkv, int level, FA3_LDS char* smem) {
    typedef AttnBwdArgs Args;
    using C = BwdCfg<D>;
    using R = RegCfg<D>;
    const auto& a = attn_args<Args>();
    const int lane = opaque_tid() & 63;
    const int w = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6);
    const int l16 = lane & 15, g4 = lane >> 4;
    const int kv = attn_kv(a.m, b, a.sk), off = kv - a.sq;
    // (keys below it are seen by every query)
    const int prefix = a.m.causal ? attn_prefix(a.m, b) : 0x7fffffff;
    constexpr int kKb = kRegWaves / kSplit;  // 32-key blocks of the job
    const int tile = fdiv(a.div_parts, level), part = level - tile * a.parts;
    const int head_part = fdiv(a.div_rparts, part), row_part = part - head_part * a.row_parts;
    const int rs = w / kKb;
    const int wg_key = tile * (32 * kKb), key0 = wg_key + 32 * (w & (kKb - 1));

    int id[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int j = key0 + 16 * n + l16;
        id[n] = -2;
        if (a.m.doc_k != nullptr && j < kv) id[n] = max(a.m.doc_k[b * a.m.doc_k_bs + j], -1);
    }
    DocSpan doc{0, 0, 0, 0, false};
    const bool docs = a.m.doc_k != nullptr;
    if (docs) doc = doc_span(id, (FA3_LDS int*)(smem + C::kRangeOff), w, lane);

    int begin = 0, end = a.sqp / 64;
    if (wg_key >= prefix && wg_key - off > 0) begin = (wg_key - off) >> 6;
    if (wg_key >= kv) end = begin;
    const int len = end - begin;
    TileWalk walk(docs ? a.m.range_q + (int64_t)b * a.m.blocks_q : nullptr,
                  begin + len * row_part / a.row_parts, begin + len * (row_part + 1) / a.row_parts,
                  doc, end);
    const int g_first = a.group * head_part / a.head_parts;
    const int g_end = a.group * (head_part + 1) / a.head_parts;
    // The step being computed -- query tile and head of the group -- and the
    // one to load.  The next one is looked up before the barrier, so that its
    // words are there when its loads go out.
    int t, g, cls;
    int ld_t = walk.next(), ld_g = g_first, ld_idle = 0;
    auto lookup = [&]() {
        if (ld_t < 0) return;
        const auto& a = attn_args<Args>();
        const int h = hkv * a.group + ld_g;
        ld_idle = scalar_load(a.flags + (((int64_t)b * a.heads_q + h) * (a.sqp >> 6) + ld_t));
    };
    auto take = [&]() {
        t = ld_t;
        g = ld_g;
        cls = walk.cls;
    };
    lookup();
    take();
    auto issue = [&](FA3_LDS char* st) {
        const int ln = opaque_tid() & 63, i0 = ld_t * 64, h = hkv * attn_args<Args>().group + ld_g;
        int64_t row;  // of the statistics
        bool whole;
        {
            const auto& a = attn_args<Args>();
            row = ((int64_t)b * a.heads_q + h) * a.sqp + i0;
            whole = a.d == D && ld_idle == 0;
        }
        auto load = [&](FA3_LDS char* tile, const auto& x) {
            const _Float16* p = x.p + b * x.bs + h * x.hs;
            if (whole) {
                attn_load_tile<D>(tile, p, x.rs, i0, w, ln);
            } else {
                const auto& a = attn_args<Args>();
                const float* nl = a.nlse2 + (row - i0);
                attn_load_tile_edge<D>(tile, p, x.rs, i0, a.sq, a.d, w, ln,
                                       [&](int i) { return nl[i] != kNegInf; });
            }
        };
        load(st, attn_args<Args>().q);
        wall();
        load(st + R::kTileBytes, attn_args<Args>().dout);
        wall();
        const auto& a = attn_args<Args>();
        if (w < 2)
            __builtin_amdgcn_global_load_lds((const void*)((w == 0 ? a.nlse2 : a.ndelta) + row + ln),
                                             (FA3_LDS void*)(st + 2 * R::kTileBytes + 256 * w), 4, 0, 0);
        else if (w == 2 && a.m.doc_q != nullptr)
            attn_load_ids(st + C::kIdsOff, a.m.doc_q + b * a.m.doc_q_bs, i0, a.sq, ln);
    };
    FA3_LDS char* s0 = smem;
    FA3_LDS char* s1 = smem + C::kStageBytes;
    if (t >= 0) issue(s0);
    f16x8 kf[2][C::kKs], vf[2][C::kKs];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int j = key0 + 16 * n + l16;
        const bool ok = j < kv && id[n] != -1;
        const int64_t r = j < kv ? j : 0;
        const _Float16* k = a.k.p + b * a.k.bs + hkv * a.k.hs + r * a.k.rs;
        const _Float16* v = a.v.p + b * a.v.bs + hkv * a.v.hs + r * a.v.rs;
#pragma unroll
        for (int s = 0; s < C::kKs; ++s) {
            kf[n][s] = attn_row8(k, p1_chunk<D>(s, g4), a.d, ok);
            vf[n][s] = attn_row8(v, p1_chunk<D>(s, g4), a.d, ok);
        }
    }
    f32x4 av[C::kDB][2], ak[C::kDB][2];
#pragma unroll
    for (int i = 0; i < C::kDB; ++i) {
        av[i][0] = av[i][1] = f32x4{};
        ak[i][0] = ak[i][1] = f32x4{};
    }
    const RegReader<D> rd0(lane, 0);
    const float c = a.m.c;

    auto sub = [&](const FA3_LDS char* st, int r, bool same) {
        const int i0 = t * 64 + 32 * r;
        // rows i0 .. i0 + 31 against keys key0 .. key0 + 31
        if (key0 >= kv || (key0 >= prefix && key0 > i0 + 31 + off)) return;
        const bool full = key0 + 32 <= kv && same &&
                          (key0 + 31 <= i0 + off || prefix - 32 >= key0);
        uint32_t vis = 0xffff;
        if (!full) {
            const int l = opaque_tid() & 63;
            vis = 0;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int j = key0 + 16 * n + (l & 15);
                // rows (m, e) with 16 m + e >= first see key j
                const int first = j >= kv ? 64
                                  : j < prefix ? -64
                                               : j - off - i0 - 4 * (l >> 4);
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    vis |= 16 * (x >> 2) + (x & 3) >= first ? 1u << (8 * n + x) : 0u;
            }
            if (walk.ranges != nullptr) {
                const auto& a = attn_args<Args>();
                uint32_t met = 0;
                int id[2];  // (read again: not worth two registers over the loop)
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    id[n] = max(a.m.doc_k[b * a.m.doc_k_bs + min(key0 + 16 * n + (l & 15), a.sk - 1)], -1);
                const FA3_LDS i32x4* ids = (const FA3_LDS i32x4*)(st + C::kIdsOff + 128 * r) + (l >> 4);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const i32x4 x = ids[4 * m];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            met |= doc_of(x[e]) == id[n] ? 1u << (8 * n + 4 * m + e) : 0u;
                }
                vis &= met;
            }
        }
        RegReader<D> rd = rd0;
        rd.opaque();
        const FA3_LDS f32x4* rows = (const FA3_LDS f32x4*)(st + 2 * R::kTileBytes + 128 * r) +
                                    ((opaque_tid() & 63) >> 4);
        f32x4 s[2][2], dp[2][2], nl[2];  // [m][n]: rows 16 m + 4 g4 + e, keys 16 n + l16
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            dp[m][0] = dp[m][1] = rows[16 + 4 * m];
            s[m][0] = s[m][1] = f32x4{};
        }
        reg_scores<D, kBf16, AttnAhead<D, D == 128 ? kCap || kBias : kFine>>(rd, st, st + R::kTileBytes, r, kf, vf, s, dp);
        nl[0] = rows[0];
        nl[1] = rows[4];
        float slope = 0.f;
        if constexpr (kBias) {
            const auto& a = attn_args<Args>();
            slope = scalar_load(a.m.slopes + (b * a.m.slopes_bs + hkv * a.group + g)) * kLog2e;
        }
        float k1 = 0.f, cap2 = 0.f;
        if constexpr (kCap) {
            const auto& a = attn_args<Args>();
            k1 = a.m.k1;
            cap2 = a.m.cap2;
        }
        float p[2][8], ds[2][8];  // [n][4 m + e]
        const int ln = opaque_tid() & 63;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            // distance of row (m, e): d0 + 16 m + e
            wall();
            const float d0 = kBias ? (float)(i0 + off + 4 * (ln >> 4) - key0 - 16 * n - (ln & 15)) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int m = j >> 2, e = j & 3;
                if (kCap && kSplit == 2 && j == 4) wall();
                attn_pds<kCap, kBias>(s[m][n][e], dp[m][n][e], nl[m][e], c, k1, cap2, kFine, slope,
                                      d0 + (float)(16 * m + e), bit_mask(vis, 8 * n + j), p[n][j],
                                      ds[n][j]);
            }
        }
        const f16x8 bp[2] = {pack8<kBf16>(p[0]), pack8<kBf16>(p[1])};
        const f16x8 bs[2] = {pack8<kBf16>(ds[0]), pack8<kBf16>(ds[1])};
        reg_grads<D, kBf16, true, AttnAhead<D, D == 128 ? kCap || kBias : kFine>>(rd, st + R::kTileBytes, st, r, bp, bs, av, ak);
    };
    auto stage = [&](FA3_LDS char* __restrict__ ld, const FA3_LDS char* __restrict__ st) {
        if (++ld_g == g_end) {
            ld_g = g_first;
            ld_t = walk.next();
        }
        lookup();
        wait_vm_lgkm0<0>();
        barrier();
        if (ld_t >= 0) issue(ld);
        if (cls & kTileMeets) {
            if constexpr (kSplit == 1) {
                sub(st, 0, cls & kTileSame);
                sub(st, 1, cls & kTileSame);
            } else {
                sub(st, rs, cls & kTileSame);
            }
        }
        take();
    };
    while (t >= 0) {
        stage(s1, s0);
        if (t < 0) break;
        stage(s0, s1);
    }
    wait_vm_lgkm0<0>();
    barrier();  // every wave is done with the stages: they take the outputs
    const auto& z = attn_args<Args>();
    const BwdJob e = bwd_job(z, blockIdx.x);  // (decoded again: not held over the loop)
    const int etile = fdiv(z.div_parts, e.level), epart = e.level - etile * z.parts;
    const int ew = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6), ers = ew / kKb;
    const int ekb = ew & (kKb - 1), ekey = (etile * kKb + ekb) * 32;
    const int eln = opaque_tid() & 63;
    auto store = [&](const f32x4 (&acc)[C::kDB][2], const auto& x, float mul, int which,
                     FA3_LDS char* stg) {
        if (z.parts > 1) {
            const int64_t first = ((int64_t)(2 * epart + which) * z.groups + e.b * z.heads_kv + e.hkv) * z.sk;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int j = ekey + 16 * n + (eln & 15);
                if (j >= z.sk) continue;
                float* p = z.part + (first + j) * D + 4 * (eln >> 4);
#pragma unroll
                for (int i = 0; i < C::kDB; ++i) *(f32x4*)(p + 16 * i) = acc[i][n];
            }
            return;
        }
        const float m2[2] = {mul, mul};
        attn_store<D, kBf16>(acc, m2, z.d, stg, [&](int r) -> _Float16* {
            return ekey + r < z.sk ? x.p + e.b * x.bs + e.hkv * x.hs + (ekey + r) * x.rs : nullptr;
        });
    };
    if constexpr (kSplit == 1) {
        FA3_LDS char* stg = smem + ew * C::kDB * 1024;
        store(av, z.dv, 1.f, 0, stg);
        store(ak, z.dk, z.scale, 1, stg);
    } else {
        // the two waves of a key block swap halves: one sums and writes dV, the other dK
        FA3_LDS char* mine = smem + ew * C::kDB * 2048;
        FA3_LDS char* other = smem + (ekb + kKb * (1 - ers)) * C::kDB * 2048;
        if (ers == 0) reg_put<C::kDB>(mine, ak, eln);
        else reg_put<C::kDB>(mine, av, eln);
        wait_vm_lgkm0<0>();
        barrier();
        if (ers == 0) {
            reg_add<C::kDB>(other, av, eln);
            store(av, z.dv, 1.f, 0, other);
        } else {
            reg_add<C::kDB>(other, ak, eln);
            store(ak, z.dk, z.scale, 1, other);
        }
    }
}

// Row tile `tile` (128 / kSplit rows).  kSplit 2: the two waves of a 32-row
// block take one 32-key half of every stage each.
template <int D, bool kBf16, bool kCap, bool kBias, bool kFine, int kSplit>
__device__ __forceinline__ void attn_dq(int b, int hkv, int tile, FA3_LDS char* smem) {
    typedef AttnBwdArgs Args;
    using C = BwdCfg<D>;
    using R = RegCfg<D>;
    const auto& a = attn_args<Args>();
    const int lane = opaque_tid() & 63;
    const int w = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6);
    const int l16 = lane & 15, g4 = lane >> 4;
    const int kv = attn_kv(a.m, b, a.sk), prefix = attn_prefix(a.m, b), off = kv - a.sq;
    const bool causal = a.m.causal;
    constexpr int kQb = kRegWaves / kSplit;  // 32-row blocks of the job
    const int rs = w / kQb;
    const int row0 = (tile * kQb + (w & (kQb - 1))) * 32;
    const bool any = row0 < a.rows;
    const int last = min(row0 + 32, a.rows) - 1, wg_last = min((tile + 1) * (32 * kQb), a.rows) - 1;
    const int lim_min = any ? attn_limit(fdiv(a.div_group, row0), off, kv, causal, prefix) : 0x7fffffff;
    const int lim_max = any ? attn_limit(fdiv(a.div_group, last), off, kv, causal, prefix) : 0;
    const int wg_max = attn_limit(fdiv(a.div_group, wg_last), off, kv, causal, prefix);

    int lim[2], id[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const AttnRow r = attn_row(row0 + 16 * n + l16, a.rows, hkv, a.group, a.div_group);
        lim[n] = r.ok ? attn_limit(r.i, off, kv, causal, prefix) : 0;
        id[n] = -2;
        if (a.m.doc_q != nullptr && r.ok) id[n] = max(a.m.doc_q[b * a.m.doc_q_bs + r.i], -1);
    }
    DocSpan doc{0, 0, 0, 0, false};
    if (a.m.doc_q != nullptr) doc = doc_span(id, (FA3_LDS int*)(smem + C::kRangeOff), w, lane);

    const _Float16* kp = a.k.p + b * a.k.bs + hkv * a.k.hs;
    const _Float16* vp = a.v.p + b * a.v.bs + hkv * a.v.hs;
    const int* ids = a.m.doc_k == nullptr ? nullptr : a.m.doc_k + b * a.m.doc_k_bs;
    TileWalk walk(ids == nullptr ? nullptr : a.m.range_k + (int64_t)b * a.m.blocks_k, 0,
                  (wg_max + 63) >> 6, doc, 1 << 30);
    auto issue = [&](FA3_LDS char* st, int t) {
        const int j0 = t * 64, ln = opaque_tid() & 63;
        const auto& a = attn_args<Args>();
        if (j0 + 64 <= kv && a.d == D && !(walk.cls & kTileHidden)) {
            attn_load_tile<D>(st, kp, a.k.rs, j0, w, ln);
            attn_load_tile<D>(st + R::kTileBytes, vp, a.v.rs, j0, w, ln);
        } else {
            auto seen = [&](int j) { return ids == nullptr || ids[j] >= 0; };
            attn_load_tile_edge<D>(st, kp, a.k.rs, j0, kv, a.d, w, ln, seen);
            attn_load_tile_edge<D>(st + R::kTileBytes, vp, a.v.rs, j0, kv, a.d, w, ln, seen);
        }
        if (ids != nullptr && w == 0) attn_load_ids(st + C::kIdsOff, ids, j0, a.sk, ln);
    };
    FA3_LDS char* s0 = smem;
    FA3_LDS char* s1 = smem + C::kStageBytes;
    int t = walk.next();
    if (t >= 0) issue(s0, t);
    f16x8 qf[2][C::kKs], df[2][C::kKs];
    float nl[2], slope[2];
    int qp[2];
    f32x4 nd[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const AttnRow r = attn_row(row0 + 16 * n + l16, a.rows, hkv, a.group, a.div_group);
        const int64_t at = ((int64_t)b * a.heads_q + r.h) * a.sqp + r.i;
        nl[n] = r.ok ? a.nlse2[at] : kNegInf;
        const float x = r.ok ? a.ndelta[at] : 0.f;
        nd[n] = f32x4{x, x, x, x};
        const bool ok = nl[n] != kNegInf;
        const _Float16* q = a.q.p + b * a.q.bs + r.h * a.q.hs + r.i * a.q.rs;
        const _Float16* o = a.dout.p + b * a.dout.bs + r.h * a.dout.hs + r.i * a.dout.rs;
#pragma unroll
        for (int s = 0; s < C::kKs; ++s) {
            qf[n][s] = attn_row8(q, p1_chunk<D>(s, g4), a.d, ok);
            df[n][s] = attn_row8(o, p1_chunk<D>(s, g4), a.d, ok);
        }
        qp[n] = 0;
        slope[n] = 0.f;
        if constexpr (kBias) {
            qp[n] = r.i + off;
            slope[n] = a.m.slopes[b * a.m.slopes_bs + r.h] * kLog2e;
        }
    }
    f32x4 acc[C::kDB][2];
#pragma unroll
    for (int i = 0; i < C::kDB; ++i) acc[i][0] = acc[i][1] = f32x4{};
    const RegReader<D> rd0(lane, 0);
    const float c = a.m.c;

    auto sub = [&](const FA3_LDS char* st, int t, int r, bool same) {
        const int j0 = t * 64 + 32 * r;
        if (j0 >= lim_max) return;
        const bool full = j0 + 32 <= lim_min && same;
        uint32_t vis = 0xffff;
        if (!full) {
            const int jl = j0 + 4 * ((opaque_tid() & 63) >> 4);
            vis = 0;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int k = lim[n] - jl;
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    vis |= 16 * (x >> 2) + (x & 3) < k ? 1u << (8 * n + x) : 0u;
            }
            if (ids != nullptr) {
                uint32_t met = 0;
                const FA3_LDS i32x4* kids = (const FA3_LDS i32x4*)(st + C::kIdsOff + 128 * r) +
                                            ((opaque_tid() & 63) >> 4);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const i32x4 x = kids[4 * m];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            met |= doc_of(x[e]) == id[n] ? 1u << (8 * n + 4 * m + e) : 0u;
                }
                vis &= met;
            }
        }
        RegReader<D> rd = rd0;
        rd.opaque();
        f32x4 s[2][2], dp[2][2];  // [m][n]: keys 16 m + 4 g4 + e, rows 16 n + l16
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                s[m][n] = f32x4{};
                dp[m][n] = nd[n];
            }
        reg_scores<D, kBf16, AttnAhead<D, D == 128 ? kCap || kBias : kFine>>(rd, st, st + R::kTileBytes, r, qf, df, s, dp);
        float k1 = 0.f, cap2 = 0.f;
        if constexpr (kCap) {
            const auto& a = attn_args<Args>();
            k1 = a.m.k1;
            cap2 = a.m.cap2;
        }
        float ds[2][8];
        const int ln = opaque_tid() & 63;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float d0 = kBias ? (float)(qp[n] - j0 - 4 * (ln >> 4)) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int m = j >> 2, e = j & 3;
                float p;
                attn_pds<kCap, kBias>(s[m][n][e], dp[m][n][e], nl[n], c, k1, cap2, kFine, slope[n],
                                      d0 - (float)(16 * m + e), bit_mask(vis, 8 * n + j), p, ds[n][j]);
            }
        }
        const f16x8 bs[2] = {pack8<kBf16>(ds[0]), pack8<kBf16>(ds[1])};
        reg_grads<D, kBf16, false, AttnAhead<D, D == 128 ? kCap || kBias : kFine>>(rd, st, st, r, bs, bs, acc, acc);
    };
    auto stage = [&](FA3_LDS char* __restrict__ ld, const FA3_LDS char* __restrict__ st) {
        const int cls = walk.cls, tn = walk.next();
        wait_vm_lgkm0<0>();
        barrier();
        if (tn >= 0) issue(ld, tn);
        if (cls & kTileMeets) {
            if constexpr (kSplit == 1) {
                sub(st, t, 0, cls & kTileSame);
                sub(st, t, 1, cls & kTileSame);
            } else {
                sub(st, t, rs, cls & kTileSame);
            }
        }
        t = tn;
    };
    while (t >= 0) {
        stage(s1, s0);
        if (t < 0) break;
        stage(s0, s1);
    }
    wait_vm_lgkm0<0>();
    barrier();
    const auto& z = attn_args<Args>();
    const BwdJob e = bwd_job(z, blockIdx.x);
    const int ew = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6), ers = ew / kQb;
    const int eqb = ew & (kQb - 1), eln = opaque_tid() & 63;
    const int erow = (dq_tile(z, e.level) * kQb + eqb) * 32;
    const float sc[2] = {z.scale, z.scale};
    FA3_LDS char* stg = smem + ew * C::kDB * 1024;
    if constexpr (kSplit == 2) {
        // the second wave's sums go to the first, which writes
        FA3_LDS char* slot = smem + eqb * C::kDB * 2048;
        stg = slot;
        if (ers == 1) reg_put<C::kDB>(slot, acc, eln);
        wait_vm_lgkm0<0>();
        barrier();
        if (ers == 1) return;
        reg_add<C::kDB>(slot, acc, eln);
    }
    // (a row that sees no key: zeros, but zeros that may have met a NaN of
    // other rows' keys)
#pragma unroll
    for (int n = 0; n < 2; ++n)
        if (nl[n] == kNegInf) {
#pragma unroll
            for (int i = 0; i < C::kDB; ++i) acc[i][n] = f32x4{};
        }
    attn_store<D, kBf16>(acc, sc, z.d, stg, [&](int r) -> _Float16* {
        const AttnRow x = attn_row(erow + r, z.rows, e.hkv, z.group, z.div_group);
        return x.ok ? z.dq.p + e.b * z.dq.bs + x.h * z.dq.hs + x.i * z.dq.rs : nullptr;
    });
}

// kCap: 0 none, 1 capped, 2 capped with tanh's series for small scores.
// kSplit: jobs of 128 / kSplit keys or rows.
template <int D, bool kBf16, int kCap, bool kBias, int kSplit>
__global__ __launch_bounds__(kRegThreads, D == 64 ? 3 : 2) void attn_bwd_kernel(AttnBwdArgs) {
    __shared__ __attribute__((aligned(1024))) char smem_raw[BwdCfg<D>::kBytes];
    FA3_LDS char* smem = (FA3_LDS char*)smem_raw;
    const auto& a = attn_args<AttnBwdArgs>();
    const BwdJob j = bwd_job(a, blockIdx.x);
    const int n = a.kv_tiles * a.parts;
    if (j.level < n)
        attn_dkv<D, kBf16, kCap != 0, kBias, kCap == 2, kSplit>(j.b, j.hkv, j.level, smem);
    else
        attn_dq<D, kBf16, kCap != 0, kBias, kCap == 2, kSplit>(j.b, j.hkv, dq_tile(a, j.level), smem);
}

// dV and dK from their parts, added in order; 8 columns a thread.
template <int D, bool kBf16>
__global__ __launch_bounds__(256) void attn_sum_kernel(AttnBwdArgs a) {
    constexpr int kLanes = D / 8;
    const int64_t rows = (int64_t)a.groups * a.sk;
    const int64_t r = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    const int which = blockIdx.y, col = (threadIdx.x % kLanes) * 8;
    if (r >= rows || col >= a.d) return;
    float x[8] = {};
    for (int p = 0; p < a.parts; ++p) {
        const float* y = a.part + ((int64_t)(2 * p + which) * rows + r) * D + col;
        const f32x4 lo = *(const f32x4*)y, hi = *(const f32x4*)(y + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] += lo[e];
            x[4 + e] += hi[e];
        }
    }
    const int grp = (int)(r / a.sk), j = (int)(r - (int64_t)grp * a.sk);
    const int b = fdiv(a.div_hkv, grp), hkv = grp - b * a.heads_kv;
    const AttnView& o = which ? a.dk : a.dv;
    const float mul = which ? a.scale : 1.f;
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to16<kBf16>(x[e] * mul);
    *(f16x8*)(o.p + b * o.bs + hkv * o.hs + j * o.rs + col) = v;
}

// The kernels of one call: delta, the jobs, and the parts' sum.
template <int D, bool kBf16>
void launch_bwd(const AttnBwdArgs& x, const AttnBwdPlan& f, int cap, bool bias, hipStream_t stream) {
    const int blocks = x.delta_blocks + ceil_div(x.q_blocks, 4) + ceil_div(x.k_blocks, 4);
    if (blocks > 0)
        hipLaunchKernelGGL((attn_delta_kernel<D, kBf16>), dim3(blocks), dim3(256), 0, stream, x);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(f.jobs), dim3(kRegThreads), 0, stream, x);
    };
    auto splits = [&](auto bi, auto split) {
        constexpr bool kBi = decltype(bi)::value;
        constexpr int kS = decltype(split)::value;
        if (cap == 2) go(attn_bwd_kernel<D, kBf16, 2, kBi, kS>);
        else if (cap == 1) go(attn_bwd_kernel<D, kBf16, 1, kBi, kS>);
        else go(attn_bwd_kernel<D, kBf16, 0, kBi, kS>);
    };
    auto biases = [&](auto bi) {
        f.split == 2 ? splits(bi, std::integral_constant<int, 2>{})
                     : splits(bi, std::integral_constant<int, 1>{});
    };
    bias ? biases(std::true_type{}) : biases(std::false_type{});
    if (x.parts > 1 && x.sk > 0)
        hipLaunchKernelGGL((attn_sum_kernel<D, kBf16>),
                           dim3(ceil_div((int64_t)x.groups * x.sk, 2048 / D), 2), dim3(256), 0,
                           stream, x);
}

}  // namespace
}  // namespace fa3
