// Forward attention with capped, biased and masked scores.
//
// One workgroup of four waves owns 128 rows of a KV head (a row is a query of
// one of its query heads) and walks the 64-key tiles that any of them sees,
// in one pass with the running maximum and sum of a softmax.  A wave owns 32
// rows: S^T = K Q^T with Q resident in registers as the B operand, the
// softmax down each lane's column, and O^T += V^T P^T, whose B operand is P
// as the score product left it, rounded (fa3_bwd_reg_kernel.h says why that
// needs no exchange).  K and V tiles go through two LDS stages.
#include "fa3_attn_device.h"

namespace fa3 {
namespace {

struct AttnFwdArgs {
    AttnView q, k, v, out;
    float* lse;
    float* part_o;  // splits > 1: [splits][groups * rows][D] fp32
    float* part_l;  //             [splits][groups * rows]
    AttnMask m;
    int heads_q, heads_kv, group, sq, sk, d;
    int rows;  // group * sq
    int tiles, splits, part, groups;
    uint32_t flip;  // XORed into Q's 16-bit pairs
    int scored;     // 0: a scale of zero, Q is taken as zeros
    FastDiv div_hkv, div_group, div_groups, div_gpart, div_splits;
};

template <int D>
struct FwdCfg {
    static constexpr int kTileBytes = 64 * D * 2;
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kRangeOff = 2 * kStageBytes;  // the waves' document ranges
    static constexpr int kBytes = kRangeOff + 64;
    static constexpr int kKs = D / 32, kDB = D / 16;
};

template <int D, bool kBf16, bool kCap, bool kBias>
__global__ __launch_bounds__(kRegThreads, D == 64 ? 3 : 2) void attn_fwd_kernel(AttnFwdArgs) {
    typedef AttnFwdArgs Args;
    const auto& a = attn_args<Args>();
    using C = FwdCfg<D>;
    __shared__ __attribute__((aligned(1024))) char smem_raw[C::kBytes];
    FA3_LDS char* smem = (FA3_LDS char*)smem_raw;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g4 = lane >> 4;

    int level, grp;
    attn_job(blockIdx.x, a.groups, a.div_groups, a.div_gpart, level, grp);
    const int b = fdiv(a.div_hkv, grp), hkv = grp - b * a.heads_kv;
    const int tl = fdiv(a.div_splits, level);
    const int split = level - tl * a.splits, tile = a.tiles - 1 - tl;
    const int kv = attn_kv(a.m, b, a.sk), prefix = attn_prefix(a.m, b), off = kv - a.sq;

    // this wave's rows, and what they see
    const int row0 = tile * kAttnRows + 32 * w;
    const bool any = row0 < a.rows;
    const int last = min(row0 + 32, a.rows) - 1, wg_last = min((tile + 1) * kAttnRows, a.rows) - 1;
    const int lim_min = any ? attn_limit(fdiv(a.div_group, row0), off, kv, a.m.causal, prefix) : 0x7fffffff;
    const int lim_max = any ? attn_limit(fdiv(a.div_group, last), off, kv, a.m.causal, prefix) : 0;
    const int wg_max = attn_limit(fdiv(a.div_group, wg_last), off, kv, a.m.causal, prefix);
    f16x8 qf[2][C::kKs];
    int lim[2], id[2];
    float qp[2], slope[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const AttnRow r = attn_row(row0 + 16 * n + l16, a.rows, hkv, a.group, a.div_group);
        id[n] = -2;
        // (documents: -1 for every negative one, -2 for rows that are not there)
        if (a.m.doc_q != nullptr && r.ok) id[n] = max(a.m.doc_q[b * a.m.doc_q_bs + r.i], -1);
        const bool ok = r.ok && a.scored && id[n] != -1;
        const _Float16* q = a.q.p + b * a.q.bs + r.h * a.q.hs + r.i * a.q.rs;
#pragma unroll
        for (int s = 0; s < C::kKs; ++s) {
            // (a scale below zero turns Q's signs)
            qf[n][s] = attn_flip(attn_row8(q, p1_chunk<D>(s, g4), a.d, ok), a.flip);
        }
        lim[n] = r.ok ? attn_limit(r.i, off, kv, a.m.causal, prefix) : 0;
        qp[n] = 0.f;
        slope[n] = 0.f;
        if constexpr (kBias) {
            qp[n] = (float)(r.i + off);
            slope[n] = a.m.slopes[b * a.m.slopes_bs + r.h] * kLog2e;
        }
    }
    DocSpan doc{0, 0, 0, 0, false};
    if (a.m.doc_q != nullptr) doc = doc_span(id, (FA3_LDS int*)(smem + C::kRangeOff), w, lane);

    const _Float16* kp = a.k.p + b * a.k.bs + hkv * a.k.hs;
    const _Float16* vp = a.v.p + b * a.v.bs + hkv * a.v.hs;
    const int* ids = a.m.doc_k == nullptr ? nullptr : a.m.doc_k + b * a.m.doc_k_bs;
    const int begin = split * a.part;
    TileWalk walk(ids == nullptr ? nullptr : a.m.range_k + (int64_t)b * a.m.blocks_k, begin,
                  min(begin + a.part, (wg_max + 63) >> 6), doc);
    auto issue = [&](FA3_LDS char* st, int t) {
        const int j0 = t * 64, lane = opaque_tid() & 63;
        const auto& a = attn_args<Args>();
        if (j0 + 64 <= kv && a.d == D && !(walk.cls & kTileHidden)) {
            attn_load_tile<D>(st, kp, a.k.rs, j0, w, lane);
            attn_load_tile<D>(st + C::kTileBytes, vp, a.v.rs, j0, w, lane);
        } else {
            auto seen = [&](int j) { return ids == nullptr || ids[j] >= 0; };
            attn_load_tile_edge<D>(st, kp, a.k.rs, j0, kv, a.d, w, lane, seen);
            attn_load_tile_edge<D>(st + C::kTileBytes, vp, a.v.rs, j0, kv, a.d, w, lane, seen);
        }
    };

    f32x4 o[C::kDB][2];
#pragma unroll
    for (int i = 0; i < C::kDB; ++i) o[i][0] = o[i][1] = f32x4{};
    float mx[2] = {kNegInf, kNegInf}, sum[2] = {0.f, 0.f};
    const RegReader<D> rd0(lane, 0);
    constexpr bool kLog2 = kCap || kBias;  // scores leave their product in the log2 domain
    const float c = a.m.c;

    auto compute = [&](const FA3_LDS char* st, int t, int cls) {
        const int j0 = t * 64;
        if (j0 >= lim_max) return;
        if (!(cls & kTileMeets)) return;
        const bool full = j0 + 64 <= lim_min && (cls & kTileSame);
        RegReader<D> rd = rd0;
        rd.opaque();
        f32x4 s[4][2];  // [m][n]: keys 16 m + 4 g4 + e, rows 16 n + l16
#pragma unroll
        for (int m = 0; m < 4; ++m) s[m][0] = s[m][1] = f32x4{};
        // (the bias-free, cap-free score is masked in its product's seed: its
        // scale is positive, and nothing that can be masked is infinite)
        auto mask = [&]() {
            const int ln = opaque_tid() & 63;
            const int jl = j0 + 4 * (ln >> 4);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int k = lim[n] - jl;
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[m][n][e] = 16 * m + e < k ? s[m][n][e] : kNegInf;
            }
            if (ids != nullptr) {
                const int sk = attn_args<Args>().sk;
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int kid = doc_of(ids[min(jl + 16 * m + e, sk - 1)]);
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            s[m][n][e] = kid == id[n] ? s[m][n][e] : kNegInf;
                    }
            }
        };
        if (!kLog2 && !full) mask();
        attn_scores<D, kBf16, 4, 4>(rd, st, 0, qf, s);
        if constexpr (kCap) {
            const auto& a = attn_args<Args>();
            const float k1 = a.m.k1, cap2 = a.m.cap2;
            if (a.m.cap_fine) {
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[m][n][e] = attn_tanh_fine(s[m][n][e], k1) * cap2;
            } else {
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[m][n][e] = attn_tanh(s[m][n][e], k1) * cap2;
            }
        }
        if constexpr (kBias) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float d0 = qp[n] - (float)(j0 + 4 * g4);
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = kCap ? s[m][n][e] : s[m][n][e] * c;
                        s[m][n][e] = __builtin_fmaf(-slope[n], __builtin_fabsf(d0 - (float)(16 * m + e)), x);
                    }
            }
        }
        if (kLog2 && !full) mask();
        float mu[2];
        bool up = false;
        float mn[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float x = mx[n];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) x = __builtin_fmaxf(x, s[m][n][e]);
            mn[n] = max_groups(x);
            up |= mn[n] > mx[n];
            mu[n] = mn[n] == kNegInf ? 0.f : mn[n];
            if (!kLog2) mu[n] *= c;
        }
        if (__ballot(up)) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                // (mx -inf: exp2(-inf) = 0; both -inf: mu 0, the same)
                const float f = fast_exp2(kLog2 ? mx[n] - mu[n] : __builtin_fmaf(mx[n], c, -mu[n]));
                mx[n] = mn[n];
                sum[n] *= f;
#pragma unroll
                for (int i = 0; i < C::kDB; ++i) o[i][n] *= f;
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            f16x8 bp[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = s[2 * r + (j >> 2)][n][j & 3];
                    p[j] = fast_exp2(kLog2 ? x - mu[n] : __builtin_fmaf(x, c, -mu[n]));
                    sum[n] += p[j];
                }
                bp[n] = pack8<kBf16>(p);
            }
            reg_grads<D, kBf16, false>(rd, st + C::kTileBytes, st + C::kTileBytes, r, bp, bp, o, o);
        }
    };

    FA3_LDS char* s0 = smem;
    FA3_LDS char* s1 = smem + C::kStageBytes;
    int t = walk.next();
    if (t >= 0) issue(s0, t);
    auto stage = [&](FA3_LDS char* __restrict__ ld, const FA3_LDS char* __restrict__ st) {
        const int cls = walk.cls;
        wait_vm_lgkm0<0>();
        barrier();
        const int tn = walk.next();
        if (tn >= 0) issue(ld, tn);
        compute(st, t, cls);
        t = tn;
    };
    while (t >= 0) {
        stage(s1, s0);
        if (t < 0) break;
        stage(s0, s1);
    }

    const auto& z = attn_args<Args>();
    float inv[2], lse2[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const float l = sum_groups(sum[n]);
        const bool none = mx[n] == kNegInf;
        inv[n] = none ? 0.f : 1.f / l;
        if (none) {  // (its Q may have been NaN)
#pragma unroll
            for (int i = 0; i < C::kDB; ++i) o[i][n] = f32x4{};
        }
        lse2[n] = none ? kNegInf : (kLog2 ? mx[n] : mx[n] * c) + __builtin_amdgcn_logf(l);
    }
    if (z.splits > 1) {
        const int64_t base = ((int64_t)split * z.groups + grp) * z.rows;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int r = row0 + 16 * n + l16;
            if (r >= z.rows) continue;
            if (g4 == 0) z.part_l[base + r] = lse2[n];
            float* p = z.part_o + (base + r) * D + 4 * g4;
#pragma unroll
            for (int i = 0; i < C::kDB; ++i) *(f32x4*)(p + 16 * i) = o[i][n] * inv[n];
        }
        return;
    }
    wait_vm_lgkm0<0>();
    barrier();  // every wave is done with the stages: they take the outputs
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const AttnRow r = attn_row(row0 + 16 * n + l16, z.rows, hkv, z.group, z.div_group);
        if (g4 == 0 && r.ok)
            z.lse[((int64_t)b * z.heads_q + r.h) * z.sq + r.i] = lse2[n] * 0.69314718055994531f;
    }
    attn_store<D, kBf16>(o, inv, z.d, smem + w * C::kDB * 1024, [&](int r) -> _Float16* {
        const AttnRow x = attn_row(row0 + r, z.rows, hkv, z.group, z.div_group);
        return x.ok ? z.out.p + b * z.out.bs + x.h * z.out.hs + x.i * z.out.rs : nullptr;
    });
}

// Joins the parts of a split key axis: with w_s = exp2(l_s - max l), out =
// sum w_s o_s / sum w_s.  16 lanes (D 128; 8 for D 64) take a row, 8 columns
// each; bound by reading the parts.
template <int D, bool kBf16>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnFwdArgs a) {
    constexpr int kLanes = D / 8;
    const int64_t total = (int64_t)a.groups * a.rows;
    const int64_t rg = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    const int col = (threadIdx.x % kLanes) * 8;
    if (rg >= total) return;
    float top = kNegInf;
    for (int s = 0; s < a.splits; ++s) top = __builtin_fmaxf(top, a.part_l[s * total + rg]);
    float z = 0.f, acc[8] = {};
    for (int s = 0; s < a.splits; ++s) {
        const float l = a.part_l[s * total + rg];
        if (l == kNegInf) continue;  // (nothing seen there)
        const float f = fast_exp2(l - top);
        z += f;
        const float* p = a.part_o + (s * total + rg) * D + col;
        const f32x4 x = *(const f32x4*)p, y = *(const f32x4*)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[e] = __builtin_fmaf(f, x[e], acc[e]);
            acc[4 + e] = __builtin_fmaf(f, y[e], acc[4 + e]);
        }
    }
    const int grp = (int)(rg / a.rows), r = (int)(rg - (int64_t)grp * a.rows);
    const int b = fdiv(a.div_hkv, grp), hkv = grp - b * a.heads_kv;
    const AttnRow x = attn_row(r, a.rows, hkv, a.group, a.div_group);
    const float inv = z > 0.f ? 1.f / z : 0.f;
    if (col == 0)
        a.lse[((int64_t)b * a.heads_q + x.h) * a.sq + x.i] =
            z > 0.f ? (top + __builtin_amdgcn_logf(z)) * 0.69314718055994531f : kNegInf;
    if (col >= a.d) return;
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to16<kBf16>(acc[e] * inv);
    *(f16x8*)(a.out.p + b * a.out.bs + x.h * a.out.hs + x.i * a.out.rs + col) = v;
}

// One wave per 64 positions.
__global__ __launch_bounds__(256) void attn_ranges_kernel(const int* ids, int64_t bs, int n,
                                                          int blocks, int total, AttnRange* out) {
    const int x = blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (x >= total) return;
    const int b = x / blocks, t = x - b * blocks, i = t * 64 + lane;
    const int id = i < n ? ids[b * bs + i] : -1;
    int lo = id >= 0 ? id : 0x7fffffff, hi = id >= 0 ? id : -1;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    if (__ballot(id < 0)) lo = ~lo;
    if (lane == 0) out[x] = AttnRange{lo, hi};
}

AttnView view(const ShaoboFa3AttnTensor& t) {
    return AttnView{(_Float16*)t.data, t.batch_stride, t.head_stride, t.row_stride};
}

}  // namespace

hipError_t launch_attn_ranges(const int* ids, int64_t bs, int batch, int n, AttnRange* out,
                              hipStream_t stream) {
    const int blocks = ceil_div(n, 64), total = batch * blocks;
    if (total > 0)
        hipLaunchKernelGGL(attn_ranges_kernel, dim3(ceil_div(total, 4)), dim3(256), 0, stream, ids,
                           bs, n, blocks, total, out);
    return hipGetLastError();
}

AttnFwdPlan plan_attn_fwd(const AttnProblem& p) {
    AttnFwdPlan f{};
    const int64_t rows = (int64_t)p.group * p.sq, groups = (int64_t)p.batch * p.heads_kv;
    const int D = p.d > 64 ? 128 : 64;
    f.tiles = ceil_div(rows, kAttnRows);
    const int n_t = ceil_div(p.sk, 64);
    f.splits = 1;
    f.part = n_t;
    const int64_t jobs = groups * f.tiles;
    // Fewer workgroups than two per CU: the key axis is cut, into parts of at
    // least four tiles.
    if (jobs > 0 && jobs < 512 && n_t >= 8) {
        const int want = (int)(512 / jobs), most = n_t / 4;
        const int s = want < most ? want : most;
        if (s > 1) {
            f.part = ceil_div(n_t, s);
            f.splits = ceil_div(n_t, f.part);
        }
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
    f.ok = rows < (1ll << 30) && jobs * f.splits < (1ll << 30);
    f.jobs = f.ok ? (int)(jobs * f.splits) : 0;
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
    const bool cap = p.softcap > 0.f, bias = p.bias;
    // The running maximum is taken over raw products where nothing else
    // enters the score: its scale must be positive.
    x.scored = 1;
    if (!cap && !bias) {
        if (m.c < 0.f) x.flip = 0x80008000u;
        x.scored = m.c != 0.f;
        m.c = m.c == 0.f ? 1.f : m.c < 0.f ? -m.c : m.c;
    }
    if (f.jobs == 0) return hipSuccess;
    if (p.docs && p.sk > 0) {
        AttnRange* r = (AttnRange*)(ws + f.range_off);
        const hipError_t e = launch_attn_ranges(m.doc_k, m.doc_k_bs, p.batch, p.sk, r, stream);
        if (e != hipSuccess) return e;
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
        if (cap) bias ? go(attn_fwd_kernel<kD, kB, true, true>) : go(attn_fwd_kernel<kD, kB, true, false>);
        else bias ? go(attn_fwd_kernel<kD, kB, false, true>) : go(attn_fwd_kernel<kD, kB, false, false>);
        if (f.splits > 1)
            hipLaunchKernelGGL((attn_join_kernel<kD, kB>),
                               dim3(ceil_div((int64_t)x.groups * x.rows, 2048 / kD)), dim3(256), 0,
                               stream, x);
    };
    using T = std::true_type;
    using F = std::false_type;
    if (p.d > 64) p.bf16 ? pick(std::integral_constant<int, 128>{}, T{}) : pick(std::integral_constant<int, 128>{}, F{});
    else p.bf16 ? pick(std::integral_constant<int, 64>{}, T{}) : pick(std::integral_constant<int, 64>{}, F{});
    return hipGetLastError();
}

}  // namespace fa3
