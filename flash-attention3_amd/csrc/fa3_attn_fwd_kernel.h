// Rows of a forward workgroup and what its launches share: the running softmax
// of a wave's 32 rows over LDS tiles of keys and values, the jobs, and the kernel
// that joins the parts of a split key axis.
#pragma once

#include "fa3_attn_device.h"

namespace fa3 {
namespace {

// (a cache's: fa3_cache_attn_kernel.h)
template <typename A>
__device__ __forceinline__ bool cache_sees(const A& z, int row, int b, int hkv, int g4);

template <int D>
struct FwdCfg {
    static constexpr int kTileBytes = 64 * D * 2;
    static constexpr int kStageBytes = 2 * kTileBytes + 256;  // K, V, the keys' documents
    static constexpr int kRangeOff = 2 * kStageBytes;  // the waves' document ranges
    static constexpr int kBytes = kRangeOff + 64;
    static constexpr int kKs = D / 32, kDB = D / 16;
};

// The rest of 8 values that their bf16 parts leave.
__device__ __forceinline__ f16x8 pack8_rest(const float* x, const f16x8& hi) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] - (float)__builtin_bit_cast(__bf16, (_Float16)hi[i]);
    return pack8<true>(y);
}

// g[db][n] += X^T (B + C) over the 32 streamed rows 32 r .., bf16: reg_grads
// with two terms for an operand.
template <int D>
__device__ __forceinline__ void two_terms(const RegReader<D>& rd, const FA3_LDS char* x, int r,
                                          const f16x8 (&b)[2], const f16x8 (&c)[2],
                                          f32x4 (&g)[D / 16][2]) {
    constexpr int kN = D / 16, kA = 2;
    f16x8 f[kN];
#pragma unroll
    for (int i = 0; i < kA; ++i) f[i] = rd.tr(x, r, i);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        wall();
        if (i + kA < kN) f[i + kA] = rd.tr(x, r, i + kA);
        wall();
#pragma unroll
        for (int n = 0; n < 2; ++n) g[i][n] = mfma_16x16x32<true>(f[i], b[n], g[i][n]);
#pragma unroll
        for (int n = 0; n < 2; ++n) g[i][n] = mfma_16x16x32<true>(f[i], c[n], g[i][n]);
    }
    wall();
}

// A wave's 32 rows: what they see, and their running softmax and output.
//
// The vector units bound the tile loop, so an element's score stays as it
// leaves its products as long as it can: the log2-domain score is
//   x = al raw + be[n],  al > 0
// with al, be the tile's -- raw the dot product (al = c), with a distance bias
// linear over the tile the product seeded by the bias's slope (be its value
// at the tile's first key), capped -1 / (exp(2 s / softcap) + 1) (al = 2 cap2,
// be = cap2).  Maxima are taken over raw, and p = exp2(al raw + (be - mx)) is
// one fma and the exponential.
//
// mx need not be the maximum: sums and outputs are rescaled only where a
// tile's maximum exceeds it by 2^kLazy, so p and the sums stay below 2^8 times
// their usual size, far inside fp16's and fp32's ranges.  With the exact
// maximum some row of the 32 rescales all of them in nearly every early tile.
//
// kFour: K's and V's tiles hold the levels of 4-bit rows, K's in Q's type and
// V's in bf16, and step() takes the rows' scales; a score is scaled and then
// masked, where others are masked in their product's seed (a scale of zero
// would make a NaN of it), and P is scaled before it is rounded, to bf16, whose
// range is fp32's (p is up to 2^kLazy, a scale a sixth of a row's largest value:
// finite up to values of 2^120); for fp16 rows to two bf16 terms, 16 bits of it,
// and two products.
template <int D, bool kBf16, bool kCap, bool kBias, typename Args_ = AttnFwdArgs, bool kFour = false>
struct FwdRows {
    typedef Args_ Args;
    static constexpr int kKs = D / 32, kDB = D / 16;
    static constexpr float kLazy = 8.f;
    // A tile whose every p is below 2^-64 of its row's largest is left: 2^30
    // keys of them, the longest axis, add less than 2^-34, fp32's half step
    // being 2^-25.  (Looked for only with a distance bias, which makes them.)
    static constexpr float kNone = 64.f;
    // A bias's seed is off by fp32's rounding of the slope over a whole tile,
    // also for the keys next to the row whose own bias is small: 64 slope e, a
    // few times over, is under 2e-5 of a score up to here.
    static constexpr float kGentle = 1.5f;
    f16x8 qf[2][kKs];
    int lim[2], id[2];
    int qp[2];  // the rows' places among the keys
    float slope[2];
    bool gentle;  // no slope of the wave over kGentle
    f32x4 o[kDB][2];  // columns 16 db + 4 g4 + e of rows 16 n + l16
    float mx[2], sum[2];
    int lim_min, lim_max;  // over the rows
    float k1, cap2;        // capped
    bool fine;
    int q_first, q_last;   // places of the first and last row among the keys

    // Rows row0 .. row0 + 31 of KV head hkv in batch entry b, of which those
    // at `rows` and behind see nothing and those at `end` are none.
    template <typename A>
    __device__ __forceinline__ void init(const A& a, int row0, int rows, int end, int b, int hkv,
                                         int kv, int prefix, int off, int lane) {
        const int l16 = lane & 15;
        const bool any = row0 < rows;
        const int first = fdiv(a.div_group, any ? row0 : 0);
        const int last = fdiv(a.div_group, any ? min(row0 + 32, rows) - 1 : 0);
        lim_min = any ? attn_limit(first, off, kv, a.m.causal, prefix) : 0x7fffffff;
        if (Args::kPaged && any && min(row0 + 32, end) > rows) lim_min = 0;
        lim_max = any ? attn_limit(last, off, kv, a.m.causal, prefix) : 0;
        k1 = kCap ? a.m.k1 : 0.f;
        cap2 = kCap ? a.m.cap2 : 0.f;
        fine = kCap && a.m.cap_fine;
        q_first = first + off;
        q_last = last + off;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const AttnRow r = attn_row(row0 + 16 * n + l16, rows, hkv, a.group, a.div_group);
            lim[n] = r.ok ? attn_limit(r.i, off, kv, a.m.causal, prefix) : 0;
            id[n] = -2;
            // (documents: -1 for every negative one, -2 for rows that are not there)
            if (a.m.doc_q != nullptr && r.ok) id[n] = max(a.m.doc_q[b * a.m.doc_q_bs + r.i], -1);
        }
    }
    // Their Q, after the first tile's loads have gone out.
    template <typename A>
    __device__ __forceinline__ void load(const A& a, int row0, int rows, int b, int hkv, int off,
                                         int lane) {
        const int l16 = lane & 15, g4 = lane >> 4;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const AttnRow r = attn_row(row0 + 16 * n + l16, rows, hkv, a.group, a.div_group);
            const bool ok = r.ok && a.scored && id[n] != -1;
            const _Float16* q = a.q.p + b * a.q.bs + r.h * a.q.hs + r.i * a.q.rs;
#pragma unroll
            for (int s = 0; s < kKs; ++s)  // (a scale below zero turns Q's signs)
                qf[n][s] = attn_flip(attn_row8(q, p1_chunk<D>(s, g4), a.d, ok), a.flip);
            qp[n] = 0;
            slope[n] = 0.f;
            if constexpr (kBias) {
                qp[n] = r.i + off;
                slope[n] = a.m.slopes[b * a.m.slopes_bs + r.h] * kLog2e;
            }
            mx[n] = kNegInf;
            sum[n] = 0.f;
        }
        gentle = !kBias || __ballot(!(__builtin_fabsf(slope[0]) <= kGentle &&
                                      __builtin_fabsf(slope[1]) <= kGentle)) == 0;
#pragma unroll
        for (int i = 0; i < kDB; ++i) o[i][0] = o[i][1] = f32x4{};
    }

    // Keys j0 .. j0 + 16 M - 1, which are rows 16 m0 .. of the tiles tk and tv.
    // ids: their documents in LDS, or null where all rows are of theirs.  kFour:
    // their scales, K's and 256 bytes behind them V's.
    template <int M>
    __device__ __forceinline__ void step(const RegReader<D>& rd0, const FA3_LDS char* tk,
                                         const FA3_LDS char* tv, int m0, int j0,
                                         const FA3_LDS char* ids, float c,
                                         const FA3_LDS char* scales = nullptr) {
        RegReader<D> rd = rd0;
        rd.opaque();
        const bool limited = j0 + 16 * M > lim_min;
        f32x4 s[M][2];  // [m][n]: keys 16 m + 4 g4 + e, rows 16 n + l16
        float al = c, be[2] = {0.f, 0.f};
        bool linear = false;  // every row of the wave on one side of every key
        if constexpr (kBias && !kCap && !kFour) {
            const bool past = q_first >= j0 + 16 * M - 1;
            linear = (past || q_last <= j0) && gentle && c > 1e-30f;
            const int j = j0 + 4 * ((opaque_tid() & 63) >> 4);
            const float inv = linear ? __builtin_amdgcn_rcpf(past ? c : -c) : 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float seed = slope[n] * inv;
                if (linear) be[n] = -slope[n] * __builtin_fabsf((float)(qp[n] - j));
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[m][n][e] = seed * (float)(16 * m + e);
            }
        } else {
#pragma unroll
            for (int m = 0; m < M; ++m) s[m][0] = s[m][1] = f32x4{};
        }
        // (a score without a cap is masked in its product's seed: al is
        // positive, and nothing that can be masked is infinite)
        auto mask = [&]() {
            const int ln = opaque_tid() & 63;
            if (limited) {
                const int jl = j0 + 4 * (ln >> 4);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int k = lim[n] - jl;
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[m][n][e] = 16 * m + e < k ? s[m][n][e] : kNegInf;
                }
            }
            if (ids != nullptr) {
                const FA3_LDS i32x4* kids = (const FA3_LDS i32x4*)ids + (ln >> 4);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    const i32x4 kid = kids[4 * m];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            s[m][n][e] = doc_of(kid[e]) == id[n] ? s[m][n][e] : kNegInf;
                }
            }
        };
        if (!kFour && !kCap && !(kBias && !linear)) mask();
        attn_scores<D, kBf16, M, 4>(rd, tk, m0, qf, s);
        if constexpr (kFour) {
            const FA3_LDS f32x4* ks = (const FA3_LDS f32x4*)scales + ((opaque_tid() & 63) >> 4);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const f32x4 k = ks[4 * m];
                s[m][0] *= k;
                s[m][1] *= k;
            }
        }
        if constexpr (kCap) {
            if (fine) {
                al = 1.f;
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[m][n][e] = attn_tanh_fine(s[m][n][e], k1) * cap2;
            } else {
                al = 2.f * cap2;
                be[0] = be[1] = cap2;
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[m][n][e] = __builtin_amdgcn_rcpf(-1.f - fast_exp2(s[m][n][e] * k1));
            }
        }
        if constexpr (kBias) {
            if (!linear) {
                const int j = j0 + 4 * ((opaque_tid() & 63) >> 4);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    // (exact: a difference of places, then fp32)
                    const float d0 = (float)(qp[n] - j), b0 = be[n];
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[m][n][e] = __builtin_fmaf(-slope[n], __builtin_fabsf(d0 - (float)(16 * m + e)),
                                                        __builtin_fmaf(s[m][n][e], al, b0));
                    be[n] = 0.f;
                }
                al = 1.f;
            }
        }
        if (kFour || kCap || (kBias && !linear)) mask();
        float top[2];
        bool up = false, some = false;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float x = s[0][n][0];
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e)  // (v_maximum3: no canonicalising before it)
                    x = __builtin_elementwise_maximum(x, s[m][n][e]);
            top[n] = max_groups(__builtin_fmaf(al, x, be[n]));
            up |= top[n] > mx[n] + kLazy;
            some |= !(top[n] <= mx[n] - kNone);  // (NaN is some)
        }
        if (kBias && !__ballot(some)) return;
        if (__ballot(up)) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float m = __builtin_fmaxf(mx[n], top[n]);
                // (mx -inf: nothing seen before, 0 times its zeros)
                const float f = mx[n] == kNegInf ? 0.f : fast_exp2(mx[n] - m);
                mx[n] = m;
                sum[n] *= f;
#pragma unroll
                for (int i = 0; i < kDB; ++i) o[i][n] *= f;
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) be[n] -= mx[n] == kNegInf ? 0.f : mx[n];
#pragma unroll
        for (int r = 0; r < M / 2; ++r) {
            f16x8 bp[2], rest[2];
            f32x4 vs[2];
            if constexpr (kFour) {
                const FA3_LDS f32x4* x =
                    (const FA3_LDS f32x4*)(scales + 256) + ((opaque_tid() & 63) >> 4);
                vs[0] = x[8 * r];
                vs[1] = x[8 * r + 4];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = fast_exp2(__builtin_fmaf(s[2 * r + (j >> 2)][n][j & 3], al, be[n]));
                    sum[n] += p[j];
                    if constexpr (kFour) p[j] *= vs[j >> 2][j & 3];
                }
                bp[n] = pack8<kBf16 || kFour>(p);
                if constexpr (kFour && !kBf16) rest[n] = pack8_rest(p, bp[n]);
            }
            if constexpr (kFour && !kBf16) two_terms<D>(rd, tv, m0 / 2 + r, bp, rest, o);
            else reg_grads<D, kBf16, false>(rd, tv, tv, m0 / 2 + r, bp, bp, o, o);
        }
    }

    // Whether row `row` of KV head hkv sees any key at all: lane g4 of its four
    // looks at every fourth, last first (with causality its own document is
    // there).  What init() read is read again: not held over the tile loop.
    template <bool kDocs, typename A>
    static __device__ __forceinline__ bool sees(const A& z, int row, int b, int hkv, int g4) {
        if constexpr (Args::kPaged) return cache_sees(z, row, b, hkv, g4);
        const AttnRow r = attn_row(row, z.rows, hkv, z.group, z.div_group);
        const int kv = attn_kv(z.m, b, z.sk);
        const int lim = r.ok ? attn_limit(r.i, kv - z.sq, kv, z.m.causal, attn_prefix(z.m, b)) : 0;
        bool any = lim > 0;
        if (kDocs && any && z.m.doc_k != nullptr) {
            const int* ids = z.m.doc_k + b * z.m.doc_k_bs;
            const int id = max(z.m.doc_q[b * z.m.doc_q_bs + r.i], -1);
            any = false;
#pragma unroll 1
            for (int j = lim - 1 - g4; j >= 0 && !any; j -= 4) any = doc_of(ids[j]) == id;
        }
        return max_groups(any ? 1.f : 0.f) > 0.f;
    }

    // After the last tile.  A row without a maximum but with a sum has met NaN:
    // in what it sees, or it sees nothing and its Q or other rows' keys held
    // it, which counts for nothing.
    template <bool kDocs>
    __device__ __forceinline__ void settle(int row0, int b, int hkv) {
        const int ln = opaque_tid() & 63;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const bool odd = mx[n] == kNegInf && sum_groups(sum[n]) != 0.f;
            if (!__ballot(odd)) continue;
            // (by all lanes: they meet in it.  finish() clears o)
            const bool some = sees<kDocs>(attn_args<Args>(), row0 + 16 * n + (ln & 15), b, hkv, ln >> 4);
            if (odd && !some) sum[n] = 0.f;
        }
    }

    // The four waves' (kSplit: of the same rows, over different keys) softmaxes
    // meet: afterwards the wave with rs 0 holds the whole.  x: 2 KiB, slots:
    // D / 16 * 2 KiB + 512 a wave of rs > 0.
    template <int kSplit>
    __device__ __forceinline__ void meet(FA3_LDS float* x, FA3_LDS char* slots, int w, int qb,
                                         int rs) {
        constexpr int kQb = kRegWaves / kSplit, kSlot = kDB * 2048 + 512;
        const int ln = opaque_tid() & 63;
#pragma unroll
        for (int n = 0; n < 2; ++n) x[(2 * w + n) * 64 + ln] = mx[n];
        wait_vm_lgkm0<0>();
        barrier();
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float top = kNegInf;
#pragma unroll
            for (int k = 0; k < kSplit; ++k)
                top = __builtin_fmaxf(top, x[(2 * (qb + kQb * k) + n) * 64 + ln]);
            const float mu = top == kNegInf ? 0.f : top;
            const float f = fast_exp2(mx[n] - mu);
            mx[n] = top;
            sum[n] *= f;
#pragma unroll
            for (int i = 0; i < kDB; ++i) o[i][n] *= f;
        }
        if (rs > 0) {
            FA3_LDS char* slot = slots + (qb + kQb * (rs - 1)) * kSlot;
            reg_put<kDB>(slot, o, ln);
            FA3_LDS float* l = (FA3_LDS float*)(slot + kDB * 2048);
            l[ln] = sum[0];
            l[64 + ln] = sum[1];
        }
        wait_vm_lgkm0<0>();
        barrier();
        if (rs > 0) return;
#pragma unroll
        for (int k = 0; k < kSplit - 1; ++k) {
            FA3_LDS char* slot = slots + (qb + kQb * k) * kSlot;
            reg_add<kDB>(slot, o, ln);
            FA3_LDS float* l = (FA3_LDS float*)(slot + kDB * 2048);
            sum[0] += l[ln];
            sum[1] += l[64 + ln];
        }
    }

    // The rows' outputs and log-sum-exps, or (splits > 1) their part of both;
    // stg: D / 16 KiB of the wave's own.
    __device__ __forceinline__ void finish(int row0, int end, int b, int hkv, int grp, int split,
                                           FA3_LDS char* stg) {
        const auto& z = attn_args<Args>();
        const int ln = opaque_tid() & 63, l16 = ln & 15, g4 = ln >> 4;
        float inv[2], lse2[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float l = sum_groups(sum[n]);
            const bool none = mx[n] == kNegInf && l == 0.f;
            inv[n] = none ? 0.f : 1.f / l;
            if (none) {  // (other rows' V may have been NaN)
#pragma unroll
                for (int i = 0; i < kDB; ++i) o[i][n] = f32x4{};
            }
            lse2[n] = none ? kNegInf : mx[n] + __builtin_amdgcn_logf(l);
        }
        if (z.splits > 1) {
            const int64_t base = ((int64_t)split * z.groups + grp) * z.rows;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int r = row0 + 16 * n + l16;
                if (r >= end) continue;
                if (g4 == 0) z.part_l[base + r] = lse2[n];
                float* p = z.part_o + (base + r) * D + 4 * g4;
#pragma unroll
                for (int i = 0; i < kDB; ++i) *(f32x4*)(p + 16 * i) = o[i][n] * inv[n];
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const AttnRow r = attn_row(row0 + 16 * n + l16, end, hkv, z.group, z.div_group);
            if (g4 == 0 && r.ok)
                z.lse[((int64_t)b * z.heads_q + r.h) * z.sq + r.i] = lse2[n] * 0.69314718055994531f;
        }
        attn_store<D, kBf16>(o, inv, z.d, stg, [&](int r) -> _Float16* {
            const AttnRow x = attn_row(row0 + r, end, hkv, z.group, z.div_group);
            return x.ok ? z.out.p + b * z.out.bs + x.h * z.out.hs + x.i * z.out.rs : nullptr;
        });
    }
};

// A workgroup's job: levels are row tiles (last rows first, causal's longest)
// times parts of the key axis.
struct FwdJob {
    int b, hkv, grp, tile, split;
};
template <typename A>
__device__ __forceinline__ FwdJob fwd_job(const A& a, int id) {
    FwdJob j;
    int level;
    attn_job(id, a.groups, a.by_group, a.div_groups, a.div_gpart, a.div_levels, a.levels, level, j.grp);
    j.b = fdiv(a.div_hkv, j.grp);
    j.hkv = j.grp - j.b * a.heads_kv;
    const int tl = fdiv(a.div_splits, level);
    j.split = level - tl * a.splits;
    j.tile = a.tiles - 1 - tl;
    return j;
}

// Joins the parts of a split key axis: with w_s = exp2(l_s - max l), out =
// sum w_s o_s / sum w_s.  D / 8 lanes hold a row, 8 columns each.  kWays
// groups of them take every kWays-th part of it, whose sums meet at the end:
// many parts are few rows, which leave only latency to win (whole calls: B1
// Hq32 Hkv8 Sk16384 D128 in 32 parts 37.1 us with one way, 19.4 with four), and
// few parts are many rows, which fill the chip (B1 Hq16 Hkv4 S2011 in two parts
// 59.2 with one way, 66.0 with four).
template <int D, bool kBf16, int kWays>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnFwdArgs a) {
    constexpr int kLanes = D / 8, kRow = kLanes * kWays;
    const int lane = threadIdx.x & (kRow - 1);
    const int64_t total = (int64_t)a.groups * a.rows;
    const int64_t rg = (int64_t)blockIdx.x * (256 / kRow) + (int)(threadIdx.x / kRow);
    if (rg >= total) return;
    float top = kNegInf;
    for (int s = lane; s < a.splits; s += kRow) top = __builtin_fmaxf(top, a.part_l[s * total + rg]);
#pragma unroll
    for (int o = kRow / 2; o > 0; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    const int col = (lane % kLanes) * 8;
    float z = 0.f, acc[8] = {};
#pragma unroll 4
    for (int s = lane / kLanes; s < a.splits; s += kWays) {
        const float l = a.part_l[s * total + rg];
        const float* p = a.part_o + (s * total + rg) * D + col;
        const f32x4 x = *(const f32x4*)p, y = *(const f32x4*)(p + 4);
        // (a part that saw nothing has no output to weigh: it may hold anything)
        const bool none = l == kNegInf;
        const float f = none ? 0.f : fast_exp2(l - top);
        z += f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[e] = __builtin_fmaf(f, none ? 0.f : x[e], acc[e]);
            acc[4 + e] = __builtin_fmaf(f, none ? 0.f : y[e], acc[4 + e]);
        }
    }
#pragma unroll
    for (int o = kRow / 2; o >= kLanes; o >>= 1) {
        z += __shfl_xor(z, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor(acc[e], o);
    }
    const int grp = (int)(rg / a.rows), r = (int)(rg - (int64_t)grp * a.rows);
    const int b = fdiv(a.div_hkv, grp), hkv = grp - b * a.heads_kv;
    const AttnRow x = attn_row(r, a.rows, hkv, a.group, a.div_group);
    const bool none = z == 0.f;  // (NaN is not)
    const float inv = none ? 0.f : 1.f / z;
    if (lane == 0)
        a.lse[((int64_t)b * a.heads_q + x.h) * a.sq + x.i] =
            none ? kNegInf : (top + __builtin_amdgcn_logf(z)) * 0.69314718055994531f;
    if (lane >= kLanes || col >= a.d) return;
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to16<kBf16>(acc[e] * inv);
    *(f16x8*)(a.out.p + b * a.out.bs + x.h * a.out.hs + x.i * a.out.rs + col) = v;
}

}  // namespace
}  // namespace fa3
