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
    int levels, by_group;
    FastDiv div_hkv, div_group, div_groups, div_gpart, div_splits, div_levels;
};

template <int D>
struct FwdCfg {
    static constexpr int kTileBytes = 64 * D * 2;
    static constexpr int kStageBytes = 2 * kTileBytes + 256;  // K, V, the keys' documents
    static constexpr int kRangeOff = 2 * kStageBytes;  // the waves' document ranges
    static constexpr int kBytes = kRangeOff + 64;
    static constexpr int kKs = D / 32, kDB = D / 16;
};

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
template <int D, bool kBf16, bool kCap, bool kBias>
struct FwdRows {
    typedef AttnFwdArgs Args;
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

    // Rows row0 .. row0 + 31 of KV head hkv in batch entry b.
    template <typename A>
    __device__ __forceinline__ void init(const A& a, int row0, int b, int hkv, int kv, int prefix,
                                         int off, int lane) {
        const int l16 = lane & 15;
        const bool any = row0 < a.rows;
        const int first = fdiv(a.div_group, any ? row0 : 0);
        const int last = fdiv(a.div_group, any ? min(row0 + 32, a.rows) - 1 : 0);
        lim_min = any ? attn_limit(first, off, kv, a.m.causal, prefix) : 0x7fffffff;
        lim_max = any ? attn_limit(last, off, kv, a.m.causal, prefix) : 0;
        k1 = kCap ? a.m.k1 : 0.f;
        cap2 = kCap ? a.m.cap2 : 0.f;
        fine = kCap && a.m.cap_fine;
        q_first = first + off;
        q_last = last + off;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const AttnRow r = attn_row(row0 + 16 * n + l16, a.rows, hkv, a.group, a.div_group);
            lim[n] = r.ok ? attn_limit(r.i, off, kv, a.m.causal, prefix) : 0;
            id[n] = -2;
            // (documents: -1 for every negative one, -2 for rows that are not there)
            if (a.m.doc_q != nullptr && r.ok) id[n] = max(a.m.doc_q[b * a.m.doc_q_bs + r.i], -1);
        }
    }
    // Their Q, after the first tile's loads have gone out.
    template <typename A>
    __device__ __forceinline__ void load(const A& a, int row0, int b, int hkv, int off, int lane) {
        const int l16 = lane & 15, g4 = lane >> 4;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const AttnRow r = attn_row(row0 + 16 * n + l16, a.rows, hkv, a.group, a.div_group);
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
    // ids: their documents in LDS, or null where all rows are of theirs.
    template <int M>
    __device__ __forceinline__ void step(const RegReader<D>& rd0, const FA3_LDS char* tk,
                                         const FA3_LDS char* tv, int m0, int j0,
                                         const FA3_LDS char* ids, float c) {
        RegReader<D> rd = rd0;
        rd.opaque();
        const bool limited = j0 + 16 * M > lim_min;
        f32x4 s[M][2];  // [m][n]: keys 16 m + 4 g4 + e, rows 16 n + l16
        float al = c, be[2] = {0.f, 0.f};
        bool linear = false;  // every row of the wave on one side of every key
        if constexpr (kBias && !kCap) {
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
        if (!kCap && !(kBias && !linear)) mask();
        attn_scores<D, kBf16, M, 4>(rd, tk, m0, qf, s);
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
        if (kCap || (kBias && !linear)) mask();
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
            f16x8 bp[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = fast_exp2(__builtin_fmaf(s[2 * r + (j >> 2)][n][j & 3], al, be[n]));
                    sum[n] += p[j];
                }
                bp[n] = pack8<kBf16>(p);
            }
            reg_grads<D, kBf16, false>(rd, tv, tv, m0 / 2 + r, bp, bp, o, o);
        }
    }

    // Whether row `row` of KV head hkv sees any key at all: lane g4 of its four
    // looks at every fourth, last first (with causality its own document is
    // there).  What init() read is read again: not held over the tile loop.
    template <bool kDocs, typename A>
    static __device__ __forceinline__ bool sees(const A& z, int row, int b, int hkv, int g4) {
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
    __device__ __forceinline__ void finish(int row0, int b, int hkv, int grp, int split,
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
                if (r >= z.rows) continue;
                if (g4 == 0) z.part_l[base + r] = lse2[n];
                float* p = z.part_o + (base + r) * D + 4 * g4;
#pragma unroll
                for (int i = 0; i < kDB; ++i) *(f32x4*)(p + 16 * i) = o[i][n] * inv[n];
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const AttnRow r = attn_row(row0 + 16 * n + l16, z.rows, hkv, z.group, z.div_group);
            if (g4 == 0 && r.ok)
                z.lse[((int64_t)b * z.heads_q + r.h) * z.sq + r.i] = lse2[n] * 0.69314718055994531f;
        }
        attn_store<D, kBf16>(o, inv, z.d, stg, [&](int r) -> _Float16* {
            const AttnRow x = attn_row(row0 + r, z.rows, hkv, z.group, z.div_group);
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
    rows.init(a, (job.tile * kQb + qb) * 32, b, hkv, kv, prefix, off, lane);
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
    rows.load(a, (job.tile * kQb + qb) * 32, b, hkv, off, lane);
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
    rows.finish((e.tile * kQb + eqb) * 32, e.b, e.hkv, e.grp, e.split,
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
    rows.init(a, 0, b, hkv, kv, prefix, off, lane);
    rows.load(a, 0, b, hkv, off, lane);
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
    rows.finish(0, e.b, e.hkv, e.grp, e.split, smem + 2048);
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
