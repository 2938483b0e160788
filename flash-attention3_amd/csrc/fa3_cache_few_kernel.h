// Few rows of a KV head: 16 kBlocks rows a workgroup, whose four waves all hold
// them and take every fourth block of 32 keys each, straight from HBM to
// registers.
//
// A lane's share of a block, with r = lane % 16 and g = lane / 16:
//   K   the channels D / 4 g .. of rows r and 16 + r: the A operand of S^T = K
//       Q^T whose k-step s stands for the channels D / 4 g + 8 s .. of each g,
//       in Q's operand too; a row is read once by four lanes that lie together;
//   V   the D / 16 channels D / 16 r .. of the rows 4 g + 0..3 and 16 + 4 g +
//       0..3, whose scores are the lane's own.  Two rows' values of a channel
//       side by side are a pair of the A operand of O^T += V^T P^T: of 16 bits
//       by one byte permutation; of 4 bits two rows' codes are put into one
//       byte (two shifts and two selects for 16 codes), which one conversion
//       makes two levels of;
//   4 bits: the scales of those rows, K's and V's.  Levels are exact, the
//       scale of K meets the fp32 score, that of V meets P before its rounding
//       to bf16 (fp16 rows: to two bf16 terms, FwdRows).
// Two blocks' loads are out at a time; there is no barrier before the waves meet.
//
// Bound by HBM: 16 sequences of up to 8192 in 16 bits 62.6 us, 5.1 TB/s; 48 of up
// to 16384 in 4 bits 108.6 us, 5.0 TB/s (the codes make 49 % of the SIMDs' cycles
// vector instructions, matrix ones 14 %).  Where few keys are left to a wave,
// its chain of loads, products and exponentials: 8 x 5 tokens over 6001 in 4
// bits 16 us, one token over 129 6.1 (kernel trace; 4.7 a call in a captured graph).
#pragma once

#include "fa3_cache_attn_kernel.h"

namespace fa3 {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Where a sequence's blocks lie.
struct FewPages {
    const char *k, *v;  // the KV head's
    int64_t k_ps, k_rs, v_ps, v_rs;
    int shift, d;
};

template <int D, bool kFour>
struct FewBlock {  // 4 bits
    typedef typename std::conditional<D == 128, u32x4, u32x2>::type Codes;
    typedef typename std::conditional<D == 128, uint32_t, uint16_t>::type Piece;
    Codes k[2];
    Piece v[8];
    f32x4 ks[2], vs[2];

    __device__ __forceinline__ void load(const FewPages& p, const CacheBlock& x, int lane) {
        const int l16 = lane & 15, g4 = lane >> 4, row = x.j0 & ((1 << p.shift) - 1);
        const char* pk = p.k + x.page * p.k_ps;
        const char* pv = p.v + x.page * p.v_ps;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            k[t] = *(const Codes*)(pk + (row + 16 * t + l16) * (D / 2) + g4 * (D / 8));
            const int at = (D / 2 << p.shift) + (row + 16 * t + 4 * g4) * 4;
            ks[t] = *(const f32x4*)(pk + at);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[4 * t + e] = *(const Piece*)(pv + (row + 16 * t + 4 * g4 + e) * (D / 2) + l16 * (D / 32));
            vs[t] = *(const f32x4*)(pv + at);
        }
    }
    // rows n and behind hold anything: none of it is to reach a product
    __device__ __forceinline__ void cut(int n, int lane) {
        const int k = n - 4 * (lane >> 4);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) vs[t][e] = 16 * t + e < k ? vs[t][e] : 0.f;
    }
    template <bool kBf16>
    __device__ __forceinline__ f16x8 key(int t, int s) const {
        return cache_levels8<kBf16>(k[t][s]);
    }
    // use(i, operand) for every channel i of the lane
    template <typename F>
    __device__ __forceinline__ void values(F use) const {
        // x[j][0]: even channels' codes of rows 2 j and 2 j + 1, a byte each; x[j][1]: odd ones'
        uint32_t x[4][2];
        if constexpr (D == 128) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t y = v[2 * j], z = v[2 * j + 1];
                x[j][0] = (y & 0x0F0F0F0Fu) | ((z << 4) & 0xF0F0F0F0u);
                x[j][1] = ((y >> 4) & 0x0F0F0F0Fu) | (z & 0xF0F0F0F0u);
            }
        } else {  // (bytes 0, 1: rows 2 j and 2 j + 1; bytes 2, 3: 2 j + 4 and 2 j + 5)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t y = v[2 * j] | ((uint32_t)v[2 * j + 4] << 16);
                const uint32_t z = v[2 * j + 1] | ((uint32_t)v[2 * j + 5] << 16);
                x[j][0] = (y & 0x0F0F0F0Fu) | ((z << 4) & 0xF0F0F0F0u);
                x[j][1] = ((y >> 4) & 0x0F0F0F0Fu) | (z & 0xF0F0F0F0u);
                x[j + 2][0] = x[j][0] >> 16;
                x[j + 2][1] = x[j][1] >> 16;
            }
        }
        auto byte = [&](auto sel) {
            constexpr int kSel = decltype(sel)::value;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 y = {cache_levels<true, kSel>(x[0][h]), cache_levels<true, kSel>(x[1][h]),
                                 cache_levels<true, kSel>(x[2][h]), cache_levels<true, kSel>(x[3][h])};
                use(2 * kSel + h, __builtin_bit_cast(f16x8, y));
            }
        };
        byte(std::integral_constant<int, 0>{});
        byte(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
            byte(std::integral_constant<int, 2>{});
            byte(std::integral_constant<int, 3>{});
        }
    }
};

template <int D>
struct FewBlock<D, false> {  // 16 bits
    typedef typename std::conditional<D == 128, u32x4, u32x2>::type Piece;
    f16x8 k[2][D / 32];
    Piece v[8];

    __device__ __forceinline__ void load(const FewPages& p, const CacheBlock& x, int lane) {
        const int l16 = lane & 15, g4 = lane >> 4, row = x.j0 & ((1 << p.shift) - 1);
        const char* pk = p.k + x.page * p.k_ps + (row + l16) * p.k_rs + g4 * (D / 2);
        const char* pv = p.v + x.page * p.v_ps + (row + 4 * g4) * p.v_rs + l16 * (D / 8);
        if (p.d == D) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int s = 0; s < D / 32; ++s) k[t][s] = *(const f16x8*)(pk + 16 * t * p.k_rs + 16 * s);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * t + e] = *(const Piece*)(pv + (16 * t + e) * p.v_rs);
            }
            return;
        }
        const bool in = l16 * (D / 16) < p.d;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int s = 0; s < D / 32; ++s)
                k[t][s] = *(const f16x8*)(g4 * (D / 4) + 8 * s < p.d ? pk + 16 * t * p.k_rs + 16 * s
                                                                    : (const char*)attn_zeros);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[4 * t + e] = *(const Piece*)(in ? pv + (16 * t + e) * p.v_rs : (const char*)attn_zeros);
        }
    }
    __device__ __forceinline__ void cut(int n, int lane) {
        const int k = n - 4 * (lane >> 4);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                    v[4 * t + e][i] = 16 * t + e < k ? v[4 * t + e][i] : 0u;
    }
    template <bool kBf16>
    __device__ __forceinline__ f16x8 key(int t, int s) const {
        return k[t][s];
    }
    template <typename F>
    __device__ __forceinline__ void values(F use) const {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            u32x4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = __builtin_amdgcn_perm(v[2 * j + 1][i / 2], v[2 * j][i / 2],
                                             i % 2 ? 0x07060302u : 0x05040100u);
            use(i, __builtin_bit_cast(f16x8, y));
        }
    }
};

template <int D, int kBlocks>
struct FewCfg {
    static constexpr int kDB = D / 16;
    static constexpr int kSlot = kBlocks * (kDB * 1024 + 256);  // a wave's outputs and sums
    static constexpr int kMax = 4 * kBlocks * 256;              // the waves' maxima
    static constexpr int kBytes = kMax + 4 * kSlot;
};

// kDealt: parts of several sequences, dealt by their lengths.  (A kernel of its
// own: as a branch it cost one token over 129 keys 0.3 us of 5.5, and 64 selected
// pages 0.9 of 21.3.)
template <int D, bool kBf16, bool kCap, bool kBias, bool kFour, int kBlocks, bool kDealt>
__global__ __launch_bounds__(kRegThreads, few_waves(D, kFour, kBlocks)) void cache_few_kernel(CacheAttnArgs) {
    typedef CacheAttnArgs Args;
    const auto& a = attn_args<Args>();
    using C = FewCfg<D, kBlocks>;
    constexpr int kKs = D / 32, kDB = D / 16;
    constexpr float kLazy = 8.f;  // as FwdRows: rescaled only past 2^8
    __shared__ __attribute__((aligned(16))) char smem_raw[C::kBytes];
    FA3_LDS char* smem = (FA3_LDS char*)smem_raw;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    CacheJob job;
    CacheSpan span;
    int slot = 0, parts = a.splits;
    if constexpr (kDealt) {
        slot = fdiv(a.div_hkv, blockIdx.x);
        const CacheDeal d = cache_deal(a, slot);
        if (d.b < 0) return;
        const int hkv = blockIdx.x - slot * a.heads_kv;
        FwdJob f;
        f.b = d.b;
        f.hkv = hkv;
        f.grp = d.b * a.heads_kv + hkv;
        f.split = d.split;
        f.tile = 0;
        job = cache_job_of(a, f, 16 * kBlocks);
        const int n = (job.lim + 31) >> 5;
        span.begin = min(d.split * d.part, n);
        span.end = min(span.begin + d.part, n);
        parts = d.parts;
        if (hkv == 0 && d.split == 0 && threadIdx.x == 0) a.x.deal[d.b] = make_int2(d.first, d.parts);
    } else {
        job = cache_job(a, blockIdx.x, 16 * kBlocks);
        span = cache_span(a, job);
    }
    const int first = span.begin + w, end = span.end;
    const int n = end > first ? (end - first + 3) >> 2 : 0;
    const FewPages at{a.x.cv.k + job.hkv * a.x.cv.k_hs, a.x.cv.v + job.hkv * a.x.cv.v_hs,
                      a.x.cv.k_ps, a.x.cv.k_rs, a.x.cv.v_ps, a.x.cv.v_rs, a.x.cv.shift, a.d};
    auto issue = [&](FewBlock<D, kFour>& f, const CacheBlock& x) {
        if (x.page >= 0) f.load(at, x, opaque_tid() & 63);
    };
    FewBlock<D, kFour> f0, f1;
    CacheBlock b0 = cache_block(a, job, first, end);
    issue(f0, b0);
    CacheBlock b1 = cache_block(a, job, first + 4, end);
    issue(f1, b1);

    f16x8 qf[kBlocks][kKs];
    int lim[kBlocks], place[kBlocks];
    float slope[kBlocks], mx[kBlocks], sum[kBlocks];
    f32x4 o[kDB][kBlocks];  // channels kDB (4 g4 + e) + i of row l16
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
        const AttnRow r = attn_row(job.row0 + 16 * q + l16, job.rows, job.hkv, a.group, a.div_group);
        const _Float16* p = a.q.p + job.b * a.q.bs + r.h * a.q.hs + r.i * a.q.rs;
#pragma unroll
        for (int s = 0; s < kKs; ++s)
            qf[q][s] = attn_flip(attn_row8(p, D / 32 * g4 + s, a.d, r.ok && a.scored), a.flip);
        lim[q] = r.ok ? attn_limit(r.i, job.off, job.kv, a.m.causal, job.prefix) : 0;
        place[q] = r.i + job.off;
        slope[q] = kBias ? a.m.slopes[job.b * a.m.slopes_bs + r.h] * kLog2e : 0.f;
        mx[q] = kNegInf;
        sum[q] = 0.f;
#pragma unroll
        for (int i = 0; i < kDB; ++i) o[i][q] = f32x4{};
    }
    // below it every row sees every key
    int lim_min = 0x7fffffff;
    if (min(job.row0 + 16 * kBlocks, job.end) > job.rows) lim_min = 0;
    else lim_min = attn_limit(fdiv(a.div_group, job.row0), job.off, job.kv, a.m.causal, job.prefix);
    const float c = a.m.c, k1 = kCap ? a.m.k1 : 0.f, cap2 = kCap ? a.m.cap2 : 0.f;
    const bool fine = kCap && a.m.cap_fine;
    const int kv = job.kv;

    auto step = [&](FewBlock<D, kFour>& f, int j0) {
        f32x4 s[2][kBlocks];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) s[t][q] = f32x4{};
#pragma unroll
            for (int i = 0; i < kKs; ++i) {
                const f16x8 x = f.template key<kBf16>(t, i);
#pragma unroll
                for (int q = 0; q < kBlocks; ++q)
                    s[t][q] = mfma_16x16x32<kBf16>(x, qf[q][i], s[t][q]);
            }
            if constexpr (kFour) {
#pragma unroll
                for (int q = 0; q < kBlocks; ++q) s[t][q] *= f.ks[t];
            }
        }
        // log2-domain scores
        float far[kBlocks];
        if constexpr (kBias) {
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) far[q] = (float)(place[q] - (j0 + 4 * g4));
        }
#pragma unroll
        for (int q = 0; q < kBlocks; ++q)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = s[t][q][e];
                    if constexpr (kCap)
                        x = (fine ? attn_tanh_fine(x, k1) : attn_tanh(x, k1)) * cap2;
                    else
                        x *= c;
                    if constexpr (kBias)  // (exact: a difference of places, then fp32)
                        x = __builtin_fmaf(-slope[q], __builtin_fabsf(far[q] - (float)(16 * t + e)), x);
                    s[t][q][e] = x;
                }
        if (j0 + 32 > lim_min) {
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) {
                const int k = lim[q] - (j0 + 4 * g4);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[t][q][e] = 16 * t + e < k ? s[t][q][e] : kNegInf;
            }
        }
        if (j0 + 32 > kv) f.cut(kv - j0, opaque_tid() & 63);
        float top[kBlocks];
        bool up = false;
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) {
            float x = s[0][q][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) x = __builtin_elementwise_maximum(x, s[t][q][e]);
            top[q] = max_groups(x);
            up |= top[q] > mx[q] + kLazy;
        }
        if (__ballot(up)) {
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) {
                const float m = __builtin_fmaxf(mx[q], top[q]);
                const float y = mx[q] == kNegInf ? 0.f : fast_exp2(mx[q] - m);
                mx[q] = m;
                sum[q] *= y;
#pragma unroll
                for (int i = 0; i < kDB; ++i) o[i][q] *= y;
            }
        }
        f16x8 bp[kBlocks], rest[kBlocks];
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) {
            const float m = mx[q] == kNegInf ? 0.f : mx[q];
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = fast_exp2(s[j >> 2][q][j & 3] - m);
                sum[q] += p[j];
                if constexpr (kFour) p[j] *= f.vs[j >> 2][j & 3];
            }
            bp[q] = pack8<kBf16 || kFour>(p);
            if constexpr (kFour && !kBf16) rest[q] = pack8_rest(p, bp[q]);
        }
        f.values([&](int i, f16x8 x) {
#pragma unroll
            for (int q = 0; q < kBlocks; ++q) {
                o[i][q] = mfma_16x16x32<kBf16 || kFour>(x, bp[q], o[i][q]);
                if constexpr (kFour && !kBf16) o[i][q] = mfma_16x16x32<true>(x, rest[q], o[i][q]);
            }
        });
    };
    for (int x = 0; x < n; x += 2) {
        const CacheBlock b2 = cache_block(attn_args<Args>(), job, first + 4 * x + 8, end);
        if (b0.page >= 0) step(f0, b0.j0);
        b0 = b2;
        issue(f0, b0);
        const CacheBlock b3 = cache_block(attn_args<Args>(), job, first + 4 * x + 12, end);
        if (b1.page >= 0) step(f1, b1.j0);
        b1 = b3;
        issue(f1, b1);
    }

    // A row without a maximum but with a sum has met NaN (FwdRows::settle).
    const auto& z = attn_args<Args>();
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
        sum[q] = sum_groups(sum[q]);
        const bool odd = mx[q] == kNegInf && sum[q] != 0.f;
        if (!__ballot(odd)) continue;
        const bool some = cache_sees(z, job.row0 + 16 * q + l16, job.b, job.hkv, g4);
        if (odd && !some) sum[q] = 0.f;
    }
    // The waves meet: sums and outputs at the largest maximum; wave w adds up
    // and writes the channels kDB (4 g4 + w) ..
    FA3_LDS float* xm = (FA3_LDS float*)smem;
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) xm[(w * kBlocks + q) * 64 + lane] = mx[q];
    wait_vm_lgkm0<0>();
    barrier();
    FA3_LDS char* slots = smem + C::kMax;
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
        float m = kNegInf;
#pragma unroll
        for (int k = 0; k < 4; ++k) m = __builtin_fmaxf(m, xm[(k * kBlocks + q) * 64 + lane]);
        const float y = mx[q] == kNegInf && sum[q] == 0.f ? 0.f : fast_exp2(mx[q] - (m == kNegInf ? 0.f : m));
        // (a NaN that is one: mx -inf, y 0, and the sum stays NaN)
        mx[q] = m;
        sum[q] *= y;
        const bool none = y == 0.f && sum[q] == 0.f;  // (other rows' V may have been NaN)
        FA3_LDS char* slot = slots + w * C::kSlot + q * kDB * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < kDB; ++i) {
            f32x4 x;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = none ? 0.f : o[4 * (i % (kDB / 4)) + c][q][i / (kDB / 4)] * y;
            *(FA3_LDS f32x4*)(slot + i * 1024) = x;
        }
        *(FA3_LDS float*)(slots + w * C::kSlot + kBlocks * kDB * 1024 + q * 256 + lane * 4) = sum[q];
    }
    wait_vm_lgkm0<0>();
    barrier();
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
        f32x4 y[kDB / 4] = {};
        float total = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            FA3_LDS char* slot = slots + k * C::kSlot;
#pragma unroll
            for (int i = 0; i < kDB / 4; ++i)
                y[i] += *(FA3_LDS f32x4*)(slot + (q * kDB + w * (kDB / 4) + i) * 1024 + lane * 16);
            total += *(FA3_LDS float*)(slot + kBlocks * kDB * 1024 + q * 256 + lane * 4);
        }
        const int row = job.row0 + 16 * q + l16;
        if (row >= job.end) continue;
        const bool none = mx[q] == kNegInf && total == 0.f;
        const float inv = none ? 0.f : 1.f / total;
        const float lse2 = none ? kNegInf : mx[q] + __builtin_amdgcn_logf(total);
        float out[kDB];
#pragma unroll
        for (int i = 0; i < kDB; ++i) out[i] = none ? 0.f : y[i / 4][i % 4] * inv;
        const int c = kDB * (4 * g4 + w);
        const bool first = g4 == 0 && w == 0;
        if (parts > 1) {
            const int64_t at = kDealt ? ((int64_t)slot * z.heads_kv + job.hkv) * z.rows + row
                                             : ((int64_t)job.split * z.groups + job.grp) * z.rows + row;
            if (first) z.part_l[at] = lse2;
#pragma unroll
            for (int i = 0; i < kDB / 4; ++i) *(f32x4*)(z.part_o + at * D + c + 4 * i) = *(const f32x4*)(out + 4 * i);
            continue;
        }
        const AttnRow r = attn_row(row, job.end, job.hkv, z.group, z.div_group);
        if (first) z.lse[((int64_t)job.b * z.heads_q + r.h) * z.sq + r.i] = lse2 * 0.69314718055994531f;
        if (c >= z.d) continue;
        _Float16* p = z.out.p + job.b * z.out.bs + r.h * z.out.hs + r.i * z.out.rs + c;
        if constexpr (kDB == 8) {
            *(f16x8*)p = pack8<kBf16>(out);
        } else {
            f16x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = to16<kBf16>(out[i]);
            *(f16x4*)p = x;
        }
    }
}

// Joins the parts of the sequences that were dealt several, as attn_join_kernel
// does: a wave has a row, D / 8 lanes of it 8 channels each of every 512 / D-th
// part.  Latency: 4.7 us for 512 rows, 4.9 for 1536, what the launch of the other
// join takes.
template <int D, bool kBf16>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttnArgs a) {
    constexpr int kLanes = D / 8, kWays = 512 / D;
    const int lane = threadIdx.x & 63;
    const int64_t rg = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rg >= (int64_t)a.groups * a.rows) return;
    const int grp = (int)(rg / a.rows), r = (int)(rg - (int64_t)grp * a.rows);
    const int b = fdiv(a.div_hkv, grp), hkv = grp - b * a.heads_kv;
    const int2 deal = a.x.deal[b];
    if (deal.y <= 1) return;  // (its only part wrote the outputs)
    auto at = [&](int s) { return ((int64_t)(deal.x + s) * a.heads_kv + hkv) * a.rows + r; };
    float top = kNegInf;
    for (int s = lane; s < deal.y; s += 64) top = __builtin_fmaxf(top, a.part_l[at(s)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    const int col = (lane % kLanes) * 8;
    float z = 0.f, acc[8] = {};
#pragma unroll 4
    for (int s = lane / kLanes; s < deal.y; s += kWays) {
        const float l = a.part_l[at(s)];
        const float* p = a.part_o + at(s) * D + col;
        const f32x4 x = *(const f32x4*)p, y = *(const f32x4*)(p + 4);
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
    for (int o = 32; o >= kLanes; o >>= 1) {
        z += __shfl_xor(z, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor(acc[e], o);
    }
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
