// What the attention kernels share: the log2-domain score, masks, the walk
// over 64-position tiles and their direct-to-LDS loads.
#pragma once

#include "fa3_attn_internal.h"
#include "fa3_bwd_reg_kernel.h"

namespace fa3 {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();

// 16 zero bytes: where the loads of rows and columns outside a tensor read.
__device__ __attribute__((aligned(16))) const uint32_t attn_zeros[4] = {0, 0, 0, 0};

// max over the four lanes of equal lane % 16, NaN if one of them is.
// v_permlane{32,16}_swap with one register on both sides leave a lane's own
// and its partner's value.
__device__ __forceinline__ float max_groups(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = __builtin_elementwise_maximum(__builtin_bit_cast(float, (uint32_t)r[0]),
                                      __builtin_bit_cast(float, (uint32_t)r[1]));
    const uint32_t v = __builtin_bit_cast(uint32_t, x);
    r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __builtin_elementwise_maximum(__builtin_bit_cast(float, (uint32_t)r[0]),
                                         __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    const uint32_t v = __builtin_bit_cast(uint32_t, x);
    r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// tanh(s / softcap) of a raw dot product s:
//   1 - 2 / (exp(2 s scale / softcap) + 1),  k1 = 2 scale log2 e / softcap.
// Both ends come out right (exp2 overflows to infinity: 1; underflows: -1).
// The result is off by about 2^-24 absolutely, the score by softcap times
// that; with a cap over kCapFine (fa3_attn_api.cpp), where that would show,
// scores below softcap / 8 take the series u - u^3 / 3 + 2 u^5 / 15 -
// 17 u^7 / 315 (next term 62 / 2835 u^9, 1.3e-9 of the value at 1 / 8).
__device__ __forceinline__ float attn_tanh(float s, float k1) {
    const float r = __builtin_amdgcn_rcpf(fast_exp2(s * k1) + 1.f);
    return __builtin_fmaf(-2.f, r, 1.f);
}
__device__ __forceinline__ float attn_tanh_fine(float s, float k1) {
    const float u = s * (k1 * 0.34657359027997265f), u2 = u * u;
    float t = __builtin_fmaf(u2, -17.f / 315.f, 2.f / 15.f);
    t = __builtin_fmaf(u2, t, -1.f / 3.f);
    t = __builtin_fmaf(u2 * u, t, u);
    float far = attn_tanh(s, k1);
    __asm__("" : "+v"(far));  // (a select, not a branch per element)
    return __builtin_fabsf(u) < 0.125f ? t : far;
}

// The AttnRange of 64-position block x of ids [batch][n], by one wave.
__device__ __forceinline__ void attn_range(const int* ids, int64_t bs, int n, int blocks, int x,
                                           AttnRange* out, int lane) {
    const int b = x / blocks, i = (x - b * blocks) * 64 + lane;
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

// A document as masks compare it: every negative one meets none.
__device__ __forceinline__ int doc_of(int id) { return id < 0 ? -3 : id; }

// Smallest and largest of ids >= 0 over a wave (two per lane), and over the
// workgroup through `x` (8 words of LDS; one barrier).
struct DocSpan {
    int lo, hi;    // of the wave
    int glo, ghi;  // of the workgroup
    bool pad;      // an id of the wave is -1
};
__device__ __forceinline__ DocSpan doc_span(const int (&id)[2], FA3_LDS int* x, int w, int lane) {
    DocSpan s;
    s.pad = __ballot(id[0] == -1 || id[1] == -1) != 0;
    s.lo = 0x7fffffff;
    s.hi = -1;
#pragma unroll
    for (int n = 0; n < 2; ++n)
        if (id[n] >= 0) {
            s.lo = min(s.lo, id[n]);
            s.hi = max(s.hi, id[n]);
        }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {  // (lanes l and l + 16 hold the same)
        s.lo = min(s.lo, __shfl_xor(s.lo, o));
        s.hi = max(s.hi, __shfl_xor(s.hi, o));
    }
    s.lo = __builtin_amdgcn_readfirstlane(s.lo);
    s.hi = __builtin_amdgcn_readfirstlane(s.hi);
    if (lane == 0) {
        x[2 * w] = s.lo;
        x[2 * w + 1] = s.hi;
    }
    wait_vm_lgkm0<0>();
    barrier();
    s.glo = 0x7fffffff;
    s.ghi = -1;
#pragma unroll
    for (int i = 0; i < kRegWaves; ++i) {
        s.glo = min(s.glo, __builtin_amdgcn_readfirstlane(x[2 * i]));
        s.ghi = max(s.ghi, __builtin_amdgcn_readfirstlane(x[2 * i + 1]));
    }
    return s;
}

// A word that no kernel running now writes, at an address that is the same in
// all lanes, through the scalar cache.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
    typedef __attribute__((address_space(4))) const T K;
    return *(K*)(uintptr_t)p;
}

// The tiles' walk: 64-position tiles t of [begin, end), those left out whose
// documents cannot meet the workgroup's.  All lanes of all waves of a
// workgroup step alike: a wave looks at the ranges of 64 tiles at a time.
constexpr int kTileMeets = 1;   // the tile's documents can meet this wave's
constexpr int kTileSame = 2;    // both have one document, the same
constexpr int kTileHidden = 4;  // the tile has positions of no document
struct TileWalk {
    const AttnRange* ranges;  // of this batch entry; null: every tile, from `near` down, then up
    int at, end;              // next tile (ranges: next tile to look up)
    int begin, up;
    int base;
    uint64_t live;            // of the tiles base .. base + 63
    DocSpan doc;
    int cls;                  // kTile* of the tile last returned

    __device__ __forceinline__ TileWalk(const AttnRange* r, int begin_, int end_, const DocSpan& d,
                                        int near)
        : ranges(r), at(begin_), end(end_), begin(begin_), base(begin_), live(0), doc(d),
          cls(kTileMeets | kTileSame) {
        near = near < end_ - 1 ? near : end_ - 1;
        if (ranges == nullptr && near >= begin_) at = near;
        if (ranges == nullptr && begin_ >= end_) at = -1;
        up = near >= begin_ ? near + 1 : begin_ + 1;
    }
    // the next tile, or -1
    __device__ __forceinline__ int next() {
        if (ranges == nullptr) {
            if (at >= begin) return at--;
            return up < end ? up++ : -1;
        }
        while (live == 0) {
            if (at >= end) return -1;
            base = at;
            at = end - at > 64 ? at + 64 : end;
            const int t = base + (int)__lane_id();
            int rlo = 0x7fffffff, rhi = -1;
            if (t < end) {
                const i32x2 r = *(const i32x2*)(ranges + t);
                rlo = r[0];
                rhi = r[1];
            }
            const int l = rlo < 0 ? ~rlo : rlo;
            live = __ballot(rhi >= doc.glo && l <= doc.ghi);
        }
        const int k = __builtin_ctzll(live);
        live &= live - 1;
        // (read once more, through the scalar cache: held per lane, the ranges
        // would cost two vector registers over the whole loop, and a vector
        // load here is waited for before the next tile's loads go out)
        const i32x2 r = scalar_load((const i32x2*)(ranges + base + k));
        const int x = r[0], hi = r[1], lo = x < 0 ? ~x : x;
        cls = (hi >= doc.lo && lo <= doc.hi ? kTileMeets : 0) |
              (x >= 0 && !doc.pad && lo == hi && doc.lo == doc.hi && lo == doc.lo ? kTileSame : 0) |
              (x < 0 ? kTileHidden : 0);
        return base + k;
    }
};

// Direct-to-LDS copy of rows [row0, row0 + 64) of a [rows][d] matrix (row
// stride rs elements) into a swizzled [64][D] tile by the 4 waves.
template <int D>
__device__ __forceinline__ void attn_load_tile(FA3_LDS char* tile, const _Float16* src, int64_t rs,
                                               int row0, int w, int lane) {
    constexpr int kLd = RegCfg<D>::kLd, kRows = 512 / D, kC = D / 8;
    const int row = lane / kC;
    const uint32_t c = ((uint32_t)(lane % kC) ^ reg_swz<D>(row)) & (kC - 1);
    const char* p = (const char*)(src + (int64_t)(row0 + 16 * w) * rs) + (int64_t)row * rs * 2;
#pragma unroll
    for (int j = 0; j < kLd; ++j)
        __builtin_amdgcn_global_load_lds(
            (const void*)(p + (int64_t)(kRows * j) * rs * 2 + ((c ^ reg_swz<D>(kRows * j)) & (kC - 1)) * 16),
            (FA3_LDS void*)(tile + (w * kLd + j) * 1024), 16, 0, 0);
}
// The same where rows end at `rows`, columns at d < D, or rows take no part
// (seen(row) is false): those read as zeros.
template <int D, typename Seen>
__device__ __forceinline__ void attn_load_tile_edge(FA3_LDS char* tile, const _Float16* src,
                                                    int64_t rs, int row0, int rows, int d, int w,
                                                    int lane, Seen seen) {
    constexpr int kLd = RegCfg<D>::kLd, kRows = 512 / D, kC = D / 8;
    const int row = lane / kC;
    const uint32_t c = ((uint32_t)(lane % kC) ^ reg_swz<D>(row)) & (kC - 1);
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
        const int r = row0 + 16 * w + kRows * j + row;
        const uint32_t cj = (c ^ reg_swz<D>(kRows * j)) & (kC - 1);
        const char* p = (const char*)attn_zeros;
        if (r < rows && (int)cj * 8 < d && seen(r)) p = (const char*)(src + (int64_t)r * rs) + cj * 16;
        __builtin_amdgcn_global_load_lds((const void*)p,
                                         (FA3_LDS void*)(tile + (w * kLd + j) * 1024), 16, 0, 0);
    }
}

// The documents of 64 positions from i0 on (n in all) to 256 bytes of LDS, by
// one wave.
__device__ __forceinline__ void attn_load_ids(FA3_LDS char* to, const int* ids, int i0, int n,
                                              int lane) {
    __builtin_amdgcn_global_load_lds((const void*)(ids + min(i0 + lane, n - 1)), (FA3_LDS void*)to,
                                     4, 0, 0);
}

// 8 elements 8 c .. of a row (d of them are there), or zeros
__device__ __forceinline__ f16x8 attn_row8(const _Float16* row, int c, int d, bool ok) {
    const _Float16* p = ok && 8 * c < d ? row + 8 * c : (const _Float16*)attn_zeros;
    return *(const f16x8*)p;
}

// Operands on their way in the backward's products (RegCfg): masks and score
// options leave fewer registers for them at D 128.
template <int D, bool kScored>
struct AttnAhead : RegCfg<D> {
    static constexpr int kAhead0 = 2;
    static constexpr int kAhead1 = kScored ? 1 : 2;
    static constexpr int kAheadG = D == 128 ? 4 : 2;
};

// Turns the sign of 8 elements where flip is 0x80008000.
__device__ __forceinline__ f16x8 attn_flip(f16x8 x, uint32_t flip) {
    return __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, x) ^ flip);
}

// s[m][n] += X B over D for M 16-row blocks of an LDS tile, from row block
// m0 on, and the two resident column blocks; kAhead operands on their way.
template <int D, bool kBf16, int M, int kAhead>
__device__ __forceinline__ void attn_scores(const RegReader<D>& rd, const FA3_LDS char* x, int m0,
                                            const f16x8 (&b)[2][D / 32], f32x4 (&s)[M][2]) {
    constexpr int kKs = D / 32, kN = M * kKs;
    f16x8 f[kN];
    auto m_of = [](int i) { return i / kKs; };
    auto ks_of = [](int i) { return i % kKs; };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = rd.row(x, m0 + m_of(i), ks_of(i));
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        wall();
        if (i + kAhead < kN) f[i + kAhead] = rd.row(x, m0 + m_of(i + kAhead), ks_of(i + kAhead));
        wall();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = j ^ (i & 1);
            s[m_of(i)][n] = mfma_16x16x32<kBf16>(f[i], b[n][ks_of(i)], s[m_of(i)][n]);
        }
    }
    wall();
}

// The kernel's arguments, read again where they are used: held in scalar
// registers over the tile loop, they do not fit.
template <typename Args>
__device__ __forceinline__ __attribute__((address_space(4))) const Args& attn_args() {
    typedef __attribute__((address_space(4))) const Args KArg;
    KArg* p = (KArg*)__builtin_amdgcn_kernarg_segment_ptr();
    __asm__ volatile("" : "+s"(p));
    return *p;
}

// Query rows of a KV head: its group * sq (query, head) pairs in that order,
// so that a tile's rows are the fewest queries and share every key.
struct AttnRow {
    int i, h;  // query and query head
    bool ok;
};
template <typename Div>
__device__ __forceinline__ AttnRow attn_row(int r, int rows, int hkv, int group, const Div& div) {
    AttnRow x;
    x.ok = r < rows;
    const int q = x.ok ? r : 0;
    x.i = fdiv(div, q);
    x.h = hkv * group + (q - x.i * group);
    return x;
}

// Keys visible to query i: those below this limit (documents aside).
__device__ __forceinline__ int attn_limit(int i, int off, int kv, int causal, int prefix) {
    if (!causal) return kv;
    int lim = i + off + 1;  // i + off + 1 <= kv
    if (prefix > lim) lim = prefix < kv ? prefix : kv;
    return lim > 0 ? lim : 0;
}

// Filled keys and prefix of batch entry b.
template <typename M>
__device__ __forceinline__ int attn_kv(const M& m, int b, int sk) {
    if (m.kv_lens == nullptr) return sk;
    const int kv = scalar_load(m.kv_lens + b);
    return kv < 0 ? 0 : kv < sk ? kv : sk;
}
template <typename M>
__device__ __forceinline__ int attn_prefix(const M& m, int b) {
    if (m.prefix == nullptr) return 0;
    const int n = scalar_load(m.prefix + b);
    return n > 0 ? n : 0;
}

// A wave's 32 x D block (acc[db][n]: row 16 n + l16, columns 16 db + 4 g + e)
// times mul[n] to 16-bit rows row(r) (null: not there), columns below d, through
// the wave's own D / 16 KiB of LDS, so that every global store writes whole
// 128-byte row segments.
template <int D, bool kBf16, typename Row>
__device__ __forceinline__ void attn_store(const f32x4 (*acc)[2], const float (&mul)[2], int d,
                                           FA3_LDS char* stg, Row row) {
    const int lane = opaque_tid() & 63, l16 = lane & 15, g4 = lane >> 4;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = to16<kBf16>(acc[i][n][e] * mul[n]);
            lds_write_b64(stg, (uint32_t)(i >> 2) * 4096 +
                                   stage128_off(16 * n + l16, 2 * (i & 3) + (g4 >> 1), g4 & 1), v);
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = 8 * j + ((lane >> 2) & 7), c = (lane & 3) | ((lane >> 5) << 2);
        _Float16* p = row(r);
        if (p == nullptr) continue;
#pragma unroll
        for (int pn = 0; pn < D / 64; ++pn)
            if (64 * pn + 8 * c < d)
                store_out(p + 64 * pn + 8 * c,
                          stage_fix(lds_read_b128(stg + pn * 4096, stage128_chunk(r, c)), r));
    }
}

// Workgroup id's job.  XCD x runs the workgroups with id % 8 == x.  With a
// multiple of 8 groups ((batch, KV head) pairs) an XCD takes every eighth one
// whole, so that its keys stay in one L2: level by level over its groups, so
// that the longest jobs start first, or (by_group, for jobs of one length) one
// group after the other.  Otherwise jobs go level by level over all groups.
template <typename Div>
__device__ __forceinline__ void attn_job(int id, int groups, bool by_group, const Div& div_groups,
                                         const Div& div_part, const Div& div_levels, int levels,
                                         int& level, int& group) {
    if (groups % 8 == 0) {
        const int part = groups / 8, pos = id / 8;
        int g;
        if (by_group) {
            g = fdiv(div_levels, pos);
            level = pos - g * levels;
        } else {
            level = fdiv(div_part, pos);
            g = pos - level * part;
        }
        group = id % 8 + 8 * g;
    } else {
        level = fdiv(div_groups, id);
        group = id - level * groups;
    }
}

}  // namespace
}  // namespace fa3
