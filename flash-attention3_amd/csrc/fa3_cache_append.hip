// Appending to a paged cache with the rotary positions applied on the way, and
// reading it back.
//
// append: a workgroup takes a run of consecutive places of one sequence, within
// one page, and some heads of q, of k or of v.  A group of lanes holds a row, 8
// channels a lane (or 8 and their partners, where those lie apart), and forms
// the cosines and sines of its pairs once for all the heads that it turns; where
// tokens are few, groups share the heads instead.  A row's largest magnitude, for
// its codes, is an exchange among its lanes.  With bounds a run of k is a whole
// page, so that one workgroup owns its bounds: lanes of equal channels compare
// their keys (as 16-bit integers of the same order, two at a time), waves meet
// in LDS.
//
// The turn is fp64 throughout: a row of codes goes by the keys' 16-bit values
// and a level's border by a few of their bits, so an fp32 turn's last bits
// would now and then decide a level.  (A double becomes 16 bits by way of fp32,
// as a cast does.)
//
// Bound by HBM where there is much to move: 8192 tokens of 32 + 8 heads of 128
// channels 46 us, 4.4 TB/s; the fp64 work shows in 4 bits with bounds, where
// each head's run forms its own angles (2 x 2048 such tokens: 29 us, their bytes
// 17).  One token 4.3 us a call in a captured graph (4.8 in a kernel trace), 2 of
// them its angles.
//
// read: a thread per 8 channels; 2 x 4096 places of 8 heads from 4 bits 10 us,
// 4.3 TB/s.
#include "fa3_cache_device.h"
#include "fa3_rotary_angle.h"

namespace fa3 {
namespace {

struct RowsView {
    char* p;
    int64_t bs, hs, rs;  // bytes
};

struct AppendArgs {
    CacheView c;
    RowsView k, v, q, q_out;
    char* bounds;
    const void* positions;  // null: places
    int64_t p_as, p_bs, p_rs;
    const float* freqs;
    int type, axes, pairs;
    int seqlen, heads_q, heads_kv, d;
    // log2 of a workgroup's places, and runs of a sequence; k's beside q's and v's
    int run, segments, run_k, segments_k;
    int hq, hk, hv;  // heads a workgroup takes
    int parts_k, parts_v, batch;
    int lanes, tokens;  // log2 of a row's lanes, and of the rows side by side
    int units;          // of a turned row: 16-byte pieces (with their partners, where those lie apart)
    FastDiv div_segments, div_segments_k, div_row, div_hv;
};

// Lengths that an append follows: past any table by more rows than a call has.
constexpr int kAppendPlaces = (1 << 30) + kMaxGrid;

constexpr int kAppendThreads = 256;
constexpr int kAppendWaves = kAppendThreads / 64;

template <bool kBf16>
__device__ __forceinline__ float value16(_Float16 x) {
    if constexpr (kBf16) return (float)__builtin_bit_cast(__bf16, x);
    else return (float)x;
}

// cos, sin of k / 64 turns.
struct TurnTable {
    double v[64][2];
    constexpr TurnTable() : v() {
        constexpr double c[17] = {
            1.0, 0x1.fd88da3d12526p-1, 0x1.f6297cff75cb0p-1, 0x1.e9f4156c62ddap-1,
            0x1.d906bcf328d46p-1, 0x1.c38b2f180bdb1p-1, 0x1.a9b66290ea1a3p-1, 0x1.8bc806b151741p-1,
            0x1.6a09e667f3bcdp-1, 0x1.44cf325091dd6p-1, 0x1.1c73b39ae68c8p-1, 0x1.e2b5d3806f63bp-2,
            0x1.87de2a6aea963p-2, 0x1.294062ed59f06p-2, 0x1.8f8b83c69a60bp-3, 0x1.917a6bc29b42cp-4,
            0.0};
        for (int j = 0; j < 16; ++j) {
            const double x = c[j], y = c[16 - j];
            v[j][0] = x, v[j][1] = y;
            v[16 + j][0] = -y, v[16 + j][1] = x;
            v[32 + j][0] = -x, v[32 + j][1] = -y;
            v[48 + j][0] = y, v[48 + j][1] = -x;
        }
    }
};
__device__ const TurnTable turn_table = TurnTable();

// Cosine and sine of rev turns, |rev| <= 1/2, off by about 2^-52: those of the
// nearest 64th of a turn, and Taylor's series of the rest r, |r| <= pi / 64 (its
// next terms are r^9 / 9! < 2^-57 and r^10 / 10! < 2^-65).
__device__ __forceinline__ double2 turn_cos_sin(double rev) {
    const double k = rint(rev * 64.0);
    const double r = (rev - k * 0.015625) * 6.283185307179586, x = r * r;
    const double* t = turn_table.v[(int)k & 63];
    const double c = t[0], s = t[1];
    double p = __builtin_fma(x, -1.0 / 5040.0, 1.0 / 120.0);
    p = __builtin_fma(x, p, -1.0 / 6.0);
    const double sr = __builtin_fma(x * r, p, r);
    double q = __builtin_fma(x, 1.0 / 40320.0, -1.0 / 720.0);
    q = __builtin_fma(x, q, 1.0 / 24.0);
    q = __builtin_fma(x, q, -0.5);
    const double cr = x * q;  // cos r - 1
    return make_double2(c + __builtin_fma(c, cr, -s * sr), s + __builtin_fma(s, cr, c * sr));
}

// Largest magnitude of 8 values, as bits: those that are not finite are above
// all others.
__device__ __forceinline__ uint32_t top8(const f16x8& x) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[i]) & 0x7FFFu);
    return top;
}
__device__ __forceinline__ uint32_t top_of_lanes(uint32_t top, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    return top;
}

// A row's scale, and 8 of its values' codes.
template <bool kBf16>
struct RowCodes {
    float scale, m, r;
    int e;
    bool wild;
    __device__ __forceinline__ explicit RowCodes(uint32_t top) {
        const float a = value16<kBf16>(__builtin_bit_cast(_Float16, (uint16_t)top));
        wild = top >= (kBf16 ? 0x7F80u : 0x7C00u);
        scale = wild ? __builtin_nanf("") : a / 6.f;
        // (a is taken into [1/2, 1) before its reciprocal)
        e = -__builtin_amdgcn_frexp_expf(a);
        m = ldexpf(a, e);
        r = top == 0 ? 0.f : 1.f / m;
    }
    // y = 6 x / a, rounded once: on a border between levels exactly, where the
    // conversion takes the even code
    __device__ __forceinline__ uint32_t operator()(const f16x8& x) const {
        if (wild) return 0;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = 6.f * ldexpf(value16<kBf16>(x[i]), e), q = t * r;
            y[i] = __builtin_fmaf(__builtin_fmaf(-q, m, t), r, q);
        }
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
    }
};

// By way of fp32, which the compiler is kept from leaving out.
template <bool kBf16>
__device__ __forceinline__ _Float16 round16(double x) {
    float y = (float)x;
    __asm__("" : "+v"(y));
    return to16<kBf16>(y);
}

template <bool kBf16, bool kInterleaved>
__device__ __forceinline__ void turn8(const f16x8& x, const f16x8& y, const double2* cs, f16x8& r,
                                      f16x8& q) {
    if constexpr (kInterleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double a = value16<kBf16>(x[2 * j]), b = value16<kBf16>(x[2 * j + 1]);
            r[2 * j] = round16<kBf16>(a * cs[j].x - b * cs[j].y);
            r[2 * j + 1] = round16<kBf16>(b * cs[j].x + a * cs[j].y);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double a = value16<kBf16>(x[j]), b = value16<kBf16>(y[j]);
            r[j] = round16<kBf16>(a * cs[j].x - b * cs[j].y);
            q[j] = round16<kBf16>(b * cs[j].x + a * cs[j].y);
        }
    }
}

// One run's rows of some heads.  (The arguments are read where they are used:
// held in scalar registers they do not fit.)
struct AppendRun {
    int b, place0, i0, i1, t1, page, h0, heads;
};

// v: D / 8 lanes a row.
template <bool kBf16, bool kFour>
__device__ __forceinline__ void append_v(const AppendRun& r) {
    const auto& a = attn_args<AppendArgs>();
    const int d = a.d, units = d / 8, shift = a.c.shift, total = (r.i1 - r.i0) * a.hv * units;
    for (int x0 = 0; x0 < total; x0 += kAppendThreads) {
        const int x = x0 + threadIdx.x, row = fdiv(a.div_row, x), u = x - row * units;
        const int t = fdiv(a.div_hv, row), h = row - t * a.hv, i = r.i0 + t;
        const bool ok = x < total && h < r.heads && i < r.t1;
        f16x8 y{};
        if (ok) y = *(const f16x8*)(a.v.p + r.b * a.v.bs + (r.h0 + h) * a.v.hs + i * a.v.rs + 16 * u);
        char* page = a.c.v + r.page * a.c.v_ps + (r.h0 + h) * a.c.v_hs;
        const int at = (r.place0 + i) & ((1 << shift) - 1);
        if constexpr (kFour) {
            const RowCodes<kBf16> codes(top_of_lanes(top8(y), units));
            if (!ok) continue;
            *(uint32_t*)(page + at * (d / 2) + 4 * u) = codes(y);
            if (u == 0) *(float*)(page + (d / 2 << shift) + 4 * at) = codes.scale;
        } else {
            if (ok) *(f16x8*)(page + at * a.c.v_rs + 16 * u) = y;
        }
    }
}

// Two 16-bit values as unsigned integers of the same order (a NaN beyond the
// infinity of its sign), and back.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t order_of(uint32_t x) {
    const uint32_t sign = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, x) >> (i16x2)15);
    return x ^ (sign | 0x80008000u);
}
__device__ __forceinline__ uint32_t of_order(uint32_t k) {
    const uint32_t sign = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, k) >> (i16x2)15);
    return k ^ (~sign | 0x80008000u);
}
template <bool kHigh>
__device__ __forceinline__ uint32_t edge16(uint32_t x, uint32_t y) {
    const u16x2 u = __builtin_bit_cast(u16x2, x), v = __builtin_bit_cast(u16x2, y);
    return __builtin_bit_cast(uint32_t, kHigh ? __builtin_elementwise_max(u, v)
                                              : __builtin_elementwise_min(u, v));
}
// A lane's smallest and largest keys of its 8 channels.
struct Edges {
    uint32_t low[4], high[4];  // channels 2 i, 2 i + 1
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < 4; ++i) low[i] = 0xFFFFFFFFu, high[i] = 0u;
    }
    __device__ __forceinline__ void take(const f16x8& x) {
        const u32x4 k = __builtin_bit_cast(u32x4, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            low[i] = edge16<false>(low[i], order_of(k[i]));
            high[i] = edge16<true>(high[i], order_of(k[i]));
        }
    }
    __device__ __forceinline__ void meet(int lanes) {  // those `lanes` apart
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            low[i] = edge16<false>(low[i], __shfl_xor((int)low[i], lanes));
            high[i] = edge16<true>(high[i], __shfl_xor((int)high[i], lanes));
        }
    }
    // to and from chunk c of [low, high][d / 2]
    __device__ __forceinline__ void put(uint32_t* e, int c, int d) const {
        *(u32x4*)(e + 4 * c) = u32x4{low[0], low[1], low[2], low[3]};
        *(u32x4*)(e + d / 2 + 4 * c) = u32x4{high[0], high[1], high[2], high[3]};
    }
    __device__ __forceinline__ void take(const uint32_t* e, int c, int d) {
        const u32x4 x = *(const u32x4*)(e + 4 * c), y = *(const u32x4*)(e + d / 2 + 4 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            low[i] = edge16<false>(low[i], x[i]);
            high[i] = edge16<true>(high[i], y[i]);
        }
    }
    // as 16-bit values, with those that the page has (unless it starts anew)
    __device__ __forceinline__ void store(char* bounds, int c, int d, const f16x8& old_low,
                                          const f16x8& old_high, bool anew) {
        const u32x4 x = __builtin_bit_cast(u32x4, old_low), y = __builtin_bit_cast(u32x4, old_high);
        u32x4 l, h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            l[i] = of_order(anew ? low[i] : edge16<false>(low[i], order_of(x[i])));
            h[i] = of_order(anew ? high[i] : edge16<true>(high[i], order_of(y[i])));
        }
        *(u32x4*)(bounds + 16 * c) = l;
        *(u32x4*)(bounds + 2 * d + 16 * c) = h;
    }
};

// q (to its output) or k (to its page) of a run.  kBounds: k with bounds, one
// head for each of the workgroup's sets of groups.
template <bool kBf16, bool kFour, bool kInterleaved, bool kQ, bool kBounds>
__device__ __forceinline__ void append_turned(const AppendRun& r, uint32_t* edges) {
    const auto& a = attn_args<AppendArgs>();
    const int lanes = 1 << a.lanes, tokens = 1 << a.tokens, group = threadIdx.x >> a.lanes;
    const int u = threadIdx.x & (lanes - 1), t = group & (tokens - 1);
    const int h_first = group >> a.tokens, h_step = kAppendThreads >> (a.lanes + a.tokens);
    const int pairs = a.pairs, turned = (kInterleaved ? 2 : 1) * pairs / 8;
    const bool in = u < a.units, turns = u < turned, two = turns && !kInterleaved;
    // chunks of the lane: c0, and where pairs lie apart c1
    const int c0 = turns ? u : pairs / 4 + u - turned, c1 = pairs / 8 + u;
    constexpr int kN = kInterleaved ? 4 : 8;
    // the page's bounds, read long before they are needed
    Edges e0, e1;
    f16x8 old[4] = {};
    char* bounds = nullptr;
    const bool anew = ((r.place0 + r.i0) & ((1 << a.c.shift) - 1)) == 0;
    const bool mine = kBounds && in && t == 0 && h_first < r.heads;
    if constexpr (kBounds) {
        e0.none();
        e1.none();
        bounds = a.bounds + ((int64_t)r.page * a.heads_kv + r.h0 + h_first) * 4 * a.d;
        if (mine && !anew) {
            old[0] = *(const f16x8*)(bounds + 16 * c0);
            old[1] = *(const f16x8*)(bounds + 2 * a.d + 16 * c0);
            if (two) {
                old[2] = *(const f16x8*)(bounds + 16 * c1);
                old[3] = *(const f16x8*)(bounds + 2 * a.d + 16 * c1);
            }
        }
    }
    for (int i0 = r.i0; i0 < (kQ ? r.i1 : r.t1); i0 += tokens) {
        const int i = i0 + t;
        const bool put = in && i < (kQ ? r.i1 : r.t1);
        // the row's places in and out, and a head's distance
        const char* from;
        char* to;
        int64_t from_hs, to_hs;
        int scale_at = 0;
        {
            const auto& z = attn_args<AppendArgs>();
            const auto& src = kQ ? z.q : z.k;
            from_hs = src.hs;
            from = src.p + r.b * src.bs + i * src.rs + (r.h0 + h_first) * from_hs;
            if constexpr (kQ) {
                to_hs = z.q_out.hs;
                to = z.q_out.p + r.b * z.q_out.bs + i * z.q_out.rs;
            } else {
                const int at = (r.place0 + i) & ((1 << z.c.shift) - 1);
                to_hs = z.c.k_hs;
                to = z.c.k + r.page * z.c.k_ps + at * (kFour ? z.d / 2 : z.c.k_rs);
                scale_at = (z.d / 2 << z.c.shift) - at * (z.d / 2 - 4);
            }
            to += (r.h0 + h_first) * to_hs;
        }
        // (a head's values are on their way while those before it are turned)
        f16x8 x{}, y{};
        auto load = [&](int h) {
            if (put && h < r.heads) {
                x = *(const f16x8*)(from + 16 * c0);
                if (two) y = *(const f16x8*)(from + 16 * c1);
            }
        };
        load(h_first);
        double2 cs[kN];
        if (turns && put) {
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const auto& a = attn_args<AppendArgs>();
                const int p = kN * u + j;
                double rev = 0.0;
                if (a.positions == nullptr) {
                    rev = axis_turns((double)(r.place0 + i), a.freqs[p]);
                } else {
                    for (int x = 0; x < a.axes; ++x)
                        rev += axis_turns(position(a.positions, a.type,
                                                   x * a.p_as + r.b * a.p_bs + i * a.p_rs),
                                          a.freqs[x * pairs + p]);
                }
                cs[j] = turn_cos_sin(rev - rint(rev));
            }
        }
        for (int h = h_first; h < r.heads; h += h_step, to += h_step * to_hs) {
            f16x8 lo = x, hi{};
            const f16x8 x0 = x, y0 = y;
            from += h_step * from_hs;
            if constexpr (!kBounds) load(h + h_step);
            if (turns) turn8<kBf16, kInterleaved>(x0, y0, cs, lo, hi);
            if constexpr (!kQ && kFour) {
                const RowCodes<kBf16> codes(top_of_lanes(put ? max(top8(lo), two ? top8(hi) : 0u) : 0u, lanes));
                if (put) {
                    *(uint32_t*)(to + 4 * c0) = codes(lo);
                    if (two) *(uint32_t*)(to + 4 * c1) = codes(hi);
                    if (u == 0) *(float*)(to + scale_at) = codes.scale;
                }
            } else if (put) {
                *(f16x8*)(to + 16 * c0) = lo;
                if (two) *(f16x8*)(to + 16 * c1) = hi;
            }
            if constexpr (kBounds) {
                if (put) {
                    e0.take(lo);
                    if (two) e1.take(hi);
                }
                break;  // (its only head)
            }
        }
    }
    if constexpr (kBounds) {
        const auto& a = attn_args<AppendArgs>();
        const int d = a.d, w = threadIdx.x >> 6;
        for (int o = lanes; o < lanes * tokens && o < 64; o *= 2) {
            e0.meet(o);
            if (two) e1.meet(o);
        }
        if (lanes * tokens > 64) {  // (a head's rows lie in several waves)
            const int waves = lanes * tokens / 64;
            uint32_t* e = edges + w * d;
            if (in && (threadIdx.x & 63) < lanes) {
                e0.put(e, c0, d);
                if (two) e1.put(e, c1, d);
            }
            __syncthreads();
            if (mine)
                for (int k = 1; k < waves; ++k) {
                    e0.take(e + k * d, c0, d);
                    if (two) e1.take(e + k * d, c1, d);
                }
        }
        if (mine) {
            e0.store(bounds, c0, d, old[0], old[1], anew);
            if (two) e1.store(bounds, c1, d, old[2], old[3], anew);
        }
    }
}

template <bool kBf16, bool kFour, bool kInterleaved, bool kBounds>
__global__ __launch_bounds__(kAppendThreads) void cache_append_kernel(AppendArgs) {
    const auto& a = attn_args<AppendArgs>();
    __shared__ __attribute__((aligned(16))) uint32_t edges[kBounds ? kAppendWaves * 128 : 4];
    // k first: with bounds its runs are the longest
    int part = blockIdx.y;
    const bool is_k = part < a.parts_k;
    if (!is_k) part -= a.parts_k;
    const bool is_v = !is_k && part < a.parts_v, is_q = !is_k && !is_v;
    if (is_q) part -= a.parts_v;
    AppendRun r;
    r.b = fdiv(is_k ? a.div_segments_k : a.div_segments, blockIdx.x);
    if (r.b >= a.batch) return;  // (k's runs may be longer, and fewer)
    const int seg = blockIdx.x - r.b * (is_k ? a.segments_k : a.segments), run = is_k ? a.run_k : a.run;
    // (not taken into the table's places: a token past them is not written, one
    // that is moved back would be, over another)
    const int kv = cache_length(scalar_load(a.c.kv_lens + r.b), kAppendPlaces);
    const int fresh = cache_new(a.c, r.b, a.seqlen);
    // rows i0 .. i1 - 1 of the call, at places place0 + i
    r.place0 = kv - fresh;
    const int run0 = ((r.place0 >> run) + seg) << run;
    r.i0 = max(run0 - r.place0, 0);
    r.i1 = min(run0 + (1 << run) - r.place0, a.seqlen);
    if (r.i0 >= r.i1) return;
    // tokens among them: i0 .. t1 - 1 (a place below 0 or past the table, or a page
    // that is none: not written)
    r.page = -1;
    if (run0 >= 0 && r.i0 < fresh && run0 < a.c.width << a.c.shift)
        r.page = cache_page_scalar(a.c, r.b, (r.place0 + r.i0) >> a.c.shift);
    r.t1 = r.page >= 0 ? min(r.i1, fresh) : r.i0;
    const int per = is_q ? a.hq : is_k ? a.hk : a.hv;
    r.h0 = part * per;
    r.heads = min(per, (is_q ? a.heads_q : a.heads_kv) - r.h0);
    if (is_q) {
        append_turned<kBf16, kFour, kInterleaved, true, false>(r, nullptr);
        return;
    }
    if (r.i0 >= r.t1) return;
    if (is_v) append_v<kBf16, kFour>(r);
    else append_turned<kBf16, kFour, kInterleaved, false, kBounds>(r, edges);
}

struct ReadArgs {
    CacheView c;
    RowsView k, v;
    int seqlen, heads_kv, d, blocks;
    FastDiv div_blocks, div_heads, div_units;
};

// A thread per 8 channels of a row, of k and of v.
template <bool kBf16, bool kFour>
__global__ __launch_bounds__(256) void cache_read_kernel(ReadArgs a) {
    const int bh = fdiv(a.div_blocks, blockIdx.x), x = (blockIdx.x - bh * a.blocks) * 256 + threadIdx.x;
    const int s = fdiv(a.div_units, x), u = x - s * (a.d / 8);
    if (s >= a.seqlen) return;
    const int b = fdiv(a.div_heads, bh), h = bh - b * a.heads_kv;
    const int shift = a.c.shift;
    int page = -1;
    if (s < cache_kv(a.c, b)) page = cache_page(a.c, b, s >> shift);
    const int row = s & ((1 << shift) - 1);
    f16x8 k{}, v{};
    if (page >= 0) {
        const char* pk = a.c.k + page * a.c.k_ps + h * a.c.k_hs;
        const char* pv = a.c.v + page * a.c.v_ps + h * a.c.v_hs;
        if constexpr (kFour) {
            auto rows = [&](const char* p) {
                const f16x8 y = cache_levels8<kBf16>(*(const uint32_t*)(p + row * (a.d / 2) + 4 * u));
                const float scale = *(const float*)(p + (a.d / 2 << shift) + 4 * row);
                f16x8 r;
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = to16<kBf16>(value16<kBf16>(y[i]) * scale);
                return r;
            };
            k = rows(pk);
            v = rows(pv);
        } else {
            k = *(const f16x8*)(pk + row * a.c.k_rs + 16 * u);
            v = *(const f16x8*)(pv + row * a.c.v_rs + 16 * u);
        }
    }
    *(f16x8*)(a.k.p + b * a.k.bs + h * a.k.hs + s * a.k.rs + 16 * u) = k;
    *(f16x8*)(a.v.p + b * a.v.bs + h * a.v.hs + s * a.v.rs + 16 * u) = v;
}

RowsView rows_view(const ShaoboFa3AttnTensor& t) {
    return RowsView{(char*)t.data, 2 * t.batch_stride, 2 * t.head_stride, 2 * t.row_stride};
}
int log2_of(int x) {
    int n = 0;
    while ((1 << n) < x) ++n;
    return n;
}

}  // namespace

CacheView cache_view(const ShaoboFa3Cache& c) {
    const int size = c.bits == 16 ? 2 : 1;
    CacheView v;
    v.k = (char*)c.k.data;
    v.v = (char*)c.v.data;
    v.k_ps = c.k.page_stride * size;
    v.k_hs = c.k.head_stride * size;
    v.k_rs = c.k.row_stride * size;
    v.v_ps = c.v.page_stride * size;
    v.v_hs = c.v.head_stride * size;
    v.v_rs = c.v.row_stride * size;
    v.table = c.page_table;
    v.table_s = c.page_table_stride;
    v.kv_lens = c.kv_lens;
    v.new_lens = c.new_lens;
    v.pages = c.pages;
    v.width = c.width;
    v.shift = log2_of(c.page_size);
    return v;
}

AppendGrid append_grid(const ShaoboFa3CacheAppendParams& p) {
    AppendGrid g{};
    const ShaoboFa3Cache& c = p.cache;
    const int pairs = p.freqs != nullptr ? p.pairs : 0;
    g.units = ((p.interleaved ? 2 : 1) * pairs + c.head_dim - 2 * pairs) / 8;
    while ((1 << g.lanes) < g.units) ++g.lanes;
    // Rows side by side: up to the call's, in a power of two; the groups of
    // lanes that are left share the heads.  A run is as many places; of k with
    // bounds a whole page.
    const int side = kAppendThreads >> g.lanes;
    int run = 1;
    while (run < side && run < p.seqlen) run *= 2;
    if (run > c.page_size) run = c.page_size;
    const int run_k = c.bounds != nullptr ? c.page_size : run;
    g.tokens = log2_of(run);
    g.run = log2_of(run);
    g.run_k = log2_of(run_k);
    auto runs = [&](int n) { return (int)(((int64_t)p.seqlen + n - 2) / n) + 1; };
    g.segments = runs(run);
    g.segments_k = runs(run_k);
    // A token's cosines are formed by every workgroup that turns some of its
    // heads, at a cost of about 8 of them: as many heads each as leave a
    // thousand workgroups to q (k and v: 512), and no fewer than its groups take
    // at once.  (8192 tokens of 32 + 8 heads 43.9 us, with half as many
    // workgroups 42.6, with twice as many 51.5; 2 x 2048 in 4 bits and read back
    // 38.2, 39.5, 43.6.)
    const int at_once = side / run;
    auto share = [&](int heads, int runs, int want) {
        int64_t x = (int64_t)heads * c.batch * runs / want;
        if (x < at_once) x = at_once;
        return (int)(x < 1 ? 1 : x < heads ? x : heads);
    };
    g.hq = p.num_heads_q > 0 ? share(p.num_heads_q, g.segments, 1024) : 1;
    g.hk = share(c.num_heads_kv, g.segments_k, 512);
    g.hv = share(c.num_heads_kv, g.segments, 512);
    if (c.bounds != nullptr) g.hk = at_once < c.num_heads_kv ? at_once : c.num_heads_kv;
    g.parts_q = p.num_heads_q > 0 ? ceil_div(p.num_heads_q, g.hq) : 0;
    g.parts_k = ceil_div(c.num_heads_kv, g.hk);
    g.parts_v = ceil_div(c.num_heads_kv, g.hv);
    const int64_t n = (int64_t)c.batch * g.segments;
    const int parts = g.parts_q + g.parts_k + g.parts_v;
    g.ok = n * parts < kMaxGrid && parts < 65536;
    return g;
}

hipError_t launch_cache_append(const ShaoboFa3CacheAppendParams& p, hipStream_t stream) {
    const AppendGrid g = append_grid(p);
    AppendArgs a{};
    a.c = cache_view(p.cache);
    a.k = rows_view(p.k);
    a.v = rows_view(p.v);
    a.q = rows_view(p.q);
    a.q_out = rows_view(p.q_out);
    a.bounds = (char*)p.cache.bounds;
    a.positions = p.positions;
    a.p_as = p.position_axis_stride;
    a.p_bs = p.position_batch_stride;
    a.p_rs = p.position_row_stride;
    a.freqs = p.freqs;
    a.type = p.position_type;
    a.axes = p.axes;
    a.pairs = p.freqs != nullptr ? p.pairs : 0;
    a.seqlen = p.seqlen;
    a.heads_q = p.num_heads_q;
    a.heads_kv = p.cache.num_heads_kv;
    a.d = p.cache.head_dim;
    a.run = g.run;
    a.segments = g.segments;
    a.run_k = g.run_k;
    a.segments_k = g.segments_k;
    a.batch = p.cache.batch;
    a.hq = g.hq;
    a.hk = g.hk;
    a.hv = g.hv;
    a.parts_k = g.parts_k;
    a.parts_v = g.parts_v;
    a.units = g.units;
    a.div_segments = make_fastdiv(g.segments);
    a.div_segments_k = make_fastdiv(g.segments_k);
    a.div_row = make_fastdiv(a.d / 8);
    a.lanes = g.lanes;
    a.tokens = g.tokens;
    a.div_hv = make_fastdiv(g.hv);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(p.cache.batch * g.segments, g.parts_q + g.parts_k + g.parts_v),
                           dim3(kAppendThreads), 0, stream, a);
    };
    auto pick = [&](auto bf, auto four) {
        constexpr bool kB = decltype(bf)::value, kF = decltype(four)::value;
        if (a.bounds != nullptr)
            p.interleaved ? go(cache_append_kernel<kB, kF, true, true>) : go(cache_append_kernel<kB, kF, false, true>);
        else
            p.interleaved ? go(cache_append_kernel<kB, kF, true, false>) : go(cache_append_kernel<kB, kF, false, false>);
    };
    using T = std::true_type;
    using F = std::false_type;
    const bool four = p.cache.bits == 4;
    if (p.cache.dtype == SHAOBO_FA3_DTYPE_BF16) four ? pick(T{}, T{}) : pick(T{}, F{});
    else four ? pick(F{}, T{}) : pick(F{}, F{});
    return hipGetLastError();
}

hipError_t launch_cache_read(const ShaoboFa3CacheReadParams& p, hipStream_t stream) {
    ReadArgs a{};
    a.c = cache_view(p.cache);
    a.k = rows_view(p.k);
    a.v = rows_view(p.v);
    a.seqlen = p.seqlen;
    a.heads_kv = p.cache.num_heads_kv;
    a.d = p.cache.head_dim;
    a.blocks = ceil_div((int64_t)p.seqlen * (a.d / 8), 256);
    a.div_blocks = make_fastdiv(a.blocks);
    a.div_heads = make_fastdiv(a.heads_kv);
    a.div_units = make_fastdiv(a.d / 8);
    const int grid = p.cache.batch * a.heads_kv * a.blocks;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, stream, a); };
    const bool four = p.cache.bits == 4;
    if (p.cache.dtype == SHAOBO_FA3_DTYPE_BF16)
        four ? go(cache_read_kernel<true, true>) : go(cache_read_kernel<true, false>);
    else four ? go(cache_read_kernel<false, true>) : go(cache_read_kernel<false, false>);
    return hipGetLastError();
}

}  // namespace fa3
