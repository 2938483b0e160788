// Appending to a paged cache with the rotary positions applied on the way, and
// reading it back.
//
// append: a workgroup takes a run of consecutive places of one sequence that
// lies in one page, 16 of them at a time, and some heads of q, of k or of v.
// Cosines and sines are formed once per token and pair, in LDS, for all its
// heads; k's turned rows pass through LDS, where a row's 16 bytes a thread
// become codes and a channel's rows become bounds (the run is then a whole
// page, so that one workgroup owns its bounds).
//
// The turn is fp64 throughout: a row of codes goes by the keys' 16-bit values
// and a level's border by a few of their bits, so an fp32 turn's last bits
// would now and then decide a level; at the vector units' fp64 rate, which is
// fp32's, it stays behind the memory.  (A double becomes 16 bits by way of
// fp32, as a cast does.)
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
    int parts_q, parts_k, batch;
    int units;          // of a turned row: 16-byte pieces (with their partners, where those lie apart)
    FastDiv div_segments, div_segments_k, div_pairs, div_units, div_row, div_hq, div_hk, div_hv;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 16;  // of a run at a time

template <bool kBf16>
__device__ __forceinline__ float value16(_Float16 x) {
    if constexpr (kBf16) return (float)__builtin_bit_cast(__bf16, x);
    else return (float)x;
}

// 8 channels of a row of which the kLanes lanes around hold all: the codes, and
// the row's scale.
template <bool kBf16>
__device__ __forceinline__ uint32_t to_codes(const f16x8& x, int lanes, float* scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[i]) & 0x7FFFu);
    for (int o = lanes / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    const float a = value16<kBf16>(__builtin_bit_cast(_Float16, (uint16_t)top));
    if (top >= (kBf16 ? 0x7F80u : 0x7C00u)) {
        *scale = __builtin_nanf("");
        return 0;
    }
    *scale = a / 6.f;
    // y = 6 x / a, rounded once: on a border between levels exactly, where the
    // conversion takes the even code.  (a is taken into [1/2, 1) first.)
    const int e = __builtin_amdgcn_frexp_expf(a);
    const float m = ldexpf(a, -e), r = top == 0 ? 0.f : 1.f / m;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = 6.f * ldexpf(value16<kBf16>(x[i]), -e), q = t * r;
        y[i] = __builtin_fmaf(__builtin_fmaf(-q, m, t), r, q);
    }
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
    return w;
}

// 8 channels 8 u .. of row `row` of a page and head
template <bool kBf16, bool kFour>
__device__ __forceinline__ void put_row(char* page, int64_t rs, int row, int u, int d, int shift,
                                        const f16x8& x, bool ok) {
    if constexpr (kFour) {
        float scale;
        const uint32_t w = to_codes<kBf16>(x, d / 8, &scale);
        if (!ok) return;
        *(uint32_t*)(page + row * (d / 2) + 4 * u) = w;
        if (u == 0) *(float*)(page + (d / 2 << shift) + 4 * row) = scale;
    } else {
        if (ok) *(f16x8*)(page + row * rs + 16 * u) = x;
    }
}

template <bool kBf16, bool kInterleaved>
__device__ __forceinline__ void turn8(const f16x8& x, const f16x8& y, const double2* cs, f16x8& r,
                                      f16x8& q) {
    if constexpr (kInterleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double a = value16<kBf16>(x[2 * j]), b = value16<kBf16>(x[2 * j + 1]);
            r[2 * j] = to16<kBf16>((float)(a * cs[j].x - b * cs[j].y));
            r[2 * j + 1] = to16<kBf16>((float)(b * cs[j].x + a * cs[j].y));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double a = value16<kBf16>(x[j]), b = value16<kBf16>(y[j]);
            r[j] = to16<kBf16>((float)(a * cs[j].x - b * cs[j].y));
            q[j] = to16<kBf16>((float)(b * cs[j].x + a * cs[j].y));
        }
    }
}

// One run's rows of some heads.  (The arguments are read where they are used:
// held in scalar registers they do not fit.)
struct AppendRun {
    int b, run0, place0, i0, i1, t0, t1, page, h0, heads;
};

// v, or k from LDS (kept): rows c0 .. c0 + n - 1 to the run's page.
template <bool kBf16, bool kFour, bool kV>
__device__ __forceinline__ void put_rows(const AppendRun& r, int c0, int n, const _Float16* kept) {
    const auto& a = attn_args<AppendArgs>();
    const int d = a.d, units = d / 8, per = kV ? a.hv : a.hk, shift = a.c.shift, total = n * per * units;
    for (int x0 = 0; x0 < total; x0 += kAppendThreads) {
        const int x = x0 + threadIdx.x, row = fdiv(a.div_row, x), u = x - row * units;
        const int t = fdiv(kV ? a.div_hv : a.div_hk, row), h = row - t * per, i = c0 + t;
        const bool ok = x < total && h < r.heads && i >= r.t0 && i < r.t1;
        f16x8 y{};
        if (ok) {
            if constexpr (kV)
                y = *(const f16x8*)(a.v.p + r.b * a.v.bs + (r.h0 + h) * a.v.hs + i * a.v.rs + 16 * u);
            else
                y = *(const f16x8*)(kept + row * d + 8 * u);
        }
        char* page = kV ? a.c.v + r.page * a.c.v_ps + (r.h0 + h) * a.c.v_hs
                        : a.c.k + r.page * a.c.k_ps + (r.h0 + h) * a.c.k_hs;
        put_row<kBf16, kFour>(page, kV ? a.c.v_rs : a.c.k_rs, (r.place0 + i) & ((1 << shift) - 1), u, d,
                              shift, y, ok);
    }
}

// Cosines and sines of rows c0 .. c0 + n - 1.
__device__ __forceinline__ void turn_table(const AppendRun& r, int c0, int n, double2* turn) {
    const auto& a = attn_args<AppendArgs>();
    for (int x = threadIdx.x; x < n * a.pairs; x += kAppendThreads) {
        const int t = fdiv(a.div_pairs, x), p = x - t * a.pairs, i = c0 + t;
        double rev = 0.0;
        if (a.positions == nullptr) {
            rev = axis_turns((double)(r.place0 + i), a.freqs[p]);
        } else {
            for (int ax = 0; ax < a.axes; ++ax)
                rev += axis_turns(position(a.positions, a.type, ax * a.p_as + r.b * a.p_bs + i * a.p_rs),
                                  a.freqs[ax * a.pairs + p]);
        }
        rev -= rint(rev);
        double sn, cs;
        sincospi(2.0 * rev, &sn, &cs);
        turn[x] = make_double2(cs, sn);
    }
}

// Rows c0 .. c0 + n - 1 of q to its output, or of k to LDS (kept).
template <bool kBf16, bool kInterleaved, bool kQ>
__device__ __forceinline__ void turn_rows(const AppendRun& r, int c0, int n, const double2* turn,
                                          _Float16* kept) {
    const auto& a = attn_args<AppendArgs>();
    const auto& in = kQ ? a.q : a.k;
    const int per = kQ ? a.hq : a.hk, pairs = a.pairs, total = n * per * a.units;
    const int turned = (kInterleaved ? 2 : 1) * pairs / 8;
    for (int x = threadIdx.x; x < total; x += kAppendThreads) {
        const int row = fdiv(a.div_units, x), u = x - row * a.units;
        const int t = fdiv(kQ ? a.div_hq : a.div_hk, row), h = row - t * per, i = c0 + t;
        if (h >= r.heads || (!kQ && (i < r.t0 || i >= r.t1))) continue;
        const char* src = in.p + r.b * in.bs + (r.h0 + h) * in.hs + i * in.rs;
        char* dst = kQ ? a.q_out.p + r.b * a.q_out.bs + (r.h0 + h) * a.q_out.hs + i * a.q_out.rs
                       : (char*)(kept + row * a.d);
        if (u >= turned) {
            const int e = 4 * pairs + 16 * (u - turned);
            *(f16x8*)(dst + e) = *(const f16x8*)(src + e);
            continue;
        }
        const f16x8 y = *(const f16x8*)(src + 16 * u);
        f16x8 z = y, lo, hi = y;
        if constexpr (!kInterleaved) z = *(const f16x8*)(src + 2 * pairs + 16 * u);
        turn8<kBf16, kInterleaved>(y, z, turn + t * pairs + (kInterleaved ? 4 : 8) * u, lo, hi);
        *(f16x8*)(dst + 16 * u) = lo;
        if constexpr (!kInterleaved) *(f16x8*)(dst + 2 * pairs + 16 * u) = hi;
    }
}

template <bool kBf16, bool kFour, bool kInterleaved>
__global__ __launch_bounds__(kAppendThreads) void cache_append_kernel(AppendArgs) {
    const auto& a = attn_args<AppendArgs>();
    extern __shared__ __attribute__((aligned(16))) char append_lds[];
    double2* turn = (double2*)append_lds;  // [tokens][pairs] cos, sin
    _Float16* kept = (_Float16*)(append_lds + kAppendTokens * a.pairs * 16);  // [tokens][heads][d]
    int part = blockIdx.y;
    const bool is_q = part < a.parts_q;
    if (!is_q) part -= a.parts_q;
    const bool is_v = !is_q && part >= a.parts_k, is_k = !is_q && !is_v;
    if (is_v) part -= a.parts_k;
    AppendRun r;
    r.b = fdiv(is_k ? a.div_segments_k : a.div_segments, blockIdx.x);
    if (r.b >= a.batch) return;  // (k's runs may be longer, and fewer)
    const int seg = blockIdx.x - r.b * (is_k ? a.segments_k : a.segments), run = is_k ? a.run_k : a.run;
    const int kv = cache_kv(a.c, r.b), fresh = cache_new(a.c, r.b, a.seqlen);
    // rows i0 .. i1 - 1 of the call, at places place0 + i
    r.place0 = kv - fresh;
    r.run0 = ((r.place0 >> run) + seg) << run;
    r.i0 = max(r.run0 - r.place0, 0);
    r.i1 = min(r.run0 + (1 << run) - r.place0, a.seqlen);
    if (r.i0 >= r.i1) return;
    // tokens among them (a place below 0 or a page that is none: not written)
    r.page = -1;
    if (r.run0 >= 0 && r.i0 < fresh) r.page = cache_page_scalar(a.c, r.b, (r.place0 + r.i0) >> a.c.shift);
    r.t0 = r.i0;
    r.t1 = r.page >= 0 ? min(r.i1, fresh) : r.t0;
    const int per = is_q ? a.hq : is_k ? a.hk : a.hv;
    r.h0 = part * per;
    r.heads = min(per, (is_q ? a.heads_q : a.heads_kv) - r.h0);
    if (is_v) {
        put_rows<kBf16, kFour, true>(r, r.i0, r.i1 - r.i0, nullptr);
        return;
    }
    // bounds: this thread's channels 2 c, 2 c + 1 of head tid / (d / 2)
    const int d = a.d, bh = threadIdx.x / (d / 2), bc = 2 * (threadIdx.x - bh * (d / 2));
    const bool bounds = !is_q && a.bounds != nullptr && bh < r.heads && r.t0 < r.t1;
    float low[2] = {__builtin_inff(), __builtin_inff()}, high[2] = {-__builtin_inff(), -__builtin_inff()};
    for (int c0 = r.i0; c0 < r.i1; c0 += kAppendTokens) {
        const int n = min(kAppendTokens, r.i1 - c0);
        if (c0 > r.i0) __syncthreads();
        turn_table(r, c0, n, turn);
        __syncthreads();
        if (is_q) {
            turn_rows<kBf16, kInterleaved, true>(r, c0, n, turn, nullptr);
            continue;
        }
        turn_rows<kBf16, kInterleaved, false>(r, c0, n, turn, kept);
        __syncthreads();
        put_rows<kBf16, kFour, false>(r, c0, n, kept);
        if (bounds) {
            const int per = attn_args<AppendArgs>().hk;
            for (int i = c0; i < min(c0 + n, r.t1); ++i) {
                const _Float16* x = kept + ((i - c0) * per + bh) * d + bc;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float y = value16<kBf16>(x[j]);
                    low[j] = __builtin_elementwise_minimum(low[j], y);
                    high[j] = __builtin_elementwise_maximum(high[j], y);
                }
            }
        }
    }
    if (!bounds) return;
    const auto& z = attn_args<AppendArgs>();
    _Float16* x = (_Float16*)z.bounds + ((int64_t)r.page * z.heads_kv + r.h0 + bh) * 2 * d + bc;
    const bool anew = ((r.place0 + r.t0) & ((1 << z.c.shift) - 1)) == 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (!anew) {
            low[j] = __builtin_elementwise_minimum(low[j], value16<kBf16>(x[j]));
            high[j] = __builtin_elementwise_maximum(high[j], value16<kBf16>(x[d + j]));
        }
        x[j] = to16<kBf16>(low[j]);
        x[d + j] = to16<kBf16>(high[j]);
    }
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
    // A run of 16 places, fewer where the call has fewer; bounds: a whole page.
    int run = 1;
    while (run < kAppendTokens && run < p.seqlen) run *= 2;
    const int run_k = c.bounds != nullptr ? c.page_size : run;
    g.run = log2_of(run);
    g.run_k = log2_of(run_k);
    auto runs = [&](int n) { return (int)(((int64_t)p.seqlen + n - 2) / n) + 1; };
    g.segments = runs(run);
    g.segments_k = runs(run_k);
    // A token's cosines are formed by every workgroup that turns some of its
    // heads, at a cost of about 8 of them: as many heads each as leave a
    // thousand workgroups to q, and few where tokens are few; of k what LDS and
    // the bounds' threads hold (8192 tokens, Hq32 Hkv8 D128: 56 us with 4 of
    // each, APPEND_US with 16 and 8).
    const int64_t n = (int64_t)c.batch * g.segments;
    auto share = [&](int heads, int least) {
        const int64_t x = heads * n / 1024;
        return (int)(x < least ? (least < heads ? least : heads) : x < heads ? x : heads);
    };
    g.hq = p.num_heads_q > 0 ? share(p.num_heads_q, 4) : 1;
    g.hk = share(c.num_heads_kv, 4);
    g.hv = share(c.num_heads_kv, 4);
    const int most = c.bounds != nullptr ? 256 / (c.head_dim / 2) : 8;
    if (g.hk > most) g.hk = most;
    g.parts_q = p.num_heads_q > 0 ? ceil_div(p.num_heads_q, g.hq) : 0;
    g.parts_k = ceil_div(c.num_heads_kv, g.hk);
    g.parts_v = ceil_div(c.num_heads_kv, g.hv);
    int tokens = run_k < kAppendTokens ? run_k : kAppendTokens;
    if (tokens > p.seqlen) tokens = p.seqlen;
    g.lds = (size_t)kAppendTokens * pairs * 16 + (size_t)tokens * g.hk * c.head_dim * 2;
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
    a.parts_q = g.parts_q;
    a.parts_k = g.parts_k;
    a.units = g.units;
    a.div_segments = make_fastdiv(g.segments);
    a.div_segments_k = make_fastdiv(g.segments_k);
    a.div_pairs = make_fastdiv(a.pairs);
    a.div_units = make_fastdiv(g.units);
    a.div_row = make_fastdiv(a.d / 8);
    a.div_hq = make_fastdiv(g.hq);
    a.div_hk = make_fastdiv(g.hk);
    a.div_hv = make_fastdiv(g.hv);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(p.cache.batch * g.segments, g.parts_q + g.parts_k + g.parts_v),
                           dim3(kAppendThreads), g.lds, stream, a);
    };
    auto pick = [&](auto bf, auto four) {
        constexpr bool kB = decltype(bf)::value, kF = decltype(four)::value;
        p.interleaved ? go(cache_append_kernel<kB, kF, true>) : go(cache_append_kernel<kB, kF, false>);
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
