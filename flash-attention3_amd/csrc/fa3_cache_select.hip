// Selecting pages of a cache by what their bounds allow.
//
// cache_score_kernel: sixteen lanes hold a page's two bounds, 8 channels each,
// and sum max(q low, q high) over the channels for four heads of the group at
// a time: the positive part of q meets the upper bound, the negative one the
// lower.  Sums are fp64, so that two pages change places only where their
// scores agree to its last bits; they leave as 64-bit keys of the same order.
// Bound by reading the bounds: a wave has sixteen pages of them on their way.
//
// cache_pick_kernel: one workgroup per token and KV head finds the key of the
// last page that is taken, by histograms of 1024 equal ranges between the
// smallest and the largest key in question (one, as a rule, leaves a few keys,
// which one wave ranks), and writes the pages at and above it in their order.
#include "fa3_cache_device.h"

namespace fa3 {
namespace {

struct SelectArgs {
    CacheView c;
    const _Float16* q;
    int64_t q_bs, q_hs, q_rs;
    const _Float16* bounds;
    uint64_t* keys;  // [batch * heads_kv * seqlen][width]
    int* selected;
    int seqlen, heads_kv, group, d, count, chunks;
    FastDiv div_chunks, div_seq, div_heads;
};

constexpr uint64_t kKeyOwn = ~0ull, kKeyTop = ~0ull - 1;  // the token's own page; a score past all numbers
constexpr int kScorePages = 64;  // a workgroup's: 16 a wave
constexpr int kGroupHeads = 4;   // of a group at a time

// Keys order as the scores do; 0 is below all.
__device__ __forceinline__ uint64_t score_key(double s) {
    if (!(__builtin_fabs(s) < __builtin_inf())) return kKeyTop;
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    return u >> 63 ? ~u : u | (1ull << 63);
}

template <bool kBf16>
__device__ __forceinline__ float value16(_Float16 x) {
    if constexpr (kBf16) return (float)__builtin_bit_cast(__bf16, x);
    else return (float)x;
}

// x + the value of the lane that a DPP control selects
template <int kCtrl>
__device__ __forceinline__ double add_dpp(double x) {
    typedef int i32x2v __attribute__((ext_vector_type(2)));
    const i32x2v u = __builtin_bit_cast(i32x2v, x);
    const i32x2v v = {__builtin_amdgcn_mov_dpp(u[0], kCtrl, 0xF, 0xF, false),
                      __builtin_amdgcn_mov_dpp(u[1], kCtrl, 0xF, 0xF, false)};
    return x + __builtin_bit_cast(double, v);
}
// over 16 lanes: all of them get the sum, in one order
__device__ __forceinline__ double sum16(double x) {
    x = add_dpp<0x128>(x);  // row_ror:8
    x = add_dpp<0x124>(x);
    x = add_dpp<0x122>(x);
    return add_dpp<0x121>(x);
}

template <bool kBf16>
__global__ __launch_bounds__(256) void cache_score_kernel(SelectArgs a) {
    const int row = fdiv(a.div_chunks, blockIdx.x), chunk = blockIdx.x - row * a.chunks;
    const int bh = fdiv(a.div_seq, row), i = row - bh * a.seqlen;
    const int b = fdiv(a.div_heads, bh), h = bh - b * a.heads_kv;
    const int kv = cache_kv(a.c, b), n = cache_new(a.c, b, a.seqlen);
    const int place = kv - n + i;
    if (i >= n || place < 0) return;  // (padding: the other kernel reads no keys)
    const int own = place >> a.c.shift;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4, w = threadIdx.x >> 6;
    const int first = chunk * kScorePages + 16 * w + g4;  // this lane's pages: every fourth
    if (chunk * kScorePages > own) return;
    const bool in = 8 * l16 < a.d;
    int page[4];
    f16x8 lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int p = first + 4 * j;
        page[j] = p <= own ? cache_page(a.c, b, p) : -1;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo[j] = hi[j] = f16x8{};
        if (page[j] >= 0 && in) {
            const _Float16* x = a.bounds + ((int64_t)page[j] * a.heads_kv + h) * 2 * a.d + 8 * l16;
            lo[j] = *(const f16x8*)x;
            hi[j] = *(const f16x8*)(x + a.d);
        }
    }
    double best[4];
    bool past[4];  // a head's score is no number, or infinite
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        best[j] = -__builtin_inf();
        past[j] = false;
    }
    const _Float16* q = a.q + b * a.q_bs + (int64_t)h * a.group * a.q_hs + i * a.q_rs + 8 * l16;
    for (int g0 = 0; g0 < a.group; g0 += kGroupHeads) {
        f16x8 qv[kGroupHeads];
#pragma unroll
        for (int g = 0; g < kGroupHeads; ++g) {
            qv[g] = f16x8{};
            // (a group's last heads again where it is no multiple of four: the same maximum)
            if (in) qv[g] = *(const f16x8*)(q + min(g0 + g, a.group - 1) * a.q_hs);
        }
        double s[4][kGroupHeads] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            double up[kGroupHeads], down[kGroupHeads];
#pragma unroll
            for (int g = 0; g < kGroupHeads; ++g) {
                const float x = value16<kBf16>(qv[g][e]);
                // (NaN is kept by one of the two)
                up[g] = x < 0.f ? 0.f : x;
                down[g] = x < 0.f ? x : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double l = value16<kBf16>(lo[j][e]), u = value16<kBf16>(hi[j][e]);
#pragma unroll
                for (int g = 0; g < kGroupHeads; ++g)
                    s[j][g] = __builtin_fma(up[g], u, __builtin_fma(down[g], l, s[j][g]));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int g = 0; g < kGroupHeads; ++g) {
                const double x = sum16(s[j][g]);
                past[j] |= !(__builtin_fabs(x) < __builtin_inf());
                best[j] = x > best[j] ? x : best[j];
            }
    }
    uint64_t* keys = a.keys + (int64_t)row * a.c.width;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int p = first + 4 * j;
        if (l16 == 0 && p <= own)
            keys[p] = page[j] < 0 ? 0 : p == own ? kKeyOwn : past[j] ? kKeyTop : score_key(best[j]);
    }
}

constexpr int kPickThreads = 512;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kBins = 1024;
constexpr int kRank = 64;         // keys that one wave ranks
constexpr int kPickKeys = 4096;   // of a row, held in LDS; longer rows are read again

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int o) {
    const uint32_t l = __shfl_xor((int)(uint32_t)x, o), h = __shfl_xor((int)(uint32_t)(x >> 32), o);
    return (uint64_t)h << 32 | l;
}

__global__ __launch_bounds__(kPickThreads) void cache_pick_kernel(SelectArgs a) {
    __shared__ uint64_t held[kPickKeys];
    __shared__ uint64_t few[kRank];
    __shared__ uint64_t edge[2];
    __shared__ uint32_t bins[kBins];
    __shared__ uint64_t wave_lo[kPickWaves], wave_hi[kPickWaves];
    __shared__ int wave_n[3 * kPickWaves];
    __shared__ int found[3];  // bin, above it, in it
    __shared__ int listed;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int bh = fdiv(a.div_seq, row), i = row - bh * a.seqlen, b = fdiv(a.div_heads, bh);
    const int kv = cache_kv(a.c, b), fresh = cache_new(a.c, b, a.seqlen);
    int* out = a.selected + (int64_t)row * a.count;
    const int place = kv - fresh + i;
    const int n = i < fresh && place >= 0 ? (place >> a.c.shift) + 1 : 0;
    const uint64_t* keys = a.keys + (int64_t)row * a.c.width;
    // smallest and largest key that is neither none nor past all numbers; how many of each
    uint64_t lo = ~0ull, hi = 0;
    int past = 0, all = 0;
    const bool held_ok = n <= kPickKeys;
    for (int p = tid; p < n; p += kPickThreads) {
        const uint64_t k = keys[p];
        if (held_ok) held[p] = k;
        if (k == 0) continue;
        ++all;
        if (k >= kKeyTop) {
            ++past;
            continue;
        }
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    }
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t l = shfl_xor64(lo, o), h = shfl_xor64(hi, o);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
        past += __shfl_xor(past, o);
        all += __shfl_xor(all, o);
    }
    if (lane == 0) {
        wave_lo[w] = lo;
        wave_hi[w] = hi;
        wave_n[w] = past;
        wave_n[kPickWaves + w] = all;
    }
    __syncthreads();
    past = all = 0;
    for (int k = 0; k < kPickWaves; ++k) {
        lo = wave_lo[k] < lo ? wave_lo[k] : lo;
        hi = wave_hi[k] > hi ? wave_hi[k] : hi;
        past += wave_n[k];
        all += wave_n[kPickWaves + k];
    }
    auto key = [&](int p) { return held_ok ? held[p] : keys[p]; };
    // Taken: keys above `last`, and of those equal to it the first `equal`.
    uint64_t last = 0;
    int equal = 0;
    if (all > a.count) {
        int need = a.count;
        if (past >= need) {  // (the own page is one, where it is there)
            last = kKeyTop;
            equal = need;
            // one key above kKeyTop at most: counted here, not by the histogram
            int own = 0;
            if (n > 0 && key(n - 1) == kKeyOwn) own = 1;
            equal -= own;
        } else {
            need -= past;
            for (;;) {  // (each round divides hi - lo by 1024)
                if (lo == hi) {
                    last = lo;
                    equal = need;
                    break;
                }
                const int bits = 64 - __builtin_clzll(hi - lo), drop = bits > 10 ? bits - 10 : 0;
                for (int k = tid; k < kBins; k += kPickThreads) bins[k] = 0;
                if (tid == 0) listed = 0;
                __syncthreads();
                for (int p = tid; p < n; p += kPickThreads) {
                    const uint64_t k = key(p);
                    if (k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> drop], 1u);
                }
                __syncthreads();
                // thread t has bins 1023 - 2 t and 1022 - 2 t: sums from the top
                const int c0 = bins[kBins - 1 - 2 * tid], c1 = bins[kBins - 2 - 2 * tid];
                int upto = c0 + c1;
                for (int o = 1; o < 64; o *= 2) {
                    const int x = __shfl_up(upto, o);
                    if (lane >= o) upto += x;
                }
                if (lane == 63) wave_n[2 * kPickWaves + w] = upto;
                __syncthreads();
                int before = upto - c0 - c1;
                for (int k = 0; k < w; ++k) before += wave_n[2 * kPickWaves + k];
                if (before < need && need <= before + c0) {
                    found[0] = kBins - 1 - 2 * tid;
                    found[1] = before;
                    found[2] = c0;
                } else if (before + c0 < need && need <= before + c0 + c1) {
                    found[0] = kBins - 2 - 2 * tid;
                    found[1] = before + c0;
                    found[2] = c1;
                }
                __syncthreads();
                const int bin = found[0], in = found[2];
                need -= found[1];
                const uint64_t bottom = lo + ((uint64_t)bin << drop);
                const uint64_t top = bottom + ((1ull << drop) - 1);
                hi = top < hi ? top : hi;
                lo = bottom;
                if (drop == 0 || in > kRank) {
                    __syncthreads();
                    continue;
                }
                for (int p = tid; p < n; p += kPickThreads) {
                    const uint64_t k = key(p);
                    if (k >= lo && k <= hi) few[atomicAdd(&listed, 1)] = k;
                }
                __syncthreads();
                if (w == 0) {
                    const uint64_t mine = lane < in ? few[lane] : 0;
                    int above = 0, same = 0;
                    for (int k = 0; k < in; ++k) {
                        above += few[k] > mine;
                        same += few[k] == mine;
                    }
                    if (lane < in && above < need && need <= above + same) {
                        edge[0] = mine;
                        edge[1] = need - above;
                    }
                }
                __syncthreads();
                last = edge[0];
                equal = (int)edge[1];
                break;
            }
        }
    }
    // In ascending order: pages before a thread's, by ballots.
    int base = 0, same = 0;
    for (int p0 = 0; p0 < n; p0 += kPickThreads) {
        const int p = p0 + tid;
        const uint64_t k = p < n ? key(p) : 0;
        const bool above = k > last, on = last != 0 && k == last;
        const uint64_t ma = __ballot(above), mo = __ballot(on), below = (1ull << lane) - 1;
        __syncthreads();  // (wave_n of the round before has been read)
        if (lane == 0) {
            wave_n[w] = __builtin_popcountll(ma);
            wave_n[kPickWaves + w] = __builtin_popcountll(mo);
        }
        __syncthreads();
        int a0 = base, s0 = same;
        for (int x = 0; x < kPickWaves; ++x) {
            if (x < w) {
                a0 += wave_n[x];
                s0 += wave_n[kPickWaves + x];
            }
            base += wave_n[x];
            same += wave_n[kPickWaves + x];
        }
        const int ra = a0 + __builtin_popcountll(ma & below), rs = s0 + __builtin_popcountll(mo & below);
        const int at = ra + (rs < equal ? rs : equal);
        if ((above || (on && rs < equal)) && at < a.count) out[at] = p;
    }
    const int taken = base + (same < equal ? same : equal);
    for (int p = taken + tid; p < a.count; p += kPickThreads) out[p] = -1;
}

}  // namespace

CacheSelectPlan plan_cache_select(const ShaoboFa3CacheSelectParams& p) {
    CacheSelectPlan f{};
    const int64_t rows = (int64_t)p.cache.batch * p.cache.num_heads_kv * p.seqlen;
    f.chunks = ceil_div(p.cache.width, kScorePages);
    f.ok = rows < kMaxGrid && rows * f.chunks < kMaxGrid;
    f.total = f.ok ? (size_t)rows * p.cache.width * 8 : 0;
    f.total = (f.total + 255) / 256 * 256;
    return f;
}

hipError_t launch_cache_select(const ShaoboFa3CacheSelectParams& p, hipStream_t stream) {
    const CacheSelectPlan f = plan_cache_select(p);
    SelectArgs a{};
    a.c = cache_view(p.cache);
    a.q = (const _Float16*)p.q.data;
    a.q_bs = p.q.batch_stride;
    a.q_hs = p.q.head_stride;
    a.q_rs = p.q.row_stride;
    a.bounds = (const _Float16*)p.cache.bounds;
    a.keys = (uint64_t*)p.workspace;
    a.selected = p.selected;
    a.seqlen = p.seqlen;
    a.heads_kv = p.cache.num_heads_kv;
    a.group = p.num_heads_q / p.cache.num_heads_kv;
    a.d = p.cache.head_dim;
    a.count = p.count;
    a.chunks = f.chunks;
    a.div_chunks = make_fastdiv(f.chunks);
    a.div_seq = make_fastdiv(p.seqlen);
    a.div_heads = make_fastdiv(a.heads_kv);
    const int rows = p.cache.batch * a.heads_kv * p.seqlen;
    if (f.chunks > 0) {
        const dim3 grid(rows * f.chunks);
        if (p.cache.dtype == SHAOBO_FA3_DTYPE_BF16)
            hipLaunchKernelGGL(cache_score_kernel<true>, grid, dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL(cache_score_kernel<false>, grid, dim3(256), 0, stream, a);
    }
    hipLaunchKernelGGL(cache_pick_kernel, dim3(rows), dim3(kPickThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace fa3
