// Selecting pages of a cache by what their bounds allow.
//
// cache_score_kernel: sixteen lanes hold a page's two bounds, 8 channels each,
// and sum max(q low, q high) over the channels for four heads of the group at
// a time: the positive part of q meets the upper bound, the negative one the
// lower.  Sums are fp64, so that two pages change places only where their
// scores agree to its last bits; they leave as 64-bit keys of the same order.
// A wave has sixteen pages of bounds on their way; q's parts wait in LDS as
// doubles.  The sixteen sums of a lane's four pages and heads meet in steps that
// halve them, so that a lane ends with one (105 operations, 192 for a sum of
// each over all lanes).  16 sequences of 512 pages, 8 KV heads: 12 us, 23 MB of
// bounds; 2048 pages of one sequence 5.7, latency.
//
// cache_pick_kernel: one workgroup per token and KV head finds the key of the
// last page that is taken, by histograms of 1024 equal ranges between the
// smallest and the largest key in question (one, as a rule, leaves a few keys,
// which one wave ranks), and writes the pages at and above it in their order.  A
// thread has neighbouring pages, in registers unless there are more than
// 4096.  48 of 512 pages, 128 rows: 5.8 us; 64 of 2048, 8 rows: 6.5; the chain
// of its steps, whose barriers wait for one workgroup's eight waves.
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

template <int kCtrl>
__device__ __forceinline__ uint64_t dpp64(uint64_t x) {
    const uint32_t l = __builtin_amdgcn_mov_dpp((int)(uint32_t)x, kCtrl, 0xF, 0xF, false);
    const uint32_t h = __builtin_amdgcn_mov_dpp((int)(uint32_t)(x >> 32), kCtrl, 0xF, 0xF, false);
    return (uint64_t)h << 32 | l;
}
// A lane keeps the upper half of x[0 .. 2 n - 1] (up) or the lower, and adds what
// the lane that a DPP control selects has of it.
template <int kCtrl, int n>
__device__ __forceinline__ void meet(double* x, bool up) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const double keep = up ? x[n + i] : x[i], give = up ? x[i] : x[n + i];
        x[i] = keep + __builtin_bit_cast(double, dpp64<kCtrl>(__builtin_bit_cast(uint64_t, give)));
    }
}
constexpr int kRor8 = 0x128, kHalfMirror = 0x141, kQuad2 = 0x4E, kQuad1 = 0xB1;  // lane ^ 8, ^ 7, ^ 2, ^ 1

template <bool kBf16>
__global__ __launch_bounds__(256, 4) void cache_score_kernel(SelectArgs a) {
    __shared__ double2 parts[kGroupHeads][8][16];  // q's positive and negative part, channel 8 l16 + e
    const int row = fdiv(a.div_chunks, blockIdx.x), chunk = blockIdx.x - row * a.chunks;
    const int bh = fdiv(a.div_seq, row), i = row - bh * a.seqlen;
    const int b = fdiv(a.div_heads, bh), h = bh - b * a.heads_kv;
    const int kv = cache_kv(a.c, b), n = cache_new(a.c, b, a.seqlen);
    const int place = kv - n + i;
    if (i >= n || place < 0) return;  // (padding: the other kernel reads no keys)
    const int own = place >> a.c.shift;
    if (chunk * kScorePages > own) return;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4, w = threadIdx.x >> 6;
    const int first = chunk * kScorePages + 16 * w + g4;  // this lane's pages: every fourth
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
    uint64_t best = 0;  // of page first + 4 (l16 / 4)
    const _Float16* q = a.q + b * a.q_bs + (int64_t)h * a.group * a.q_hs + i * a.q_rs;
    for (int g0 = 0; g0 < a.group; g0 += kGroupHeads) {
        if (g0 > 0) __syncthreads();
        for (int x = threadIdx.x; x < kGroupHeads * 128; x += 256) {
            const int g = x >> 7, c = x & 127;
            // (a group's last heads again where it is no multiple of four: the same maximum)
            const float y = c < a.d ? value16<kBf16>(q[min(g0 + g, a.group - 1) * a.q_hs + c]) : 0.f;
            // (NaN is kept by one of the two)
            parts[g][c & 7][c >> 3] = make_double2(y < 0.f ? 0.f : y, y < 0.f ? y : 0.f);
        }
        __syncthreads();
        double s[4 * kGroupHeads] = {};  // [page][head]
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            wall();  // (one channel's parts at a time in registers)
            double2 y[kGroupHeads];
#pragma unroll
            for (int g = 0; g < kGroupHeads; ++g) y[g] = parts[g][e][l16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // (not unpacked before their turn)
                uint32_t x = __builtin_bit_cast(u32x4, lo[j])[e / 2], z = __builtin_bit_cast(u32x4, hi[j])[e / 2];
                __asm__ volatile("" : "+v"(x), "+v"(z));
                const double l = value16<kBf16>(__builtin_bit_cast(f16x2, x)[e % 2]);
                const double u = value16<kBf16>(__builtin_bit_cast(f16x2, z)[e % 2]);
#pragma unroll
                for (int g = 0; g < kGroupHeads; ++g)
                    s[4 * j + g] = __builtin_fma(y[g].x, u, __builtin_fma(y[g].y, l, s[4 * j + g]));
            }
        }
        wall();
        meet<kRor8, 8>(s, l16 & 8);        // pages 0, 1 or 2, 3
        meet<kHalfMirror, 4>(s, l16 & 4);  // one page
        meet<kQuad2, 2>(s, l16 & 2);
        meet<kQuad1, 1>(s, l16 & 1);       // one head
        uint64_t k = score_key(s[0]);
        const uint64_t k2 = dpp64<kQuad2>(k);
        k = k2 > k ? k2 : k;
        const uint64_t k1 = dpp64<kQuad1>(k);
        k = k1 > k ? k1 : k;
        best = k > best ? k : best;
    }
    const int j = l16 >> 2, p = first + 4 * j;
    int mine = page[0];
#pragma unroll
    for (int x = 1; x < 4; ++x) mine = j == x ? page[x] : mine;
    if ((l16 & 3) == 0 && p <= own)
        a.keys[(int64_t)row * a.c.width + p] = mine < 0 ? 0 : p == own ? kKeyOwn : best;
}

constexpr int kPickThreads = 512;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kBins = 1024;
constexpr int kRank = 64;  // keys that one wave ranks

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int o) {
    const uint32_t l = __shfl_xor((int)(uint32_t)x, o), h = __shfl_xor((int)(uint32_t)(x >> 32), o);
    return (uint64_t)h << 32 | l;
}

// kPer: pages a thread has in registers; 0: as many as there are, read again.
template <int kPer>
__global__ __launch_bounds__(kPickThreads) void cache_pick_kernel(SelectArgs a) {
    __shared__ uint64_t few[kRank];
    __shared__ uint64_t edge[2];
    __shared__ uint32_t bins[kBins];
    __shared__ uint64_t wave_lo[kPickWaves], wave_hi[kPickWaves];
    __shared__ int wave_n[4 * kPickWaves];
    __shared__ int found[3];  // bin, above it, in it
    __shared__ int listed;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int bh = fdiv(a.div_seq, row), i = row - bh * a.seqlen, b = fdiv(a.div_heads, bh);
    const int kv = cache_kv(a.c, b), fresh = cache_new(a.c, b, a.seqlen);
    int* out = a.selected + (int64_t)row * a.count;
    const int place = kv - fresh + i;
    const int n = i < fresh && place >= 0 ? (place >> a.c.shift) + 1 : 0;
    const uint64_t* keys = a.keys + (int64_t)row * a.c.width;
    const int per = kPer > 0 ? kPer : (n + kPickThreads - 1) / kPickThreads;
    // this thread's pages per tid .. (0: none, also past the last)
    uint64_t held[kPer > 0 ? kPer : 1];
    if constexpr (kPer > 0) {
#pragma unroll
        for (int x = 0; x < kPer; ++x) held[x] = kPer * tid + x < n ? keys[kPer * tid + x] : 0;
    }
    auto each = [&](auto use) {
        if constexpr (kPer > 0) {
#pragma unroll
            for (int x = 0; x < kPer; ++x) use(x, held[x]);
        } else {
            for (int x = 0; x < per; ++x) use(x, per * tid + x < n ? keys[per * tid + x] : 0);
        }
    };
    if (tid == 0) listed = 0;
    for (int k = tid; k < kBins; k += kPickThreads) bins[k] = 0;
    // smallest and largest key that is neither none nor past all numbers; how
    // many are past them, and how many there are (in one word)
    uint64_t lo = ~0ull, hi = 0;
    int past = 0, all = 0;
    each([&](int, uint64_t k) {
        all += k != 0;
        past += k >= kKeyTop;
        const bool number = k != 0 && k < kKeyTop;
        lo = number && k < lo ? k : lo;
        hi = number && k > hi ? k : hi;
    });
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
#pragma unroll
    for (int k = 0; k < kPickWaves; ++k) {
        lo = wave_lo[k] < lo ? wave_lo[k] : lo;
        hi = wave_hi[k] > hi ? wave_hi[k] : hi;
        past += wave_n[k];
        all += wave_n[kPickWaves + k];
    }
    // Taken: keys above `last`, and of those equal to it the first `equal`.
    uint64_t last = 0;
    int equal = 0;
    if (all > a.count) {
        int need = a.count;
        if (past >= need) {
            // (one key is above kKeyTop, the own page's, where that is one)
            last = kKeyTop;
            equal = need - (keys[n - 1] == kKeyOwn ? 1 : 0);
        } else {
            need -= past;
            for (;;) {  // (each round divides hi - lo by 1024)
                if (lo == hi) {
                    last = lo;
                    equal = need;
                    break;
                }
                const int bits = 64 - __builtin_clzll(hi - lo), drop = bits > 10 ? bits - 10 : 0;
                each([&](int, uint64_t k) {
                    if (k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> drop], 1u);
                });
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
                bins[kBins - 1 - 2 * tid] = bins[kBins - 2 - 2 * tid] = 0;  // (for another round)
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
                each([&](int, uint64_t k) {
                    if (k >= lo && k <= hi) few[atomicAdd(&listed, 1)] = k;
                });
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
    // In ascending order: how many are above and equal before a thread's own.
    int above = 0, on = 0;
    each([&](int, uint64_t k) {
        above += k > last;
        on += last != 0 && k == last;
    });
    int above0 = above, on0 = on;
    for (int o = 1; o < 64; o *= 2) {
        const int x = __shfl_up(above0, o), y = __shfl_up(on0, o);
        if (lane >= o) {
            above0 += x;
            on0 += y;
        }
    }
    if (lane == 63) {
        wave_n[2 * kPickWaves + w] = above0;
        wave_n[3 * kPickWaves + w] = on0;
    }
    above0 -= above;
    on0 -= on;
    __syncthreads();
    int above_all = 0, on_all = 0;
#pragma unroll
    for (int k = 0; k < kPickWaves; ++k) {
        const int x = wave_n[2 * kPickWaves + k], y = wave_n[3 * kPickWaves + k];
        if (k < w) {
            above0 += x;
            on0 += y;
        }
        above_all += x;
        on_all += y;
    }
    each([&](int x, uint64_t k) {
        const bool is_above = k > last, is_on = last != 0 && k == last;
        const int at = above0 + (on0 < equal ? on0 : equal);
        if ((is_above || (is_on && on0 < equal)) && at < a.count) out[at] = per * tid + x;
        above0 += is_above;
        on0 += is_on;
    });
    const int taken = above_all + (on_all < equal ? on_all : equal);
    for (int p = taken + tid; p < a.count; p += kPickThreads) out[p] = -1;
}

}  // namespace

CacheSelectPlan plan_cache_select(const ShaoboFa3CacheSelectParams& p) {
    CacheSelectPlan f{};
    const int64_t rows = (int64_t)p.cache.batch * p.cache.num_heads_kv * p.seqlen;
    f.chunks = ceil_div(p.cache.width, kScorePages);
    // (kMaxGrid is of workgroups of 256 threads)
    f.ok = rows * (kPickThreads / 256) < kMaxGrid && rows * f.chunks < kMaxGrid;
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
    auto pick = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(rows), dim3(kPickThreads), 0, stream, a);
    };
    if (a.c.width <= kPickThreads) pick(cache_pick_kernel<1>);
    else if (a.c.width <= 2 * kPickThreads) pick(cache_pick_kernel<2>);
    else if (a.c.width <= 4 * kPickThreads) pick(cache_pick_kernel<4>);
    else if (a.c.width <= 8 * kPickThreads) pick(cache_pick_kernel<8>);
    else pick(cache_pick_kernel<0>);
    return hipGetLastError();
}

}  // namespace fa3
