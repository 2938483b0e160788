// Rotary positions on several axes for one or two tensors (q and k).
//
// A workgroup takes one to eight tokens: it forms their cosines and sines
// once, in LDS, and turns every head's row with them, 16 bytes (or 16 and
// their partners') a thread at a time.  Bound by HBM, x read once and written
// once: B2 S8192 Hq32 + Hkv8 D128 bf16 66-69 us, 4.9-5.1 TB/s, a large copy's
// rate.  Angles are sum_a positions[a] freqs[a][p], reduced to [-1/2, 1/2] turns in
// fp64 with what its products round off carried along (axis_turns): at a
// million positions an fp32 product would be off by 0.06 radians, at 2^40 an
// fp64 one by 0.0002.
#include "fa3_attn_internal.h"
#include "fa3_bwd_device.h"

namespace fa3 {
namespace {

struct RotaryView {
    char* in;
    char* out;
    int64_t ib, ih, ir, ob, oh, orow;  // strides in bytes
    int heads;
    FastDiv div_heads;
    int token_inner;  // rows of a head lie closer than heads of a row
};

struct RotaryArgs {
    RotaryView x[2];
    int tensors;
    const void* positions;
    int64_t p_as, p_bs, p_rs;
    const float* freqs;
    int seqlen, total;  // batch * seqlen
    int axes, pairs, inverse;
    int units;  // of a row: 16-byte pieces turned (with their partners, where those lie apart) or copied
    int tokens;
    FastDiv div_seq, div_pairs, div_units, div_tokens;
};

constexpr int kRotaryThreads = 256;

struct Half {};
struct Bf {};
template <typename T>
struct Chunk {  // 16 bytes
    static constexpr int kN = 8;
    f16x8 v;
};
template <>
struct Chunk<float> {
    static constexpr int kN = 4;
    f32x4 v;
};

template <typename T>
__device__ __forceinline__ void to_f32(const Chunk<T>& c, float (&x)[Chunk<T>::kN]) {
#pragma unroll
    for (int i = 0; i < Chunk<T>::kN; ++i) {
        if constexpr (std::is_same<T, Bf>::value) x[i] = (float)__builtin_bit_cast(__bf16, (_Float16)c.v[i]);
        else x[i] = (float)c.v[i];
    }
}
template <typename T>
__device__ __forceinline__ Chunk<T> from_f32(const float (&x)[Chunk<T>::kN]) {
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < Chunk<T>::kN; ++i) {
        if constexpr (std::is_same<T, float>::value) c.v[i] = x[i];
        else if constexpr (std::is_same<T, Bf>::value) c.v[i] = __builtin_bit_cast(_Float16, (__bf16)x[i]);
        else c.v[i] = (_Float16)x[i];
    }
    return c;
}

__device__ __forceinline__ double position(const void* p, int type, int64_t i) {
    if (type == SHAOBO_FA3_POSITIONS_INT32) return (double)((const int32_t*)p)[i];
    if (type == SHAOBO_FA3_POSITIONS_INT64) return (double)((const int64_t*)p)[i];
    return (double)((const float*)p)[i];
}

// x f / (2 pi) less a whole number of turns, for |x f| up to 2^53 within 2^-50
// of a turn.  g + gl is f / (2 pi), gl what g's rounding left off (an fma gives
// a product's exactly) with the constant's second half; t + tl likewise is its
// product with x.  Whole turns come off t exactly.
__device__ __forceinline__ double axis_turns(double x, double f) {
#pragma clang fp contract(off)
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLow = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
    const double g = f * kTurn, gl = __builtin_fma(f, kTurn, -g) + f * kTurnLow;
    const double t = x * g, tl = __builtin_fma(x, g, -t) + x * gl;
    return (t - rint(t)) + (tl - rint(tl));
}

template <typename T, bool kInterleaved>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a, int type) {
    extern __shared__ __attribute__((aligned(16))) float2 turn[];  // [tokens][pairs] cos, sin
    const int n0 = blockIdx.x * a.tokens, n = min(a.tokens, a.total - n0);
    for (int i = threadIdx.x; i < n * a.pairs; i += kRotaryThreads) {
        const int t = fdiv(a.div_pairs, i), p = i - t * a.pairs;
        const int b = fdiv(a.div_seq, n0 + t), s = n0 + t - b * a.seqlen;
        double rev = 0.0;
        for (int x = 0; x < a.axes; ++x)
            rev += axis_turns(position(a.positions, type, x * a.p_as + b * a.p_bs + s * a.p_rs),
                              a.freqs[x * a.pairs + p]);
        rev -= rint(rev);
        float sn, cs;
        sincospif(2.f * (float)rev, &sn, &cs);
        turn[i] = make_float2(cs, a.inverse ? -sn : sn);
    }
    __syncthreads();
    constexpr int kN = Chunk<T>::kN;
    const int turned = (kInterleaved ? 2 : 1) * a.pairs / kN;
    for (int k = 0; k < a.tensors; ++k) {
        const RotaryView& v = a.x[k];
        const int total = n * v.heads * a.units;
        for (int i = threadIdx.x; i < total; i += kRotaryThreads) {
            const int row = fdiv(a.div_units, i), u = i - row * a.units;
            int t, h;
            if (v.token_inner && n == a.tokens) {
                h = fdiv(a.div_tokens, row);
                t = row - h * a.tokens;
            } else {
                t = fdiv(v.div_heads, row);
                h = row - t * v.heads;
            }
            const int b = fdiv(a.div_seq, n0 + t), s = n0 + t - b * a.seqlen;
            const char* in = v.in + b * v.ib + h * v.ih + s * v.ir;
            char* out = v.out + b * v.ob + h * v.oh + s * v.orow;
            if (u >= turned) {
                const int e = 2 * a.pairs * (16 / kN) + 16 * (u - turned);
                *(Chunk<T>*)(out + e) = *(const Chunk<T>*)(in + e);
                continue;
            }
            const float2* cs = turn + t * a.pairs + (kInterleaved ? kN / 2 : kN) * u;
            float x[kN], r[kN];
            to_f32(*(const Chunk<T>*)(in + 16 * u), x);
            if constexpr (kInterleaved) {
#pragma unroll
                for (int j = 0; j < kN / 2; ++j) {
                    const float2 c = cs[j];
                    r[2 * j] = x[2 * j] * c.x - x[2 * j + 1] * c.y;
                    r[2 * j + 1] = x[2 * j + 1] * c.x + x[2 * j] * c.y;
                }
            } else {
                const int far = a.pairs * (16 / kN);
                float y[kN], q[kN];
                to_f32(*(const Chunk<T>*)(in + far + 16 * u), y);
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    const float2 c = cs[j];
                    r[j] = x[j] * c.x - y[j] * c.y;
                    q[j] = y[j] * c.x + x[j] * c.y;
                }
                *(Chunk<T>*)(out + far + 16 * u) = from_f32<T>(q);
            }
            *(Chunk<T>*)(out + 16 * u) = from_f32<T>(r);
        }
    }
}

}  // namespace

hipError_t launch_rotary(const ShaoboFa3RotaryParams& p, hipStream_t stream) {
    const int size = p.dtype == SHAOBO_FA3_DTYPE_FP32 ? 4 : 2;
    RotaryArgs a{};
    a.tensors = p.tensors;
    for (int k = 0; k < p.tensors; ++k) {
        RotaryView& v = a.x[k];
        const ShaoboFa3AttnTensor &i = p.in[k], &o = p.out[k];
        v.in = (char*)i.data;
        v.out = (char*)o.data;
        v.ib = i.batch_stride * size;
        v.ih = i.head_stride * size;
        v.ir = i.row_stride * size;
        v.ob = o.batch_stride * size;
        v.oh = o.head_stride * size;
        v.orow = o.row_stride * size;
        v.heads = p.heads[k];
        v.div_heads = make_fastdiv(v.heads);
        v.token_inner = i.row_stride < i.head_stride;
    }
    a.positions = p.positions;
    a.p_as = p.position_axis_stride;
    a.p_bs = p.position_batch_stride;
    a.p_rs = p.position_row_stride;
    a.freqs = p.freqs;
    a.seqlen = p.seqlen;
    a.total = p.batch * p.seqlen;
    a.axes = p.axes;
    a.pairs = p.pairs;
    const int n = 16 / size;
    a.units = ((p.interleaved ? 2 : 1) * p.pairs + p.head_dim - 2 * p.pairs) / n;
    a.inverse = p.inverse;
    // As many tokens as keep a workgroup's threads busy a few times over, and
    // workgroups enough for the chip.
    int heads = 0;
    for (int k = 0; k < p.tensors; ++k) heads += p.heads[k];
    a.tokens = 1;
    while (a.tokens < 8 && a.tokens * heads * a.units < 2048 && a.total / (2 * a.tokens) >= 1024)
        a.tokens *= 2;
    a.div_seq = make_fastdiv(p.seqlen);
    a.div_pairs = make_fastdiv(p.pairs);
    a.div_units = make_fastdiv(a.units);
    a.div_tokens = make_fastdiv(a.tokens);
    const size_t lds = (size_t)a.tokens * p.pairs * 8;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(ceil_div(a.total, a.tokens)), dim3(kRotaryThreads), lds,
                           stream, a, (int)p.position_type);
    };
    if (p.dtype == SHAOBO_FA3_DTYPE_FP32) p.interleaved ? go(rotary_kernel<float, true>) : go(rotary_kernel<float, false>);
    else if (p.dtype == SHAOBO_FA3_DTYPE_BF16) p.interleaved ? go(rotary_kernel<Bf, true>) : go(rotary_kernel<Bf, false>);
    else p.interleaved ? go(rotary_kernel<Half, true>) : go(rotary_kernel<Half, false>);
    return hipGetLastError();
}

}  // namespace fa3
