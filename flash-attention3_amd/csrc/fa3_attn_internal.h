// Host-side interface between the attention layer's C entries
// (fa3_attn_api.cpp) and its kernels.  Nothing here is exported.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "fa3_bwd_internal.h"
#include "shaobo_fa3_attn.h"

namespace fa3 {

// One [batch, heads, rows, head_dim] 16-bit tensor; strides in elements.
struct AttnView {
    _Float16* p;
    int64_t bs, hs, rs;
};

// Smallest and largest document of 64 consecutive positions, those with a
// negative one left out: {INT32_MAX, -1} where that leaves none.  Where any
// was left out (or the block ends behind the sequence) lo is complemented.
struct AttnRange {
    int lo, hi;
};

// Masks and score options as the kernels take them (pointers null: absent).
struct AttnMask {
    const int* doc_q;
    const int* doc_k;
    int64_t doc_q_bs, doc_k_bs;
    const AttnRange* range_q;  // [batch][blocks_q], backward only
    const AttnRange* range_k;  // [batch][blocks_k]
    int blocks_q, blocks_k;
    const int* prefix;
    const int* kv_lens;
    const float* slopes;
    int64_t slopes_bs;
    int causal;
    // x = log2-domain score: s c, or with a cap cap2 tanh(s / softcap) from
    // e = exp2(s k1) (see attn_tanh)
    float c, k1, cap2;
    int cap_fine;  // caps large enough that small scores need tanh's series
};

// Caps over this take tanh's series for small scores (fa3_attn_device.h,
// attn_tanh_fine): below it the plain form's error, the cap times 2^-23, is
// under 1.2e-5 of a score's unit.
constexpr float kCapFine = 100.f;
// A mask's score options from a scale and a cap (0: none).
inline void set_scores(AttnMask* m, float scale, float softcap) {
    constexpr float kLog2E = 1.44269504088896340736f;
    m->c = scale * kLog2E;
    if (softcap > 0.f) {
        // (a tiny cap: the largest fp32, so that a score of zero stays one)
        const double k1 = 2.0 * scale / softcap * kLog2E;
        m->k1 = (float)(k1 < -3e38 ? -3e38 : k1 > 3e38 ? 3e38 : k1);
        m->cap2 = softcap * kLog2E;
        m->cap_fine = softcap > kCapFine;
    }
}

// A resolved problem: checked, default scale applied.
struct AttnProblem {
    int batch, heads_q, heads_kv, group, sq, sk, d;
    bool bf16;
    float scale, softcap;
    bool causal, bias, docs;
};

// Workgroups of a launch are held below this: their 256 threads count in 32 bits.
constexpr int64_t kMaxGrid = 1 << 24;
constexpr int kAttnRows = 128;  // rows (or keys) resident per workgroup

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// The forward kernels' arguments.
struct AttnFwdArgs {
    static constexpr bool kPaged = false;
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

struct AttnFwdPlan {
    bool token;  // the kernel for few rows
    int split;   // otherwise: workgroups of 128 / split rows
    int tiles;   // row tiles of a KV head's group * sq rows
    int splits;  // parts of the key axis
    int part;    // 64-key tiles per part
    int jobs;
    size_t range_off, po_off, pl_off, total;
    bool ok;
};
AttnFwdPlan plan_attn_fwd(const AttnProblem& p);

struct AttnBwdPlan {
    int split;     // jobs of 128 / split keys or rows
    int kv_tiles;  // key tiles
    int q_tiles;   // row tiles of a KV head's group * sq rows
    int head_parts, row_parts;  // dKV jobs per key tile: their product
    int sqp;       // rows of the statistics, padded to whole 64-row blocks
    int jobs;
    size_t nlse2_off, ndelta_off, flag_off, range_k_off, range_q_off, part_off, total;
    bool ok;
};
AttnBwdPlan plan_attn_bwd(const AttnProblem& p);

struct AttnBwdArgs {
    AttnView q, k, v, dout, out, dq, dk, dv;
    const float* lse;
    float* softmax_d;
    float* nlse2;   // [batch * heads_q][sqp]
    float* ndelta;
    int* flags;     // [batch * heads_q][sqp / 64]: a row that takes no part
    AttnMask m;
    float scale;
    int heads_q, heads_kv, group, sq, sk, d, sqp;
    int rows;  // group * sq
    int kv_tiles, q_tiles, groups;
    int delta_blocks, q_blocks, k_blocks;  // attn_delta_kernel's: rows, then document ranges
    // dKV jobs per key tile: head_parts ranges of the group's heads times
    // row_parts ranges of the query tiles.  More than one: their fp32 sums go
    // to part [head_parts * row_parts][dV, dK][groups][sk][D] and attn_sum_kernel
    // adds them in order.
    int head_parts, row_parts, parts;
    float* part;
    int rising;
    FastDiv div_hkv, div_group, div_groups, div_gpart, div_hq, div_blocks, div_parts, div_rparts;
};
void launch_attn_bwd_d64_fp16(const AttnBwdArgs&, const AttnBwdPlan&, int cap, bool bias, hipStream_t);
void launch_attn_bwd_d64_bf16(const AttnBwdArgs&, const AttnBwdPlan&, int cap, bool bias, hipStream_t);
void launch_attn_bwd_d128_fp16(const AttnBwdArgs&, const AttnBwdPlan&, int cap, bool bias, hipStream_t);
void launch_attn_bwd_d128_bf16(const AttnBwdArgs&, const AttnBwdPlan&, int cap, bool bias, hipStream_t);

hipError_t launch_attn_fwd(const AttnProblem& p, const ShaoboFa3AttnParams& a, AttnMask m,
                           hipStream_t stream);
hipError_t launch_attn_bwd(const AttnProblem& p, const ShaoboFa3AttnParams& a, AttnMask m,
                           hipStream_t stream);
hipError_t launch_rotary(const ShaoboFa3RotaryParams& p, hipStream_t stream);

}  // namespace fa3
