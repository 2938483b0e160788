// Host side of the attention backward: how a problem is cut, and its launch.
#include "fa3_attn_internal.h"

namespace fa3 {
namespace {

AttnView view(const ShaoboFa3AttnTensor& t) {
    return AttnView{(_Float16*)t.data, t.batch_stride, t.head_stride, t.row_stride};
}

}  // namespace

AttnBwdPlan plan_attn_bwd(const AttnProblem& p) {
    AttnBwdPlan f{};
    const int64_t rows = (int64_t)p.group * p.sq, groups = (int64_t)p.batch * p.heads_kv;
    const int D = p.d > 64 ? 128 : 64;
    f.sqp = ceil_div(p.sq, 64) * 64;
    const int64_t q_steps = f.sqp / 64, k_steps = ceil_div(p.sk, 64);
    // How the work is cut: the candidate with the smallest estimate.  In units
    // of 16 products of a 32 x 32 block (a dKV job takes 4 a block, a dQ job 3,
    // and a wave streams 2 / split of them a stage), a launch takes the
    // longer of the work's share of a workgroup slot and the longest job, then
    // the parts' way through memory.  us per unit measured on full chips and
    // on long single jobs; bf16, us, as split / head parts / row parts:
    //   B2 Hq32 Hkv8 S4096 D128 causal   1/1/1  919  2/1/1 1038  2/2/1 1073
    //   B4 Hq16 Hkv4 S1024 D128 capped   1/1/1  228  2/1/1  148  2/2/1  109  1/4/1 107
    //   B1 Hq8 Hkv1 S4096 D128 causal    1/1/1 1373  2/1/1  884  2/8/1  157  2/4/1 250
    //   B1 H7 S1923 D128 causal          1/1/1   98  2/1/1   73  2/1/2   65  2/1/4  85
    //   B8 H8 S512 D128                  1/1/1   41  2/1/1   49  2/1/2   76
    //   B2 H4 S2048 D64 causal           1/1/1   70  2/1/1   52  2/1/2   55
    const double unit = D == 128 ? 0.51 : 0.34, job_unit = D == 128 ? 0.45 : 0.3;
    const double alone_unit = D == 128 ? 0.335 : 0.25;
    const int slots = D == 128 ? 512 : 768;
    const double seen = p.causal ? 0.5 : 1.0;
    double best = 1e30;
    f.split = f.head_parts = f.row_parts = 1;
    for (int split = 1; split <= 2; ++split)
        for (int hp = 1; hp <= p.group; hp = hp * 2 > p.group && hp < p.group ? p.group : hp * 2)
            for (int rp = 1; rp <= 4 && (rp == 1 || rp <= q_steps); rp *= 2) {
                if (hp < p.group && rp > 1) continue;  // (heads are cut first: no step is shared)
                const int64_t kt = ceil_div(p.sk, kAttnRows / split), qt = ceil_div(rows, kAttnRows / split);
                const double per = 2.0 / split;
                const double kv = (double)ceil_div(p.group, hp) * ceil_div(q_steps, rp) * per * 4;
                const double q = (double)k_steps * per * 3;
                const double work = groups * seen *
                                    (kt * (double)p.group * q_steps * per * 4 + qt * q) *
                                    (split == 2 ? 1.13 : 1.0);
                const double jobs = (double)groups * (kt * hp * rp + qt);
                const double job = (kv > q ? kv : q) * (jobs <= 256 ? alone_unit : job_unit);
                const double even = work / slots * unit;
                double us = job > even ? job : even;
                if (hp * rp > 1)
                    us += 4.0 + 16.0 * hp * rp * (double)groups * p.sk * D / 4e6;
                if (us < best) {
                    best = us;
                    f.split = split;
                    f.head_parts = hp;
                    f.row_parts = rp;
                }
            }
    const int keys = kAttnRows / f.split;
    f.kv_tiles = ceil_div(p.sk, keys);
    f.q_tiles = ceil_div(rows, keys);
    const int parts = f.head_parts * f.row_parts;
    const int64_t jobs = groups * ((int64_t)f.kv_tiles * parts + f.q_tiles);
    const int64_t blocks = groups * p.group * q_steps;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t x = at;
        at += (n + 255) / 256 * 256;
        return x;
    };
    f.nlse2_off = take((size_t)blocks * 64 * 4);
    f.ndelta_off = take((size_t)blocks * 64 * 4);
    f.flag_off = take((size_t)blocks * 4);
    f.range_k_off = take(p.docs ? (size_t)p.batch * k_steps * sizeof(AttnRange) : 0);
    f.range_q_off = take(p.docs ? (size_t)p.batch * q_steps * sizeof(AttnRange) : 0);
    f.part_off = take(parts > 1 ? (size_t)2 * parts * groups * p.sk * D * 4 : 0);
    f.total = at;
    const int64_t delta = blocks + ((int64_t)p.batch * (q_steps + k_steps) + 8) / 4;
    f.ok = rows < (1ll << 30) && jobs < kMaxGrid && delta < kMaxGrid &&
           groups * p.sk / 4 < kMaxGrid;
    f.jobs = f.ok ? (int)jobs : 0;
    return f;
}

hipError_t launch_attn_bwd(const AttnProblem& p, const ShaoboFa3AttnParams& a, AttnMask m,
                           hipStream_t stream) {
    const AttnBwdPlan f = plan_attn_bwd(p);
    if (f.jobs == 0) return hipSuccess;
    char* ws = (char*)a.workspace;
    AttnBwdArgs x{};
    x.q = view(a.q);
    x.k = view(a.k);
    x.v = view(a.v);
    x.out = view(a.out);
    x.dout = view(a.dout);
    x.dq = view(a.dq);
    x.dk = view(a.dk);
    x.dv = view(a.dv);
    x.lse = a.softmax_lse;
    x.softmax_d = a.softmax_d;
    x.nlse2 = (float*)(ws + f.nlse2_off);
    x.ndelta = (float*)(ws + f.ndelta_off);
    x.flags = (int*)(ws + f.flag_off);
    x.scale = p.scale;
    x.heads_q = p.heads_q;
    x.heads_kv = p.heads_kv;
    x.group = p.group;
    x.sq = p.sq;
    x.sk = p.sk;
    x.d = p.d;
    x.sqp = f.sqp;
    x.rows = p.group * p.sq;
    x.kv_tiles = f.kv_tiles;
    x.q_tiles = f.q_tiles;
    x.groups = p.batch * p.heads_kv;
    x.div_hkv = make_fastdiv(p.heads_kv);
    x.div_group = make_fastdiv(p.group);
    x.div_groups = make_fastdiv(x.groups);
    x.div_gpart = make_fastdiv(x.groups / 8);
    x.div_hq = make_fastdiv(p.heads_q);
    x.div_blocks = make_fastdiv(f.sqp / 64);
    x.head_parts = f.head_parts;
    x.row_parts = f.row_parts;
    x.parts = f.head_parts * f.row_parts;
    x.div_parts = make_fastdiv(x.parts);
    x.rising = p.causal && f.jobs <= 512;
    x.div_rparts = make_fastdiv(f.row_parts);
    x.part = (float*)(ws + f.part_off);
    x.delta_blocks = x.groups * p.group * (f.sqp / 64);
    if (p.docs) {
        m.range_k = (AttnRange*)(ws + f.range_k_off);
        m.range_q = (AttnRange*)(ws + f.range_q_off);
        m.blocks_k = ceil_div(p.sk, 64);
        m.blocks_q = f.sqp / 64;
        x.q_blocks = p.batch * m.blocks_q;
        // (one set of documents for both: one set of ranges)
        if (m.doc_k == m.doc_q && m.doc_k_bs == m.doc_q_bs && p.sk == p.sq) m.range_k = m.range_q;
        else x.k_blocks = p.batch * m.blocks_k;
    }
    x.m = m;
    const int cap = p.softcap > 0.f ? m.cap_fine ? 2 : 1 : 0;
    auto launch = p.d > 64 ? p.bf16 ? launch_attn_bwd_d128_bf16 : launch_attn_bwd_d128_fp16
                           : p.bf16 ? launch_attn_bwd_d64_bf16 : launch_attn_bwd_d64_fp16;
    launch(x, f, cap, p.bias, stream);
    return hipGetLastError();
}

}  // namespace fa3
