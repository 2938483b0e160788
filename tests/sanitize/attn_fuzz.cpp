// Host-side fuzz of the attention layer's C entries under AddressSanitizer /
// UndefinedBehaviorSanitizer (built by tests/sanitize/Makefile; no GPU needed).
// Random parameter structs -- valid ones, single-field mutations and absurd
// values -- go through every check, plan and workspace query, and with null
// tensors through the entries themselves, so that each call returns before any
// HIP call.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "shaobo_fa3_attn.h"

namespace {

std::mt19937_64 rng(20261206);

int32_t pick_int() {
    static const int32_t edge[] = {0,    1,     -1,      2,       7,       8,          64,         128,
                                   1000, 65536, 1 << 20, 1 << 24, 1 << 30, (1 << 30) + 8, 0x7FFFFFF8, 0x7FFFFFFF,
                                   INT32_MIN};
    if (rng() % 3 == 0) return (int32_t)rng();
    return edge[rng() % (sizeof(edge) / sizeof(edge[0]))];
}
int64_t pick_stride() {
    static const int64_t edge[] = {0, 8, -8, 4, 128, 1ll << 40, INT64_MAX, INT64_MIN, INT64_MAX - 7};
    return edge[rng() % (sizeof(edge) / sizeof(edge[0]))];
}
float pick_float() {
    static const float edge[] = {0.f, 1.f, -1.f, 1e-45f, 1e30f, 1e31f, -1e30f, INFINITY, NAN, 30.f};
    return edge[rng() % (sizeof(edge) / sizeof(edge[0]))];
}
// somewhere: its place counts, what it holds is not read
template <typename T>
T* maybe(T* p) {
    return rng() % 2 ? p : nullptr;
}

void strides(ShaoboFa3AttnTensor* t) {
    t->batch_stride = pick_stride();
    t->head_stride = pick_stride();
    t->row_stride = pick_stride();
}

int32_t word;
float number;

void random_attn(ShaoboFa3AttnParams* p) {
    shaobo_fa3_attn_params_init(p);
    const bool plausible = rng() % 3 != 0;
    if (plausible) {
        p->batch = 1 + (int)(rng() % 64);
        p->num_heads_kv = 1 + (int)(rng() % 16);
        p->num_heads_q = p->num_heads_kv * (1 << (rng() % 8));
        p->seqlen_q = (int)(rng() >> (34 + rng() % 29));
        p->seqlen_k = (int)(rng() >> (34 + rng() % 29));
        p->head_dim = 8 * (1 + (int)(rng() % 16));
        p->causal = (int)(rng() % 2);
        p->dtype = (int)(rng() % 2);
        if (p->causal) p->prefix_lens = maybe(&word);
        p->documents_q = p->documents_k = maybe(&word);
        p->slopes = maybe(&number);
        p->kv_lens = maybe(&word);
        if (rng() % 4 == 0) p->softcap = 50.f;
    }
    const int n = plausible ? (int)(rng() % 3) : 4 + (int)(rng() % 12);
    for (int i = 0; i < n; ++i) {
        switch (rng() % 14) {
            case 0: p->batch = pick_int(); break;
            case 1: p->seqlen_q = pick_int(); break;
            case 2: p->seqlen_k = pick_int(); break;
            case 3: p->num_heads_q = pick_int(); break;
            case 4: p->num_heads_kv = pick_int(); break;
            case 5: p->head_dim = pick_int(); break;
            case 6: p->dtype = pick_int(); break;
            case 7: p->causal = pick_int(); break;
            case 8: p->softmax_scale_is_set = (int)(rng() % 3); p->softmax_scale = pick_float(); break;
            case 9: p->softcap = pick_float(); break;
            case 10: strides(&p->q); break;
            case 11: strides(&p->dk); break;
            case 12: p->struct_size = (uint32_t)pick_int(); break;
            default: p->documents_q = maybe(&word); break;
        }
    }
    p->workspace_bytes = rng() % 2 ? 0 : ~(size_t)0;
}

void random_rotary(ShaoboFa3RotaryParams* p) {
    shaobo_fa3_rotary_params_init(p);
    p->batch = 1 + (int)(rng() % 8);
    p->seqlen = 1 + (int)(rng() % 8192);
    p->head_dim = 8 * (2 + (int)(rng() % 63));
    p->pairs = 8 * (1 + (int)(rng() % 32));
    p->axes = 1 + (int)(rng() % 4);
    p->tensors = 1 + (int)(rng() % 2);
    p->heads[0] = p->heads[1] = 1 + (int)(rng() % 32);
    const int n = (int)(rng() % 4);
    for (int i = 0; i < n; ++i) {
        switch (rng() % 12) {
            case 0: p->batch = pick_int(); break;
            case 1: p->seqlen = pick_int(); break;
            case 2: p->head_dim = pick_int(); break;
            case 3: p->dtype = pick_int(); break;
            case 4: p->axes = pick_int(); break;
            case 5: p->pairs = pick_int(); break;
            case 6: p->interleaved = pick_int(); break;
            case 7: p->position_type = pick_int(); break;
            case 8: p->tensors = pick_int(); break;
            case 9: p->heads[rng() % 2] = pick_int(); break;
            case 10: strides(&p->in[rng() % 2]); break;
            default: p->struct_size = (uint32_t)pick_int(); break;
        }
    }
}

bool status_ok(int st) { return st >= SHAOBO_FA3_STATUS_SUCCESS && st <= SHAOBO_FA3_STATUS_UNSUPPORTED; }

}  // namespace

int main(int argc, char** argv) {
    const int iters = argc > 1 ? std::atoi(argv[1]) : 20000;
    int seen[3] = {}, rotary_seen[3] = {};
    for (int it = 0; it < iters; ++it) {
        ShaoboFa3AttnParams p;
        random_attn(&p);
        const int fwd = shaobo_fa3_attn_fwd_validate(&p), bwd = shaobo_fa3_attn_bwd_validate(&p);
        const size_t nf = shaobo_fa3_attn_fwd_workspace_bytes(&p);
        const size_t nb = shaobo_fa3_attn_bwd_workspace_bytes(&p);
        if (!status_ok(fwd) || !status_ok(bwd)) return std::printf("status %d %d\n", fwd, bwd), 1;
        if ((fwd && nf) || (bwd && nb)) return std::printf("a workspace for refused parameters\n"), 1;
        // (as much memory as the card has, many times over, is a plan gone wrong)
        if (nf > (1ull << 45) || nb > (1ull << 45)) return std::printf("%zu %zu bytes\n", nf, nb), 1;
        ++seen[fwd];
        // null tensors: refused, or nothing to do
        const int st = shaobo_fa3_attn_fwd(&p, nullptr), sb = shaobo_fa3_attn_bwd(&p, nullptr);
        if (!status_ok(st) || !status_ok(sb)) return std::printf("entries %d %d\n", st, sb), 1;
        ShaoboFa3RotaryParams r;
        random_rotary(&r);
        const int sr = shaobo_fa3_rotary(&r, nullptr);
        if (!status_ok(sr)) return std::printf("rotary %d\n", sr), 1;
        ++rotary_seen[sr];
    }
    std::printf("%d structs: attention %d %d %d, rotary %d %d %d (success, invalid, unsupported)\n",
                iters, seen[0], seen[1], seen[2], rotary_seen[0], rotary_seen[1], rotary_seen[2]);
    return seen[0] && seen[1] && seen[2] && rotary_seen[1] && rotary_seen[2] ? 0 : 1;
}
