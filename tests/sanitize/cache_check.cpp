// What the cache's kernels make of a page table's entries and of lengths, the
// launches' plans over random problems, and a fuzz of the C entries, under
// AddressSanitizer / UndefinedBehaviorSanitizer (built by
// tests/sanitize/Makefile; no GPU needed: null tensors end every call before
// any HIP call).
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "fa3_cache_internal.h"

namespace {

std::mt19937_64 rng(20261208);

int32_t pick_int() {
    static const int32_t edge[] = {0, 1, -1, 2, 3, 4, 8, 16, 32, 64, 65, 128, 1000, 1024, 2048, 65536, 1 << 20,
                                   1 << 24, 1 << 30, 0x7FFFFFF8, 0x7FFFFFFF, INT32_MIN};
    if (rng() % 3 == 0) return (int32_t)rng();
    return edge[rng() % (sizeof(edge) / sizeof(edge[0]))];
}
int64_t pick_stride() {
    static const int64_t edge[] = {0, 8, -8, 4, 16, 128, 1ll << 40, INT64_MAX, INT64_MIN, INT64_MAX - 7};
    return edge[rng() % (sizeof(edge) / sizeof(edge[0]))];
}
float pick_float() {
    static const float edge[] = {0.f, 1.f, -1.f, 1e-45f, 1e30f, 1e31f, -1e30f, INFINITY, NAN, 30.f};
    return edge[rng() % (sizeof(edge) / sizeof(edge[0]))];
}
float number;
int32_t word;

void random_cache(ShaoboFa3Cache* c, bool plausible) {
    if (plausible) {
        c->batch = 1 + (int)(rng() % 64);
        c->num_heads_kv = 1 + (int)(rng() % 16);
        c->head_dim = rng() % 2 ? 128 : 64;
        c->dtype = (int)(rng() % 2);
        c->bits = rng() % 2 ? 16 : 4;
        c->pages = (int)(rng() >> 40);
        c->page_size = 32 << (rng() % 6);
        c->width = (int)(rng() >> (50 + rng() % 10));
    }
    const int n = plausible ? (int)(rng() % 3) : 4 + (int)(rng() % 10);
    for (int i = 0; i < n; ++i) {
        switch (rng() % 12) {
            case 0: c->batch = pick_int(); break;
            case 1: c->num_heads_kv = pick_int(); break;
            case 2: c->head_dim = pick_int(); break;
            case 3: c->dtype = pick_int(); break;
            case 4: c->bits = pick_int(); break;
            case 5: c->pages = pick_int(); break;
            case 6: c->page_size = pick_int(); break;
            case 7: c->width = pick_int(); break;
            case 8: c->k.page_stride = pick_stride(); break;
            case 9: c->v.head_stride = pick_stride(); break;
            case 10: c->k.row_stride = pick_stride(); break;
            default: c->bounds = rng() % 2 ? (void*)(1 << 20) : nullptr; break;
        }
    }
}
void random_rows(ShaoboFa3AttnTensor* t) {
    if (rng() % 8 == 0) t->head_stride = pick_stride();
}
bool status_ok(int st) { return st >= SHAOBO_FA3_STATUS_SUCCESS && st <= SHAOBO_FA3_STATUS_UNSUPPORTED; }

int fail(const char* what) {
    std::printf("%s\n", what);
    return 1;
}

// Every key of every row is in one part, for any length a sequence may have
// (what cache_span and cache_tile_kernel cut on the GPU).
bool parts_cover(int n, int splits, int least, int round) {
    const int part = std::max(((n + splits - 1) / splits + round - 1) / round * round, least);
    int64_t seen = 0;
    for (int s = 0; s < splits; ++s) {
        const int64_t at = (int64_t)s * part;
        const int begin = at < n ? (int)at : n;
        const int end = n - begin > part ? begin + part : n;
        if (begin < seen || (begin > seen && begin < n)) return false;
        seen = end;
    }
    return seen == n;
}

}  // namespace

int main(int argc, char** argv) {
    const int iters = argc > 1 ? std::atoi(argv[1]) : 20000;
    const int entries[] = {INT32_MIN, -2, -1, 0, 1, 9, 10, 11, INT32_MAX};
    for (int e : entries)
        for (int pages : {0, 1, 10, INT32_MAX}) {
            const int p = fa3::cache_page_of(e, pages), n = fa3::cache_length(e, pages);
            if (p != (e >= 0 && e < pages ? e : -1)) return fail("page");
            if (n < 0 || n > pages || (e >= 0 && e <= pages && n != e)) return fail("length");
        }
    int seen[3] = {}, dealt = 0;
    for (int it = 0; it < iters; ++it) {
        const bool plausible = rng() % 4 != 0;
        ShaoboFa3CacheAttnParams a;
        shaobo_fa3_cache_attn_params_init(&a);
        random_cache(&a.cache, plausible);
        a.seqlen = plausible ? (int)(rng() >> (48 + rng() % 15)) : pick_int();
        a.num_heads_q = plausible ? (int32_t)((uint32_t)a.cache.num_heads_kv << (rng() % 7)) : pick_int();
        a.causal = (int)(rng() % (plausible ? 2 : 4));
        if (rng() % 6 == 0) a.softmax_scale = pick_float(), a.softmax_scale_is_set = (int)(rng() % 3);
        if (rng() % 6 == 0) a.softcap = pick_float();
        if (rng() % 3 == 0) a.slopes = &number;
        if (rng() % 3 == 0) a.selected = &word, a.count = plausible ? 1 + (int)(rng() % 200) : pick_int();
        random_rows(&a.q);
        random_rows(&a.out);
        const int st = shaobo_fa3_cache_attn_validate(&a);
        const size_t need = shaobo_fa3_cache_attn_workspace_bytes(&a);
        if (!status_ok(st)) return fail("status");
        if (st && need) return fail("a workspace for refused parameters");
        if (need > (1ull << 45)) return std::printf("%zu bytes\n", need), 1;
        ++seen[st];
        if (!status_ok(shaobo_fa3_cache_attn(&a, nullptr))) return fail("attn");
        if (st == SHAOBO_FA3_STATUS_SUCCESS && plausible) {
            fa3::CacheProblem p{};
            p.batch = a.cache.batch;
            p.heads_q = a.num_heads_q;
            p.heads_kv = a.cache.num_heads_kv;
            p.group = p.heads_q / p.heads_kv;
            p.sq = a.seqlen;
            p.d = a.cache.head_dim;
            p.sk = a.cache.width * a.cache.page_size;
            p.page = a.cache.page_size;
            p.count = a.selected ? a.count : 0;
            p.four = a.cache.bits == 4;
            p.causal = a.causal != 0;
            const fa3::CachePlan f = fa3::plan_cache_attn(p);
            if (!f.ok || f.splits < 1) return fail("plan");
            if (f.slots > 0) {
                if (f.slots <= p.batch || p.batch > fa3::kDealBatch || f.splits > 1 ||
                    f.jobs != f.slots * p.heads_kv)
                    return fail("slots");
                uint32_t total = 0;
                std::vector<uint32_t> n(p.batch);
                const int shape = (int)(rng() % 3);
                for (uint32_t& x : n) {
                    const uint32_t most = p.sk / 32 + 1;
                    x = (uint32_t)(rng() % (shape == 0 || (shape == 1 && rng() % 8 == 0) ? most : most < 16 ? most : 16));
                    total += x;
                }
                auto count = [&](uint32_t part) {
                    uint32_t s = 0;
                    for (uint32_t x : n) s += std::max(1u, (x + part - 1) / part);
                    return s;
                };
                const uint32_t part = fa3::deal_part(total, f.slots, p.batch, 2, count);
                if (part < 2 || count(4 * part) > (uint32_t)f.slots) return fail("a part without a slot");
                ++dealt;
            }
            const int64_t rows = (int64_t)p.group * p.sq;
            if (p.count > 0 ? f.tiles < (int64_t)p.sq || f.per_query * f.row_tile < p.group
                            : (int64_t)f.tiles * (f.token ? f.row_tile : 128 / f.split) < rows)
                return fail("rows without a job");
            for (int k = 0; k < 4; ++k) {
                const int n = p.sk ? (int)(rng() % (p.sk + 1)) : 0;
                if (!parts_cover((n + 31) / 32, f.splits, 8, 4) || !parts_cover((n + 63) / 64, f.splits, 4, 1))
                    return fail("parts");
            }
        }
        ShaoboFa3CacheSelectParams s;
        shaobo_fa3_cache_select_params_init(&s);
        random_cache(&s.cache, plausible);
        s.seqlen = plausible ? 1 + (int)(rng() % 8) : pick_int();
        s.num_heads_q = plausible ? (int32_t)(2u * (uint32_t)s.cache.num_heads_kv) : pick_int();
        s.count = plausible ? 1 + (int)(rng() % 100) : pick_int();
        const int ss = shaobo_fa3_cache_select_validate(&s);
        const size_t sn = shaobo_fa3_cache_select_workspace_bytes(&s);
        if (!status_ok(ss) || (ss && sn) || sn > (1ull << 45)) return fail("select");
        if (!status_ok(shaobo_fa3_cache_select(&s, nullptr))) return fail("select entry");
        ShaoboFa3CacheAppendParams p;
        shaobo_fa3_cache_append_params_init(&p);
        random_cache(&p.cache, plausible);
        p.seqlen = plausible ? (int)(rng() >> (48 + rng() % 15)) : pick_int();
        p.num_heads_q = plausible ? (int)(rng() % 64) : pick_int();
        if (rng() % 2) {
            p.freqs = &number;
            p.pairs = plausible ? 8 * (1 + (int)(rng() % 8)) : pick_int();
            p.axes = plausible ? 1 : pick_int();
            p.interleaved = (int)(rng() % (plausible ? 2 : 3));
        }
        if (rng() % 4 == 0) p.positions = &word;
        if (rng() % 16 == 0) p.struct_size = (uint32_t)pick_int();
        if (!status_ok(shaobo_fa3_cache_append(&p, nullptr))) return fail("append");
        ShaoboFa3CacheReadParams r;
        shaobo_fa3_cache_read_params_init(&r);
        random_cache(&r.cache, plausible);
        r.seqlen = pick_int();
        if (!status_ok(shaobo_fa3_cache_read(&r, nullptr))) return fail("read");
    }
    std::printf("ok %d %d %d\n", seen[0], seen[1], seen[2]);
    return seen[0] > iters / 20 && seen[1] > 0 && seen[2] > 0 && dealt > iters / 500 ? 0 : fail("the fuzz is one-sided");
}
