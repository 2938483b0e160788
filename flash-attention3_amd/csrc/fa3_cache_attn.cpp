// Attention to a paged cache: which kernel, how many jobs, and their launch.
#include "fa3_cache_internal.h"

namespace fa3 {

CachePlan plan_cache_attn(const CacheProblem& p) {
    CachePlan f{};
    const int64_t rows = (int64_t)p.group * p.sq, groups = (int64_t)p.batch * p.heads_kv;
    const int D = p.d > 64 ? 128 : 64;
    // Selected pages are a query's own, and its heads few rows.
    f.token = p.count > 0 || rows <= 32;
    const int64_t at_once = p.count > 0 ? p.group : rows;
    f.row_tile = at_once <= 16 ? 16 : 32;
    f.split = !f.token && groups * ceil_div(rows, kAttnRows) < 512 ? 2 : 1;
    f.per_query = ceil_div(p.group, f.row_tile);
    const int64_t tiles = p.count > 0 ? (int64_t)p.sq * f.per_query
                          : f.token   ? 1
                                      : ceil_div(rows, kAttnRows / f.split);
    f.splits = 1;
    const int64_t jobs = groups * tiles;
    // Jobs that leave the chip half empty cut the key axis, as long as a part
    // keeps 256 keys (tiles: 512).  How many parts there are goes by the places
    // that the pages have; a sequence's own length is cut into them on the GPU.
    const int fill = f.token ? 256 * ((p.four || D == 64 ? 4 : 3) - f.row_tile / 16) : 512;
    const int64_t keys = p.count > 0 ? (int64_t)p.count * p.page : p.sk;
    const int least = f.token ? 256 : 512;
    if (jobs > 0 && 2 * jobs <= fill && keys >= 2 * least) {
        const int64_t want = fill / jobs, most = keys / least;
        f.splits = (int)(want < most ? want : most);
    }
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t x = at;
        at += (n + 255) / 256 * 256;
        return x;
    };
    const int64_t all = jobs * f.splits;
    f.ok = rows < (1ll << 30) && tiles < (1ll << 30) && all < kMaxGrid && groups * rows / 4 < kMaxGrid;
    if (!f.ok) return f;
    f.tiles = (int)tiles;
    f.jobs = (int)all;
    if (f.splits > 1) {
        f.po_off = take((size_t)f.splits * groups * rows * D * 4);
        f.pl_off = take((size_t)f.splits * groups * rows * 4);
    }
    f.total = at;
    return f;
}

hipError_t launch_cache_attn(const CacheProblem& p, const ShaoboFa3CacheAttnParams& a, AttnMask m,
                             hipStream_t stream) {
    const CachePlan f = plan_cache_attn(p);
    if (f.jobs == 0) return hipSuccess;
    char* ws = (char*)a.workspace;
    auto view = [](const ShaoboFa3AttnTensor& t) {
        return AttnView{(_Float16*)t.data, t.batch_stride, t.head_stride, t.row_stride};
    };
    CacheAttnArgs x{};
    x.q = view(a.q);
    x.out = view(a.out);
    x.lse = a.softmax_lse;
    x.part_o = (float*)(ws + f.po_off);
    x.part_l = (float*)(ws + f.pl_off);
    x.heads_q = p.heads_q;
    x.heads_kv = p.heads_kv;
    x.group = p.group;
    x.sq = p.sq;
    x.sk = p.sk;
    x.d = p.d;
    x.rows = p.group * p.sq;
    x.tiles = f.tiles;
    x.splits = f.splits;
    x.part = 8;  // a part has at least 8 blocks of 32 keys, or 8 tiles of 64
    x.groups = p.batch * p.heads_kv;
    x.levels = f.tiles * f.splits;
    // (longest first, or jobs of one length group by group, as plan_attn_fwd)
    x.by_group = f.token || !p.causal;
    x.div_hkv = make_fastdiv(p.heads_kv);
    x.div_group = make_fastdiv(p.group);
    x.div_groups = make_fastdiv(x.groups);
    x.div_gpart = make_fastdiv(x.groups / 8);
    x.div_splits = make_fastdiv(f.splits);
    x.div_levels = make_fastdiv(x.levels);
    // Maxima are taken over raw products: their scale must be positive.
    x.scored = 1;
    if (!(p.softcap > 0.f)) {
        if (m.c < 0.f) x.flip = 0x80008000u;
        x.scored = m.c != 0.f;
        m.c = m.c == 0.f ? 1.f : m.c < 0.f ? -m.c : m.c;
    }
    x.m = m;
    x.x.cv = cache_view(a.cache);
    x.x.selected = a.selected;
    x.x.count = p.count;
    x.x.per_query = f.per_query;
    x.x.div_per_query = make_fastdiv(f.per_query);
    if (p.d > 64) p.four ? launch_cache_d128_4(x, p, f, stream) : launch_cache_d128_16(x, p, f, stream);
    else p.four ? launch_cache_d64_4(x, p, f, stream) : launch_cache_d64_16(x, p, f, stream);
    return hipGetLastError();
}

}  // namespace fa3
