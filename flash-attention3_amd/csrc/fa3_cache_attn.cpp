// Attention to a paged cache: which kernel, how many jobs, and their launch.
#include "fa3_cache_internal.h"

namespace fa3 {

namespace {

int64_t ceil64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Parts of the key axis for jobs of few rows that are not dealt (few_slots says
// which are): one sequence, more than 256, selected pages.  As many as fill the
// chip once, and then up to twice as many where those leave the CUs less uneven
// (the most jobs a CU has, by the parts' length); one where the jobs fill it
// already.  A part keeps 256 keys.  Whole calls, us, the rule's choice first, D
// 128.  One token and 8 KV heads, over 2048 keys in 16 bits: 10.3 in 8 parts, 13.2
// in 4, 23.3 whole; over 16384: 21.7 in 64, 20.2 in 32, 22.0 in 16, 170 whole; over
// 131072: 100 in 64, 105 in 128, 100 in 32; the same in 4 bits: 36.6 in 96, 41.0
// in 128, 35.5 in 64, 44.5 in 32.  64 pages of 2048 in 4 bits: 21.7 in 16, 24.0 in
// 8, 45.7 whole; 48 pages, 16 sequences: 63.2 in 4, 64.0 in 2, 65.7 in 6.  300
// sequences of one KV head, over 8192: 246 in 2, 270 whole, 223 in 4.
int few_splits(int64_t jobs, int fill, int64_t keys) {
    const int64_t most = keys / 256, least = fill / jobs;
    if (least < 1 || jobs >= fill || most < 2) return 1;
    int64_t best = least < most ? least : most;
    for (int64_t s = best + 1; s <= 2 * least && s <= most; ++s)
        if (ceil64(jobs * s, 256) * best < ceil64(jobs * best, 256) * s) best = s;
    return (int)best;
}

// Slots of a KV head for parts of several sequences, dealt on the GPU by their
// lengths (cache_deal); 0: every sequence in as many parts (few_splits), which
// costs a launch less where those are one.  As many slots as fill the chip, and
// half as many at least beyond one a sequence: a part is then no longer than
// twice what an even share would be.  16 bits, 8 KV heads, D 128: 32768 keys
// beside 63 times 512 54 us, whole sequences 359; 4 of 32768 beside 124 of 1024
// 206 and 518; 16 of up to 8192 70.4, in four parts each 71.9; but 64 of 512 under
// a table of 32768 27.8 and 24.9, hence not where no sequence can be long.  As
// many slots again as fill the chip: 64 of 4096 to 32768 896 for 950, 64 of
// 2048 118 for 109.
int few_slots(const CacheProblem& p, int64_t jobs, int fill) {
    if (p.batch < 2 || p.batch > kDealBatch || p.sk < 512) return 0;
    if ((int64_t)p.batch * (p.sk / 32) >= (1ll << 31) || (jobs >= fill && p.sk < 8192)) return 0;
    const int per = fill / p.heads_kv, half = per > 2 ? per / 2 : 1;
    return per > p.batch + half ? per : p.batch + half;
}

// Rows and parts for jobs of many rows, by an estimate of the launch, us: a
// 64-key step of a job of 128 rows (64) takes 1.96 (1.42) where the CU has one
// job and 1.33 (0.86) a job where it has more; parts of a sequence write their
// sums and read them again at 4 TB/s, in a launch of 5; a job's beginning and
// end are four steps.  How much of the places
// is filled is not known here: all of them are taken to be.  (D 128; measured,
// the estimate's choice first: 1531 tokens over 9211, 8 KV heads, in 4 bits 300
// us in 128 rows and 2 parts, 293 in 4, 350 whole, 366 in 64 rows and 2, in 16 bits
// 280, 270, 310, 315; 8 times 64 over 8192, 110 in 128 rows and 4 parts, 128 in 64
// and 2; 2011 of 4 KV heads, 50 in 64 rows, 52 in 128 and 2 parts, 67 in 128; 512
// of 8 KV heads, 18 in 64 rows, 21 in 128, 26 in 2 parts of either.  The choice is
// within 4 % of the best of these.)
void tile_plan(const CacheProblem& p, CachePlan* f) {
    const int64_t rows = (int64_t)p.group * p.sq, groups = (int64_t)p.batch * p.heads_kv;
    const double last = p.sk / 64.0;  // steps of the longest job, and of them all in the mean
    const double mean = p.causal && p.sk > 0 ? last - (p.sq < p.sk ? p.sq : p.sk) / 128.0 : last;
    double best = 1e300;
    for (int split = 1; split <= 2; ++split) {
        const int64_t jobs = groups * ceil64(rows, kAttnRows / split);
        const double alone = split == 1 ? 1.96 : 1.42, among = split == 1 ? 1.33 : 0.86;
        for (int parts = 1; parts <= 32 && (parts == 1 || last >= 4 * parts); ++parts) {
            const int64_t a_cu = ceil64(jobs * parts, 256);
            const double step = a_cu <= 1 ? alone : 2 * among;  // of a job beside another
            double t = (a_cu <= 1 ? alone : a_cu * among) * (mean / parts + 4);
            if ((last / parts + 4) * step > t) t = (last / parts + 4) * step;
            if (parts > 1) t += 5 + (double)parts * groups * rows * 8.0 * (p.d > 64 ? 128 : 64) / 4e6;
            if (t < best) {
                best = t;
                f->split = split;
                f->splits = parts;
            }
        }
    }
}

}  // namespace

CachePlan plan_cache_attn(const CacheProblem& p) {
    CachePlan f{};
    const int64_t rows = (int64_t)p.group * p.sq, groups = (int64_t)p.batch * p.heads_kv;
    const int D = p.d > 64 ? 128 : 64;
    if (groups >= kMaxGrid || rows >= (1ll << 30)) return f;
    // Selected pages are a query's own, and its heads few rows.
    f.token = p.count > 0 || rows <= 32;
    const int64_t at_once = p.count > 0 ? p.group : rows;
    f.row_tile = at_once <= 16 ? 16 : 32;
    f.per_query = ceil_div(p.group, f.row_tile);
    f.split = f.splits = 1;
    if (!f.token) tile_plan(p, &f);
    const int64_t tiles = p.count > 0 ? (int64_t)p.sq * f.per_query
                          : f.token   ? 1
                                      : ceil_div(rows, kAttnRows / f.split);
    const int64_t jobs = groups * tiles;
    if (f.token && jobs > 0) {
        const int fill = 256 * few_waves(D, p.four, f.row_tile / 16);
        f.slots = p.count > 0 ? 0 : few_slots(p, jobs, fill);
        if (f.slots == 0)
            f.splits = few_splits(jobs, fill, p.count > 0 ? (int64_t)p.count * p.page : p.sk);
    }
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t x = at;
        at += (n + 255) / 256 * 256;
        return x;
    };
    const int64_t all = f.slots > 0 ? (int64_t)f.slots * p.heads_kv : jobs * f.splits;
    f.ok = tiles < (1ll << 30) && all < kMaxGrid && groups * rows / 4 < kMaxGrid;
    if (!f.ok) return f;
    f.tiles = (int)tiles;
    f.jobs = (int)all;
    if (f.splits > 1 || f.slots > 0) {
        const size_t parts = f.slots > 0 ? (size_t)f.slots * p.heads_kv : (size_t)f.splits * groups;
        f.po_off = take(parts * rows * D * 4);
        f.pl_off = take(parts * rows * 4);
    }
    if (f.slots > 0) f.deal_off = take((size_t)p.batch * 8);
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
    x.part = f.token ? 8 : 4;  // a part's least, 256 keys: blocks of 32, or tiles of 64
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
    x.x.slots = f.slots;
    x.x.batch = p.batch;
    x.x.deal = (int2*)(ws + f.deal_off);
    if (p.d > 64) p.four ? launch_cache_d128_4(x, p, f, stream) : launch_cache_d128_16(x, p, f, stream);
    else p.four ? launch_cache_d64_4(x, p, f, stream) : launch_cache_d64_16(x, p, f, stream);
    return hipGetLastError();
}

}  // namespace fa3
