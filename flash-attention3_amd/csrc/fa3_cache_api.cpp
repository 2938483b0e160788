// C entries of the paged cache (shaobo_fa3_cache.h): parameter checks,
// workspace sizes and launches.
#include <cmath>
#include <cstring>

#include "fa3_cache_internal.h"

namespace {

using fa3::AttnMask;
using fa3::CacheProblem;

constexpr int kOk = SHAOBO_FA3_STATUS_SUCCESS;
constexpr int kInvalid = SHAOBO_FA3_STATUS_INVALID_VALUE;
constexpr int kUnsupported = SHAOBO_FA3_STATUS_UNSUPPORTED;
// Places of a sequence, heads and listed pages are held below these, so that
// rows, blocks and jobs count in 32 bits.
constexpr int64_t kMaxPlaces = 1 << 30;
constexpr int32_t kMaxHeads = 1 << 16;
constexpr int32_t kMaxCount = 1 << 20;
constexpr float kMaxScore = 1e30f;

bool strides_ok(const ShaoboFa3AttnTensor& t) {
    return t.batch_stride % 8 == 0 && t.head_stride % 8 == 0 && t.row_stride % 8 == 0;
}
bool aligned(const void* p) { return p != nullptr && (uintptr_t)p % 16 == 0; }
bool flag(int32_t x) { return x == 0 || x == 1; }

// Sizes and strides of a cache and of a call's rows, pointers aside.
int check_cache(const ShaoboFa3Cache& c, int32_t seqlen, bool pages) {
    if (c.batch < 0 || seqlen < 0 || c.num_heads_kv <= 0 || c.head_dim <= 0 || c.pages < 0 ||
        c.width < 0 || c.page_size <= 0 || (c.bits != 16 && c.bits != 4))
        return kInvalid;
    if (c.dtype != SHAOBO_FA3_DTYPE_FP16 && c.dtype != SHAOBO_FA3_DTYPE_BF16) return kUnsupported;
    if (c.head_dim > 128 || c.head_dim % 8 != 0) return kUnsupported;
    if (c.bits == 4 && c.head_dim != 64 && c.head_dim != 128) return kUnsupported;
    if (c.page_size < 32 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)) != 0)
        return kUnsupported;
    if ((int64_t)c.width * c.page_size > kMaxPlaces || c.num_heads_kv > kMaxHeads) return kUnsupported;
    if ((int64_t)c.batch * seqlen >= fa3::kMaxGrid || (int64_t)c.batch * c.num_heads_kv >= fa3::kMaxGrid)
        return kUnsupported;
    if (pages) {
        const int by = c.bits == 16 ? 8 : 16;
        for (const ShaoboFa3CachePages* p : {&c.k, &c.v})
            if (p->page_stride % by != 0 || p->head_stride % by != 0 ||
                (c.bits == 16 && p->row_stride % by != 0))
                return kUnsupported;
    }
    return kOk;
}
// Its pointers, where a call reads them.
bool cache_there(const ShaoboFa3Cache& c, bool pages) {
    if (c.kv_lens == nullptr || (c.width > 0 && c.page_table == nullptr)) return false;
    return !pages || c.pages == 0 || (aligned(c.k.data) && aligned(c.v.data));
}
int heads_ok(int32_t heads_q, int32_t heads_kv) {
    if (heads_q <= 0 || heads_q % heads_kv != 0) return kInvalid;
    return heads_q <= kMaxHeads ? kOk : kUnsupported;
}

// Runs `launch` on the stream's device.
template <typename F>
int on_stream(void* stream, F launch) {
    int dev = -1;
    const hipError_t d = fa3::launch_device((hipStream_t)stream, &dev);
    if (d == hipErrorInvalidDevice) return kInvalid;
    if (d != hipSuccess) return SHAOBO_FA3_STATUS_HIP_ERROR;
    return launch((hipStream_t)stream) == hipSuccess ? kOk : SHAOBO_FA3_STATUS_HIP_ERROR;
}

int check_append(const ShaoboFa3CacheAppendParams* p) {
    if (p == nullptr || p->struct_size < sizeof(*p)) return kInvalid;
    const int st = check_cache(p->cache, p->seqlen, true);
    if (st != kOk) return st;
    if (p->num_heads_q < 0) return kInvalid;
    if (p->num_heads_q > kMaxHeads) return kUnsupported;
    if (p->freqs != nullptr) {
        if (p->axes < 1 || p->pairs < 0 || !flag(p->interleaved) ||
            (p->positions != nullptr && (p->position_type < SHAOBO_FA3_POSITIONS_INT32 ||
                                         p->position_type > SHAOBO_FA3_POSITIONS_FP32)))
            return kInvalid;
        if (p->axes > 4 || p->pairs < 8 || p->pairs % 8 != 0 || p->pairs > p->cache.head_dim / 2)
            return kUnsupported;
        if (p->positions == nullptr && p->axes != 1) return kInvalid;
    } else if (p->positions != nullptr) {
        return kInvalid;
    }
    if (!strides_ok(p->k) || !strides_ok(p->v)) return kUnsupported;
    if (p->num_heads_q > 0 && (!strides_ok(p->q) || !strides_ok(p->q_out))) return kUnsupported;
    return p->seqlen == 0 || p->cache.batch == 0 || fa3::append_grid(*p).ok ? kOk : kUnsupported;
}

int check_attn(const ShaoboFa3CacheAttnParams* a, CacheProblem* p) {
    if (a == nullptr || a->struct_size < sizeof(*a)) return kInvalid;
    const ShaoboFa3Cache& c = a->cache;
    int st = check_cache(c, a->seqlen, true);
    if (st == kOk) st = heads_ok(a->num_heads_q, c.num_heads_kv);
    if (st != kOk) return st;
    if (!flag(a->causal) || !flag(a->softmax_scale_is_set)) return kInvalid;
    if (a->softmax_scale_is_set && !(std::fabs(a->softmax_scale) <= kMaxScore)) return kInvalid;
    if (!(a->softcap >= 0.f && a->softcap <= kMaxScore)) return kInvalid;
    if (a->prefix_lens != nullptr && !a->causal) return kInvalid;
    if (a->count < 0 || (a->selected != nullptr && a->count == 0)) return kInvalid;
    if (a->count > kMaxCount) return kUnsupported;
    if (!strides_ok(a->q) || !strides_ok(a->out)) return kUnsupported;
    p->batch = c.batch;
    p->heads_q = a->num_heads_q;
    p->heads_kv = c.num_heads_kv;
    p->group = a->num_heads_q / c.num_heads_kv;
    p->sq = a->seqlen;
    p->d = c.head_dim;
    p->sk = c.width * c.page_size;
    p->page = c.page_size;
    p->count = a->selected != nullptr ? a->count : 0;
    p->bf16 = c.dtype == SHAOBO_FA3_DTYPE_BF16;
    p->four = c.bits == 4;
    p->causal = a->causal != 0;
    p->bias = a->slopes != nullptr;
    p->scale = a->softmax_scale_is_set ? a->softmax_scale : 1.f / std::sqrt((float)c.head_dim);
    p->softcap = a->softcap;
    if ((int64_t)p->batch * p->heads_q >= fa3::kMaxGrid) return kUnsupported;
    return fa3::plan_cache_attn(*p).ok ? kOk : kUnsupported;
}

int check_select(const ShaoboFa3CacheSelectParams* p) {
    if (p == nullptr || p->struct_size < sizeof(*p)) return kInvalid;
    int st = check_cache(p->cache, p->seqlen, false);
    if (st == kOk) st = heads_ok(p->num_heads_q, p->cache.num_heads_kv);
    if (st != kOk) return st;
    if (p->count < 1) return kInvalid;
    if (p->count > kMaxCount || !strides_ok(p->q)) return kUnsupported;
    return fa3::plan_cache_select(*p).ok ? kOk : kUnsupported;
}

template <typename P>
void init(P* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = (uint32_t)sizeof(*p);
    p->cache.dtype = SHAOBO_FA3_DTYPE_FP16;
    p->cache.bits = 16;
    p->cache.page_size = 64;
}

}  // namespace

extern "C" {

void shaobo_fa3_cache_append_params_init(ShaoboFa3CacheAppendParams* params) {
    init(params);
    if (params != nullptr) params->axes = 1;
}
void shaobo_fa3_cache_attn_params_init(ShaoboFa3CacheAttnParams* params) { init(params); }
void shaobo_fa3_cache_select_params_init(ShaoboFa3CacheSelectParams* params) { init(params); }
void shaobo_fa3_cache_read_params_init(ShaoboFa3CacheReadParams* params) { init(params); }

int shaobo_fa3_cache_append(const ShaoboFa3CacheAppendParams* params, void* stream) {
    const ShaoboFa3CacheAppendParams* p = params;
    const int st = check_append(p);
    if (st != kOk) return st;
    if (p->cache.batch == 0 || p->seqlen == 0) return kOk;
    if (!cache_there(p->cache, true) || !aligned(p->k.data) || !aligned(p->v.data) ||
        (p->num_heads_q > 0 && (!aligned(p->q.data) || !aligned(p->q_out.data))) ||
        (uintptr_t)p->cache.bounds % 16 != 0)
        return kInvalid;
    return on_stream(stream, [&](hipStream_t s) { return fa3::launch_cache_append(*p, s); });
}

int shaobo_fa3_cache_attn_validate(const ShaoboFa3CacheAttnParams* params) {
    CacheProblem p;
    return check_attn(params, &p);
}
size_t shaobo_fa3_cache_attn_workspace_bytes(const ShaoboFa3CacheAttnParams* params) {
    CacheProblem p;
    return check_attn(params, &p) == kOk ? fa3::plan_cache_attn(p).total : 0;
}
int shaobo_fa3_cache_attn(const ShaoboFa3CacheAttnParams* params, void* stream) {
    const ShaoboFa3CacheAttnParams* a = params;
    CacheProblem p;
    const int st = check_attn(a, &p);
    if (st != kOk) return st;
    if (p.batch == 0 || p.sq == 0) return kOk;
    const size_t need = fa3::plan_cache_attn(p).total;
    if (!cache_there(a->cache, true) || !aligned(a->q.data) || !aligned(a->out.data) ||
        a->softmax_lse == nullptr)
        return kInvalid;
    if (need > 0 && (a->workspace == nullptr || (uintptr_t)a->workspace % 256 != 0 ||
                     a->workspace_bytes < need))
        return kInvalid;
    AttnMask m{};
    m.prefix = a->prefix_lens;
    m.kv_lens = a->cache.kv_lens;
    m.slopes = a->slopes;
    m.slopes_bs = a->slopes_batch_stride;
    m.causal = a->causal;
    fa3::set_scores(&m, p.scale, p.softcap);
    return on_stream(stream, [&](hipStream_t s) { return fa3::launch_cache_attn(p, *a, m, s); });
}

int shaobo_fa3_cache_select_validate(const ShaoboFa3CacheSelectParams* params) {
    return check_select(params);
}
size_t shaobo_fa3_cache_select_workspace_bytes(const ShaoboFa3CacheSelectParams* params) {
    return check_select(params) == kOk ? fa3::plan_cache_select(*params).total : 0;
}
int shaobo_fa3_cache_select(const ShaoboFa3CacheSelectParams* params, void* stream) {
    const ShaoboFa3CacheSelectParams* p = params;
    const int st = check_select(p);
    if (st != kOk) return st;
    if (p->cache.batch == 0 || p->seqlen == 0) return kOk;
    const size_t need = fa3::plan_cache_select(*p).total;
    if (!cache_there(p->cache, false) || !aligned(p->q.data) || p->selected == nullptr ||
        (p->cache.pages > 0 && !aligned(p->cache.bounds)))
        return kInvalid;
    if (need > 0 && (p->workspace == nullptr || (uintptr_t)p->workspace % 256 != 0 ||
                     p->workspace_bytes < need))
        return kInvalid;
    return on_stream(stream, [&](hipStream_t s) { return fa3::launch_cache_select(*p, s); });
}

int shaobo_fa3_cache_read(const ShaoboFa3CacheReadParams* params, void* stream) {
    const ShaoboFa3CacheReadParams* p = params;
    if (p == nullptr || p->struct_size < sizeof(*p)) return kInvalid;
    const int st = check_cache(p->cache, p->seqlen, true);
    if (st != kOk) return st;
    if (!strides_ok(p->k) || !strides_ok(p->v)) return kUnsupported;
    const int64_t blocks = ((int64_t)p->seqlen * (p->cache.head_dim / 8) + 255) / 256;
    if (blocks * p->cache.batch * p->cache.num_heads_kv >= fa3::kMaxGrid) return kUnsupported;
    if (p->cache.batch == 0 || p->seqlen == 0) return kOk;
    if (!cache_there(p->cache, true) || !aligned(p->k.data) || !aligned(p->v.data)) return kInvalid;
    return on_stream(stream, [&](hipStream_t s) { return fa3::launch_cache_read(*p, s); });
}

}  // extern "C"
