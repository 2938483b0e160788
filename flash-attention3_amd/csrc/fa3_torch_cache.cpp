// PyTorch operators of the paged cache: shaobo_fa3::cache_append (and
// ::cache_append_into), ::cache_attn, ::cache_select and ::cache_read
// (shaobo_fa3_torch.py adds their fake implementations).  Built into the
// attention layer's library.
#include "fa3_torch_common.h"
#include "shaobo_fa3_cache.h"

#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>

#include <initializer_list>

namespace {

int32_t dtype_of(at::ScalarType t) {
    return t == at::kBFloat16 ? SHAOBO_FA3_DTYPE_BF16 : SHAOBO_FA3_DTYPE_FP16;
}

void check_type(at::ScalarType t, const char* name) {
    TORCH_CHECK_VALUE(t == at::kHalf || t == at::kBFloat16, name, " must be fp16 or bf16");
}

// No operator here has a gradient: a call that would leave one out is refused.
// (Looked at first: what autograd knows nothing of, nearly every tensor here.)
void no_gradient(std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors) {
        if (t == nullptr || t->unsafeGetTensorImpl()->autograd_meta() == nullptr) continue;
        const bool wanted =
            (at::GradMode::is_enabled() && t->requires_grad()) ||
            (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined());
        TORCH_CHECK_VALUE(!wanted, "the cache's operators have no gradient: pass detached tensors");
    }
}
const Tensor* given(const optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

// Two elements of what an append writes must not share memory: the call would
// leave either one's value there.
void check_written(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(at::has_internal_overlap(t) != at::MemOverlap::Yes, name,
                      ": written to, it must not overlap itself");
}

// Counts a write as autograd does, so that a backward that saved t misses its
// values.  (Tensors made under inference mode have no counter.)
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// [B] lengths
const int32_t* lens_of(const Tensor& t, int64_t B, const Tensor& like, const char* name) {
    check_int32(t, {B}, like, name);
    TORCH_CHECK_VALUE(B <= 1 || t.stride(0) == 1, name, " must be contiguous");
    return t.data_ptr<int32_t>();
}

ShaoboFa3CachePages pages_of(const Tensor& t, bool four, const char* name) {
    ShaoboFa3CachePages p;
    p.data = t.data_ptr();
    const int64_t align = 16 / t.element_size();
    int64_t s[3];
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) <= 1 ? 0 : t.stride(i);
    TORCH_CHECK_VALUE(t.size(3) <= 1 || t.stride(3) == 1, name, ": rows must be contiguous");
    if (four) {
        TORCH_CHECK_VALUE(t.size(2) <= 1 || t.stride(2) == t.size(3), name,
                          ": held in 4 bits, the last two axes must be contiguous");
        s[2] = 0;
    }
    for (int i = 0; i < 3; ++i)
        TORCH_CHECK_VALUE(s[i] % align == 0, name, ": strides must be multiples of 16 bytes");
    TORCH_CHECK_VALUE(t.numel() == 0 || (uintptr_t)p.data % 16 == 0, name, ": must be 16-byte aligned");
    p.page_stride = s[0];
    p.head_stride = s[1];
    p.row_stride = s[2];
    return p;
}

// A cache and its sequences, checked against rows of type `type` and head_dim
// D (0: taken from the pages) in B sequences on like's device.
ShaoboFa3Cache cache_of(const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                        const Tensor& kv_lens, const optional<Tensor>& new_lens, at::ScalarType type,
                        int64_t D) {
    TORCH_CHECK_VALUE(k_pages.is_cuda() && v_pages.device() == k_pages.device(),
                      "k_pages and v_pages must be on the same GPU");
    TORCH_CHECK_VALUE(k_pages.dim() == 4 && v_pages.sizes() == k_pages.sizes() &&
                          v_pages.scalar_type() == k_pages.scalar_type(),
                      "k_pages and v_pages must be alike, [pages, heads, page_size, row]");
    const bool four = k_pages.scalar_type() == at::kByte;
    TORCH_CHECK_VALUE(four || k_pages.scalar_type() == type,
                      "pages must have the rows' type (16 bits) or be uint8 (4 bits)");
    const int64_t row = k_pages.size(3), d = four ? 2 * (row - 4) : row;
    TORCH_CHECK_VALUE(D == 0 || d == D, "pages of head_dim ", d, ", rows of ", D);
    TORCH_CHECK_VALUE(!four || d == 64 || d == 128, "4 bits: head_dim must be 64 or 128");
    TORCH_CHECK_VALUE(d % 8 == 0 && d >= 8 && d <= 128, "head_dim must be a multiple of 8 up to 128");
    const int64_t size = k_pages.size(2);
    TORCH_CHECK_VALUE(size >= 32 && size <= 1024 && (size & (size - 1)) == 0,
                      "page_size must be 32, 64, 128, 256, 512 or 1024");
    TORCH_CHECK_VALUE(k_pages.size(1) >= 1, "no heads");
    TORCH_CHECK_VALUE(page_table.dim() == 2 && page_table.scalar_type() == at::kInt &&
                          page_table.device() == k_pages.device(),
                      "page_table must be int32 [batch, width] on the same GPU");
    TORCH_CHECK_VALUE(page_table.size(1) <= 1 || page_table.stride(1) == 1,
                      "page_table's rows must be contiguous");
    const int64_t B = page_table.size(0);
    constexpr int64_t kMost = 1 << 30;  // (what fits a launch is the library's to say)
    TORCH_CHECK_VALUE(B < kMost && page_table.size(1) * size <= kMost && k_pages.size(0) <= kMost &&
                          k_pages.size(1) <= (1 << 16),
                      "too many sequences, pages or heads");
    ShaoboFa3Cache c{};
    c.batch = (int32_t)B;
    c.num_heads_kv = (int32_t)k_pages.size(1);
    c.head_dim = (int32_t)d;
    c.dtype = dtype_of(type);
    c.bits = four ? 4 : 16;
    c.pages = (int32_t)k_pages.size(0);
    c.page_size = (int32_t)size;
    c.width = (int32_t)page_table.size(1);
    c.k = pages_of(k_pages, four, "k_pages");
    c.v = pages_of(v_pages, four, "v_pages");
    c.page_table = page_table.data_ptr<int32_t>();
    c.page_table_stride = B > 1 ? page_table.stride(0) : 0;
    c.kv_lens = lens_of(kv_lens, B, k_pages, "kv_lens");
    if (new_lens.has_value()) c.new_lens = lens_of(*new_lens, B, k_pages, "new_lens");
    return c;
}

void check_bounds(const Tensor& bounds, int64_t pages, const ShaoboFa3Cache& c, at::ScalarType type,
                  const Tensor& like) {
    TORCH_CHECK_VALUE(bounds.sizes() == at::IntArrayRef({pages, c.num_heads_kv, 2, c.head_dim}) &&
                          bounds.scalar_type() == type && bounds.is_contiguous() &&
                          bounds.device() == like.device(),
                      "bounds must be contiguous [pages, heads_kv, 2, head_dim] of the rows' type");
    TORCH_CHECK_VALUE(bounds.numel() == 0 || (uintptr_t)bounds.data_ptr() % 16 == 0,
                      "bounds must be 16-byte aligned");
}

// A call's rows x: [B, H, S, D] like the first of them.
void check_rows(const Tensor& x, const Tensor& first, const Tensor& page_table, const char* name) {
    TORCH_CHECK_VALUE(x.dim() == 4 && x.size(0) == page_table.size(0) && x.size(2) == first.size(2) &&
                          x.size(3) == first.size(3) && x.scalar_type() == first.scalar_type() &&
                          x.device() == page_table.device(),
                      name, " must be [batch, heads, sequence, head_dim] as the other rows are, with the "
                      "page table's batch and GPU");
}

// The append; turned q goes to q_out, or (fresh) to a tensor made there.
void append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
            const Tensor& page_table, const Tensor& kv_lens, const optional<Tensor>& new_lens,
            const optional<Tensor>& q, const optional<Tensor>& positions, const optional<Tensor>& freqs,
            bool interleaved, const optional<Tensor>& bounds, Tensor& q_out, bool fresh) {
    no_gradient({&k, &v, &k_pages, &v_pages, given(q), given(positions), given(freqs), given(bounds),
                 q_out.defined() ? &q_out : nullptr});
    TORCH_CHECK_VALUE(k.dim() == 4, "k must be [batch, heads, sequence, head_dim]");
    check_type(k.scalar_type(), "k");
    ShaoboFa3CacheAppendParams p;
    shaobo_fa3_cache_append_params_init(&p);
    p.cache = cache_of(k_pages, v_pages, page_table, kv_lens, new_lens, k.scalar_type(), k.size(3));
    check_written(k_pages, "k_pages");
    check_written(v_pages, "v_pages");
    // (that overlap in part may be one pool whose pages the table tells apart)
    TORCH_CHECK_VALUE(at::get_overlap_status(k_pages, v_pages) != at::MemOverlapStatus::Full,
                      "k_pages and v_pages must not overlap");
    const int64_t B = k.size(0), S = k.size(2);
    check_rows(k, k, page_table, "k");
    check_rows(v, k, page_table, "v");
    TORCH_CHECK_VALUE(k.size(1) == p.cache.num_heads_kv && v.size(1) == k.size(1),
                      "k and v must have the pages' heads");
    TORCH_CHECK_VALUE(B < (1 << 24) && S < (1 << 24) && B * S < (1 << 24), "too many new tokens");
    p.seqlen = (int32_t)S;
    p.k = view(k, "k");
    p.v = view(v, "v");
    if (q.has_value()) {
        check_rows(*q, k, page_table, "q");
        TORCH_CHECK_VALUE(q->size(1) >= 1 && q->size(1) <= (1 << 16), "too many heads, or none");
        p.num_heads_q = (int32_t)q->size(1);
        p.q = view(*q, "q");
    }
    if (freqs.has_value()) {
        TORCH_CHECK_VALUE(freqs->dim() == 2 && freqs->scalar_type() == at::kFloat &&
                              freqs->is_contiguous() && freqs->device() == k.device(),
                          "freqs must be contiguous fp32 [axes, pairs] on the same GPU");
        const int64_t A = freqs->size(0), P = freqs->size(1);
        TORCH_CHECK_VALUE(A >= 1 && A <= 4, "one to four axes");
        TORCH_CHECK_VALUE(P >= 8 && P % 8 == 0 && 2 * P <= k.size(3),
                          "pairs must be a multiple of 8, and twice as many at most head_dim");
        TORCH_CHECK_VALUE(positions.has_value() || A == 1, "several axes need positions");
        p.axes = (int32_t)A;
        p.pairs = (int32_t)P;
        p.interleaved = interleaved;
        p.freqs = freqs->data_ptr<float>();
    }
    if (positions.has_value()) {
        TORCH_CHECK_VALUE(freqs.has_value(), "positions need freqs");
        TORCH_CHECK_VALUE(positions->dim() == 3 && positions->size(0) == p.axes &&
                              positions->size(1) == B && positions->size(2) == S &&
                              positions->device() == k.device(),
                          "positions must be [axes, batch, sequence] on the same GPU");
        switch (positions->scalar_type()) {
            case at::kInt: p.position_type = SHAOBO_FA3_POSITIONS_INT32; break;
            case at::kLong: p.position_type = SHAOBO_FA3_POSITIONS_INT64; break;
            case at::kFloat: p.position_type = SHAOBO_FA3_POSITIONS_FP32; break;
            default: TORCH_CHECK_VALUE(false, "positions must be int32, int64 or fp32");
        }
        // (without elements there is no address: the call does nothing)
        p.positions = positions->numel() > 0 ? positions->data_ptr() : nullptr;
        if (positions->numel() == 0) p.freqs = nullptr;
        p.position_axis_stride = positions->stride(0);
        p.position_batch_stride = positions->stride(1);
        p.position_row_stride = positions->stride(2);
    }
    if (bounds.has_value()) {
        check_bounds(*bounds, k_pages.size(0), p.cache, k.scalar_type(), k);
        p.cache.bounds = bounds->data_ptr();
    }
    const Guard guard(k.device());
    if (fresh && q.has_value()) q_out = like(*q);
    TORCH_CHECK_VALUE(q.has_value() == q_out.defined(), "q and q_out: both or neither");
    if (!fresh && q.has_value()) {
        check_rows(q_out, k, page_table, "q_out");
        TORCH_CHECK_VALUE(q_out.size(1) == q->size(1), "q_out must have q's heads");
        check_written(q_out, "q_out");
        TORCH_CHECK_VALUE(at::get_overlap_status(q_out, *q) != at::MemOverlapStatus::Partial,
                          "q_out must be q or lie apart from it");
    }
    if (q.has_value()) p.q_out = view(q_out, "q_out");
    check_status(shaobo_fa3_cache_append(&p, stream_of(k)), "shaobo_fa3_cache_append");
    written(k_pages);
    written(v_pages);
    if (bounds.has_value()) written(*bounds);
    if (!fresh && q.has_value()) written(q_out);
}

std::vector<Tensor> cache_append(const Tensor& k, const Tensor& v, Tensor k_pages, Tensor v_pages,
                                 const Tensor& page_table, const Tensor& kv_lens,
                                 const optional<Tensor>& new_lens, const optional<Tensor>& q,
                                 const optional<Tensor>& positions, const optional<Tensor>& freqs,
                                 bool interleaved, const optional<Tensor>& bounds) {
    std::vector<Tensor> out(q.has_value() ? 1 : 0);
    Tensor none;
    append(k, v, k_pages, v_pages, page_table, kv_lens, new_lens, q, positions, freqs, interleaved, bounds,
           out.empty() ? none : out[0], true);
    return out;
}

// The same with q's output given and nothing returned: the form that a traced
// graph holds (functionalization knows no operator that writes and returns a list).
void cache_append_into(const Tensor& k, const Tensor& v, Tensor k_pages, Tensor v_pages,
                       const Tensor& page_table, const Tensor& kv_lens,
                       const optional<Tensor>& new_lens, const optional<Tensor>& q,
                       const optional<Tensor>& positions, const optional<Tensor>& freqs,
                       bool interleaved, const optional<Tensor>& bounds, const optional<Tensor>& q_out) {
    Tensor to = q_out.has_value() ? *q_out : Tensor();
    append(k, v, k_pages, v_pages, page_table, kv_lens, new_lens, q, positions, freqs, interleaved, bounds, to,
           false);
}

std::tuple<Tensor, Tensor> cache_attn(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                                      const Tensor& page_table, const Tensor& kv_lens,
                                      const optional<Tensor>& new_lens, bool causal,
                                      optional<double> scale, double softcap,
                                      const optional<Tensor>& slopes,
                                      const optional<Tensor>& prefix_lens,
                                      const optional<Tensor>& selected) {
    no_gradient({&q, &k_pages, &v_pages, given(slopes)});
    TORCH_CHECK_VALUE(q.dim() == 4, "q must be [batch, heads, sequence, head_dim]");
    check_type(q.scalar_type(), "q");
    ShaoboFa3CacheAttnParams p;
    shaobo_fa3_cache_attn_params_init(&p);
    p.cache = cache_of(k_pages, v_pages, page_table, kv_lens, new_lens, q.scalar_type(), q.size(3));
    check_rows(q, q, page_table, "q");
    const int64_t B = q.size(0), Hq = q.size(1), S = q.size(2), Hkv = p.cache.num_heads_kv;
    TORCH_CHECK_VALUE(Hq > 0 && Hq % Hkv == 0, "q's heads must be a multiple of the pages'");
    TORCH_CHECK_VALUE(Hq <= (1 << 16) && S < (1 << 24) && B * S < (1 << 24), "too many heads or new tokens");
    p.seqlen = (int32_t)S;
    p.num_heads_q = (int32_t)Hq;
    p.causal = causal;
    if (scale.has_value()) {
        TORCH_CHECK_VALUE(std::fabs(*scale) <= 1e30, "softmax_scale must be finite (1e30 at most)");
        p.softmax_scale = (float)*scale;
        p.softmax_scale_is_set = 1;
    }
    TORCH_CHECK_VALUE(softcap >= 0.0 && softcap <= 1e30,
                      "softcap must be 0 (none) or positive and finite (1e30 at most)");
    p.softcap = (float)softcap;
    TORCH_CHECK_VALUE(softcap == 0.0 || p.softcap > 0.f, "softcap is too small for fp32");
    p.q = view(q, "q");
    if (slopes.has_value()) p.slopes = slopes_of(*slopes, q, &p.slopes_batch_stride);
    if (prefix_lens.has_value()) {
        TORCH_CHECK_VALUE(causal, "prefix_lens needs causal=True");
        p.prefix_lens = lens_of(*prefix_lens, B, q, "prefix_lens");
    }
    if (selected.has_value()) {
        TORCH_CHECK_VALUE(selected->dim() == 4 && selected->scalar_type() == at::kInt &&
                              selected->size(0) == B && selected->size(1) == Hkv &&
                              selected->size(2) == S && selected->is_contiguous() &&
                              selected->device() == q.device(),
                          "selected must be contiguous int32 [batch, heads_kv, sequence, count]");
        TORCH_CHECK_VALUE(selected->size(3) >= 1 && selected->size(3) <= (1 << 20),
                          "selected must list 1 to 2^20 pages");
        p.count = (int32_t)selected->size(3);
        p.selected = selected->data_ptr<int32_t>();
        if (selected->numel() == 0) p.count = 0;
    }
    check_status(shaobo_fa3_cache_attn_validate(&p), "shaobo_fa3_cache_attn");  // (before it takes memory)
    const Guard guard(q.device());
    const Tensor out = like(q);
    const Tensor lse = at::empty({B, Hq, S}, q.options().dtype(at::kFloat));
    p.out = view(out, "out");
    p.softmax_lse = lse.data_ptr<float>();
    const Tensor ws = workspace(shaobo_fa3_cache_attn_workspace_bytes(&p), q, &p);
    check_status(shaobo_fa3_cache_attn(&p, stream_of(q)), "shaobo_fa3_cache_attn");
    return {out, lse};
}

Tensor cache_select(const Tensor& q, const Tensor& bounds, const Tensor& page_table,
                    const Tensor& kv_lens, int64_t page_size, int64_t count,
                    const optional<Tensor>& new_lens) {
    no_gradient({&q, &bounds});
    TORCH_CHECK_VALUE(q.dim() == 4 && q.is_cuda(), "q must be [batch, heads, sequence, head_dim] on a GPU");
    check_type(q.scalar_type(), "q");
    TORCH_CHECK_VALUE(bounds.dim() == 4, "bounds must be [pages, heads_kv, 2, head_dim]");
    TORCH_CHECK_VALUE(page_size >= 32 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
                      "page_size must be 32, 64, 128, 256, 512 or 1024");
    TORCH_CHECK_VALUE(page_table.dim() == 2 && page_table.scalar_type() == at::kInt &&
                          page_table.device() == q.device() &&
                          (page_table.size(1) <= 1 || page_table.stride(1) == 1),
                      "page_table must be int32 [batch, width] on the same GPU, rows contiguous");
    check_rows(q, q, page_table, "q");
    const int64_t B = q.size(0), Hq = q.size(1), S = q.size(2), D = q.size(3), Hkv = bounds.size(1);
    TORCH_CHECK_VALUE(D % 8 == 0 && D >= 8 && D <= 128, "head_dim must be a multiple of 8 up to 128");
    TORCH_CHECK_VALUE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "q's heads must be a multiple of the bounds'");
    TORCH_CHECK_VALUE(count >= 1 && count <= (1 << 20), "count must be 1 to 2^20");
    constexpr int64_t kMost = 1 << 30;
    TORCH_CHECK_VALUE(B < kMost && page_table.size(1) * page_size <= kMost && bounds.size(0) <= kMost &&
                          Hq <= (1 << 16) && S < (1 << 24) && B * S < (1 << 24),
                      "too many sequences, pages, heads or new tokens");
    ShaoboFa3CacheSelectParams p;
    shaobo_fa3_cache_select_params_init(&p);
    p.seqlen = (int32_t)S;
    p.num_heads_q = (int32_t)Hq;
    p.count = (int32_t)count;
    ShaoboFa3Cache& c = p.cache;
    c.batch = (int32_t)B;
    c.num_heads_kv = (int32_t)Hkv;
    c.head_dim = (int32_t)D;
    c.dtype = dtype_of(q.scalar_type());
    c.pages = (int32_t)bounds.size(0);
    c.page_size = (int32_t)page_size;
    c.width = (int32_t)page_table.size(1);
    c.page_table = page_table.data_ptr<int32_t>();
    c.page_table_stride = B > 1 ? page_table.stride(0) : 0;
    c.kv_lens = lens_of(kv_lens, B, q, "kv_lens");
    if (new_lens.has_value()) c.new_lens = lens_of(*new_lens, B, q, "new_lens");
    check_bounds(bounds, bounds.size(0), c, q.scalar_type(), q);
    c.bounds = bounds.data_ptr();
    p.q = view(q, "q");
    check_status(shaobo_fa3_cache_select_validate(&p), "shaobo_fa3_cache_select");
    const Guard guard(q.device());
    const Tensor out = at::empty({B, Hkv, S, count}, q.options().dtype(at::kInt));
    p.selected = out.data_ptr<int32_t>();
    const Tensor ws = workspace(shaobo_fa3_cache_select_workspace_bytes(&p), q, &p);
    check_status(shaobo_fa3_cache_select(&p, stream_of(q)), "shaobo_fa3_cache_select");
    return out;
}

std::tuple<Tensor, Tensor> cache_read(const Tensor& k_pages, const Tensor& v_pages,
                                      const Tensor& page_table, const Tensor& kv_lens, int64_t seqlen,
                                      at::ScalarType dtype) {
    no_gradient({&k_pages, &v_pages});
    check_type(dtype, "dtype");
    ShaoboFa3CacheReadParams p;
    shaobo_fa3_cache_read_params_init(&p);
    p.cache = cache_of(k_pages, v_pages, page_table, kv_lens, c10::nullopt, dtype, 0);
    TORCH_CHECK_VALUE(seqlen >= 0 && seqlen < (1 << 24) && p.cache.batch * seqlen < (1 << 24),
                      "seqlen must be 0 or more, and fit a launch");
    p.seqlen = (int32_t)seqlen;
    const Guard guard(k_pages.device());
    const auto options = k_pages.options().dtype(dtype);
    const std::vector<int64_t> sizes{p.cache.batch, p.cache.num_heads_kv, seqlen, p.cache.head_dim};
    const Tensor k = at::empty(sizes, options), v = at::empty(sizes, options);
    p.k = view(k, "k");
    p.v = view(v, "v");
    check_status(shaobo_fa3_cache_read(&p, stream_of(k_pages)), "shaobo_fa3_cache_read");
    return {k, v};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(shaobo_fa3, m) {
    m.def(
        "cache_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, "
        "Tensor kv_lens, Tensor? new_lens=None, Tensor? q=None, Tensor? positions=None, "
        "Tensor? freqs=None, bool interleaved=False, Tensor(c!)? bounds=None) -> Tensor[]");
    m.def(
        "cache_append_into(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, "
        "Tensor kv_lens, Tensor? new_lens=None, Tensor? q=None, Tensor? positions=None, "
        "Tensor? freqs=None, bool interleaved=False, Tensor(c!)? bounds=None, Tensor(d!)? q_out=None) "
        "-> ()");
    m.def(
        "cache_attn(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens, "
        "Tensor? new_lens=None, bool causal=True, float? softmax_scale=None, float softcap=0.0, "
        "Tensor? slopes=None, Tensor? prefix_lens=None, Tensor? selected=None) -> (Tensor, Tensor)");
    m.def(
        "cache_select(Tensor q, Tensor bounds, Tensor page_table, Tensor kv_lens, int page_size, "
        "int count, Tensor? new_lens=None) -> Tensor");
    m.def(
        "cache_read(Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens, int seqlen, "
        "ScalarType dtype) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(shaobo_fa3, CUDA, m) {
    m.impl("cache_append", &cache_append);
    m.impl("cache_append_into", &cache_append_into);
    m.impl("cache_attn", &cache_attn);
    m.impl("cache_select", &cache_select);
    m.impl("cache_read", &cache_read);
}
