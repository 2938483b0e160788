// PyTorch operators of the attention layer: shaobo_fa3::rotary,
// ::attn_forward and ::attn_backward (shaobo_fa3_torch.py loads this library,
// adds their fake implementations and the autograd functions on top).
//
// Registered from C++, a call stays out of Python below torch's dispatch:
// what bounds the smallest calls is the host.
#include "fa3_torch_common.h"

namespace {

struct Options {
    bool causal;
    optional<double> scale;
    double softcap;
    const optional<Tensor>&slopes, &documents, &documents_k, &prefix_lens, &kv_lens;
};

// Parameters of a call, its inputs checked.
ShaoboFa3AttnParams params_of(const Tensor& q, const Tensor& k, const Tensor& v,
                              const Options& o) {
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                      "q, k and v must be [batch, heads, sequence, head_dim]");
    const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3), Hkv = k.size(1),
                  Sk = k.size(2);
    TORCH_CHECK_VALUE(k.size(0) == B && k.size(3) == D && v.sizes() == k.sizes() && Hkv > 0 &&
                          Hq > 0 && Hq % Hkv == 0,
                      "k / v shape ", k.sizes(), " / ", v.sizes(), " does not match q ", q.sizes());
    const auto dt = q.scalar_type();
    TORCH_CHECK_VALUE((dt == at::kHalf || dt == at::kBFloat16) && k.scalar_type() == dt &&
                          v.scalar_type() == dt,
                      "q, k and v must share one type, fp16 or bf16");
    TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() && v.device() == q.device(),
                      "q, k and v must be on the same GPU");
    TORCH_CHECK_VALUE(D % 8 == 0 && D >= 8 && D <= 128, "head_dim must be a multiple of 8 up to 128");
    constexpr int64_t kMost = 1 << 30;  // (what fits a launch is the library's to say)
    TORCH_CHECK_VALUE(B < kMost && B * Hq < kMost && Sq <= kMost && Sk <= kMost && Hq <= (1 << 16),
                      "too many batch entries, heads or positions");
    ShaoboFa3AttnParams p;
    shaobo_fa3_attn_params_init(&p);
    p.batch = (int32_t)B;
    p.seqlen_q = (int32_t)Sq;
    p.seqlen_k = (int32_t)Sk;
    p.num_heads_q = (int32_t)Hq;
    p.num_heads_kv = (int32_t)Hkv;
    p.head_dim = (int32_t)D;
    p.dtype = dt == at::kBFloat16 ? SHAOBO_FA3_DTYPE_BF16 : SHAOBO_FA3_DTYPE_FP16;
    p.causal = o.causal ? 1 : 0;
    if (o.scale.has_value()) {
        TORCH_CHECK_VALUE(std::fabs(*o.scale) <= 1e30, "softmax_scale must be finite (1e30 at most)");
        p.softmax_scale = (float)*o.scale;
        p.softmax_scale_is_set = 1;
    }
    TORCH_CHECK_VALUE(o.softcap >= 0.0 && o.softcap <= 1e30,
                      "softcap must be 0 (none) or positive and finite (1e30 at most)");
    p.softcap = (float)o.softcap;
    TORCH_CHECK_VALUE(o.softcap == 0.0 || p.softcap > 0.f, "softcap is too small for fp32");
    p.q = view(q, "q");
    p.k = view(k, "k");
    p.v = view(v, "v");
    if (o.slopes.has_value()) p.slopes = slopes_of(*o.slopes, q, &p.slopes_batch_stride);
    auto ids = [&](const Tensor& t, int64_t n, const char* name, const int32_t** out, int64_t* bs) {
        check_int32(t, {B, n}, q, name);
        TORCH_CHECK_VALUE(n <= 1 || t.stride(1) == 1, name, " must be contiguous along the sequence");
        *out = t.data_ptr<int32_t>();
        *bs = B > 1 ? t.stride(0) : 0;
    };
    TORCH_CHECK_VALUE(o.documents.has_value() || !o.documents_k.has_value(),
                      "documents_k needs documents");
    if (o.documents.has_value()) {
        TORCH_CHECK_VALUE(o.documents_k.has_value() || Sq == Sk,
                          "documents_k must be given where queries and keys differ in number");
        ids(*o.documents, Sq, "documents", &p.documents_q, &p.documents_q_batch_stride);
        ids(o.documents_k.has_value() ? *o.documents_k : *o.documents, Sk, "documents_k",
            &p.documents_k, &p.documents_k_batch_stride);
        if (Sq == 0 || Sk == 0) p.documents_q = p.documents_k = nullptr;  // (nothing to mask)
    }
    auto lens = [&](const Tensor& t, const char* name) {
        check_int32(t, {B}, q, name);
        TORCH_CHECK_VALUE(B <= 1 || t.stride(0) == 1, name, " must be contiguous");
        return t.data_ptr<int32_t>();
    };
    if (o.prefix_lens.has_value()) {
        TORCH_CHECK_VALUE(o.causal, "prefix_lens needs causal=True");
        p.prefix_lens = lens(*o.prefix_lens, "prefix_lens");
    }
    if (o.kv_lens.has_value()) p.kv_lens = lens(*o.kv_lens, "kv_lens");
    return p;
}

std::tuple<Tensor, Tensor> attn_forward(
    const Tensor& q, const Tensor& k, const Tensor& v, bool causal, optional<double> scale,
    double softcap, const optional<Tensor>& slopes, const optional<Tensor>& documents,
    const optional<Tensor>& documents_k, const optional<Tensor>& prefix_lens,
    const optional<Tensor>& kv_lens) {
    ShaoboFa3AttnParams p = params_of(
        q, k, v, Options{causal, scale, softcap, slopes, documents, documents_k, prefix_lens, kv_lens});
    check_status(shaobo_fa3_attn_fwd_validate(&p), "shaobo_fa3_attn_fwd");  // (before it takes memory)
    const Guard guard(q.device());
    const Tensor out = like(q);
    const Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    p.out = view(out, "out");
    p.softmax_lse = lse.data_ptr<float>();
    const Tensor ws = workspace(shaobo_fa3_attn_fwd_workspace_bytes(&p), q, &p);
    check_status(shaobo_fa3_attn_fwd(&p, stream_of(q)), "shaobo_fa3_attn_fwd");
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attn_backward(
    const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
    const Tensor& softmax_lse, bool causal, optional<double> scale, double softcap,
    const optional<Tensor>& slopes, const optional<Tensor>& documents,
    const optional<Tensor>& documents_k, const optional<Tensor>& prefix_lens,
    const optional<Tensor>& kv_lens) {
    ShaoboFa3AttnParams p = params_of(
        q, k, v, Options{causal, scale, softcap, slopes, documents, documents_k, prefix_lens, kv_lens});
    for (const Tensor* t : {&dout, &out})
        TORCH_CHECK_VALUE(t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type() &&
                              t->device() == q.device(),
                          "dout and out must be like q");
    TORCH_CHECK_VALUE(softmax_lse.scalar_type() == at::kFloat &&
                          softmax_lse.sizes() == q.sizes().slice(0, 3) &&
                          softmax_lse.is_contiguous() && softmax_lse.device() == q.device(),
                      "softmax_lse must be contiguous fp32 [batch, heads_q, sequence]");
    p.dout = view(dout, "dout");
    p.out = view(out, "out");
    check_status(shaobo_fa3_attn_bwd_validate(&p), "shaobo_fa3_attn_bwd");
    const Guard guard(q.device());
    p.softmax_lse = softmax_lse.data_ptr<float>();
    const Tensor dq = like(q), dk = like(k), dv = like(v);
    const Tensor delta = at::empty_like(softmax_lse);
    p.dq = view(dq, "dq");
    p.dk = view(dk, "dk");
    p.dv = view(dv, "dv");
    p.softmax_d = delta.data_ptr<float>();
    const Tensor ws = workspace(shaobo_fa3_attn_bwd_workspace_bytes(&p), q, &p);
    check_status(shaobo_fa3_attn_bwd(&p, stream_of(q)), "shaobo_fa3_attn_bwd");
    return {dq, dk, dv, delta};
}

std::vector<Tensor> rotary(at::TensorList xs, const Tensor& positions, const Tensor& freqs,
                           bool interleaved, bool inverse) {
    TORCH_CHECK_VALUE(xs.size() == 1 || xs.size() == 2, "rotary takes one or two tensors");
    const Tensor& x = xs[0];
    TORCH_CHECK_VALUE(x.dim() == 4, "rotary's tensors must be [batch, heads, sequence, head_dim]");
    const int64_t B = x.size(0), S = x.size(2), D = x.size(3);
    const auto dt = x.scalar_type();
    TORCH_CHECK_VALUE(dt == at::kHalf || dt == at::kBFloat16 || dt == at::kFloat,
                      "rotary's tensors must be fp16, bf16 or fp32");
    TORCH_CHECK_VALUE(x.is_cuda(), "rotary's tensors must be on a GPU");
    for (const Tensor& t : xs)
        TORCH_CHECK_VALUE(t.dim() == 4 && t.size(0) == B && t.size(2) == S && t.size(3) == D &&
                              t.scalar_type() == dt && t.device() == x.device(),
                          "rotary's tensors must differ in their heads only");
    TORCH_CHECK_VALUE(D % 8 == 0 && D >= 8 && D <= 512, "head_dim must be a multiple of 8 up to 512");
    TORCH_CHECK_VALUE(freqs.dim() == 2 && freqs.scalar_type() == at::kFloat &&
                          freqs.is_contiguous() && freqs.device() == x.device(),
                      "freqs must be contiguous fp32 [axes, pairs] on the same GPU");
    const int64_t A = freqs.size(0), P = freqs.size(1);
    TORCH_CHECK_VALUE(A >= 1 && A <= 4, "rotary takes one to four axes");
    TORCH_CHECK_VALUE(P >= 8 && P % 8 == 0 && 2 * P <= D,
                      "pairs must be a multiple of 8, and twice as many at most head_dim");
    TORCH_CHECK_VALUE(positions.dim() == 3 && positions.size(0) == A && positions.size(1) == B &&
                          positions.size(2) == S && positions.device() == x.device(),
                      "positions must be [axes, batch, sequence] on the same GPU");
    ShaoboFa3RotaryParams p;
    shaobo_fa3_rotary_params_init(&p);
    switch (positions.scalar_type()) {
        case at::kInt: p.position_type = SHAOBO_FA3_POSITIONS_INT32; break;
        case at::kLong: p.position_type = SHAOBO_FA3_POSITIONS_INT64; break;
        case at::kFloat: p.position_type = SHAOBO_FA3_POSITIONS_FP32; break;
        default: TORCH_CHECK_VALUE(false, "positions must be int32, int64 or fp32");
    }
    TORCH_CHECK_VALUE(B < (1 << 24) && S < (1 << 24) && B * S < (1 << 24), "too many positions");
    p.batch = (int32_t)B;
    p.seqlen = (int32_t)S;
    p.head_dim = (int32_t)D;
    p.dtype = dt == at::kFloat ? SHAOBO_FA3_DTYPE_FP32
              : dt == at::kBFloat16 ? SHAOBO_FA3_DTYPE_BF16 : SHAOBO_FA3_DTYPE_FP16;
    p.axes = (int32_t)A;
    p.pairs = (int32_t)P;
    p.interleaved = interleaved;
    p.inverse = inverse;
    p.positions = positions.data_ptr();
    p.position_axis_stride = positions.stride(0);
    p.position_batch_stride = positions.stride(1);
    p.position_row_stride = positions.stride(2);
    p.freqs = freqs.data_ptr<float>();
    p.tensors = (int32_t)xs.size();
    const Guard guard(x.device());
    std::vector<Tensor> ys;
    for (size_t i = 0; i < xs.size(); ++i) {
        TORCH_CHECK_VALUE(xs[i].size(1) >= 1 && xs[i].size(1) <= (1 << 16), "too many heads, or none");
        ys.push_back(like(xs[i]));
        p.heads[i] = (int32_t)xs[i].size(1);
        p.in[i] = view(xs[i], "rotary's tensors");
        p.out[i] = view(ys[i], "rotary's outputs");
    }
    check_status(shaobo_fa3_rotary(&p, stream_of(x)), "shaobo_fa3_rotary");
    return ys;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(shaobo_fa3, m) {
    m.def(
        "attn_forward(Tensor q, Tensor k, Tensor v, bool causal, float? softmax_scale=None, "
        "float softcap=0.0, Tensor? slopes=None, Tensor? documents=None, "
        "Tensor? documents_k=None, Tensor? prefix_lens=None, Tensor? kv_lens=None) -> "
        "(Tensor, Tensor)");
    m.def(
        "attn_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor softmax_lse, "
        "bool causal, float? softmax_scale=None, float softcap=0.0, Tensor? slopes=None, "
        "Tensor? documents=None, Tensor? documents_k=None, Tensor? prefix_lens=None, "
        "Tensor? kv_lens=None) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def(
        "rotary(Tensor[] xs, Tensor positions, Tensor freqs, bool interleaved=False, "
        "bool inverse=False) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(shaobo_fa3, CUDA, m) {
    m.impl("attn_forward", &attn_forward);
    m.impl("attn_backward", &attn_backward);
    m.impl("rotary", &rotary);
}
