// C entries of the attention layer (shaobo_fa3_attn.h): parameter checks,
// workspace sizes and launches.
#include "shaobo_fa3_attn.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "fa3_attn_internal.h"

namespace {

using fa3::AttnMask;
using fa3::AttnProblem;

// Sequences and head counts are held below these, so that rows, tiles and
// jobs count in 32 bits (their products are checked by the plans).
constexpr int32_t kMaxLen = 1 << 30;
constexpr int32_t kMaxHeads = 1 << 16;
// Scales and caps are held where their products with log2 e stay in fp32.
constexpr float kMaxScore = 1e30f;

bool strides_ok(const ShaoboFa3AttnTensor& t, int elements) {
    return t.batch_stride % elements == 0 && t.head_stride % elements == 0 &&
           t.row_stride % elements == 0;
}
bool tensor_ok(const ShaoboFa3AttnTensor& t) {
    return t.data != nullptr && (uintptr_t)t.data % 16 == 0;
}

// Sizes, options and strides, pointers aside.
int check(const ShaoboFa3AttnParams* a, bool backward, AttnProblem* p) {
    if (a == nullptr || a->struct_size < sizeof(ShaoboFa3AttnParams))
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (a->batch < 0 || a->seqlen_q < 0 || a->seqlen_k < 0 || a->num_heads_q <= 0 ||
        a->num_heads_kv <= 0 || a->num_heads_q % a->num_heads_kv != 0 || a->head_dim <= 0)
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if ((a->causal != 0 && a->causal != 1) ||
        (a->softmax_scale_is_set != 0 && a->softmax_scale_is_set != 1))
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (a->softmax_scale_is_set && !(std::fabs(a->softmax_scale) <= kMaxScore))
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (!(a->softcap >= 0.f && a->softcap <= kMaxScore)) return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if ((a->documents_q == nullptr) != (a->documents_k == nullptr))
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (a->prefix_lens != nullptr && !a->causal) return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (a->dtype != SHAOBO_FA3_DTYPE_FP16 && a->dtype != SHAOBO_FA3_DTYPE_BF16)
        return SHAOBO_FA3_STATUS_UNSUPPORTED;
    if (a->head_dim > 128 || a->head_dim % 8 != 0) return SHAOBO_FA3_STATUS_UNSUPPORTED;
    if (a->seqlen_q > kMaxLen || a->seqlen_k > kMaxLen || a->num_heads_q > kMaxHeads)
        return SHAOBO_FA3_STATUS_UNSUPPORTED;
    if (!strides_ok(a->q, 8) || !strides_ok(a->k, 8) || !strides_ok(a->v, 8) ||
        !strides_ok(a->out, 8))
        return SHAOBO_FA3_STATUS_UNSUPPORTED;
    if (backward && (!strides_ok(a->dout, 8) || !strides_ok(a->dq, 8) || !strides_ok(a->dk, 8) ||
                     !strides_ok(a->dv, 8)))
        return SHAOBO_FA3_STATUS_UNSUPPORTED;
    p->batch = a->batch;
    p->heads_q = a->num_heads_q;
    p->heads_kv = a->num_heads_kv;
    p->group = a->num_heads_q / a->num_heads_kv;
    p->sq = a->seqlen_q;
    p->sk = a->seqlen_k;
    p->d = a->head_dim;
    p->bf16 = a->dtype == SHAOBO_FA3_DTYPE_BF16;
    p->scale = a->softmax_scale_is_set ? a->softmax_scale : 1.f / std::sqrt((float)a->head_dim);
    p->softcap = a->softcap;
    p->causal = a->causal != 0;
    p->bias = a->slopes != nullptr;
    p->docs = a->documents_q != nullptr;
    if ((int64_t)p->batch * p->heads_q >= fa3::kMaxGrid) return SHAOBO_FA3_STATUS_UNSUPPORTED;
    const bool fits = backward ? fa3::plan_attn_bwd(*p).ok : fa3::plan_attn_fwd(*p).ok;
    return fits ? SHAOBO_FA3_STATUS_SUCCESS : SHAOBO_FA3_STATUS_UNSUPPORTED;
}

AttnMask mask_of(const ShaoboFa3AttnParams& a, const AttnProblem& p) {
    AttnMask m{};
    m.doc_q = a.documents_q;
    m.doc_k = a.documents_k;
    m.doc_q_bs = a.documents_q_batch_stride;
    m.doc_k_bs = a.documents_k_batch_stride;
    m.prefix = a.prefix_lens;
    m.kv_lens = a.kv_lens;
    m.slopes = a.slopes;
    m.slopes_bs = a.slopes_batch_stride;
    m.causal = a.causal;
    fa3::set_scores(&m, p.scale, p.softcap);
    return m;
}

int run(const ShaoboFa3AttnParams* a, bool backward, void* stream) {
    AttnProblem p;
    const int st = check(a, backward, &p);
    if (st != SHAOBO_FA3_STATUS_SUCCESS) return st;
    // (a tensor without elements needs no memory)
    const bool rows = p.batch > 0 && p.sq > 0, keys = p.batch > 0 && p.sk > 0;
    if (!rows && !(backward && keys)) return SHAOBO_FA3_STATUS_SUCCESS;
    bool ok = true;
    if (rows) ok = tensor_ok(a->q) && tensor_ok(a->out) && a->softmax_lse != nullptr;
    if (keys) ok = ok && tensor_ok(a->k) && tensor_ok(a->v);
    if (backward && rows) ok = ok && tensor_ok(a->dout) && tensor_ok(a->dq);
    if (backward && keys) ok = ok && tensor_ok(a->dk) && tensor_ok(a->dv);
    const size_t need = backward ? fa3::plan_attn_bwd(p).total : fa3::plan_attn_fwd(p).total;
    if (need > 0)
        ok = ok && a->workspace != nullptr && (uintptr_t)a->workspace % 256 == 0 &&
             a->workspace_bytes >= need;
    if (!ok) return SHAOBO_FA3_STATUS_INVALID_VALUE;
    int dev = -1;
    const hipError_t d = fa3::launch_device((hipStream_t)stream, &dev);
    if (d == hipErrorInvalidDevice) return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (d != hipSuccess) return SHAOBO_FA3_STATUS_HIP_ERROR;
    const AttnMask m = mask_of(*a, p);
    const hipError_t e = backward ? fa3::launch_attn_bwd(p, *a, m, (hipStream_t)stream)
                                  : fa3::launch_attn_fwd(p, *a, m, (hipStream_t)stream);
    return e == hipSuccess ? SHAOBO_FA3_STATUS_SUCCESS : SHAOBO_FA3_STATUS_HIP_ERROR;
}

size_t workspace_bytes(const ShaoboFa3AttnParams* a, bool backward) {
    AttnProblem p;
    if (check(a, backward, &p) != SHAOBO_FA3_STATUS_SUCCESS) return 0;
    return backward ? fa3::plan_attn_bwd(p).total : fa3::plan_attn_fwd(p).total;
}

}  // namespace

extern "C" {

void shaobo_fa3_attn_params_init(ShaoboFa3AttnParams* params) {
    if (params == nullptr) return;
    std::memset(params, 0, sizeof(*params));
    params->struct_size = (uint32_t)sizeof(*params);
    params->dtype = SHAOBO_FA3_DTYPE_FP16;
}

int shaobo_fa3_attn_fwd_validate(const ShaoboFa3AttnParams* params) {
    AttnProblem p;
    return check(params, false, &p);
}
int shaobo_fa3_attn_bwd_validate(const ShaoboFa3AttnParams* params) {
    AttnProblem p;
    return check(params, true, &p);
}
size_t shaobo_fa3_attn_fwd_workspace_bytes(const ShaoboFa3AttnParams* params) {
    return workspace_bytes(params, false);
}
size_t shaobo_fa3_attn_bwd_workspace_bytes(const ShaoboFa3AttnParams* params) {
    return workspace_bytes(params, true);
}
int shaobo_fa3_attn_fwd(const ShaoboFa3AttnParams* params, void* stream) {
    return run(params, false, stream);
}
int shaobo_fa3_attn_bwd(const ShaoboFa3AttnParams* params, void* stream) {
    return run(params, true, stream);
}

void shaobo_fa3_rotary_params_init(ShaoboFa3RotaryParams* params) {
    if (params == nullptr) return;
    std::memset(params, 0, sizeof(*params));
    params->struct_size = (uint32_t)sizeof(*params);
    params->dtype = SHAOBO_FA3_DTYPE_FP16;
    params->axes = 1;
    params->tensors = 1;
}

int shaobo_fa3_rotary(const ShaoboFa3RotaryParams* params, void* stream) {
    const ShaoboFa3RotaryParams* p = params;
    if (p == nullptr || p->struct_size < sizeof(ShaoboFa3RotaryParams))
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (p->batch < 0 || p->seqlen < 0 || p->head_dim <= 0 || p->pairs < 0 || p->axes < 1 ||
        (p->interleaved != 0 && p->interleaved != 1) || (p->inverse != 0 && p->inverse != 1) ||
        p->position_type < SHAOBO_FA3_POSITIONS_INT32 ||
        p->position_type > SHAOBO_FA3_POSITIONS_FP32 || p->tensors < 1 || p->tensors > 2)
        return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (p->dtype != SHAOBO_FA3_DTYPE_FP16 && p->dtype != SHAOBO_FA3_DTYPE_BF16 &&
        p->dtype != SHAOBO_FA3_DTYPE_FP32)
        return SHAOBO_FA3_STATUS_UNSUPPORTED;
    if (p->head_dim > 512 || p->head_dim % 8 != 0 || p->pairs % 8 != 0 || p->pairs < 8 ||
        p->pairs > p->head_dim / 2 || p->axes > 4)
        return SHAOBO_FA3_STATUS_UNSUPPORTED;
    const int align = p->dtype == SHAOBO_FA3_DTYPE_FP32 ? 4 : 8;
    for (int k = 0; k < p->tensors; ++k) {
        if (p->heads[k] <= 0) return SHAOBO_FA3_STATUS_INVALID_VALUE;
        if (p->heads[k] > kMaxHeads || !strides_ok(p->in[k], align) ||
            !strides_ok(p->out[k], align))
            return SHAOBO_FA3_STATUS_UNSUPPORTED;
    }
    if ((int64_t)p->batch * p->seqlen >= fa3::kMaxGrid) return SHAOBO_FA3_STATUS_UNSUPPORTED;
    if (p->batch == 0 || p->seqlen == 0) return SHAOBO_FA3_STATUS_SUCCESS;
    bool ok = p->positions != nullptr && p->freqs != nullptr;
    for (int k = 0; k < p->tensors; ++k) ok = ok && tensor_ok(p->in[k]) && tensor_ok(p->out[k]);
    if (!ok) return SHAOBO_FA3_STATUS_INVALID_VALUE;
    int dev = -1;
    const hipError_t d = fa3::launch_device((hipStream_t)stream, &dev);
    if (d == hipErrorInvalidDevice) return SHAOBO_FA3_STATUS_INVALID_VALUE;
    if (d != hipSuccess) return SHAOBO_FA3_STATUS_HIP_ERROR;
    return fa3::launch_rotary(*p, (hipStream_t)stream) == hipSuccess ? SHAOBO_FA3_STATUS_SUCCESS
                                                                     : SHAOBO_FA3_STATUS_HIP_ERROR;
}

}  // extern "C"
