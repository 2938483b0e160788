// What the PyTorch operators of the attention layer and of its cache share:
// checks of tensors and the views the library takes.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <cmath>
#include <string>
#include <tuple>
#include <vector>

#include "shaobo_fa3_attn.h"

namespace {

using at::Tensor;
using c10::optional;
using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

void* stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// What the library refuses is a ValueError as the checks here are (they leave
// it what does not fit a launch); a HIP error is not.
void check_status(int st, const char* entry) {
    TORCH_CHECK_VALUE(st != SHAOBO_FA3_STATUS_INVALID_VALUE, entry, ": ", shaobo_fa3_status_string(st));
    TORCH_CHECK_VALUE(st != SHAOBO_FA3_STATUS_UNSUPPORTED, entry, ": ", shaobo_fa3_status_string(st),
                      ", more rows, heads or positions than a launch takes");
    TORCH_CHECK(st == SHAOBO_FA3_STATUS_SUCCESS, entry, ": ", shaobo_fa3_status_string(st));
}

// A [B, H, S, D] tensor as the library takes it: rows contiguous, every row
// 16-byte aligned.
ShaoboFa3AttnTensor view(const Tensor& t, const char* name) {
    const int64_t align = 16 / t.element_size();
    TORCH_CHECK_VALUE(t.size(3) <= 1 || t.stride(3) == 1, name, ": head_dim must be contiguous");
    ShaoboFa3AttnTensor v;
    v.data = t.data_ptr();
    int64_t s[3];
    for (int i = 0; i < 3; ++i) {
        s[i] = t.size(i) <= 1 ? 0 : t.stride(i);  // (a stride that is never taken)
        TORCH_CHECK_VALUE(s[i] % align == 0, name, ": strides must be multiples of 16 bytes");
    }
    TORCH_CHECK_VALUE(t.numel() == 0 || (uintptr_t)v.data % 16 == 0, name,
                      ": must be 16-byte aligned");
    v.batch_stride = s[0];
    v.head_stride = s[1];
    v.row_stride = s[2];
    return v;
}

void check_int32(const Tensor& t, at::IntArrayRef shape, const Tensor& like, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt, name, " must be int32");
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", not ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == like.device(), name, " must be on the same GPU");
}

// A distance bias of q's heads, fp32 [heads_q] or [batch, heads_q].
const float* slopes_of(const Tensor& t, const Tensor& q, int64_t* batch_stride) {
    const int64_t B = q.size(0), Hq = q.size(1);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "slopes must be fp32");
    TORCH_CHECK_VALUE((t.dim() == 1 && t.size(0) == Hq) ||
                          (t.dim() == 2 && t.size(0) == B && t.size(1) == Hq),
                      "slopes must be [heads_q] or [batch, heads_q]");
    TORCH_CHECK_VALUE(t.device() == q.device(), "slopes must be on the same GPU");
    TORCH_CHECK_VALUE(Hq == 1 || t.stride(-1) == 1, "slopes of one batch entry must be contiguous");
    *batch_stride = t.dim() == 2 && B > 1 ? t.stride(0) : 0;
    return t.data_ptr<float>();
}

// A dense tensor of t's shape and, where t is dense, its layout in memory.
// (head_dim is a multiple of 8 and contiguous in t: its rows are whole chunks.)
Tensor like(const Tensor& t) { return at::empty_like(t); }

template <typename P>
Tensor workspace(size_t n, const Tensor& t, P* p) {
    if (n == 0) return Tensor();
    Tensor ws = at::empty({(int64_t)n}, t.options().dtype(at::kByte));
    p->workspace = ws.data_ptr();
    p->workspace_bytes = n;
    return ws;
}

}  // namespace
