/*
 * shaobo_fa3_attn.h -- the attention layer around the backward of
 * shaobo_fa3_api.h: rotary positions on several axes, and softmax attention
 * with capped, biased and masked scores, forward and backward, for any
 * sequence lengths (a prompt, a training batch, a single token against a
 * long cache).  No counterpart in the reference, whose ABI rejects softcap,
 * key lengths and every mask but the causal one
 * (reference src/shaobo_fa3_bwd_api.cpp:70-120).
 *
 * Attention.  For query head h (KV head h / (num_heads_q / num_heads_kv)),
 * query i and key j of batch entry b, with kv = kv_lens[b] (seqlen_k where
 * there is none) and d = i + kv - seqlen_q - j, the distance back to the key
 * when the queries are the last seqlen_q of the kv positions:
 *   s       = softmax_scale q_i . k_j
 *   s       = softcap tanh(s / softcap)            where softcap > 0
 *   s       = s - slopes[h] |d|                    where there are slopes
 *   visible = j < kv
 *             and (not causal or d >= 0 or j < prefix_lens[b])
 *             and (no documents or documents_q[b][i] == documents_k[b][j] >= 0)
 *   out_i   = sum_j softmax(s)_ij v_j over the visible keys; 0 if none is
 *   lse_i   = log sum_j exp(s_ij);                        -inf if none is
 * The backward returns dq, dk, dv of these outputs from out and lse; slopes
 * have no gradient.  Sums, softmax statistics, dot products and biases are
 * fp32; P and dS are rounded to the tensors' type before their products with
 * V, dO, Q and K, and the outputs once more (in fp16 a dS below 2^-14 loses
 * bits as gradients do: scale the loss).  Results are bitwise reproducible.
 *
 * Keys at kv and behind, and keys with a negative document, take no part
 * whatever their K and V hold (NaN included), and neither do queries that
 * see no key, whatever their Q and dO hold.  A NaN in a row's Q or in a key
 * it sees makes the row's outputs NaN (but V of keys that a distance bias
 * leaves less than 2^-64 of the row's largest weight may not be looked at);
 * a NaN or infinity in one visible key or row can also reach other rows and
 * keys of its batch entry and KV head, rows that see no key excepted.
 *
 * Nothing is allocated; launches go to `stream` (a hipStream_t of the
 * current GPU, NULL = the null stream) and are not waited for, so they can
 * be captured into a graph.  Two calls that may overlap in time must not
 * share a workspace.
 */
#ifndef SHAOBO_FA3_ATTN_H_
#define SHAOBO_FA3_ATTN_H_

#include "shaobo_fa3_api.h"

#ifdef __cplusplus
extern "C" {
#endif

/* An element type of shaobo_fa3_rotary, beside ShaoboFa3DType. */
#define SHAOBO_FA3_DTYPE_FP32 3

/* A [batch, heads, rows, head_dim] tensor on the GPU: 16-byte aligned, the
 * elements of a row contiguous, the other strides given in elements, each a
 * multiple of 16 bytes (0 and negative ones included; outputs must not
 * overlap themselves). */
typedef struct ShaoboFa3AttnTensor {
    void* data;
    int64_t batch_stride;
    int64_t head_stride;
    int64_t row_stride;
} ShaoboFa3AttnTensor;

typedef struct ShaoboFa3AttnParams {
    uint32_t struct_size;
    int32_t batch;
    int32_t seqlen_q;
    int32_t seqlen_k;
    int32_t num_heads_q;
    int32_t num_heads_kv;
    int32_t head_dim;  /* a multiple of 8, 8 to 128 */
    int32_t dtype;     /* SHAOBO_FA3_DTYPE_FP16 or _BF16 */
    int32_t causal;    /* 0 or 1 */
    int32_t softmax_scale_is_set; /* 0: 1 / sqrt(head_dim) */
    float softmax_scale;          /* -1e30 to 1e30 */
    float softcap;                /* 0: none; up to 1e30 */

    ShaoboFa3AttnTensor q, k, v;   /* inputs */
    ShaoboFa3AttnTensor out;       /* forward: written; backward: read */
    ShaoboFa3AttnTensor dout;      /* backward: read */
    ShaoboFa3AttnTensor dq, dk, dv;/* backward: written */
    float* softmax_lse; /* [batch, num_heads_q, seqlen_q], contiguous; forward writes it */
    float* softmax_d;   /* the same, or NULL; backward writes rowsum(dout * out) */

    const float* slopes;           /* [batch or 1, num_heads_q], or NULL */
    int64_t slopes_batch_stride;   /* 0: one set for the batch */
    const int32_t* documents_q;    /* [batch, seqlen_q]; both or neither */
    const int32_t* documents_k;    /* [batch, seqlen_k] */
    int64_t documents_q_batch_stride;
    int64_t documents_k_batch_stride;
    const int32_t* prefix_lens;    /* [batch] or NULL; needs causal */
    const int32_t* kv_lens;        /* [batch] or NULL; taken into 0 .. seqlen_k */

    void* workspace;               /* 256-byte aligned scratch, need not be cleared */
    size_t workspace_bytes;
} ShaoboFa3AttnParams;

/* Zero the struct, then set struct_size, FP16 and causal = 0. */
void shaobo_fa3_attn_params_init(ShaoboFa3AttnParams* params);

/* Check sizes, options and strides only (no pointer is read, nothing is
 * launched): SUCCESS, INVALID_VALUE (malformed) or UNSUPPORTED. */
int shaobo_fa3_attn_fwd_validate(const ShaoboFa3AttnParams* params);
int shaobo_fa3_attn_bwd_validate(const ShaoboFa3AttnParams* params);

/* Workspace of one call, a function of sizes and options (which of the
 * optional pointers are set counts, not where they point); 0 may mean that
 * none is needed, and is what invalid parameters give. */
size_t shaobo_fa3_attn_fwd_workspace_bytes(const ShaoboFa3AttnParams* params);
size_t shaobo_fa3_attn_bwd_workspace_bytes(const ShaoboFa3AttnParams* params);

/* out and softmax_lse from q, k, v. */
int shaobo_fa3_attn_fwd(const ShaoboFa3AttnParams* params, void* stream);

/* dq, dk, dv (and softmax_d) from dout, q, k, v, out and softmax_lse.  dk
 * and dv of keys that no query sees are written as zeros. */
int shaobo_fa3_attn_bwd(const ShaoboFa3AttnParams* params, void* stream);

/* Rotary positions.  The first 2 pairs elements of each row are turned in
 * pairs (p, pairs + p), or (2 p, 2 p + 1) where `interleaved`, by
 *   angle[b][s][p] = sum_a positions[a][b][s] freqs[a][p]
 *   (x, y) -> (x cos - y sin, y cos + x sin),
 * by the negative angle where `inverse` (the gradient, and the way back);
 * the other elements are copied.  freqs in one row per axis cover positions
 * of one axis as well as time, height and width that own pairs each (zeros
 * elsewhere) or share them.  Angles are reduced to a turn before they become
 * fp32, off by 2^-50 of a turn at most an axis where |position| and |position
 * freq| are up to 2^53 (integers past that are rounded to fp64 first), so far
 * positions lose nothing; the rotation is fp32, rounded to 16 bits once. */
#define SHAOBO_FA3_POSITIONS_INT32 0
#define SHAOBO_FA3_POSITIONS_INT64 1
#define SHAOBO_FA3_POSITIONS_FP32 2

typedef struct ShaoboFa3RotaryParams {
    uint32_t struct_size;
    int32_t batch;
    int32_t seqlen;
    int32_t head_dim;        /* a multiple of 8, 8 to 512 */
    int32_t dtype;           /* SHAOBO_FA3_DTYPE_FP16, _BF16 or _FP32 */
    int32_t axes;            /* 1 to 4 */
    int32_t pairs;           /* a multiple of 8; 2 pairs <= head_dim */
    int32_t interleaved;     /* 0 or 1 */
    int32_t inverse;         /* 0 or 1 */
    int32_t position_type;   /* SHAOBO_FA3_POSITIONS_* */
    const void* positions;   /* [axes, batch, seqlen], strides in elements */
    int64_t position_axis_stride;
    int64_t position_batch_stride;
    int64_t position_row_stride;
    const float* freqs;      /* [axes, pairs], contiguous */
    int32_t tensors;         /* 1 or 2 (q and k in one launch) */
    int32_t heads[2];
    ShaoboFa3AttnTensor in[2];
    ShaoboFa3AttnTensor out[2];  /* may be the same tensor as in */
} ShaoboFa3RotaryParams;

void shaobo_fa3_rotary_params_init(ShaoboFa3RotaryParams* params);
int shaobo_fa3_rotary(const ShaoboFa3RotaryParams* params, void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* SHAOBO_FA3_ATTN_H_ */
