/*
 * shaobo_fa3_cache.h -- a paged cache of keys and values for the attention
 * layer of shaobo_fa3_attn.h: appending to it with the rotary positions
 * applied on the way, attention to it (all of it, or selected pages), the
 * selection, and reading it back.  Held in 16 bits or in 4.  For serving: no
 * gradients.  No counterpart in the reference.
 *
 * Pages.  Positions [n page_size, (n + 1) page_size) of sequence b are rows of
 * page page_table[b][n]; a number outside [0, pages) is no page: nothing is
 * written there, and its keys take no part.  A page belongs to one sequence
 * where it is written; sequences may share pages that are only read.  The rows
 * that a call writes (of k, of v, of q_out) must not share memory.
 *
 * Lengths.  kv_lens[b] tokens are in the cache after the call's tokens are
 * (taken into 0 .. width page_size).  Of the seqlen rows of q, k and v the
 * first new_lens[b] (taken into 0 .. seqlen; all, where there are none) are
 * tokens, the rest padding: token i is at place kv_lens[b] - new_lens[b] + i.
 * An append alone follows lengths past the table, up to 2^30 + 2^24: it writes
 * no token whose place is not in the table, and none over an earlier one.
 *
 * 16 bits: k and v are [pages, num_heads_kv, page_size, head_dim] in dtype.
 *
 * 4 bits: a row x of head_dim values is head_dim codes and one fp32 scale,
 * a / 6 for a = max |x|.  A code is a sign (8, of values below 0) and a level of
 * 0, 1/2, 1, 3/2, 2, 3, 4, 6, the nearest to 6 |x| / a (halfway: the even code); it stands for
 * level * scale.  Channels 2 c and 2 c + 1 share byte c, the first in its low
 * half.  The page_size * (head_dim / 2 + 4) bytes of a page and head are the
 * codes of all its rows, then their scales.  A row with a value that is not
 * finite stands for NaN.
 *
 * Bounds: [pages, num_heads_kv, 2, head_dim] in dtype, contiguous: for each
 * channel the smallest and the largest key (before it becomes 4 bits) that
 * appends have written to the page; a row at a page's first place starts them
 * anew.  Rows written over otherwise leave them as wide as they were.  A NaN is
 * beyond the infinity of its sign.
 *
 * Streams, launches and workspaces are as in shaobo_fa3_attn.h.
 */
#ifndef SHAOBO_FA3_CACHE_H_
#define SHAOBO_FA3_CACHE_H_

#include "shaobo_fa3_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Pages on the GPU, 16-byte aligned; strides in elements (4 bits: in bytes),
 * multiples of 16 bytes; row_stride is of 16 bits only. */
typedef struct ShaoboFa3CachePages {
    void* data;
    int64_t page_stride;
    int64_t head_stride;
    int64_t row_stride;
} ShaoboFa3CachePages;

typedef struct ShaoboFa3Cache {
    int32_t batch;
    int32_t num_heads_kv;
    int32_t head_dim;   /* a multiple of 8, 8 to 128; 4 bits: 64 or 128 */
    int32_t dtype;      /* SHAOBO_FA3_DTYPE_FP16 or _BF16 */
    int32_t bits;       /* 16 or 4 */
    int32_t pages;
    int32_t page_size;  /* 32, 64, 128, 256, 512 or 1024 */
    int32_t width;      /* pages per sequence in the table */
    ShaoboFa3CachePages k, v;
    const int32_t* page_table;  /* [batch, width], rows contiguous */
    int64_t page_table_stride;
    const int32_t* kv_lens;     /* [batch] */
    const int32_t* new_lens;    /* [batch], or NULL */
    void* bounds;               /* or NULL */
} ShaoboFa3Cache;

/* Writes k and v of the new tokens into the cache, k turned by its position
 * (bounds, where they are given, follow), and q_out = q turned likewise.
 * freqs NULL: nothing is turned.  positions NULL: one axis, a token's place;
 * otherwise as shaobo_fa3_rotary takes them.  Every row of q is turned,
 * padding too.  The turn is formed in fp64 and becomes dtype by way of fp32, as a
 * cast does. */
typedef struct ShaoboFa3CacheAppendParams {
    uint32_t struct_size;
    int32_t seqlen;
    int32_t num_heads_q;     /* 0: no queries */
    int32_t axes;            /* 1 to 4 */
    int32_t pairs;           /* a multiple of 8; 2 pairs <= head_dim */
    int32_t interleaved;     /* 0 or 1 */
    int32_t position_type;   /* SHAOBO_FA3_POSITIONS_* */
    ShaoboFa3Cache cache;
    ShaoboFa3AttnTensor k, v, q;
    ShaoboFa3AttnTensor q_out; /* may be q */
    const void* positions;   /* [axes, batch, seqlen], strides in elements, or NULL */
    int64_t position_axis_stride;
    int64_t position_batch_stride;
    int64_t position_row_stride;
    const float* freqs;      /* [axes, pairs], contiguous, or NULL */
} ShaoboFa3CacheAppendParams;

void shaobo_fa3_cache_append_params_init(ShaoboFa3CacheAppendParams* params);
int shaobo_fa3_cache_append(const ShaoboFa3CacheAppendParams* params, void* stream);

/* Attention of the new tokens' queries to their sequences, as in
 * shaobo_fa3_attn.h without documents: token i is at its place, a key at its
 * own, and visible = j < kv, its page is one, and (not causal or j <= place or
 * j < prefix).  With `selected` only keys of the pages listed for (b, KV head,
 * i) are looked at: page numbers of the sequence, those outside [0, width) left
 * out, one that is listed twice counted twice.  Padding rows give zeros and -inf.
 * As there, sums of V are finite where |v| times 2^8 times the visible keys is
 * below 2^127.
 *
 * 4 bits: scores are of what the codes stand for, in fp32 (levels are exact in
 * 16 bits, the scale is applied to the product); P times a value's scale is
 * rounded for its product with the levels, to bf16, or to 16 bits (two bf16
 * terms) in fp16. */
typedef struct ShaoboFa3CacheAttnParams {
    uint32_t struct_size;
    int32_t seqlen;
    int32_t num_heads_q;
    int32_t causal;                /* 0 or 1 */
    int32_t softmax_scale_is_set;  /* 0: 1 / sqrt(head_dim) */
    float softmax_scale;           /* -1e30 to 1e30 */
    float softcap;                 /* 0: none; up to 1e30 */
    int32_t count;                 /* pages listed per row of `selected` */
    ShaoboFa3Cache cache;
    ShaoboFa3AttnTensor q;
    ShaoboFa3AttnTensor out;
    float* softmax_lse;            /* [batch, num_heads_q, seqlen], contiguous */
    const float* slopes;           /* [batch or 1, num_heads_q], or NULL */
    int64_t slopes_batch_stride;
    const int32_t* prefix_lens;    /* [batch] or NULL; needs causal */
    const int32_t* selected;       /* [batch, num_heads_kv, seqlen, count], contiguous, or NULL */
    void* workspace;               /* 256-byte aligned */
    size_t workspace_bytes;
} ShaoboFa3CacheAttnParams;

void shaobo_fa3_cache_attn_params_init(ShaoboFa3CacheAttnParams* params);
int shaobo_fa3_cache_attn_validate(const ShaoboFa3CacheAttnParams* params);
size_t shaobo_fa3_cache_attn_workspace_bytes(const ShaoboFa3CacheAttnParams* params);
int shaobo_fa3_cache_attn(const ShaoboFa3CacheAttnParams* params, void* stream);

/* Selects `count` pages for every new token and KV head: the token's own page
 * and, of those before it, the ones whose bounds allow the largest score:
 *   score = max over the group's query heads of
 *           sum_c max(q_c low_c, q_c high_c),    in fp64
 * (equal scores: the lower page; a page and head with a bound or a score that
 * is not finite comes before all that are).
 * Page numbers of the sequence, ascending, -1 behind them; pages that are none,
 * the token's own among them, are left out, the others still listed.  All -1
 * for padding and for a token whose place is below 0.
 * For a positive softmax scale; the cache's k and v are not looked at. */
typedef struct ShaoboFa3CacheSelectParams {
    uint32_t struct_size;
    int32_t seqlen;
    int32_t num_heads_q;
    int32_t count;
    ShaoboFa3Cache cache;
    ShaoboFa3AttnTensor q;
    int32_t* selected;             /* [batch, num_heads_kv, seqlen, count], contiguous */
    void* workspace;               /* 256-byte aligned */
    size_t workspace_bytes;
} ShaoboFa3CacheSelectParams;

void shaobo_fa3_cache_select_params_init(ShaoboFa3CacheSelectParams* params);
int shaobo_fa3_cache_select_validate(const ShaoboFa3CacheSelectParams* params);
size_t shaobo_fa3_cache_select_workspace_bytes(const ShaoboFa3CacheSelectParams* params);
int shaobo_fa3_cache_select(const ShaoboFa3CacheSelectParams* params, void* stream);

/* k and v [batch, num_heads_kv, seqlen, head_dim] in dtype: the first seqlen
 * places of every sequence as the cache holds them (4 bits: level times scale in
 * fp32, rounded to dtype), zeros at and behind kv_lens[b] and where there is no
 * page. */
typedef struct ShaoboFa3CacheReadParams {
    uint32_t struct_size;
    int32_t seqlen;
    ShaoboFa3Cache cache;
    ShaoboFa3AttnTensor k, v;
} ShaoboFa3CacheReadParams;

void shaobo_fa3_cache_read_params_init(ShaoboFa3CacheReadParams* params);
int shaobo_fa3_cache_read(const ShaoboFa3CacheReadParams* params, void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* SHAOBO_FA3_CACHE_H_ */
