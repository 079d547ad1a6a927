/*
 * gdn_attention_hip.h — C ABI of libgdn_hip.so, third part: softmax attention over a window, the norm and rotation of its queries and
 * keys, its paged cache in 8 bits, and attention over that cache.
 *
 * Conventions are those of gdn_hip.h: every pointer is a DEVICE pointer owned by the caller, the library holds no state,
 * never allocates, frees or synchronises, and launches asynchronously on the stream it is given (current device of the
 * calling thread).  Return value of every int-returning entry point: 0, a negative gdn_status, or a positive hipError_t.
 * Zero a struct before filling it.
 */
#ifndef GDN_ATTENTION_HIP_H
#define GDN_ATTENTION_HIP_H

#include "gdn_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GDN_ATTENTION_ABI_VERSION 1

int gdn_attention_abi_version(void);

/*
 * RMS norm of every head of q and k, and the rotation by position, in one pass.  For each row x [D] (one head of one token):
 *     n = x / sqrt(mean(x^2) + eps) * weight
 *     y_i = n_i cos_i - n_{i + R/2} sin_i,   y_{i + R/2} = n_{i + R/2} cos_i + n_i sin_i   (i < R / 2),   y_i = n_i (i >= R)
 * with row `pos` of the tables.  Index 0 is q, 1 is k.
 *
 *   x          [B, T, heads, D]   element strides, last dim contiguous; rows aligned to 8 elements (fp32: 4)
 *   y          the same shape, contiguous
 *   weight     [D] of w_dtype, or NULL
 *   cos, sin   [table_rows, R / 2] fp32, contiguous
 *   pos        [B, T] int32, pos_stride_b elements between rows (0: one row for all), or NULL: token t has position t.  A position
 *              that the tables do not have makes its rows NaN
 *
 * D and R multiples of 8, R <= D <= 512.
 */
#define GDN_QK_ROTARY_MAX_D 512

typedef struct gdn_qk_rotary_args {
    const void *x[2];
    const void *weight[2];
    void *y[2];
    const float *cos;
    const float *sin;
    const int32_t *pos;
    int64_t pos_stride_b;
    int64_t x_stride_b[2], x_stride_t[2], x_stride_h[2];
    int32_t heads[2];
    int32_t B, T, D, R, table_rows;
    int32_t dtype;
    int32_t w_dtype;
    float eps;
} gdn_qk_rotary_args;

int gdn_qk_norm_rotary_fwd(const gdn_qk_rotary_args *args, void *stream);

/*
 * Its gradients from the forward's inputs and dy (strides and alignment as x): dx (contiguous), and the sums over rows for the
 * weights' gradients as partial_blocks partial rows [partial_blocks, D] fp32 each (NULL: not wanted), which gdn_column_sums
 * adds up in a fixed order.  fwd.y is not used.  partial_blocks: gdn_qk_rotary_partial_blocks.
 */
typedef struct gdn_qk_rotary_bwd_args {
    gdn_qk_rotary_args fwd;
    const void *dy[2];
    void *dx[2];
    float *dweight_partial[2];
    int64_t dy_stride_b[2], dy_stride_t[2], dy_stride_h[2];
    int32_t partial_blocks;
    int32_t reserved;
} gdn_qk_rotary_bwd_args;

int gdn_qk_norm_rotary_bwd(const gdn_qk_rotary_bwd_args *args, void *stream);

/* Workgroups, and with them partial rows, that gdn_qk_norm_rotary_bwd uses for these sizes on the current device; 0 for sizes it refuses. */
int gdn_qk_rotary_partial_blocks(const gdn_qk_rotary_args *args);

/*
 * Softmax attention over a window.  A query at key position p sees the keys j <= p of its sequence with j > p - window or among the
 * sequence's first `sinks`:   o = sum_j softmax_j(scale q . k_j) v_j;   zeros where no key is visible.
 *
 *   q, o   [B, T, H, D]    element strides, last dim contiguous; query head h reads head h / (H / HK) of k and v
 *   k, v   [B, S, HK, D]   query t stands at key position t + S - T; with cu_seqlens T == S
 *   lse    fp32 or NULL: what the backward needs.  dtype bf16: [B, T, H], log2 of the sum of 2^(scale log2(e) q . k_j), +inf where no
 *          key is visible; dtype fp32: [B, T, H, 2], the largest exponent m and 1 / sum 2^(scale log2(e) q . k_j - m)
 *   cu_seqlens, N, GDN_FLAG_LEFT_PADDED   as in gdn_args: packed sequences (B == 1) or a left-padded batch (N == B)
 *   window  0: every key up to the query's own
 *
 * Tokens of no sequence (padding, tokens in front of and behind the packed sequences) read as zeros in o and in the gradients.
 * D a multiple of 8 up to 256, dtype bf16 or fp32.  Rows, and with them strides, 16-byte aligned; tokens 0 to 2^23 elements apart, the heads
 * of a token within 2^28.
 */
typedef struct gdn_window_attn_args {
    const void *q;
    const void *k;
    const void *v;
    void *o;
    float *lse;
    const int32_t *cu_seqlens;
    void *workspace;
    uint64_t workspace_bytes;

    int64_t q_stride_b, q_stride_t, q_stride_h;
    int64_t k_stride_b, k_stride_t, k_stride_h;
    int64_t v_stride_b, v_stride_t, v_stride_h;
    int64_t o_stride_b, o_stride_t, o_stride_h;

    int32_t B, T, S, H, HK, D, N;
    int32_t window, sinks;
    int32_t dtype;
    int32_t flags; /* GDN_FLAG_LEFT_PADDED */
    float scale;
} gdn_window_attn_args;

int gdn_window_attn_fwd(const gdn_window_attn_args *args, void *stream);

/* Bytes of args->workspace for gdn_window_attn_fwd (may be 0); reads shape fields, window, sinks, dtype, whether cu_seqlens is NULL, and the
 * current device. */
uint64_t gdn_window_attn_workspace_bytes(const gdn_window_attn_args *args);

/*
 * Gradients from the forward's inputs, its o and lse, and dout [B, T, H, D]: dq [B, T, H, D], dk and dv [B, S, HK, D] (the gradients of
 * query heads that share one of k and v are added up in fp32), all in the inputs' dtype, with element strides, written whole.  In bf16 at most
 * 65280 query heads share one.
 */
typedef struct gdn_window_attn_bwd_args {
    gdn_window_attn_args fwd;
    const void *dout;
    void *dq;
    void *dk;
    void *dv;
    void *workspace;
    uint64_t workspace_bytes;

    int64_t dout_stride_b, dout_stride_t, dout_stride_h;
    int64_t dq_stride_b, dq_stride_t, dq_stride_h;
    int64_t dk_stride_b, dk_stride_t, dk_stride_h;
    int64_t dv_stride_b, dv_stride_t, dv_stride_h;
} gdn_window_attn_bwd_args;

int gdn_window_attn_bwd(const gdn_window_attn_bwd_args *args, void *stream);
uint64_t gdn_window_attn_bwd_workspace_bytes(const gdn_window_attn_bwd_args *args);

/*
 * A paged cache of keys and values in 8 bits.  A page holds P tokens of all HK heads; a code c (e4m3) of a page and head whose scale is s
 * stands for c 2^(s - 127).
 *
 *   k_codes    [pages, HK, P, D]            v_codes   [pages, HK, P / 16, D, 16]   (16 tokens of a column together)
 *   k_scales, v_scales   [pages, HK] uint8, 27 to 247
 *   table      [N, table_pages] int32, table_stride elements between rows: the pages of sequence n in order.  A page that is not in
 *              [0, pages) is not followed: what would be written there is dropped, what would be read there is NaN
 *
 * All contiguous.  P a multiple of 16 from 16 to 256, D a multiple of 16 up to 256; HK at most 65535; k_codes and v_codes 16-byte aligned.
 */
typedef struct gdn_paged_cache {
    void *k_codes;
    void *v_codes;
    uint8_t *k_scales;
    uint8_t *v_scales;
    const int32_t *table;
    int64_t table_stride;
    int32_t pages, P, HK, D;
    int32_t N, table_pages;
} gdn_paged_cache;

/*
 * Writes new tokens behind those that the cache holds: token i of sequence n at position start[n] + i.  A page's scale is the smallest with
 * which none of its values passes 448 (at least 27, an exponent of -100); a page that held tokens before keeps its scale or takes a larger one,
 * the older codes rounded to it.  Codes are rounded to nearest, ties to even; values that are not finite become NaN and do not count
 * for the scale.  Behind the last new token of a page its codes are left as they were.
 *
 *   k, v   [B, T, HK, D]   element strides, last dim contiguous, rows 16-byte aligned; bf16 or fp32
 *   start  [N] int32; tokens that would lie in front of position 0 or past table_pages * P are dropped
 *   cu_seqlens, GDN_FLAG_LEFT_PADDED   as in gdn_args (of the new tokens)
 */
typedef struct gdn_cache_write_args {
    gdn_paged_cache cache;
    const void *k;
    const void *v;
    const int32_t *start;
    const int32_t *cu_seqlens;
    int64_t k_stride_b, k_stride_t, k_stride_h;
    int64_t v_stride_b, v_stride_t, v_stride_h;
    int32_t B, T;
    int32_t dtype;
    int32_t flags;
} gdn_cache_write_args;

int gdn_cache_write(const gdn_cache_write_args *args, void *stream);

/* What the first min(lengths[n], T) tokens of every sequence stand for, k and v [N, T, HK, D] contiguous of dtype, zeros behind them. */
typedef struct gdn_cache_read_args {
    gdn_paged_cache cache;
    void *k;
    void *v;
    const int32_t *lengths;
    int32_t T;
    int32_t dtype;
} gdn_cache_read_args;

int gdn_cache_read(const gdn_cache_read_args *args, void *stream);

/*
 * Attention of the last T tokens of every sequence over its pages: query i of sequence n stands at position lengths[n] - T + i
 * and sees what a query of gdn_window_attn_fwd sees.  q, o [N, T, H, D] bf16, element strides, rows 16-byte aligned.
 */
typedef struct gdn_cache_attn_args {
    gdn_paged_cache cache;
    const void *q;
    void *o;
    const int32_t *lengths;
    void *workspace;
    uint64_t workspace_bytes;
    int64_t q_stride_b, q_stride_t, q_stride_h;
    int64_t o_stride_b, o_stride_t, o_stride_h;
    int32_t T, H;
    int32_t window, sinks;
    float scale;
    int32_t reserved;
} gdn_cache_attn_args;

int gdn_cache_attn(const gdn_cache_attn_args *args, void *stream);

/* Bytes of args->workspace (may be 0); reads shape fields, window, sinks, and the current device. */
uint64_t gdn_cache_attn_workspace_bytes(const gdn_cache_attn_args *args);

#ifdef __cplusplus
}
#endif

#endif /* GDN_ATTENTION_HIP_H */
