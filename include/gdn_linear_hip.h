/*
 * gdn_linear_hip.h — C ABI of libgdn_hip.so, second part: linear attention with a decay for each head, and layer norm.
 *
 * Conventions are those of gdn_hip.h: every pointer is a DEVICE pointer owned by the caller, the library holds no state,
 * never allocates, frees or synchronises, and launches asynchronously on the stream it is given (current device of the
 * calling thread).  Return value of every int-returning entry point: 0, a negative gdn_status, or a positive hipError_t.
 * Zero a struct before filling it.
 */
#ifndef GDN_LINEAR_HIP_H
#define GDN_LINEAR_HIP_H

#include "gdn_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GDN_LINEAR_ABI_VERSION 1

int gdn_linear_abi_version(void);

/*
 * Linear attention, per (sequence, value head), with w = e^{g[h]} and the state S [K, V] in fp32:
 *     S_t = w S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t
 * (the reference's linear attention, sequence_mixer_blocks/linear_attention/op.py:10-44, with a constant decay per head).
 *
 *   q, k   [B, T, qk_heads, K]   element strides, last dim contiguous; value head h reads head h / (H / qk_heads)
 *   v, o   [B, T, H, V]          element strides, last dim contiguous
 *   g      [H] fp32, the log-decay of one token (<= 0), or NULL: no decay
 *   h0     [N, H, K, V] fp32 contiguous or NULL (zero);   ht   the same or NULL (not written); ht == h0 is allowed for
 *          gdn_linear_attn_recurrent_fwd only
 *   cu_seqlens, GDN_FLAG_LEFT_PADDED   as in gdn_args: packed sequences (B == 1) or a left-padded batch (N == B)
 *   flags  GDN_FLAG_LEFT_PADDED, GDN_FLAG_ZERO_PADDING: zeros are written at tokens that belong to no sequence (the
 *          padding, tokens behind the last packed sequence); without it nothing is written there
 *
 * K a multiple of 8 up to 256, V a multiple of 8.  dtype: of q, k, v, o.  Rows, and with them strides, 16-byte aligned;
 * tokens 0 to 2^24 elements apart.
 */
typedef struct gdn_linear_attn_args {
    const void *q;
    const void *k;
    const void *v;
    const float *g;
    const float *h0;
    float *ht;
    void *o;
    const int32_t *cu_seqlens;
    void *workspace;
    uint64_t workspace_bytes;

    int64_t q_stride_b, q_stride_t, q_stride_h;
    int64_t k_stride_b, k_stride_t, k_stride_h;
    int64_t v_stride_b, v_stride_t, v_stride_h;
    int64_t o_stride_b, o_stride_t, o_stride_h;

    int32_t B, T, H, K, V, N;
    int32_t qk_heads; /* 0 = H */
    int32_t dtype;    /* gdn_dtype */
    int32_t flags;
    float scale;
} gdn_linear_attn_args;

/*
 * Whole sequences: prompts, evaluation, training.  bf16: chunks of 64 tokens on the matrix units, the state in fp32; fp32: token
 * by token in fp32.  Long sequences are cut into segments when there are too few (sequence, head) pairs to fill the GPU: every
 * segment's own contribution to the state first, their sums, then all segments at once.
 */
int gdn_linear_attn_chunk_fwd(const gdn_linear_attn_args *args, void *stream);

/* Bytes of args->workspace for gdn_linear_attn_chunk_fwd (may be 0); reads shape fields, dtype, flags, whether cu_seqlens is NULL,
 * and the current device. */
uint64_t gdn_linear_attn_workspace_bytes(const gdn_linear_attn_args *args);

/* A few tokens per sequence, the state streamed through registers once: decoding.  ht == h0 updates the state in place. */
int gdn_linear_attn_recurrent_fwd(const gdn_linear_attn_args *args, void *stream);

/*
 * Gradients of gdn_linear_attn_chunk_fwd (and of the recurrent form, which is the same function): from the forward's inputs, dout
 * and dht (NULL: zero) it writes
 *   dq, dk [B, T, qk_heads, K]  (the gradients of value heads that share one of q and k are added up in fp32; where heads
 *                              are shared, tokens of no sequence get zeros with or without GDN_FLAG_ZERO_PADDING)
 *   dv     [B, T, H, V]
 *   dh0    [N, H, K, V] fp32 or NULL
 *   dg     [H] fp32 or NULL: the derivative with respect to g[h], over all sequences
 * in the inputs' dtype, with element strides.  fwd.o, fwd.ht and fwd.workspace are not used; every result that is not NULL is
 * written whole (tokens of no sequence: GDN_FLAG_ZERO_PADDING).
 */
typedef struct gdn_linear_attn_bwd_args {
    gdn_linear_attn_args fwd;
    const void *dout;
    const float *dht;
    void *dq;
    void *dk;
    void *dv;
    float *dh0;
    float *dg;
    void *workspace;
    uint64_t workspace_bytes;

    int64_t dout_stride_b, dout_stride_t, dout_stride_h;
    int64_t dq_stride_b, dq_stride_t, dq_stride_h;
    int64_t dk_stride_b, dk_stride_t, dk_stride_h;
    int64_t dv_stride_b, dv_stride_t, dv_stride_h;
} gdn_linear_attn_bwd_args;

int gdn_linear_attn_bwd(const gdn_linear_attn_bwd_args *args, void *stream);

/* Bytes of args->workspace; reads of args what gdn_linear_attn_workspace_bytes reads, and whether dg is NULL. */
uint64_t gdn_linear_attn_bwd_workspace_bytes(const gdn_linear_attn_bwd_args *args);

/*
 * Layer norm over rows of D elements:  y = (x - mean) / sqrt(var + eps) * weight + bias, var over D (not D - 1).
 * x, y: rows with one stride each, last dim contiguous; dtype bf16 or fp32.  weight, bias [D] or NULL, both of w_dtype; a bias
 * comes with a weight or alone.  1 <= D <= GDN_LAYER_NORM_MAX_D; any alignment that the element type has.
 */
#define GDN_LAYER_NORM_MAX_D 16384

typedef struct gdn_layer_norm_args {
    const void *x;
    const void *weight;
    const void *bias;
    void *y;
    int64_t x_stride, y_stride; /* elements between rows */
    int64_t rows;
    int32_t D;
    int32_t dtype;
    int32_t w_dtype;
    float eps;
} gdn_layer_norm_args;

int gdn_layer_norm_fwd(const gdn_layer_norm_args *args, void *stream);

/*
 * dx (dtype of x) and the sums over rows for dweight and dbias, as partial_blocks partial rows [partial_blocks, D] fp32 each
 * (NULL: not wanted), which gdn_column_sums adds up in a fixed order.  partial_blocks: gdn_layer_norm_partial_blocks.
 */
typedef struct gdn_layer_norm_bwd_args {
    const void *x;
    const void *dy;
    const void *weight;
    void *dx;
    float *dweight_partial;
    float *dbias_partial;
    int64_t x_stride, dy_stride, dx_stride;
    int64_t rows;
    int32_t D;
    int32_t dtype;
    int32_t w_dtype;
    float eps;
    int32_t partial_blocks;
    int32_t reserved;
} gdn_layer_norm_bwd_args;

int gdn_layer_norm_bwd(const gdn_layer_norm_bwd_args *args, void *stream);

/* Workgroups, and with them partial rows, that gdn_layer_norm_bwd uses for these sizes on the current device; 0 for sizes it refuses. */
int gdn_layer_norm_partial_blocks(int64_t rows, int32_t D, int32_t dtype);

#ifdef __cplusplus
}
#endif

#endif /* GDN_LINEAR_HIP_H */
