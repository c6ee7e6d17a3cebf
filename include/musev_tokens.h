/*
 * musev_tokens.h -- C ABI of the token-transformer operators of libmusev_hip.so (gfx950): packed attention, rotary positions with
 * several axes, the gated residual norm and the int8 projection.  Conventions of musev_hip.h: extern "C", plain device pointers and
 * explicit strides, no hidden allocation, no global mutable state except the thread-local last-error string, every launch on the
 * hipStream_t passed as `stream` of the CURRENT device, 0 = ok / negative = MV_ERR_* with mv_last_error().  A call whose launch would have 2^32 work
 * items or more is refused (2^24 blocks of 256: rows of the norm from 2^24, of 2048 columns, to 2^28, of up to 128).
 * Matrices are rows x columns with unit inner stride; row strides (ld*) are in elements.  Element type: MV_F16 or MV_BF16.
 */
#ifndef MUSEV_TOKENS_H
#define MUSEV_TOKENS_H

#include "musev_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MV_TOKENS_ABI_VERSION 1
int mv_tokens_abi_version(void);

#define MV_F16 0
#define MV_BF16 1

/* ---- packed attention -------------------------------------------------------------------------------------------------------
 * Sequences of different lengths packed row after row; query head h reads key / value head h / (heads / kv_heads).
 *   out[i] = sum_j softmax_j(scale * q_i . k_j) v_j   over the keys j < kv_len of i's sequence, with `causal` only
 *   j <= i + kv_len - q_len (the last query sees every key);  a row that sees no key is 0.
 * A (sequence, key / value head) has q_len * group packed rows: row r is query r / group, head r % group of the group.
 * `items` (device, 8 int32 each), made by musev_amd.token_ops.attention_plan, 128 packed rows each:
 *   {first query row, q_len, first key row, kv_len, first packed row, key begin, key end, first workspace row or -1}
 * An item with a workspace row writes its unnormalised sums and the rows' references (in scores) and sums of weights there; `joins` (device, 8 int32 each:
 *   {first query row, q_len, kv_len, first packed row, first workspace row, parts, rows per part, 0}) says which parts make up which rows.
 * Rows must be 16-byte aligned.                                                                                                        */
typedef struct mv_attn_packed_desc {
    const void *q, *k, *v;
    void* out;
    const int32_t *items, *joins;
    void* workspace;               /* with joins: mv_attention_packed_workspace_bytes(ws_rows, kv_heads, d) bytes, 16-byte aligned */
    int64_t workspace_bytes, ws_rows;
    int32_t n_items, n_joins, join_rows;   /* join_rows: the most rows of a join */
    int32_t ldq, ldk, ldv, ldo;
    int32_t heads, kv_heads, d, dtype, causal;
    float scale;
} mv_attn_packed_desc;
int64_t mv_attention_packed_workspace_bytes(int64_t ws_rows, int32_t kv_heads, int32_t d);
int mv_attention_packed(const mv_attn_packed_desc* d, void* stream);

/* ---- rotary positions with several axes ----------------------------------------------------------------------------------------
 * Pair p of a head (p < pairs) turns by position[token, axis[p]] * turns[p] full turns:
 *   (a, b) -> (a cos - b sin, a sin + b cos);  elements 2 p, 2 p + 1 (halves = 0) or p, p + pairs (halves = 1) of the head;
 * elements from 2 * pairs on pass through.  k may be null.  Outputs may be the inputs themselves.                                 */
typedef struct mv_rotary_desc {
    const void *q, *k;
    void *out_q, *out_k;
    const void* positions;         /* [tokens, axes] int32 or fp32 (positions_f32), row stride ldp */
    const double* turns;           /* [pairs] turns per position step */
    const int32_t* axis;           /* [pairs] */
    int64_t tokens;
    int32_t ldq, ldk, ldoq, ldok, ldp;
    int32_t heads, kv_heads, d, pairs, axes, halves, positions_f32, dtype;
} mv_rotary_desc;
int mv_rotary_axes(const mv_rotary_desc* d, void* stream);

/* ---- gated residual norm ---------------------------------------------------------------------------------------------------------
 *   y = post ? N(f) * post_gamma + post_beta : f          N: rms (x / sqrt(mean x^2 + eps)) or layer ((x - mean) / sqrt(var + eps))
 *   s = alpha * x + gate[g] * y                            g: group_index[row], or row / rows_per_group; gate null: 1
 *   h = (N(s) * pre_gamma + pre_beta) * (1 + scale[g]) + shift[g]   (only with norm_out)
 * stream_out = s, norm_out = h; every statistic and s itself in fp32 (rows whose squares sum within its range: values up to about 1e16 in size),
 * each output rounded once.  A row whose group_index lies outside
 * [0, groups) is filled with NaN.  stream_out may be x or f, norm_out may be f or x.                                                  */
typedef struct mv_gated_norm_desc {
    const void *x, *f;
    void *stream_out, *norm_out;
    const void *post_gamma, *post_beta, *pre_gamma, *pre_beta, *gate, *scale, *shift;
    const int32_t* group_index;
    int64_t rows, groups, rows_per_group;
    int32_t c, ldx, ldf, lds, ldh, ldg, ldsc, ldsh;
    int32_t post, layer, dtype;
    float alpha, post_eps, pre_eps;
} mv_gated_norm_desc;
int mv_gated_residual_norm(const mv_gated_norm_desc* d, void* stream);

/* ---- int8 projection -----------------------------------------------------------------------------------------------------------------
 * mv_quantize_rows_i8: scale[m] = max_k |x[m, k]| / 127, code = round-to-nearest-even(127 x / max|x|); columns K .. ldc - 1 of the codes
 * become 0; a row of zeros has scale 0; a row that holds an infinity or NaN has that scale and codes 0 (its products are NaN).
 * mv_gemm_i8: out = act(a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k] + bias[n]) + residual[m, n];  the sum is exact (int32: K <= 131071),
 * what follows is fp32 from left to right (sum * a_scale first).
 * lda, ldw: multiples of 128, the columns from K on are 0.                                                                             */
int mv_quantize_rows_i8(const void* x, int64_t ldx, int64_t rows, int32_t k, int32_t dtype, int8_t* codes, int64_t ldc, float* scale,
                        void* stream);
typedef struct mv_gemm_i8_desc {
    const int8_t *a, *w;
    const float *a_scale, *w_scale;
    const void *bias, *residual;
    void* out;
    int64_t M;
    int32_t N, kp;                 /* kp: K rounded up to 128 */
    int64_t lda, ldw, ldr, ldo;
    int32_t act, dtype;
} mv_gemm_i8_desc;
int mv_gemm_i8(const mv_gemm_i8_desc* d, void* stream);
/* both in one call: x [M, K] of the element type; workspace: M * kp bytes of codes and M fp32 scales, 16-byte aligned;
 * not used (null) where M <= 4 and M * kp <= 16384, or M <= 16 and M * kp <= 8192: one launch quantises and multiplies */
typedef struct mv_linear_i8_desc {
    const void* x;
    const int8_t* w;
    const float* w_scale;
    const void *bias, *residual;
    void *out, *workspace;
    int64_t M;
    int32_t N, K;
    int64_t kp, ldx, ldw, ldr, ldo;
    int32_t act, dtype;
} mv_linear_i8_desc;
int mv_linear_i8(const mv_linear_i8_desc* d, void* stream);

#ifdef __cplusplus
}
#endif
#endif
