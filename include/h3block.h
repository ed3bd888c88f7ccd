/*
 * C ABI of the operators around an H3 DiT block's attention and MLP that go
 * beyond the reference's kernels: key-block selection and attention over the
 * selected blocks, the matrix product with a fused epilogue, and the norms
 * before and after a branch. Conventions (argument structs, element strides,
 * device pointers, streams, return codes, h3a_last_error) are those of
 * h3attn.h; nothing is allocated, nothing waits for the device, and every
 * buffer is the caller's. Inference only, as the rest of the library.
 */
#ifndef H3BLOCK_H
#define H3BLOCK_H

#include "h3attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Matrix product with its epilogue. For every row r of x and feature f < n:
 *   z[f] = sum_k x[r, k] * weight[f, k] (+ bias[f])
 *   a    = act(z[f]),  or gated: z[f] * act(z[n + f])  (weight and bias then
 *          have 2 n rows: the values, then their gates)
 *   y[r, f] = residual[r, f] + gate[t, f] * a,  t = index[r % n_index]
 * accumulated and finished in fp32 and rounded to bf16 once; without residual
 * or gate those terms are left out. t is clamped to [0, table_rows).
 * x, weight, residual and y are bf16 with rows of unit column stride; bias and
 * gate bf16 or fp32; index int32 or int64. k and n are positive multiples of 8;
 * rows are 16-byte aligned (strides multiples of 8 elements; fp32 gate rows of
 * 4); 256 rows of x and of weight span less than 2^31 bytes; a launch of 2^32
 * work items or more is refused (for at most 32 rows of x: of some 2^30 rows of
 * weight). y may be the residual, and must not overlap any other operand.
 * A launch whose last round of tiles would leave CUs idle cuts those tiles into
 * pieces along k, whose sums (fp32) take a workspace of
 * h3a_linear_workspace_size bytes, 256-byte aligned; without one every tile runs
 * whole. workspace NULL with workspace_bytes H3A_WORKSPACE_ASK: the call
 * launches, or returns H3A_NEED_WORKSPACE without launching where it takes one.
 */
#define H3A_ACT_NONE 0
#define H3A_ACT_SILU 1
#define H3A_ACT_GELU 2      /* z * Phi(z) */
#define H3A_ACT_GELU_TANH 3 /* z * (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2 */
#define H3A_ACT_RELU 4

typedef struct h3a_linear_args {
    int32_t abi_version;
    const void *x;
    const void *weight;
    const void *bias;     /* or NULL */
    int32_t bias_dtype;   /* H3A_DTYPE_BF16 or H3A_DTYPE_F32 */
    const void *residual; /* or NULL */
    const void *gate;     /* or NULL */
    int32_t gate_dtype;
    int64_t gate_stride;
    int64_t table_rows;
    const void *index;    /* with gate */
    int32_t index_dtype;  /* H3A_DTYPE_I32 or H3A_DTYPE_I64 */
    int64_t n_index;
    void *y;
    int64_t m;
    int64_t k;
    int64_t n;
    int64_t x_stride;
    int64_t weight_stride;
    int64_t residual_stride;
    int64_t y_stride;
    int32_t activation;
    int32_t gated;
    void *workspace;
    int64_t workspace_bytes;
} h3a_linear_args;

H3A_API int64_t h3a_linear_workspace_size(const h3a_linear_args *args);
H3A_API int h3a_linear(const h3a_linear_args *args, void *stream);

/*
 * The norms before and after a branch. Per row r with t = index[r % n_index]:
 *   n             = branch[r] * rsqrt(sum(branch[r]^2) / cols + eps) * branch_weight
 *   h             = residual_scale * residual[r] + gate[t] * n      (fp32)
 *   hidden_out[r] = h                                               (bf16)
 *   normed_out[r] = h * rsqrt(sum(h^2) / cols + eps) * weight
 *                   * (1 + scale[t]) + shift[t]                     (bf16)
 * The second norm uses the unrounded h. gate may be NULL (1); normed_out may be
 * NULL (weight, scale and shift are then not read); index may be NULL only when
 * no table is read. Layouts and dtypes as for h3a_rmsnorm_modulate; the two
 * weights share w_dtype, the tables table_dtype. hidden_out may be the residual.
 */
typedef struct h3a_rmsnorm_residual_gate_rmsnorm_modulate_args {
    int32_t abi_version;
    const void *residual;
    const void *branch;
    void *hidden_out;
    void *normed_out;
    const void *branch_weight;
    const void *weight;
    int32_t w_dtype;
    const void *gate;
    const void *scale;
    const void *shift;
    int32_t table_dtype;
    int64_t gate_stride;
    int64_t scale_stride;
    int64_t shift_stride;
    int64_t table_rows;
    const void *index;
    int32_t index_dtype;
    int64_t n_index;
    int64_t rows;
    int64_t cols;
    int64_t residual_stride;
    int64_t branch_stride;
    int64_t hidden_stride;
    int64_t normed_stride;
    float residual_scale;
    float eps;
} h3a_rmsnorm_residual_gate_rmsnorm_modulate_args;

H3A_API int h3a_rmsnorm_residual_gate_rmsnorm_modulate(const h3a_rmsnorm_residual_gate_rmsnorm_modulate_args *args,
                                                       void *stream);

/*
 * Key blocks of each query block by a cheap score. Query blocks are
 * H3A_BLOCK_Q rows, key blocks H3A_BLOCK_K (the last of either may be shorter);
 * nq and nk are their numbers.
 *   qm[i], km[j] = fp32(mean of the rows of query block i, key block j)
 *   s[i, j]      = fp32(<qm[i], km[j]>)       sums in 64 bits
 * index[b, h, i, :] receives the topk blocks of the largest s[i, :], in
 * ascending order: blocks with a non-zero byte in `always` come before all
 * others (among themselves by their index alone), NaN counts as -inf, equal
 * scores are taken from the lowest index on.
 * q and k are bf16 (batch, seq, head) views as for h3a_attn_fwd; always is
 * (nk,) bytes or NULL; index is contiguous int32 (batch, heads, nq, topk) with
 * 1 <= topk <= nk (none is written when nq or nk is 0). nk is at most 32,768,
 * batch x heads at most 65,535 and batch x heads x (nq + nk) below 2^22.
 * The workspace holds the means and scores: h3a_block_select_workspace_size
 * bytes, 256-byte aligned, free again once the call's work has run.
 */
#define H3A_BLOCK_Q 256
#define H3A_BLOCK_K 64

typedef struct h3a_block_select_args {
    int32_t abi_version;
    const void *q;
    const void *k;
    const void *always;
    int32_t *index;
    int64_t batch;
    int64_t heads;
    int64_t seqlen_q;
    int64_t seqlen_k;
    int64_t head_dim;
    int64_t q_stride[3]; /* batch, seq, head */
    int64_t k_stride[3];
    int64_t topk;
    void *workspace;
    int64_t workspace_bytes;
} h3a_block_select_args;

H3A_API int64_t h3a_block_select_workspace_size(const h3a_block_select_args *args);
H3A_API int h3a_block_select(const h3a_block_select_args *args, void *stream);

/*
 * Attention over lists of key blocks: query block i of (b, h) attends to the
 * keys of the blocks block_index[b, h, i, 0 .. c), c = block_count[b, h, i]
 * clamped to [0, max_blocks] (block_count NULL: max_blocks).
 *   O = softmax(scale * Q K_L^T) V_L,  LSE = log(sum(exp(scale * Q K_L^T)))
 * Entries may come in any order; one named twice counts twice, one outside
 * [0, nk) names nothing, and a row without keys gives O = 0 and LSE = -inf.
 * Scores, sums and LSE are fp32; the weights are rounded to bf16 for the product
 * with V, as in h3a_attn_fwd, and the result once more.
 * q, k, v, o and lse as for h3a_attn_fwd (dense, head_dim 128), o and lse apart
 * from every input; block_index is int32 with unit stride between a row's entries
 * and index_stride (batch, head, query block) between rows; count_stride likewise.
 * max_blocks is at most H3A_SPARSE_MAX_BLOCKS, and batch x heads x query blocks
 * below 2^20. A launch of few query blocks cuts the lists into pieces, whose
 * partial results (fp32) take a workspace of h3a_attn_sparse_workspace_size
 * bytes, 256-byte aligned; without one the lists run whole. workspace NULL with
 * workspace_bytes H3A_WORKSPACE_ASK: the call launches, or returns
 * H3A_NEED_WORKSPACE without launching where it takes one.
 */
#define H3A_SPARSE_MAX_BLOCKS 7168

typedef struct h3a_attn_sparse_args {
    int32_t abi_version;
    const void *q;
    const void *k;
    const void *v;
    void *o;
    float *lse; /* may be NULL */
    int64_t batch;
    int64_t heads;
    int64_t seqlen_q;
    int64_t seqlen_k;
    int64_t head_dim;
    int64_t q_stride[3]; /* batch, seq, head */
    int64_t k_stride[3];
    int64_t v_stride[3];
    int64_t o_stride[3];
    int64_t lse_stride[2]; /* batch, head */
    float softmax_scale;
    const int32_t *block_index;
    int64_t index_stride[3];
    const int32_t *block_count;
    int64_t count_stride[3];
    int64_t max_blocks;
    void *workspace;
    int64_t workspace_bytes;
} h3a_attn_sparse_args;

H3A_API int64_t h3a_attn_sparse_workspace_size(const h3a_attn_sparse_args *args);
H3A_API int h3a_attn_sparse(const h3a_attn_sparse_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* H3BLOCK_H */
