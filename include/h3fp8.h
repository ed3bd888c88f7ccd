/*
 * C ABI of the 8-bit linear layers of an H3 DiT block: rounding rows and weights to
 * 8 bits, the norms before a branch with their result in 8 bits, and the matrix
 * product of 8-bit operands with its epilogue. Conventions (argument structs, device
 * pointers, streams, return codes, h3a_last_error) are those of h3attn.h; nothing is
 * allocated, nothing waits for the device, and every buffer is the caller's.
 * Inference only, as the rest of the library.
 *
 * A matrix in 8 bits is e4m3 (the variant without infinities), one byte a value, and
 * its scales are e8m0: a byte e stands for 2^(e - 127), 255 for NaN. Rows of
 * activations have a scale for every 128 columns, weights one for every block of 128
 * rows x 128 columns (the last ones shorter):
 *   s = the smallest power of two, 2^-126 at the least, with max |x| <= 448 s
 *   q = e4m3(x / s), to nearest, ties to even
 * A group that holds a value that is not finite is NaN throughout, scale and values.
 * Columns are positive multiples of 16, rows of values 16-byte aligned. Rows of scales
 * start at multiples of 16 bytes; rows x stride bytes of them are readable, and what
 * lies behind a row's scales is neither used nor written. Outputs overlap nothing
 * unless an entry point says so.
 */
#ifndef H3FP8_H
#define H3FP8_H

#include "h3block.h"

#ifdef __cplusplus
extern "C" {
#endif

#define H3A_DTYPE_F8E4M3 4

/*
 * Rounds x (rows, cols; bf16 or fp32) to 8 bits. block_rows 1: a scale for every row
 * and 128 columns, scale has `rows` rows. block_rows 128: one for every block; the
 * rows are `parts` matrices of rows / parts each, whose blocks start anew (a gated
 * weight's values, then its gates), and scale has parts * ceil(rows / parts / 128)
 * rows. A row of scale holds ceil(cols / 128). Strides in elements (x) and bytes.
 */
typedef struct h3a_quantize_fp8_args {
    int32_t abi_version;
    const void *x;
    int32_t x_dtype; /* H3A_DTYPE_BF16 or H3A_DTYPE_F32 */
    void *q;
    void *scale;
    int64_t rows;
    int64_t cols;
    int64_t block_rows;
    int64_t parts;
    int64_t x_stride;
    int64_t q_stride;
    int64_t scale_stride;
} h3a_quantize_fp8_args;

H3A_API int h3a_quantize_fp8(const h3a_quantize_fp8_args *args, void *stream);

/*
 * h3a_rmsnorm_modulate with its result in 8 bits: the fp32 row is rounded in groups of
 * 128 columns. Rows, weight and table rows are 16-byte aligned; cols at most
 * H3A_NORM_FP8_MAX_COLS.
 */
#define H3A_NORM_FP8_MAX_COLS 16384

typedef struct h3a_rmsnorm_modulate_fp8_args {
    int32_t abi_version;
    const void *x;
    void *q_out;
    void *scale_out;
    const void *weight;
    int32_t w_dtype;
    const void *scale;
    const void *shift;
    int32_t table_dtype;
    int64_t scale_stride;
    int64_t shift_stride;
    int64_t table_rows;
    const void *index;
    int32_t index_dtype;
    int64_t n_index;
    int64_t rows;
    int64_t cols;
    int64_t x_stride;
    int64_t q_stride;         /* bytes */
    int64_t scale_out_stride; /* bytes */
    float eps;
} h3a_rmsnorm_modulate_fp8_args;

H3A_API int h3a_rmsnorm_modulate_fp8(const h3a_rmsnorm_modulate_fp8_args *args, void *stream);

/*
 * h3a_residual_gate_rmsnorm_modulate with its normed rows in 8 bits; hidden_out is
 * bf16 and may be the residual or the branch.
 */
typedef struct h3a_residual_gate_rmsnorm_modulate_fp8_args {
    int32_t abi_version;
    const void *residual;
    const void *branch;
    void *hidden_out;
    void *q_out;
    void *scale_out;
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
    int64_t q_stride;         /* bytes */
    int64_t scale_out_stride; /* bytes */
    float eps;
} h3a_residual_gate_rmsnorm_modulate_fp8_args;

H3A_API int h3a_residual_gate_rmsnorm_modulate_fp8(const h3a_residual_gate_rmsnorm_modulate_fp8_args *args, void *stream);

/*
 * h3a_linear with 8-bit operands:
 *   z[f] = sum_k x[r, k] x_scale[r, k / 128] * weight[f, k] weight_scale[f / 128, k / 128]
 *          (+ bias[f])
 * and y from z as there. x is in 8 bits with its scales, or bf16 (x_dtype) and rounded
 * to 8 bits first, as h3a_quantize_fp8 does with block_rows 1; y is bf16, or in 8 bits
 * with its scales (y_dtype), rounded from the fp32 result. weight_scale is
 * h3a_quantize_fp8's with block_rows 128 and, gated, parts 2: of the values' blocks,
 * then of their gates'. Products of 8-bit values are summed by the matrix cores: eight
 * neighbouring k are lined up to the largest of their products, with 13 bits kept below
 * it, and those sums are accumulated in fp32.
 * k is a positive multiple of 16, n of 8 (of 16 with y in 8 bits); rows are 16-byte
 * aligned; 256 rows of an operand or result, and all scales of weight, span less than
 * 2^31 bytes. y may be the residual (bf16) and overlaps no other operand.
 * Workspace: h3a_linear_fp8_workspace_size bytes, 256-byte aligned.
 * h3a_linear_fp8_required_workspace of them (x's or y's other form) it cannot do
 * without; with less than the whole, tiles are not cut along k. workspace NULL with
 * workspace_bytes H3A_WORKSPACE_ASK: the call launches, or returns H3A_NEED_WORKSPACE
 * without launching where it takes one.
 */
typedef struct h3a_linear_fp8_args {
    int32_t abi_version;
    const void *x;
    int32_t x_dtype;          /* H3A_DTYPE_BF16 or H3A_DTYPE_F8E4M3 */
    const void *x_scale;      /* with H3A_DTYPE_F8E4M3 */
    const void *weight;
    const void *weight_scale;
    const void *bias;         /* or NULL */
    int32_t bias_dtype;       /* H3A_DTYPE_BF16 or H3A_DTYPE_F32 */
    const void *residual;     /* or NULL */
    const void *gate;         /* or NULL */
    int32_t gate_dtype;
    int64_t gate_stride;
    int64_t table_rows;
    const void *index;        /* with gate */
    int32_t index_dtype;      /* H3A_DTYPE_I32 or H3A_DTYPE_I64 */
    int64_t n_index;
    void *y;
    int32_t y_dtype;          /* H3A_DTYPE_BF16 or H3A_DTYPE_F8E4M3 */
    void *y_scale;            /* with H3A_DTYPE_F8E4M3 */
    int64_t m;
    int64_t k;
    int64_t n;
    int64_t x_stride;         /* elements */
    int64_t x_scale_stride;   /* bytes */
    int64_t weight_stride;
    int64_t weight_scale_stride;
    int64_t residual_stride;
    int64_t y_stride;
    int64_t y_scale_stride;
    int32_t activation;
    int32_t gated;
    void *workspace;
    int64_t workspace_bytes;
} h3a_linear_fp8_args;

H3A_API int64_t h3a_linear_fp8_workspace_size(const h3a_linear_fp8_args *args);
H3A_API int64_t h3a_linear_fp8_required_workspace(const h3a_linear_fp8_args *args);
H3A_API int h3a_linear_fp8(const h3a_linear_fp8_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* H3FP8_H */
