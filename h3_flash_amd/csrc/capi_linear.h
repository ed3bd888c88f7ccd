// Argument checks that the entry points of the linear layers share.
#pragma once

#include "capi_util.h"
#include "h3block.h"
#include "kernels.h"

namespace {

using h3a::aligned16;
using h3a::aligned4;
using h3a::fail;

constexpr int64_t kMaxSpan = (int64_t)1 << 31;  // buffer offsets are 32-bit

inline bool bf16_or_f32(int32_t dtype) { return dtype == H3A_DTYPE_BF16 || dtype == H3A_DTYPE_F32; }

// The index that picks a modulation-table row per token.
inline int check_index(const char* fn, const void* index, int32_t dtype, int64_t n_index, int64_t table_rows) {
    if (!index || n_index <= 0 || table_rows <= 0) return fail(H3A_EINVAL, "%s: a table needs rows and an index of at least one entry", fn);
    if (dtype != H3A_DTYPE_I32 && dtype != H3A_DTYPE_I64) return fail(H3A_EINVAL, "%s: unknown index dtype %d", fn, dtype);
    if (((uintptr_t)index & (dtype == H3A_DTYPE_I64 ? 7u : 3u)) != 0) return fail(H3A_EINVAL, "%s: index is not aligned to its type", fn);
    return H3A_OK;
}

// Rows of memory: `rows` of `bytes` each, `pitch` apart.
struct RowSpan {
    const void* ptr;
    int64_t rows, bytes, pitch;
};

// Whether two sets of rows share a byte. At one pitch (a single row has any) they
// may lie side by side, as columns of one buffer; at two, rows in a common range
// count as shared.
inline bool overlap(const RowSpan& a, const RowSpan& b) {
    const int64_t d = (int64_t)((uintptr_t)b.ptr - (uintptr_t)a.ptr);
    if (d >= (a.rows - 1) * a.pitch + a.bytes || -d >= (b.rows - 1) * b.pitch + b.bytes) return false;
    if (a.rows == 1 && b.rows == 1) return true;
    const int64_t pitch = a.rows == 1 ? b.pitch : a.pitch;
    if (b.rows > 1 && b.pitch != pitch) return true;
    const int64_t at = (d % pitch + pitch) % pitch;  // where b's rows start in a's
    return at < a.bytes || at + b.bytes > pitch;
}

// The epilogue's operands (bias, residual, gate): checks them and fills their fields
// of p. Args: an argument struct that names them as h3a_linear_args does.
template <typename Args>
int check_epilogue(const char* fn, const Args& a, h3a::LinearParams& p) {
    if (a.bias != nullptr) {
        if (!bf16_or_f32(a.bias_dtype)) return fail(H3A_EINVAL, "%s: unknown bias dtype %d", fn, a.bias_dtype);
        if (!aligned16(a.bias)) return fail(H3A_EINVAL, "%s: bias must be 16-byte aligned", fn);
        p.bias = a.bias;
        p.bias_f32 = a.bias_dtype == H3A_DTYPE_F32;
    }
    if (a.residual != nullptr) {
        if (!aligned16(a.residual)) return fail(H3A_EINVAL, "%s: residual must be 16-byte aligned", fn);
        if (a.residual_stride < a.n || a.residual_stride % 8)
            return fail(H3A_EINVAL, "%s: residual_stride must be a multiple of 8 elements covering the row", fn);
        p.residual = a.residual;
        p.res_rs = a.residual_stride * 2;
    }
    if (a.gate != nullptr) {
        if (!bf16_or_f32(a.gate_dtype)) return fail(H3A_EINVAL, "%s: unknown gate dtype %d", fn, a.gate_dtype);
        if (!aligned16(a.gate)) return fail(H3A_EINVAL, "%s: gate must be 16-byte aligned", fn);
        const int64_t size = a.gate_dtype == H3A_DTYPE_F32 ? 4 : 2;
        if (a.gate_stride < a.n || a.gate_stride * size % 16)
            return fail(H3A_EINVAL, "%s: gate rows must be 16-byte aligned and cover n", fn);
        const int rc = check_index(fn, a.index, a.index_dtype, a.n_index, a.table_rows);
        if (rc != H3A_OK) return rc;
        p.gate = a.gate;
        p.gate_f32 = size == 4;
        p.gate_rs = a.gate_stride * size;
        p.table_rows = a.table_rows;
        p.index = a.index;
        p.index_i64 = a.index_dtype == H3A_DTYPE_I64;
        p.n_index = a.n_index;
    }
    return H3A_OK;
}

// Whether y shares a byte with them; in_place: it may be the residual itself.
inline bool overlaps_epilogue(const RowSpan& y, const h3a::LinearParams& p, bool in_place) {
    const int64_t w_rows = (p.gated ? 2 : 1) * (int64_t)p.n;
    if (p.bias != nullptr && overlap(y, RowSpan{p.bias, 1, w_rows * (p.bias_f32 ? 4 : 2), 0})) return true;
    if (p.gate != nullptr && overlap(y, RowSpan{p.gate, p.table_rows, (int64_t)p.n * (p.gate_f32 ? 4 : 2), p.gate_rs})) return true;
    if (p.residual == nullptr) return false;
    const RowSpan res{p.residual, p.m, 2 * (int64_t)p.n, p.res_rs};
    if (in_place && res.ptr == y.ptr && (p.m == 1 || res.pitch == y.pitch)) return false;
    return overlap(y, res);
}

}  // namespace
