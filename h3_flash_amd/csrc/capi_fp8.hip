// extern "C" entry points declared in include/h3fp8.h but the norms' (capi.hip):
// argument validation and launch, as capi_block.hip does for h3block.h.
#include "capi_linear.h"
#include "h3fp8.h"

namespace {

constexpr int64_t kGroup = 128;  // values that share a scale

int64_t groups_of(int64_t n) { return (n + kGroup - 1) / kGroup; }

// e4m3 rows and their scales.
int check_fp8(const char* fn, const char* name, const void* q, int64_t q_stride, const void* scale, int64_t scale_stride, int64_t cols) {
    if (!q || !aligned16(q) || q_stride < cols || q_stride % 16)
        return fail(H3A_EINVAL, "%s: %s must have 16-byte aligned rows of at least %lld bytes", fn, name, (long long)cols);
    if (!scale || !aligned16(scale) || scale_stride < groups_of(cols) || scale_stride % 16)
        return fail(H3A_EINVAL, "%s: %s's rows of scales must start at multiples of 16 bytes and hold %lld", fn, name,
                    (long long)groups_of(cols));
    return H3A_OK;
}

// Fills the launch description; *required and *need: the workspace that the call
// cannot do without, and with the sums of tiles in pieces; *empty: nothing to launch.
int prepare_linear_fp8(const h3a_linear_fp8_args* a, h3a::LinearFp8Params& p, int64_t* required, int64_t* need, bool* empty) {
    *required = *need = 0;
    *empty = false;
    const char* fn = "h3a_linear_fp8";
    if (a == nullptr) return fail(H3A_EINVAL, "%s: args is NULL", fn);
    if (a->abi_version != H3A_ABI_VERSION)
        return fail(H3A_EINVAL, "%s: abi_version %d, library is %d", fn, a->abi_version, H3A_ABI_VERSION);
    if (a->m < 0 || a->k <= 0 || a->n <= 0)
        return fail(H3A_EINVAL, "%s: bad extents (m=%lld k=%lld n=%lld)", fn, (long long)a->m, (long long)a->k, (long long)a->n);
    const bool x8 = a->x_dtype == H3A_DTYPE_F8E4M3, y8 = a->y_dtype == H3A_DTYPE_F8E4M3;
    if (!x8 && a->x_dtype != H3A_DTYPE_BF16) return fail(H3A_EINVAL, "%s: unknown x dtype %d", fn, a->x_dtype);
    if (!y8 && a->y_dtype != H3A_DTYPE_BF16) return fail(H3A_EINVAL, "%s: unknown y dtype %d", fn, a->y_dtype);
    if (a->k % 16 != 0 || a->n % (y8 ? 16 : 8) != 0)
        return fail(H3A_EUNSUPPORTED, "%s: k must be a multiple of 16 and n of %d, got %lld and %lld", fn, y8 ? 16 : 8, (long long)a->k,
                    (long long)a->n);
    if (a->activation < H3A_ACT_NONE || a->activation > H3A_ACT_RELU) return fail(H3A_EINVAL, "%s: unknown activation %d", fn, a->activation);
    if (a->m >= ((int64_t)1 << 31) - 256 || a->n >= ((int64_t)1 << 30) || a->k >= ((int64_t)1 << 30))
        return fail(H3A_EUNSUPPORTED, "%s: extents too large", fn);
    if (a->m == 0) {
        *empty = true;
        return H3A_OK;
    }
    int rc;
    if (x8) {
        if ((rc = check_fp8(fn, "x", a->x, a->x_stride, a->x_scale, a->x_scale_stride, a->k)) != H3A_OK) return rc;
    } else if (!a->x || !aligned16(a->x) || a->x_stride < a->k || a->x_stride % 8) {
        return fail(H3A_EINVAL, "%s: x must have 16-byte aligned rows of at least k elements", fn);
    }
    if ((rc = check_fp8(fn, "weight", a->weight, a->weight_stride, a->weight_scale, a->weight_scale_stride, a->k)) != H3A_OK) return rc;
    if (y8) {
        if ((rc = check_fp8(fn, "y", a->y, a->y_stride, a->y_scale, a->y_scale_stride, a->n)) != H3A_OK) return rc;
    } else if (!a->y || !aligned16(a->y) || a->y_stride < a->n || a->y_stride % 8) {
        return fail(H3A_EINVAL, "%s: y must have 16-byte aligned rows of at least n elements", fn);
    }
    const int64_t rows = h3a::linear_max_tile(), x_size = x8 ? 1 : 2;
    if (a->weight_scale_stride >= kMaxSpan / (2 * groups_of(a->n)))
        return fail(H3A_EUNSUPPORTED, "%s: the scales of weight must span less than 2^31 bytes", fn);
    if (a->x_stride > (kMaxSpan - 1) / (x_size * rows) || a->weight_stride > (kMaxSpan - 1) / rows ||
        a->y_stride > (kMaxSpan - 1) / ((y8 ? 1 : 2) * rows) || (a->residual != nullptr && a->residual_stride > (kMaxSpan - 1) / (2 * rows)) ||
        (x8 && a->x_scale_stride > (kMaxSpan - 1) / rows) || (y8 && a->y_scale_stride > (kMaxSpan - 1) / rows))
        return fail(H3A_EUNSUPPORTED, "%s: %lld rows of an operand must span less than 2^31 bytes", fn, (long long)rows);
    if ((rc = check_epilogue(fn, *a, p)) != H3A_OK) return rc;
    if (p.table_rows >= (int64_t)1 << 31) return fail(H3A_EUNSUPPORTED, "%s: the gate's table must have fewer than 2^31 rows", fn);
    p.x = a->x; p.w = a->weight; p.y = a->y;
    p.x_rs = a->x_stride * x_size; p.w_rs = a->weight_stride; p.y_rs = a->y_stride * (y8 ? 1 : 2);
    p.x_scale = x8 ? (const uint8_t*)a->x_scale : nullptr;
    p.w_scale = (const uint8_t*)a->weight_scale;
    p.x_scale_rs = a->x_scale_stride; p.w_scale_rs = a->weight_scale_stride;
    p.w_blocks = (int32_t)groups_of(a->n);
    p.y_scale = y8 ? (uint8_t*)a->y_scale : nullptr;
    p.y_scale_rs = a->y_scale_stride;
    p.m = (int32_t)a->m; p.k = (int32_t)a->k; p.n = (int32_t)a->n;
    p.act = a->activation; p.gated = a->gated != 0;
    h3a::plan_linear_fp8(p, h3a::device_cus(), required, need);
    if (p.shape < -1) return fail(H3A_EUNSUPPORTED, "%s: grid too large", fn);
    return H3A_OK;
}

}  // namespace

extern "C" {

int h3a_quantize_fp8(const h3a_quantize_fp8_args* a, void* stream) {
    h3a::clear_error();
    const char* fn = "h3a_quantize_fp8";
    if (a == nullptr) return fail(H3A_EINVAL, "%s: args is NULL", fn);
    if (a->abi_version != H3A_ABI_VERSION)
        return fail(H3A_EINVAL, "%s: abi_version %d, library is %d", fn, a->abi_version, H3A_ABI_VERSION);
    if (!bf16_or_f32(a->x_dtype)) return fail(H3A_EINVAL, "%s: unknown x dtype %d", fn, a->x_dtype);
    if (a->rows < 0 || a->cols <= 0) return fail(H3A_EINVAL, "%s: bad extents (rows=%lld cols=%lld)", fn, (long long)a->rows, (long long)a->cols);
    if (a->cols % 16 != 0) return fail(H3A_EUNSUPPORTED, "%s: cols must be a multiple of 16, got %lld", fn, (long long)a->cols);
    const bool blocks = a->block_rows == kGroup;
    if (!blocks && a->block_rows != 1) return fail(H3A_EINVAL, "%s: block_rows must be 1 or 128, got %lld", fn, (long long)a->block_rows);
    if (a->parts < 1 || a->rows % a->parts != 0 || (!blocks && a->parts != 1))
        return fail(H3A_EINVAL, "%s: rows must be `parts` matrices (1 with block_rows 1), got %lld and %lld", fn, (long long)a->rows,
                    (long long)a->parts);
    const int64_t scale_rows = blocks ? a->parts * groups_of(a->rows / a->parts) : a->rows;
    if (a->rows >= ((int64_t)1 << 31) || a->cols >= ((int64_t)1 << 30) || scale_rows * groups_of(a->cols) > h3a::quantize_max_groups(blocks))
        return fail(H3A_EUNSUPPORTED, "%s: extents too large", fn);
    if (a->rows == 0) return H3A_OK;
    const int64_t size = a->x_dtype == H3A_DTYPE_F32 ? 4 : 2;
    if (!a->x || !aligned16(a->x) || a->x_stride < a->cols || a->x_stride * size % 16)
        return fail(H3A_EINVAL, "%s: x must have 16-byte aligned rows of at least cols elements", fn);
    const int rc = check_fp8(fn, "q", a->q, a->q_stride, a->scale, a->scale_stride, a->cols);
    if (rc != H3A_OK) return rc;
    h3a::QuantizeParams p{};
    p.x = a->x; p.q = a->q; p.scale = (uint8_t*)a->scale;
    p.x_rs = a->x_stride * size; p.q_rs = a->q_stride; p.scale_rs = a->scale_stride;
    p.rows = a->rows; p.part_rows = a->rows / a->parts;
    p.cols = (int32_t)a->cols; p.x_f32 = size == 4; p.blocks = blocks;
    const RowSpan x{p.x, p.rows, size * a->cols, p.x_rs}, q{p.q, p.rows, a->cols, p.q_rs},
        s{p.scale, scale_rows, groups_of(a->cols), p.scale_rs};
    if (overlap(q, x) || overlap(s, x) || overlap(s, q)) return fail(H3A_EINVAL, "%s: x, q and scale overlap", fn);
    const hipError_t e = h3a::launch_quantize(p, (hipStream_t)stream);
    if (e != hipSuccess) return fail(H3A_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return H3A_OK;
}

int64_t h3a_linear_fp8_workspace_size(const h3a_linear_fp8_args* a) {
    h3a::clear_error();
    h3a::LinearFp8Params p{};
    int64_t required = 0, need = 0;
    bool empty = false;
    const int rc = prepare_linear_fp8(a, p, &required, &need, &empty);
    return rc != H3A_OK ? rc : need;
}

int64_t h3a_linear_fp8_required_workspace(const h3a_linear_fp8_args* a) {
    h3a::clear_error();
    h3a::LinearFp8Params p{};
    int64_t required = 0, need = 0;
    bool empty = false;
    const int rc = prepare_linear_fp8(a, p, &required, &need, &empty);
    return rc != H3A_OK ? rc : required;
}

int h3a_linear_fp8(const h3a_linear_fp8_args* a, void* stream) {
    h3a::clear_error();
    const char* fn = "h3a_linear_fp8";
    h3a::LinearFp8Params p{};
    int64_t required = 0, need = 0;
    bool empty = false;
    const int rc = prepare_linear_fp8(a, p, &required, &need, &empty);
    if (rc != H3A_OK || empty) return rc;
    // y and its scales apart from what other workgroups still read (a bf16 y may be
    // the residual, whose elements are read by the lanes that store them).
    const int64_t w_blocks = (p.gated ? 2 : 1) * (int64_t)p.w_blocks, kb = groups_of(p.k), y_size = p.y_scale != nullptr ? 1 : 2;
    const RowSpan operands[4] = {{p.x, p.m, (p.x_scale != nullptr ? 1 : 2) * (int64_t)p.k, p.x_rs},
                                 {p.w, (p.gated ? 2 : 1) * (int64_t)p.n, p.k, p.w_rs},
                                 {p.w_scale, w_blocks, kb, p.w_scale_rs},
                                 {p.x_scale, p.m, kb, p.x_scale_rs}};
    const RowSpan y{p.y, p.m, y_size * p.n, p.y_rs}, ys{p.y_scale, p.m, groups_of(p.n), p.y_scale_rs};
    bool shared = overlaps_epilogue(y, p, p.y_scale == nullptr);
    for (int i = 0; i < (p.x_scale != nullptr ? 4 : 3); ++i)
        shared = shared || overlap(y, operands[i]) || (p.y_scale != nullptr && overlap(ys, operands[i]));
    if (p.y_scale != nullptr) shared = shared || overlap(y, ys) || overlaps_epilogue(ys, p, false);
    if (shared) return fail(H3A_EINVAL, "%s: y overlaps an operand (in bf16 it may be the residual itself)", fn);
    if (need > 0) {
        if (a->workspace == nullptr && a->workspace_bytes == H3A_WORKSPACE_ASK) return H3A_NEED_WORKSPACE;
        const bool given = a->workspace != nullptr && ((uintptr_t)a->workspace & 255u) == 0;
        if (required > 0 && (!given || a->workspace_bytes < required))
            return fail(H3A_EINVAL, "%s: the workspace must hold %lld bytes, 256-byte aligned", fn, (long long)required);
        if (given && a->workspace_bytes >= required) p.ws = a->workspace;
        if (!given || a->workspace_bytes < need) {
            p.n_full = p.m_tiles * p.n_tiles;  // every tile whole
            p.split = 1;
        }
    }
    const hipError_t e = h3a::launch_linear_fp8(p, h3a::device_cus(), (hipStream_t)stream);
    if (e != hipSuccess) return fail(H3A_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return H3A_OK;
}

}  // extern "C"
