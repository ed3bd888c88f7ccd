// extern "C" entry points declared in include/h3block.h: argument validation and
// launch, as capi.hip does for h3attn.h.
#include <math.h>

#include "capi_linear.h"
#include "h3block.h"

namespace {

// A (batch, seq, head, 128) bf16 view of `rows` rows a head.
int check_view(const char* fn, const char* name, const void* ptr, const int64_t* st, int64_t window) {
    if (!ptr || !aligned16(ptr)) return fail(H3A_EINVAL, "%s: %s must be a 16-byte aligned device pointer", fn, name);
    for (int d = 0; d < 3; ++d)
        if (st[d] < 0 || st[d] % 8 != 0)
            return fail(H3A_EINVAL, "%s: %s strides must be non-negative multiples of 8 elements", fn, name);
    if (st[1] < 128) return fail(H3A_EINVAL, "%s: %s sequence stride %lld < head_dim", fn, name, (long long)st[1]);
    if (st[1] >= (kMaxSpan + window * 2 - 1) / (window * 2))
        return fail(H3A_EUNSUPPORTED, "%s: %s row stride %lld elements is too large (%lld rows must span < 2^31 bytes)", fn, name,
                    (long long)st[1], (long long)window);
    return H3A_OK;
}

int check_attn_extents(const char* fn, int64_t batch, int64_t heads, int64_t sq, int64_t sk, int64_t head_dim) {
    if (head_dim != 128) return fail(H3A_EUNSUPPORTED, "%s: head_dim must be 128, got %lld", fn, (long long)head_dim);
    if (batch < 0 || heads <= 0 || sq < 0 || sk < 0)
        return fail(H3A_EINVAL, "%s: negative or zero extent (batch=%lld heads=%lld sq=%lld sk=%lld)", fn, (long long)batch,
                    (long long)heads, (long long)sq, (long long)sk);
    if (batch > INT32_MAX || heads > INT32_MAX) return fail(H3A_EUNSUPPORTED, "%s: batch and heads must be below 2^31", fn);
    if (sq > INT32_MAX / 2 || sk > INT32_MAX / 2) return fail(H3A_EINVAL, "%s: sequence length too large", fn);
    return H3A_OK;
}

constexpr int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// Fills the launch description but for the workspace; *need: its bytes.
int prepare_select(const h3a_block_select_args* a, h3a::SelectParams& p, int64_t* need) {
    const char* fn = "h3a_block_select";
    *need = 0;
    if (a == nullptr) return fail(H3A_EINVAL, "%s: args is NULL", fn);
    if (a->abi_version != H3A_ABI_VERSION)
        return fail(H3A_EINVAL, "%s: abi_version %d, library is %d", fn, a->abi_version, H3A_ABI_VERSION);
    int rc = check_attn_extents(fn, a->batch, a->heads, a->seqlen_q, a->seqlen_k, a->head_dim);
    if (rc != H3A_OK) return rc;
    const int64_t nq = (a->seqlen_q + H3A_BLOCK_Q - 1) / H3A_BLOCK_Q, nk = (a->seqlen_k + H3A_BLOCK_K - 1) / H3A_BLOCK_K;
    if (a->batch == 0 || nq == 0 || nk == 0) return H3A_OK;  // nothing to choose
    if (a->topk < 1 || a->topk > nk)
        return fail(H3A_EINVAL, "%s: topk must be in [1, %lld], got %lld", fn, (long long)nk, (long long)a->topk);
    if (nk > h3a::select_max_blocks())
        return fail(H3A_EUNSUPPORTED, "%s: at most %d key blocks, got %lld", fn, h3a::select_max_blocks(), (long long)nk);
    // (Work items of the three launches: 256 per block, 256 per 16 x 128 scores of
    // a head, at most 1,024 per query block.)
    if ((__int128)a->batch * a->heads > 65535 || (__int128)a->batch * a->heads * (nq + nk) >= ((int64_t)1 << 22) ||
        ((nq + 15) / 16) * ((nk + 127) / 128) >= ((int64_t)1 << 24))
        return fail(H3A_EUNSUPPORTED, "%s: batch x heads must be at most 65535, and with the blocks below 2^22", fn);
    if ((rc = check_view(fn, "q", a->q, a->q_stride, 1)) != H3A_OK) return rc;
    if ((rc = check_view(fn, "k", a->k, a->k_stride, 1)) != H3A_OK) return rc;
    if (!a->index || !aligned4(a->index)) return fail(H3A_EINVAL, "%s: index must be a 4-byte aligned device pointer", fn);
    p.q = a->q; p.k = a->k;
    p.q_sb = a->q_stride[0]; p.q_rs = a->q_stride[1] * 2; p.q_sh = a->q_stride[2];
    p.k_sb = a->k_stride[0]; p.k_rs = a->k_stride[1] * 2; p.k_sh = a->k_stride[2];
    p.always = (const uint8_t*)a->always;
    p.index = a->index;
    p.batch = (int32_t)a->batch; p.heads = (int32_t)a->heads;
    p.seqlen_q = (int32_t)a->seqlen_q; p.seqlen_k = (int32_t)a->seqlen_k;
    p.nq = (int32_t)nq; p.nk = (int32_t)nk; p.topk = (int32_t)a->topk;
    const int64_t bh = a->batch * a->heads;
    *need = round256(bh * nq * 512) + round256(bh * nk * 512) + round256(bh * nq * nk * 4);
    return H3A_OK;
}

// Fills the launch description; *need: the workspace that its pieces would take.
int prepare_sparse(const h3a_attn_sparse_args* a, h3a::SparseParams& p, int64_t* need, bool* empty) {
    const char* fn = "h3a_attn_sparse";
    *need = 0;
    *empty = false;
    if (a == nullptr) return fail(H3A_EINVAL, "%s: args is NULL", fn);
    if (a->abi_version != H3A_ABI_VERSION)
        return fail(H3A_EINVAL, "%s: abi_version %d, library is %d", fn, a->abi_version, H3A_ABI_VERSION);
    int rc = check_attn_extents(fn, a->batch, a->heads, a->seqlen_q, a->seqlen_k, a->head_dim);
    if (rc != H3A_OK) return rc;
    if (!(a->softmax_scale > 0.f) || !isfinite(a->softmax_scale)) return fail(H3A_EINVAL, "%s: softmax_scale must be finite and > 0", fn);
    if (a->max_blocks < 0 || a->max_blocks > H3A_SPARSE_MAX_BLOCKS)
        return fail(a->max_blocks < 0 ? H3A_EINVAL : H3A_EUNSUPPORTED, "%s: a list holds at most %d blocks, got %lld", fn,
                    H3A_SPARSE_MAX_BLOCKS, (long long)a->max_blocks);
    if (a->batch == 0 || a->seqlen_q == 0) {
        *empty = true;
        return H3A_OK;
    }
    const int64_t window = h3a::attn_fwd_window_rows();
    if ((rc = check_view(fn, "q", a->q, a->q_stride, window)) != H3A_OK) return rc;
    if ((rc = check_view(fn, "o", a->o, a->o_stride, window)) != H3A_OK) return rc;
    // (Without keys K and V are not read.)
    if (a->seqlen_k > 0 && a->max_blocks > 0) {
        if ((rc = check_view(fn, "k", a->k, a->k_stride, window)) != H3A_OK) return rc;
        if ((rc = check_view(fn, "v", a->v, a->v_stride, window)) != H3A_OK) return rc;
        if (!a->block_index || !aligned4(a->block_index)) return fail(H3A_EINVAL, "%s: block_index must be a 4-byte aligned device pointer", fn);
        for (int d = 0; d < 3; ++d)
            if (a->index_stride[d] < 0) return fail(H3A_EINVAL, "%s: index strides must be non-negative", fn);
    }
    if (a->block_count != nullptr) {
        if (!aligned4(a->block_count)) return fail(H3A_EINVAL, "%s: block_count must be 4-byte aligned", fn);
        for (int d = 0; d < 3; ++d)
            if (a->count_stride[d] < 0) return fail(H3A_EINVAL, "%s: count strides must be non-negative", fn);
    }
    if (a->lse != nullptr && (!aligned4(a->lse) || a->lse_stride[0] < 0 || a->lse_stride[1] < 0))
        return fail(H3A_EINVAL, "%s: lse must be 4-byte aligned with non-negative strides", fn);
    const int64_t nq = (a->seqlen_q + H3A_BLOCK_Q - 1) / H3A_BLOCK_Q;
    const __int128 tiles = (__int128)a->batch * a->heads * nq;
    // (512 work items for each of a tile's 8 units: 2^32 a launch.)
    if (tiles >= ((int64_t)1 << 20)) return fail(H3A_EUNSUPPORTED, "%s: grid too large", fn);
    p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.lse = a->lse;
    p.q_sb = a->q_stride[0]; p.q_sh = a->q_stride[2]; p.q_rs = (int32_t)(a->q_stride[1] * 2);
    p.k_sb = a->k_stride[0]; p.k_sh = a->k_stride[2]; p.k_rs = (int32_t)(a->k_stride[1] * 2);
    p.v_sb = a->v_stride[0]; p.v_sh = a->v_stride[2]; p.v_rs = (int32_t)(a->v_stride[1] * 2);
    p.o_sb = a->o_stride[0]; p.o_sh = a->o_stride[2]; p.o_rs = (int32_t)(a->o_stride[1] * 2);
    p.lse_sb = a->lse_stride[0]; p.lse_sh = a->lse_stride[1];
    p.heads = (int32_t)a->heads;
    p.seqlen_q = (int32_t)a->seqlen_q; p.seqlen_k = (int32_t)a->seqlen_k;
    p.n_qtiles = (int32_t)nq; p.n_groups = (int32_t)a->batch;
    p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
    p.list = a->block_index; p.count = a->block_count;
    p.list_sb = a->index_stride[0]; p.list_sh = a->index_stride[1]; p.list_sq = a->index_stride[2];
    p.count_sb = a->count_stride[0]; p.count_sh = a->count_stride[1]; p.count_sq = a->count_stride[2];
    p.max_blocks = a->seqlen_k > 0 ? (int32_t)a->max_blocks : 0;
    p.pieces = 1;
    p.split_tiles = (int32_t)tiles;
    h3a::plan_attn_sparse(p, h3a::device_cus());
    if (p.pieces > 1) *need = (int64_t)p.pieces * (int64_t)tiles * h3a::attn_fwd_piece_bytes(true);
    return H3A_OK;
}

// Fills the launch description; *need: the workspace of its pieces, *empty:
// nothing to launch.
int prepare_linear(const h3a_linear_args* a, h3a::LinearParams& p, int64_t* need, bool* empty) {
    *need = 0;
    *empty = false;
    const char* fn = "h3a_linear";
    if (a == nullptr) return fail(H3A_EINVAL, "%s: args is NULL", fn);
    if (a->abi_version != H3A_ABI_VERSION)
        return fail(H3A_EINVAL, "%s: abi_version %d, library is %d", fn, a->abi_version, H3A_ABI_VERSION);
    if (a->m < 0 || a->k <= 0 || a->n <= 0)
        return fail(H3A_EINVAL, "%s: bad extents (m=%lld k=%lld n=%lld)", fn, (long long)a->m, (long long)a->k, (long long)a->n);
    if (a->k % 8 != 0 || a->n % 8 != 0)
        return fail(H3A_EUNSUPPORTED, "%s: k and n must be multiples of 8, got %lld and %lld", fn, (long long)a->k, (long long)a->n);
    if (a->activation < H3A_ACT_NONE || a->activation > H3A_ACT_RELU) return fail(H3A_EINVAL, "%s: unknown activation %d", fn, a->activation);
    if (a->m >= ((int64_t)1 << 31) - 256 || a->n >= ((int64_t)1 << 30) || a->k >= ((int64_t)1 << 30))
        return fail(H3A_EUNSUPPORTED, "%s: extents too large", fn);
    if (a->m == 0) {
        *empty = true;
        return H3A_OK;
    }
    const void* ptrs[3] = {a->x, a->weight, a->y};
    for (const void* q : ptrs)
        if (!q || !aligned16(q)) return fail(H3A_EINVAL, "%s: x, weight and y must be 16-byte aligned device pointers", fn);
    if (a->x_stride < a->k || a->weight_stride < a->k || a->y_stride < a->n || a->x_stride % 8 || a->weight_stride % 8 || a->y_stride % 8)
        return fail(H3A_EINVAL, "%s: strides must be multiples of 8 elements covering the row", fn);
    const int64_t rows = h3a::linear_max_tile();
    if (a->x_stride > (kMaxSpan - 1) / (2 * rows) || a->weight_stride > (kMaxSpan - 1) / (2 * rows))
        return fail(H3A_EUNSUPPORTED, "%s: %lld rows of x and of weight must span less than 2^31 bytes", fn, (long long)rows);
    const int rc = check_epilogue(fn, *a, p);
    if (rc != H3A_OK) return rc;
    p.x = a->x; p.w = a->weight; p.y = a->y;
    p.x_rs = a->x_stride * 2; p.w_rs = a->weight_stride * 2; p.y_rs = a->y_stride * 2;
    p.m = (int32_t)a->m; p.k = (int32_t)a->k; p.n = (int32_t)a->n;
    p.act = a->activation; p.gated = a->gated != 0;
    h3a::plan_linear(p, h3a::device_cus(), need);
    if (p.shape < -1) return fail(H3A_EUNSUPPORTED, "%s: grid too large", fn);
    return H3A_OK;
}

}  // namespace

extern "C" {

int64_t h3a_linear_workspace_size(const h3a_linear_args* a) {
    h3a::clear_error();
    h3a::LinearParams p{};
    int64_t need = 0;
    bool empty = false;
    const int rc = prepare_linear(a, p, &need, &empty);
    return rc != H3A_OK ? rc : need;
}

int h3a_linear(const h3a_linear_args* a, void* stream) {
    h3a::clear_error();
    const char* fn = "h3a_linear";
    h3a::LinearParams p{};
    int64_t need = 0;
    bool empty = false;
    const int rc = prepare_linear(a, p, &need, &empty);
    if (rc != H3A_OK || empty) return rc;
    // y apart from what other workgroups still read (it may be the residual, whose
    // elements are read by the lanes that store them).
    const RowSpan y{p.y, p.m, 2 * (int64_t)p.n, p.y_rs};
    if (overlap(y, RowSpan{p.x, p.m, 2 * (int64_t)p.k, p.x_rs}) ||
        overlap(y, RowSpan{p.w, (p.gated ? 2 : 1) * (int64_t)p.n, 2 * (int64_t)p.k, p.w_rs}) || overlaps_epilogue(y, p, true))
        return fail(H3A_EINVAL, "%s: y overlaps an operand (it may be the residual itself)", fn);
    if (need > 0) {
        if (a->workspace == nullptr && a->workspace_bytes == H3A_WORKSPACE_ASK) return H3A_NEED_WORKSPACE;
        if (a->workspace != nullptr && ((uintptr_t)a->workspace & 255u) == 0 && a->workspace_bytes >= need) {
            p.ws = a->workspace;
        } else {
            p.n_full = p.m_tiles * p.n_tiles;  // every tile whole
            p.split = 1;
        }
    }
    const hipError_t e = h3a::launch_linear(p, h3a::device_cus(), (hipStream_t)stream);
    if (e != hipSuccess) return fail(H3A_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return H3A_OK;
}

int h3a_rmsnorm_residual_gate_rmsnorm_modulate(const h3a_rmsnorm_residual_gate_rmsnorm_modulate_args* a, void* stream) {
    h3a::clear_error();
    const char* fn = "h3a_rmsnorm_residual_gate_rmsnorm_modulate";
    if (a == nullptr) return fail(H3A_EINVAL, "%s: args is NULL", fn);
    if (a->abi_version != H3A_ABI_VERSION)
        return fail(H3A_EINVAL, "%s: abi_version %d, library is %d", fn, a->abi_version, H3A_ABI_VERSION);
    if (a->rows < 0 || a->cols <= 0) return fail(H3A_EINVAL, "%s: bad extents (rows=%lld cols=%lld)", fn, (long long)a->rows, (long long)a->cols);
    // (A workgroup of 256 per row: 2^32 work items a launch.)
    if (a->rows >= ((int64_t)1 << 24) || a->cols >= ((int64_t)1 << 30)) return fail(H3A_EUNSUPPORTED, "%s: extents too large", fn);
    if (!(a->eps >= 0.f) || !isfinite(a->eps)) return fail(H3A_EINVAL, "%s: eps must be finite and not negative", fn);
    if (!isfinite(a->residual_scale)) return fail(H3A_EINVAL, "%s: residual_scale must be finite", fn);
    if (!bf16_or_f32(a->w_dtype)) return fail(H3A_EINVAL, "%s: unknown weight dtype %d", fn, a->w_dtype);
    if (!bf16_or_f32(a->table_dtype)) return fail(H3A_EINVAL, "%s: unknown table dtype %d", fn, a->table_dtype);
    if (a->rows == 0) return H3A_OK;
    const bool norm = a->normed_out != nullptr, tables = norm || a->gate != nullptr;
    h3a::SandwichParams p{};
    bool vec = a->cols % 8 == 0 && aligned16(a->branch_weight) && (!norm || aligned16(a->weight));
    struct Rows {
        const char* name;
        const void* ptr;
        int64_t stride;
    };
    const Rows rows[4] = {{"residual", a->residual, a->residual_stride}, {"branch", a->branch, a->branch_stride},
                          {"hidden_out", a->hidden_out, a->hidden_stride}, {"normed_out", a->normed_out, a->normed_stride}};
    for (int i = 0; i < (norm ? 4 : 3); ++i) {
        if (!rows[i].ptr) return fail(H3A_EINVAL, "%s: NULL %s pointer", fn, rows[i].name);
        if (((uintptr_t)rows[i].ptr & 1u) != 0) return fail(H3A_EINVAL, "%s: %s must be 2-byte aligned", fn, rows[i].name);
        if (rows[i].stride < a->cols) return fail(H3A_EINVAL, "%s: %s row stride %lld < cols", fn, rows[i].name, (long long)rows[i].stride);
        vec = vec && aligned16(rows[i].ptr) && rows[i].stride % 8 == 0;
    }
    const unsigned wa = a->w_dtype == H3A_DTYPE_F32 ? 3u : 1u;
    if (!a->branch_weight || ((uintptr_t)a->branch_weight & wa) || (norm && (!a->weight || ((uintptr_t)a->weight & wa))))
        return fail(H3A_EINVAL, "%s: weights must be device pointers aligned to their type", fn);
    const int64_t size = a->table_dtype == H3A_DTYPE_F32 ? 4 : 2;
    const Rows tabs[3] = {{"gate", a->gate, a->gate_stride}, {"scale", a->scale, a->scale_stride}, {"shift", a->shift, a->shift_stride}};
    for (int i = a->gate != nullptr ? 0 : 1; i < (norm ? 3 : 1); ++i) {
        if (!tabs[i].ptr || ((uintptr_t)tabs[i].ptr & (uintptr_t)(size - 1)) != 0)
            return fail(H3A_EINVAL, "%s: %s must be a device pointer aligned to its type", fn, tabs[i].name);
        if (tabs[i].stride < a->cols) return fail(H3A_EINVAL, "%s: %s row stride %lld < cols", fn, tabs[i].name, (long long)tabs[i].stride);
        vec = vec && aligned16(tabs[i].ptr) && tabs[i].stride * size % 16 == 0;
    }
    if (tables) {
        const int rc = check_index(fn, a->index, a->index_dtype, a->n_index, a->table_rows);
        if (rc != H3A_OK) return rc;
        p.index = a->index;
        p.index_i64 = a->index_dtype == H3A_DTYPE_I64;
        p.n_index = a->n_index;
        p.table_rows = a->table_rows;
    }
    p.branch = a->branch; p.residual = a->residual; p.hidden = a->hidden_out; p.out = a->normed_out;
    p.branch_weight = a->branch_weight; p.weight = a->weight;
    p.gate = a->gate; p.scale = a->scale; p.shift = a->shift;
    p.branch_stride = a->branch_stride; p.residual_stride = a->residual_stride;
    p.hidden_stride = a->hidden_stride; p.out_stride = a->normed_stride;
    p.gate_stride = a->gate_stride; p.scale_stride = a->scale_stride; p.shift_stride = a->shift_stride;
    p.rows = a->rows; p.cols = (int32_t)a->cols;
    p.w_f32 = a->w_dtype == H3A_DTYPE_F32; p.table_f32 = size == 4;
    p.residual_scale = a->residual_scale; p.eps = a->eps;
    const hipError_t e = h3a::launch_sandwich(p, vec, (hipStream_t)stream);
    if (e != hipSuccess) return fail(H3A_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return H3A_OK;
}

int64_t h3a_block_select_workspace_size(const h3a_block_select_args* a) {
    h3a::clear_error();
    h3a::SelectParams p{};
    int64_t need = 0;
    const int rc = prepare_select(a, p, &need);
    return rc != H3A_OK ? rc : need;
}

int h3a_block_select(const h3a_block_select_args* a, void* stream) {
    h3a::clear_error();
    const char* fn = "h3a_block_select";
    h3a::SelectParams p{};
    int64_t need = 0;
    const int rc = prepare_select(a, p, &need);
    if (rc != H3A_OK || need == 0) return rc;
    if (!a->workspace || ((uintptr_t)a->workspace & 255u) != 0 || a->workspace_bytes < need)
        return fail(H3A_EINVAL, "%s: the workspace must hold %lld bytes, 256-byte aligned", fn, (long long)need);
    const int64_t bh = a->batch * a->heads;
    p.qm = (float*)a->workspace;
    p.km = (float*)((char*)p.qm + round256(bh * p.nq * 512));
    p.score = (float*)((char*)p.km + round256(bh * p.nk * 512));
    const hipError_t e = h3a::launch_block_select(p, (hipStream_t)stream);
    if (e != hipSuccess) return fail(H3A_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return H3A_OK;
}

int64_t h3a_attn_sparse_workspace_size(const h3a_attn_sparse_args* a) {
    h3a::clear_error();
    h3a::SparseParams p{};
    int64_t need = 0;
    bool empty = false;
    const int rc = prepare_sparse(a, p, &need, &empty);
    return rc != H3A_OK ? rc : need;
}

int h3a_attn_sparse(const h3a_attn_sparse_args* a, void* stream) {
    h3a::clear_error();
    const char* fn = "h3a_attn_sparse";
    h3a::SparseParams p{};
    int64_t need = 0;
    bool empty = false;
    const int rc = prepare_sparse(a, p, &need, &empty);
    if (rc != H3A_OK || empty) return rc;
    if (need > 0) {
        if (a->workspace == nullptr && a->workspace_bytes == H3A_WORKSPACE_ASK) return H3A_NEED_WORKSPACE;
        if (a->workspace != nullptr && ((uintptr_t)a->workspace & 255u) == 0 && a->workspace_bytes >= need) {
            p.ws_o = a->workspace;
            p.ws_lse = (float*)((char*)a->workspace + (int64_t)p.pieces * p.split_tiles * H3A_BLOCK_Q * 512);
        } else {
            p.pieces = 1;  // every list whole
        }
    }
    const hipError_t e = h3a::launch_attn_sparse(p, (hipStream_t)stream);
    if (e != hipSuccess) return fail(H3A_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return H3A_OK;
}

}  // extern "C"
