// Row-wise fusions of the MiniMax H3 DiT block around attention (gfx950).
//
// Arithmetic follows the reference Triton kernels
// (src/h3_flash/runtime/kernels/fusions.py), in fp32 with one rounding on
// store:
//   rmsnorm_modulate (:69-96)
//       n   = x * rsqrt(sum(x^2) / C + eps)
//       out = n * w * (1 + scale[t]) + shift[t]
//   residual_gate_rmsnorm_modulate (:23-67)
//       h      = residual + gate[t] * branch          -> hidden_out
//       n      = h * rsqrt(sum(h^2) / C + eps) * w    (h in fp32, unrounded)
//       normed = n * (1 + scale[t]) + shift[t]        -> normed_out
//   swiglu (:98-123)
//       out = value * (gate * sigmoid(gate)),  value = x[:, :C], gate = x[:, C:]
// with t = index[row % n_index] the modulation-table row of a token.
//
// Layout and roofline: each row kernel keeps its row in VGPRs (one 256-thread
// workgroup per row, 16 bytes per lane per vector), so x (and residual,
// branch) are read from HBM once and the outputs written once; weight and the
// small modulation tables are re-read by every row and served from L2. All
// kernels are HBM-bound. Indices outside the table are clamped to it (the
// reference reads out of bounds there).
#include "kernels.h"
#include "modulate.h"
#include "row_util.h"

namespace h3a {
namespace {

constexpr int kSwigluThreads = 128;  // measured 4.5% faster than 256 for swiglu

// Element path (any C, any alignment): two passes over the row, the second
// re-reading x (or the unrounded residual + gate * branch) from cache.
template <bool kResidual>
__global__ __launch_bounds__(kThreads) void modulate_elem_kernel(ModulateParams p) {
    __shared__ float red[kWaves];
    const int64_t row = blockIdx.x;
    const int C = p.cols;
    const int64_t t = table_row(p, row);
    auto value = [&](int c) {
        if constexpr (kResidual) {
            const float r = bf16_to_f32(((const uint16_t*)p.residual)[row * p.residual_stride + c]);
            const float b = bf16_to_f32(((const uint16_t*)p.x)[row * p.x_stride + c]);
            return r + load1(p.gate, t * p.gate_stride + c, p.table_f32) * b;
        } else {
            return bf16_to_f32(((const uint16_t*)p.x)[row * p.x_stride + c]);
        }
    };
    float ss = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
        const float h = value(c);
        ss += h * h;
        if constexpr (kResidual) {
            const uint32_t bits = pack_bf16x2(h, 0.f);
            ((uint16_t*)p.hidden)[row * p.hidden_stride + c] = (uint16_t)(bits & 0xffffu);
        }
    }
    const float r = rsqrtf(block_sum(ss, red) / (float)C + p.eps);
    for (int c = threadIdx.x; c < C; c += kThreads) {
        const float o = value(c) * r * load1(p.weight, c, p.w_f32) * (1.0f + load1(p.scale, t * p.scale_stride + c, p.table_f32)) +
                        load1(p.shift, t * p.shift_stride + c, p.table_f32);
        const uint32_t bits = pack_bf16x2(o, 0.f);
        ((uint16_t*)p.out)[row * p.out_stride + c] = (uint16_t)(bits & 0xffffu);
    }
}

__device__ __forceinline__ float silu_mul(float v, float g) { return v * (g * (1.0f / (1.0f + __expf(-g)))); }

// out[r, c] = x[r, c] * silu(x[r, C + c]); vector o covers 8 columns.
__global__ __launch_bounds__(kSwigluThreads) void swiglu_kernel(SwigluParams p) {
    const int64_t per_row = p.cols / 8;
    const int64_t total = p.rows * per_row;
    for (int64_t o = blockIdx.x * (int64_t)kSwigluThreads + threadIdx.x; o < total; o += (int64_t)gridDim.x * kSwigluThreads) {
        const int64_t row = o / per_row;
        const int64_t c = (o - row * per_row) * 8;
        const uint16_t* x = (const uint16_t*)p.x + row * p.x_stride + c;
        float v[8], g[8], out[8];
        unpack8(__builtin_nontemporal_load((const i32x4*)x), v);
        unpack8(__builtin_nontemporal_load((const i32x4*)(x + p.cols)), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = silu_mul(v[e], g[e]);
        __builtin_nontemporal_store(pack8(out), (i32x4*)((uint16_t*)p.out + row * p.out_stride + c));
    }
}

__global__ __launch_bounds__(kSwigluThreads) void swiglu_elem_kernel(SwigluParams p) {
    const int64_t total = p.rows * p.cols;
    for (int64_t o = blockIdx.x * (int64_t)kSwigluThreads + threadIdx.x; o < total; o += (int64_t)gridDim.x * kSwigluThreads) {
        const int64_t row = o / p.cols;
        const int64_t c = o - row * p.cols;
        const uint16_t* x = (const uint16_t*)p.x + row * p.x_stride;
        const uint32_t bits = pack_bf16x2(silu_mul(bf16_to_f32(x[c]), bf16_to_f32(x[p.cols + c])), 0.f);
        ((uint16_t*)p.out)[row * p.out_stride + c] = (uint16_t)(bits & 0xffffu);
    }
}

unsigned stride_grid(int64_t work) {
    const int64_t blocks = (work + kSwigluThreads - 1) / kSwigluThreads;
    return (unsigned)(blocks < 65536 ? (blocks > 0 ? blocks : 1) : 65536);
}

template <bool kResidual>
hipError_t launch_modulate_t(const ModulateParams& p, bool vec, hipStream_t stream) {
    const int nv = (int)((p.cols + 8 * kThreads - 1) / (8 * kThreads));
    if (!vec || nv < 1 || nv > 8) {
        hipLaunchKernelGGL((modulate_elem_kernel<kResidual>), dim3((unsigned)p.rows), dim3(kThreads), 0, stream, p);
    } else if (p.table_f32) {
        if (p.w_f32)
            launch_modulate_vec<kResidual, true, true, false>(p, nv, stream);
        else
            launch_modulate_vec<kResidual, true, false, false>(p, nv, stream);
    } else {
        if (p.w_f32)
            launch_modulate_vec<kResidual, false, true, false>(p, nv, stream);
        else
            launch_modulate_vec<kResidual, false, false, false>(p, nv, stream);
    }
    return hipGetLastError();
}

}  // namespace

int modulate_max_vector_cols() { return 8 * 8 * kThreads; }

hipError_t launch_modulate(const ModulateParams& p, bool vec, hipStream_t stream) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    return p.residual != nullptr ? launch_modulate_t<true>(p, vec, stream) : launch_modulate_t<false>(p, vec, stream);
}

hipError_t launch_swiglu(const SwigluParams& p, bool vec, hipStream_t stream) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    if (vec)
        hipLaunchKernelGGL(swiglu_kernel, dim3(stride_grid(p.rows * (p.cols / 8))), dim3(kSwigluThreads), 0, stream, p);
    else
        hipLaunchKernelGGL(swiglu_elem_kernel, dim3(stride_grid(p.rows * p.cols)), dim3(kSwigluThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace h3a
