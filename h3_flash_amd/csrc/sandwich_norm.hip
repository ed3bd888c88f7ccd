// The norms before and after a branch of a DiT block (gfx950): the norm of the
// branch, its gate and the scaled residual, the norm and modulation that the
// next branch starts with, in one pass over the rows.
//
//   n      = branch * rsqrt(sum(branch^2) / C + eps) * branch_weight
//   h      = residual_scale * residual + gate[t] * n           -> hidden_out
//   normed = h * rsqrt(sum(h^2) / C + eps) * weight * (1 + scale[t]) + shift[t]
//                                                               -> normed_out
// with t = index[row % n_index] clamped to the table, in fp32 with one rounding
// on each store (the second norm takes h unrounded). Without a gate table the
// gate is 1; without normed_out the pass ends at h.
//
// HBM-bound: two rows read, two written; weights and table rows come from LDS
// and the caches. The two sums follow one another, so a row stays in registers
// from its loads to its last store.
#include "kernels.h"
#include "row_util.h"

namespace h3a {
namespace {

// W waves per row, 4 / W rows per workgroup, which share the two weight rows
// through LDS (bf16 tables). Vectors 0 .. NV-2 of a lane lie inside the row (NV =
// ceil(C / (512 W))); the last one, where it does not, is loaded from the row's
// last vector and dropped. Branch, residual and gate are all in flight before the
// first sum, scale and shift before the second.
template <int W, int NV, bool kNorm, bool kWF32>
__global__ __launch_bounds__(kThreads, 2) void sandwich_row_kernel(SandwichParams p) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = (threadIdx.x & 63) + 64 * (wave % W);  // of the row's W waves
    const int64_t row_id = (int64_t)blockIdx.x * (kWaves / W) + wave / W;  // uniform
    const bool live = row_id < p.rows;
    const int64_t row = live ? row_id : p.rows - 1;  // a wave past the rows loads the last one, stores nothing
    const int C = p.cols;
    uint32_t off[NV];  // byte offset of vector k in a bf16 row
#pragma unroll
    for (int k = 0; k < NV; ++k) off[k] = (uint32_t)(lane + 64 * W * k) * 16u;
    const bool last = (int)(off[NV - 1] / 2) < C;
    if (!last) off[NV - 1] = (uint32_t)(C - 8) * 2u;

    const char* const br = (const char*)p.branch + row * p.branch_stride * 2;
    const char* const rr = (const char*)p.residual + row * p.residual_stride * 2;
    i32x4 rx[NV], rres[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) rx[k] = __builtin_nontemporal_load((const i32x4*)(br + off[k]));
#pragma unroll
    for (int k = 0; k < NV; ++k) rres[k] = __builtin_nontemporal_load((const i32x4*)(rr + off[k]));
    // The weight rows: vector i (columns 8i .. 8i+7, the last clamped into the
    // row) of row j at wl[(j * kWv + i) * kWl].
    constexpr int kWv = NV * 64 * W, kWl = kWF32 ? 2 : 1, kWr = kNorm ? 2 : 1;
    __shared__ i32x4 wl[kWr * kWv * kWl];
#pragma unroll
    for (int j = 0; j < kWr; ++j) {
        const char* const src = (const char*)(j == 0 ? p.branch_weight : p.weight);
#pragma unroll
        for (int it = 0; it < (kWv + kThreads - 1) / kThreads; ++it) {
            const int i = min((int)threadIdx.x + it * kThreads, kWv - 1);
            const Raw8<kWF32> v = fetch8o<kWF32>(src, (uint32_t)min(i * 8, C - 8) * 2u);
            wl[(j * kWv + i) * kWl] = v.a;
            if constexpr (kWF32) wl[(j * kWv + i) * kWl + 1] = v.b;
        }
    }
    auto weight = [&](int j, int k, float* out) __attribute__((always_inline)) {
        Raw8<kWF32> w;
        w.a = wl[(j * kWv + lane + 64 * W * k) * kWl];
        if constexpr (kWF32) w.b = wl[(j * kWv + lane + 64 * W * k) * kWl + 1];
        unpack_raw8<kWF32>(w, out);
    };
    const int64_t t = p.index != nullptr ? table_row(p, row) : 0;
    i32x4 g[NV];
    if (p.gate != nullptr) {
        const char* const gr = (const char*)p.gate + t * p.gate_stride * 2;
#pragma unroll
        for (int k = 0; k < NV; ++k) g[k] = *(const i32x4*)(gr + off[k]);
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) g[k] = i32x4{0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80};
    }
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float b[8];
        unpack8(rx[k], b);
        if (k < NV - 1 || last)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += b[e] * b[e];
    }
    // Sum over the row's waves, in wave order.
    __shared__ float red[2][kWaves];
    auto row_sum = [&](float v, int i) __attribute__((always_inline)) {
        if constexpr (W == 1) return v;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += red[i][wave / W * W + w];
        return s;
    };
    ss = wave_sum(ss);
    if (W > 1 && (threadIdx.x & 63) == 0) red[0][wave] = ss;
    __syncthreads();  // the weight rows are in LDS
    const float r1 = rsqrtf(row_sum(ss, 0) / (float)C + p.eps);
    if (W == 1 && !live) return;
    i32x4 sc[kNorm ? NV : 1], sh[kNorm ? NV : 1];
    if constexpr (kNorm) {
        const char* const scr = (const char*)p.scale + t * p.scale_stride * 2;
        const char* const shr = (const char*)p.shift + t * p.shift_stride * 2;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            sc[k] = *(const i32x4*)(scr + off[k]);
            sh[k] = *(const i32x4*)(shr + off[k]);
        }
    }
    char* const hr = (char*)p.hidden + row * p.hidden_stride * 2;
    auto hidden = [&](int k, float* h) __attribute__((always_inline)) {
        float b[8], r[8], gv[8], wv[8];
        unpack8(rx[k], b);
        unpack8(rres[k], r);
        unpack8(g[k], gv);
        weight(0, k, wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = p.residual_scale * r[e] + gv[e] * (b[e] * r1 * wv[e]);
    };
    float s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float h[8];
        hidden(k, h);
        if (k < NV - 1 || last) {
            if (W == 1 || live) __builtin_nontemporal_store(pack8(h), (i32x4*)(hr + off[k]));
#pragma unroll
            for (int e = 0; e < 8; ++e) s2 += h[e] * h[e];
        }
    }
    if constexpr (kNorm) {
        // h is formed again below from the raw vectors rather than held in fp32
        // through the sum (half the registers: two waves per SIMD at NV = 11).
#pragma unroll
        for (int k = 0; k < NV; ++k) asm volatile("" : "+v"(rx[k]), "+v"(rres[k]), "+v"(g[k]));
        s2 = wave_sum(s2);
        if constexpr (W > 1) {
            if ((threadIdx.x & 63) == 0) red[1][wave] = s2;
            __syncthreads();
            if (!live) return;
        }
        const float r2 = rsqrtf(row_sum(s2, 1) / (float)C + p.eps);
        char* const orow = (char*)p.out + row * p.out_stride * 2;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float h[8], wv[8], scv[8], shv[8], o[8];
            hidden(k, h);
            weight(1, k, wv);
            unpack8(sc[k], scv);
            unpack8(sh[k], shv);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = h[e] * r2 * wv[e] * (1.0f + scv[e]) + shv[e];
            if (k < NV - 1 || last) __builtin_nontemporal_store(pack8(o), (i32x4*)(orow + off[k]));
        }
    }
}

// One row per workgroup, NV vectors of 8 per thread: few rows, wide rows, fp32
// tables.
template <int NV, bool kTabF32, bool kWF32>
__global__ __launch_bounds__(kThreads) void sandwich_block_kernel(SandwichParams p) {
    __shared__ float red[2][kWaves];
    const int64_t row = blockIdx.x;
    const int C = p.cols;
    const int64_t t = p.index != nullptr ? table_row(p, row) : 0;
    int col[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) col[k] = (threadIdx.x + k * kThreads) * 8;
    const bool last = col[NV - 1] < C;
    if (!last) col[NV - 1] = C - 8;
    const uint16_t* const br = (const uint16_t*)p.branch + row * p.branch_stride;
    const uint16_t* const rr = (const uint16_t*)p.residual + row * p.residual_stride;
    i32x4 rx[NV], rres[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) rx[k] = __builtin_nontemporal_load((const i32x4*)(br + col[k]));
#pragma unroll
    for (int k = 0; k < NV; ++k) rres[k] = __builtin_nontemporal_load((const i32x4*)(rr + col[k]));
    const bool gated = p.gate != nullptr, norm = p.out != nullptr;
    Raw8<kTabF32> g[NV];
    Raw8<kWF32> w[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        w[k] = fetch8<kWF32>(p.branch_weight, col[k]);
        if (gated) g[k] = fetch8<kTabF32>(p.gate, t * p.gate_stride + col[k]);
    }
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float b[8];
        unpack8(rx[k], b);
        if (k < NV - 1 || last)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += b[e] * b[e];
    }
    const float r1 = rsqrtf(block_sum(ss, red[0]) / (float)C + p.eps);
    uint16_t* const hr = (uint16_t*)p.hidden + row * p.hidden_stride;
    float h[NV][8];
    float s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float b[8], r[8], gv[8], wv[8];
        unpack8(rx[k], b);
        unpack8(rres[k], r);
        unpack_raw8<kTabF32>(g[k], gv);
        unpack_raw8<kWF32>(w[k], wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[k][e] = p.residual_scale * r[e] + (gated ? gv[e] : 1.0f) * (b[e] * r1 * wv[e]);
        if (k < NV - 1 || last) {
            __builtin_nontemporal_store(pack8(h[k]), (i32x4*)(hr + col[k]));
#pragma unroll
            for (int e = 0; e < 8; ++e) s2 += h[k][e] * h[k][e];
        }
    }
    if (!norm) return;
    Raw8<kTabF32> sc[NV], sh[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        w[k] = fetch8<kWF32>(p.weight, col[k]);
        sc[k] = fetch8<kTabF32>(p.scale, t * p.scale_stride + col[k]);
        sh[k] = fetch8<kTabF32>(p.shift, t * p.shift_stride + col[k]);
    }
    const float r2 = rsqrtf(block_sum(s2, red[1]) / (float)C + p.eps);
    uint16_t* const orow = (uint16_t*)p.out + row * p.out_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (k == NV - 1 && !last) break;
        float wv[8], scv[8], shv[8], o[8];
        unpack_raw8<kWF32>(w[k], wv);
        unpack_raw8<kTabF32>(sc[k], scv);
        unpack_raw8<kTabF32>(sh[k], shv);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = h[k][e] * r2 * wv[e] * (1.0f + scv[e]) + shv[e];
        __builtin_nontemporal_store(pack8(o), (i32x4*)(orow + col[k]));
    }
}

// Any width and alignment: three passes over the row, the later ones from cache.
__global__ __launch_bounds__(kThreads) void sandwich_elem_kernel(SandwichParams p) {
    __shared__ float red[2][kWaves];
    const int64_t row = blockIdx.x;
    const int C = p.cols;
    const int64_t t = p.index != nullptr ? table_row(p, row) : 0;
    const uint16_t* const br = (const uint16_t*)p.branch + row * p.branch_stride;
    const uint16_t* const rr = (const uint16_t*)p.residual + row * p.residual_stride;
    float ss = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
        const float b = bf16_to_f32(br[c]);
        ss += b * b;
    }
    const float r1 = rsqrtf(block_sum(ss, red[0]) / (float)C + p.eps);
    // (hidden_out may be the residual: a column's h is formed again from what
    // was read, before its store.)
    auto value = [&](int c, float r) {
        const float g = p.gate != nullptr ? load1(p.gate, t * p.gate_stride + c, p.table_f32) : 1.0f;
        return p.residual_scale * r + g * (bf16_to_f32(br[c]) * r1 * load1(p.branch_weight, c, p.w_f32));
    };
    float s2 = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
        const float h = value(c, bf16_to_f32(rr[c]));
        s2 += h * h;
        if (p.out == nullptr) ((uint16_t*)p.hidden)[row * p.hidden_stride + c] = (uint16_t)(pack_bf16x2(h, 0.f) & 0xffffu);
    }
    if (p.out == nullptr) return;
    const float r2 = rsqrtf(block_sum(s2, red[1]) / (float)C + p.eps);
    for (int c = threadIdx.x; c < C; c += kThreads) {
        const float h = value(c, bf16_to_f32(rr[c]));
        const float o = h * r2 * load1(p.weight, c, p.w_f32) * (1.0f + load1(p.scale, t * p.scale_stride + c, p.table_f32)) +
                        load1(p.shift, t * p.shift_stride + c, p.table_f32);
        ((uint16_t*)p.hidden)[row * p.hidden_stride + c] = (uint16_t)(pack_bf16x2(h, 0.f) & 0xffffu);
        ((uint16_t*)p.out)[row * p.out_stride + c] = (uint16_t)(pack_bf16x2(o, 0.f) & 0xffffu);
    }
}

template <int W, bool kNorm, bool kWF32>
void launch_rows(const SandwichParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)((p.rows + kWaves / W - 1) / (kWaves / W))), block(kThreads);
    const int nv = (p.cols + 512 * W - 1) / (512 * W);
#define H3A_NW(n) \
    if (nv == n) hipLaunchKernelGGL((sandwich_row_kernel<W, n, kNorm, kWF32>), grid, block, 0, stream, p);
    if constexpr (W == 1) {
        H3A_NW(1) H3A_NW(2) H3A_NW(3) H3A_NW(4) H3A_NW(8)
    }
    H3A_NW(5) H3A_NW(6) H3A_NW(7)
#undef H3A_NW
}

template <bool kTabF32, bool kWF32>
void launch_block(const SandwichParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.rows), block(kThreads);
    switch ((p.cols + 8 * kThreads - 1) / (8 * kThreads)) {
#define H3A_NV(n)                                                                                     \
    case n:                                                                                           \
        hipLaunchKernelGGL((sandwich_block_kernel<n, kTabF32, kWF32>), grid, block, 0, stream, p);   \
        break;
        H3A_NV(1) H3A_NV(2) H3A_NV(3) H3A_NV(4) H3A_NV(5) H3A_NV(6) H3A_NV(7) H3A_NV(8)
#undef H3A_NV
    }
}

}  // namespace

hipError_t launch_sandwich(const SandwichParams& p, bool vec, hipStream_t stream) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    const bool w = p.w_f32 != 0;
    // us by graph replays, a workgroup per row / one wave / two waves: 1,024 rows
    // of 1,024 4.3 / 4.4 / 4.5, 2,048 of 1,024 6.4 / 5.3 / 5.6, 49,920 of 1,024 95 /
    // 68 / 71, 2,048 of 4,096 16 / 14 / 17, 6,240 of 5,376 56 / - / 60, 12,480 of
    // 5,376 103 / - / 105, 20,000 of 5,376 164 / - / 162, 30,000 of 6,144 276 / - /
    // 259, 49,920 of 5,120 398 / 355 / 362. Past 4,096 columns a row takes a wave
    // over 256 registers, past 7,168 two.
    const int waves = !vec || p.table_f32 || p.rows <= 1024 ? 0 : p.cols <= 4096 ? 1 : p.rows > 16384 && p.cols <= 7168 ? 2 : 0;
    if (waves == 1) {
        if (p.out != nullptr)
            w ? launch_rows<1, true, true>(p, stream) : launch_rows<1, true, false>(p, stream);
        else
            w ? launch_rows<1, false, true>(p, stream) : launch_rows<1, false, false>(p, stream);
    } else if (waves == 2) {
        if (p.out != nullptr)
            w ? launch_rows<2, true, true>(p, stream) : launch_rows<2, true, false>(p, stream);
        else
            w ? launch_rows<2, false, true>(p, stream) : launch_rows<2, false, false>(p, stream);
    } else if (vec && p.cols <= 8 * 8 * kThreads) {
        if (p.table_f32)
            w ? launch_block<true, true>(p, stream) : launch_block<true, false>(p, stream);
        else
            w ? launch_block<false, true>(p, stream) : launch_block<false, false>(p, stream);
    } else {
        hipLaunchKernelGGL(sandwich_elem_kernel, dim3((unsigned)p.rows), dim3(kThreads), 0, stream, p);
    }
    return hipGetLastError();
}

}  // namespace h3a
