// Kernels of the norm and modulation before a branch (gfx950), and after one its
// gate and residual, for rows that fit a workgroup's or a wave's registers. The
// normed row is stored in bf16, or (kQuant) in 8 bits: e4m3 with a power of two for
// each 128 columns, which are the 8 columns each of 16 neighbouring lanes.
#pragma once

#include "fp8_util.h"
#include "kernels.h"
#include "row_util.h"

namespace h3a {
namespace {

// Eight normed values of a row from column c on, in 8 bits. Lanes past the row (in
// false) hold another lane's columns: they count for no group and store nothing. All
// lanes of the wave call it.
__device__ __forceinline__ void store_fp8(const ModulateParams& p, int64_t row, int c, const float (&o)[8], bool in) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(o[e]) & 0x7fffffffu);
    const int s = fp8_exponent(group16_max(in ? top : 0));
    if (!in) return;
    const float inv = fp8_inverse(s);
    __builtin_nontemporal_store(i32x2{fp8x4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv),
                                      fp8x4(o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv)},
                                (i32x2*)((char*)p.q + row * p.q_stride + c));
    if ((c & 127) == 0) p.q_scale[row * p.q_scale_stride + (c >> 7)] = (uint8_t)s;
}

// Vector path: C % 8 == 0, every row and table row 16-byte aligned.
// NV = vectors of 8 per thread, the fewest with NV * 8 * kThreads >= C, so a
// thread's vectors 0 .. NV-2 always lie inside the row and only the last may
// not. That one is loaded from the row's last vector instead and dropped.
// Every load of a phase is then issued without a branch between loads, and
// all of them are in flight together (a load behind a bounds branch is
// waited for before the next one is issued). Table dtypes are template
// arguments for the same reason.
template <int NV, bool kResidual, bool kTabF32, bool kWF32, bool kQuant>
__global__ __launch_bounds__(kThreads) void modulate_kernel(ModulateParams p) {
    __shared__ float red[kWaves];
    const int64_t row = blockIdx.x;
    const int C = p.cols;
    const int64_t t = table_row(p, row);
    int col[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) col[k] = (threadIdx.x + k * kThreads) * 8;
    const bool last = col[NV - 1] < C;  // the last vector lies inside the row
    if (!last) col[NV - 1] = C - 8;

    const uint16_t* xr = (const uint16_t*)p.x + row * p.x_stride;
    i32x4 rx[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) rx[k] = __builtin_nontemporal_load((const i32x4*)(xr + col[k]));
    float h[NV][8];
    float ss = 0.f;
    if constexpr (kResidual) {
        const uint16_t* rr = (const uint16_t*)p.residual + row * p.residual_stride;
        i32x4 rres[NV];
        Raw8<kTabF32> g[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) rres[k] = __builtin_nontemporal_load((const i32x4*)(rr + col[k]));
#pragma unroll
        for (int k = 0; k < NV; ++k) g[k] = fetch8<kTabF32>(p.gate, t * p.gate_stride + col[k]);
        uint16_t* hr = (uint16_t*)p.hidden + row * p.hidden_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float r[8], b[8], gv[8];
            unpack8(rres[k], r);
            unpack8(rx[k], b);
            unpack_raw8<kTabF32>(g[k], gv);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[k][e] = r[e] + gv[e] * b[e];
            if (k < NV - 1 || last) {
                __builtin_nontemporal_store(pack8(h[k]), (i32x4*)(hr + col[k]));
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += h[k][e] * h[k][e];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            unpack8(rx[k], h[k]);
            if (k < NV - 1 || last)
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += h[k][e] * h[k][e];
        }
    }
    // Weight and table rows are issued before the reduction, so their latency
    // overlaps it.
    Raw8<kWF32> w[NV];
    Raw8<kTabF32> sc[NV], sh[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        w[k] = fetch8<kWF32>(p.weight, col[k]);
        sc[k] = fetch8<kTabF32>(p.scale, t * p.scale_stride + col[k]);
        sh[k] = fetch8<kTabF32>(p.shift, t * p.shift_stride + col[k]);
    }
    const float r = rsqrtf(block_sum(ss, red) / (float)C + p.eps);
    uint16_t* orow = (uint16_t*)p.out + row * p.out_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (!kQuant && k == NV - 1 && !last) break;
        float wv[8], scv[8], shv[8], o[8];
        unpack_raw8<kWF32>(w[k], wv);
        unpack_raw8<kTabF32>(sc[k], scv);
        unpack_raw8<kTabF32>(sh[k], shv);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = h[k][e] * r * wv[e] * (1.0f + scv[e]) + shv[e];
        if constexpr (kQuant)
            store_fp8(p, row, col[k], o, k < NV - 1 || last);
        else
            __builtin_nontemporal_store(pack8(o), (i32x4*)(orow + col[k]));
    }
}

// Wave path (C % 8 == 0, C <= 64 * 8 * kRowVecMax, 16-byte aligned rows):
// one wave per row, four rows per workgroup, which share the weight row
// through LDS (one barrier). Each wave issues its row's loads (x, or
// residual and branch, and the gate row) and then every scale and shift
// vector it will need, all before the first wait, and holds its outputs
// until the end: on gfx9 one counter covers loads and stores, so a store
// issued ahead of a load would make that load's wait also wait for the
// store. The row index, and so the row bases and the modulation-table row,
// are wave-uniform (scalar registers; lanes add 32-bit offsets). Measured
// against the one-row-per-workgroup kernel above on 49,920 x 5,120 rows:
// 5.4 -> 6.0 TB/s (rmsnorm_modulate) and 5.3 -> 6.1 TB/s (residual
// variant); at 6,240 rows within 2%. Used for bf16 tables up to 11 vectors
// per lane (C <= 5,632), where it keeps two waves per SIMD; the block kernel
// takes the rest.
constexpr int kRowVecMax = 11;

template <bool kTabF32>
struct RowTabs {
    Raw8<kTabF32> sc, sh;
};

template <int NV, bool kResidual, bool kTabF32, bool kWF32, bool kQuant>
__global__ __launch_bounds__(kThreads) void modulate_row_kernel(ModulateParams p) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t row_id = (int64_t)blockIdx.x * kWaves + wave;  // uniform: row bases and t in scalar registers
    const bool live = row_id < p.rows;
    const int64_t row = live ? row_id : p.rows - 1;  // a wave past the rows loads the last one, stores nothing
    const int C = p.cols;
    // Vectors 0 .. NV-2 of a lane lie inside the row (NV = ceil(C / 512));
    // the last one, where it does not, is loaded from the row's last vector
    // and dropped. off[k]: byte offset of vector k in a bf16 row.
    uint32_t off[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) off[k] = (uint32_t)(lane + 64 * k) * 16u;
    const bool last = (int)(off[NV - 1] / 2) < C;
    if (!last) off[NV - 1] = (uint32_t)(C - 8) * 2u;

    const char* xr = (const char*)p.x + row * p.x_stride * 2;
    i32x4 rx[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) rx[k] = __builtin_nontemporal_load((const i32x4*)(xr + off[k]));
    i32x4 rres[kResidual ? NV : 1];
    if constexpr (kResidual) {
        const char* rr = (const char*)p.residual + row * p.residual_stride * 2;
#pragma unroll
        for (int k = 0; k < NV; ++k) rres[k] = __builtin_nontemporal_load((const i32x4*)(rr + off[k]));
    }
    const int64_t t = table_row(p, row);
    const int tb_sz = kTabF32 ? 4 : 2;
    const char* const wrow = (const char*)p.weight;
    const char* const scrow = (const char*)p.scale + t * p.scale_stride * tb_sz;
    const char* const shrow = (const char*)p.shift + t * p.shift_stride * tb_sz;
    // The weight row, shared by the workgroup's four rows, goes through LDS:
    // vector i (columns 8i .. 8i+7, the last clamped into the row) at wl[i].
    constexpr int kWv = NV * 64, kWl = kWF32 ? 2 : 1;
    __shared__ i32x4 wl[kWv * kWl];
    {
        constexpr int kIt = (kWv + kThreads - 1) / kThreads;
        Raw8<kWF32> wv[kIt];
#pragma unroll
        for (int it = 0; it < kIt; ++it) {
            const int i = min((int)threadIdx.x + it * kThreads, kWv - 1);
            wv[it] = fetch8o<kWF32>(wrow, (uint32_t)min(i * 8, C - 8) * 2u);
        }
#pragma unroll
        for (int it = 0; it < kIt; ++it) {
            const int i = min((int)threadIdx.x + it * kThreads, kWv - 1);
            wl[i * kWl] = wv[it].a;
            if constexpr (kWF32) wl[i * kWl + 1] = wv[it].b;
        }
    }
    auto tabs = [&](int k) __attribute__((always_inline)) {
        return RowTabs<kTabF32>{fetch8o<kTabF32>(scrow, off[k]), fetch8o<kTabF32>(shrow, off[k])};
    };
    float ss = 0.f;
    float h[kResidual ? NV : 1][8];
    if constexpr (kResidual) {
        const char* const grow = (const char*)p.gate + t * p.gate_stride * tb_sz;
        Raw8<kTabF32> g[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) g[k] = fetch8o<kTabF32>(grow, off[k]);
        char* const hr = (char*)p.hidden + row * p.hidden_stride * 2;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float r[8], b[8], gv[8];
            unpack_raw8<kTabF32>(g[k], gv);
            unpack8(rres[k], r);
            unpack8(rx[k], b);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[k][e] = r[e] + gv[e] * b[e];
            if (live && (k < NV - 1 || last)) {
                __builtin_nontemporal_store(pack8(h[k]), (i32x4*)(hr + off[k]));
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += h[k][e] * h[k][e];
            }
        }
    }
    RowTabs<kTabF32> tb[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) tb[k] = tabs(k);
    if constexpr (!kResidual) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float v[8];
            unpack8(rx[k], v);
            if (k < NV - 1 || last)
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
        }
        // Unpack x again below rather than keep the fp32 values of the sum
        // live through it (twice the registers of the raw vectors).
#pragma unroll
        for (int k = 0; k < NV; ++k) asm volatile("" : "+v"(rx[k]));
    }
    const float r = rsqrtf(wave_sum(ss) / (float)C + p.eps);
    __syncthreads();  // the weight row is in LDS
    if (!live) return;
    i32x4 ov[kQuant ? 1 : NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float v[8], wv[8], scv[8], shv[8], o[8];
        if constexpr (kResidual) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = h[k][e];
        } else {
            unpack8(rx[k], v);
        }
        {
            Raw8<kWF32> w;
            w.a = wl[(lane + 64 * k) * kWl];
            if constexpr (kWF32) w.b = wl[(lane + 64 * k) * kWl + 1];
            unpack_raw8<kWF32>(w, wv);
        }
        unpack_raw8<kTabF32>(tb[k].sc, scv);
        unpack_raw8<kTabF32>(tb[k].sh, shv);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e] * r * wv[e] * (1.0f + scv[e]) + shv[e];
        if constexpr (kQuant)
            store_fp8(p, row, (int)off[k] / 2, o, k < NV - 1 || last);
        else
            ov[k] = pack8(o);
    }
    if constexpr (kQuant) return;
    char* const orow = (char*)p.out + row * p.out_stride * 2;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (k < NV - 1 || last) __builtin_nontemporal_store(ov[kQuant ? 0 : k], (i32x4*)(orow + off[k]));
}

// The rows up to which the 8-bit forms take a workgroup per row: few rows leave CUs idle,
// and a row's loads and sum are done the sooner the more waves share it (us, wave /
// workgroup: 257 x 5,376 6.2 / 3.6, with the residual 8.0 / 4.2; 512 rows 6.6 / 4.5 and 8.5
// / 6.1, of 1,024 columns 2.9 / 2.7; 1,024 rows 7.0 / 6.0 but with the residual 9.0 / 10.3).
// One limit for both: the residual's; without it a workgroup still gains 1 us at 1,024 rows.
constexpr int kFewRows = 512;

template <bool kResidual, bool kTabF32, bool kWF32, bool kQuant>
void launch_modulate_vec(const ModulateParams& p, int nv, hipStream_t stream) {
    const int nw = (int)((p.cols + 511) / 512);  // vectors per lane with one wave per row
    if constexpr (!kTabF32) {
        if (nw <= kRowVecMax && (!kQuant || p.rows > kFewRows)) {
            const dim3 grid((unsigned)((p.rows + kWaves - 1) / kWaves)), block(kThreads);
            switch (nw) {
#define H3A_NW(n)                                                                                                     \
    case n:                                                                                                           \
        hipLaunchKernelGGL((modulate_row_kernel<n, kResidual, kTabF32, kWF32, kQuant>), grid, block, 0, stream, p);         \
        break;
                H3A_NW(1) H3A_NW(2) H3A_NW(3) H3A_NW(4) H3A_NW(5) H3A_NW(6) H3A_NW(7) H3A_NW(8)
                H3A_NW(9) H3A_NW(10) H3A_NW(11)
#undef H3A_NW
            }
            return;
        }
    }
    const dim3 grid((unsigned)p.rows), block(kThreads);
    switch (nv) {
#define H3A_NV(n)                                                                                                     \
    case n:                                                                                                           \
        hipLaunchKernelGGL((modulate_kernel<n, kResidual, kTabF32, kWF32, kQuant>), grid, block, 0, stream, p);             \
        break;
        H3A_NV(1) H3A_NV(2) H3A_NV(3) H3A_NV(4) H3A_NV(5) H3A_NV(6) H3A_NV(7) H3A_NV(8)
#undef H3A_NV
    }
}

}  // namespace
}  // namespace h3a
