// Matrix product of 8-bit operands with bias, activation, gate and residual in its
// epilogue (gfx950): linear.hip's layers with e4m3 values and a power of two for each
// 128 values of K (fp8_util.h).
//
//   z[m, f] = sum_b xs[m, b] ws[f / 128, b] sum_{k in block b} x[m, k] * w[f, k]
// and then as in linear.hip, the result in bf16 or in 8 bits in groups of 128
// features. The matrix instructions take both scales with their operands
// (v_mfma_scale_f32_*_f8f6f4: one e8m0 for each row's 32 values of K), so a scaled
// sum accumulates as an unscaled one does, without a separate sum per block.
#include "fp8_util.h"
#include "kernels.h"
#include "linear_util.h"

namespace h3a {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------- few tokens

// linear.hip's row form on bytes: NA blocks of 16 rows of w x 16 NB tokens per
// workgroup, K split over its waves by chunks of 128 bytes, a scale's block each. Lane
// l holds of row l & 15 the 16-byte pieces l >> 4 and 4 + (l >> 4) of a chunk, of w and
// of x alike (which of the chunk's K they are does not matter to a sum over all).
// bf16 rows of x are rounded to 8 bits as they come in: the four lanes of a row hold a
// whole group.
constexpr int kRowsMaxTokens = 32;

template <int NA, int NB, bool kGated, bool kXBf16>
__global__ __launch_bounds__(NA == 1 ? 1024 : 512) void linear_fp8_rows_kernel(LinearFp8Params p) {
    constexpr int kS = kGated ? 2 : 1, NF = NA / kS;  // blocks of output features
    constexpr int kU = NA * NB >= 4 || kXBf16 ? 1 : 4;
    constexpr int kX = kXBf16 ? 4 : 2;  // 16-byte loads of a row's pieces
    extern __shared__ f32x4 part[];  // [wave][NA * NB][64]
    const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, l15 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)blockDim.x >> 6;
    const int f0 = (int)blockIdx.x * 16 * NF, m0 = (int)blockIdx.y * 16 * NB;
    const char* wr[NA];
#pragma unroll
    for (int a = 0; a < NA; ++a)
        wr[a] = (const char*)p.w + ((int64_t)(a % kS) * p.n + min(f0 + 16 * (a / kS) + l15, p.n - 1)) * p.w_rs;
    const uint8_t* ws[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) ws[s] = p.w_scale + (int64_t)(s * p.w_blocks + f0 / kFp8Group) * p.w_scale_rs;
    const char* xr[NB];
    const uint8_t* xs[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t m = min(m0 + 16 * b + l15, p.m - 1);
        xr[b] = (const char*)p.x + m * p.x_rs;
        xs[b] = p.x_scale + m * p.x_scale_rs;
    }
    f32x4 acc[NA][NB];
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{};
    const int chunks = (p.k + kFp8Group - 1) / kFp8Group;
    for (int c0 = wave; c0 < chunks; c0 += waves * kU) {
        i32x4 w[kU][2][NA], x[kU][kX][NB];
        int sw[kU][kS], sx[kU][NB];
        bool in[kU][2];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int c = c0 + u * waves;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = c * kFp8Group + h * 64 + q * 16;
                in[u][h] = at < p.k;
                const int o = in[u][h] ? at : p.k - 16;
#pragma unroll
                for (int a = 0; a < NA; ++a) w[u][h][a] = *(const i32x4*)(wr[a] + o);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if constexpr (kXBf16) {
                        x[u][2 * h][b] = *(const i32x4*)(xr[b] + 2 * o);
                        x[u][2 * h + 1][b] = *(const i32x4*)(xr[b] + 2 * o + 16);
                    } else {
                        x[u][h][b] = *(const i32x4*)(xr[b] + o);
                    }
                }
            }
            const int cs = min(c, chunks - 1);
#pragma unroll
            for (int s = 0; s < kS; ++s) sw[u][s] = ws[s][cs];
            if constexpr (!kXBf16) {
#pragma unroll
                for (int b = 0; b < NB; ++b) sx[u][b] = xs[b][cs];
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            i32x8 xv[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (kXBf16) {
                    float v[4][8];
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const i32x4 raw = in[u][i / 2] ? x[u][i][b] : i32x4{};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[i][2 * e] = __uint_as_float((uint32_t)raw[e] << 16);
                            v[i][2 * e + 1] = __uint_as_float((uint32_t)raw[e] & 0xffff0000u);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
                    }
                    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
                    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
                    sx[u][b] = fp8_exponent(top);
                    const float inv = fp8_inverse(sx[u][b]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        xv[b][2 * i] = fp8x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
                        xv[b][2 * i + 1] = fp8x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) xv[b][4 * h + e] = in[u][h] ? x[u][h][b][e] : 0;
                }
            }
#pragma unroll
            for (int a = 0; a < NA; ++a) {
                i32x8 wv;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) wv[4 * h + e] = in[u][h] ? w[u][h][a][e] : 0;
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv[b], acc[a][b], 0, 0, 0, sw[u][a % kS], 0, sx[u][b]);
            }
        }
    }
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) part[(wave * NA * NB + a * NB + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    // Wave i finishes block i of the NF x NB: lane l holds token l & 15, features 4 (l >> 4) + e.
    for (int i = wave; i < NF * NB; i += waves) {
        const int a = i / NB, b = i % NB;
        const int m = m0 + 16 * b + l15, f = f0 + 16 * a + 4 * q;
        f32x4 z[kS];
#pragma unroll
        for (int s = 0; s < kS; ++s) {
            z[s] = f32x4{};
            for (int v = 0; v < waves; ++v) z[s] += part[(v * NA * NB + (kS * a + s) * NB + b) * 64 + lane];
        }
        if (m >= p.m || f >= p.n) continue;
        if (p.y32 != nullptr)
            *(f32x4*)(p.y32 + (int64_t)m * p.n + f) = finished4<kS>(p, z, m, f);
        else
            finish4<kS>(p, z, m, f);
    }
}

template <int NA, int NB, bool kGated, bool kXBf16>
hipError_t launch_rows_t(const LinearFp8Params& p, int waves, hipStream_t stream) {
    constexpr int kFeatures = 16 * NA / (kGated ? 2 : 1);
    const dim3 grid((unsigned)((p.n + kFeatures - 1) / kFeatures), (unsigned)((p.m + 16 * NB - 1) / (16 * NB)));
    const size_t lds = (size_t)waves * NA * NB * 1024;
    hipLaunchKernelGGL((linear_fp8_rows_kernel<NA, NB, kGated, kXBf16>), grid, dim3(64 * waves), lds, stream, p);
    return hipGetLastError();
}

// Blocks of rows per workgroup and its waves, as linear.hip chooses them.
struct RowsForm {
    int na, waves;
    int64_t groups;  // workgroups
};

RowsForm rows_form(const LinearFp8Params& p, int cus) {
    const int64_t blocks = (int64_t)((p.n + 15) / 16) * (p.gated ? 2 : 1);
    RowsForm f;
    f.na = blocks >= 4ll * cus ? 4 : blocks >= cus || p.gated ? 2 : 1;
    f.groups = (blocks + f.na - 1) / f.na;
    f.waves = 4;
    while (f.waves < (f.na == 1 ? 16 : 8) && f.groups * f.waves < 16ll * cus && f.waves * kFp8Group < p.k) f.waves *= 2;
    return f;
}

template <int NB, bool kXBf16>
hipError_t launch_rows(const LinearFp8Params& p, int cus, hipStream_t stream) {
    const RowsForm f = rows_form(p, cus);
    if (p.gated) return f.na == 4 ? launch_rows_t<4, NB, true, kXBf16>(p, f.waves, stream) : launch_rows_t<2, NB, true, kXBf16>(p, f.waves, stream);
    return f.na == 4   ? launch_rows_t<4, NB, false, kXBf16>(p, f.waves, stream)
           : f.na == 2 ? launch_rows_t<2, NB, false, kXBf16>(p, f.waves, stream)
                       : launch_rows_t<1, NB, false, kXBf16>(p, f.waves, stream);
}

// y32's rounding to 8 bits.
hipError_t launch_result(const LinearFp8Params& p, hipStream_t stream) {
    QuantizeParams q{};
    q.x = p.y32; q.q = p.y; q.scale = p.y_scale;
    q.x_rs = 4 * (int64_t)p.n; q.q_rs = p.y_rs; q.scale_rs = p.y_scale_rs;
    q.rows = p.m; q.part_rows = p.m; q.cols = p.n; q.x_f32 = 1;
    return launch_quantize(q, stream);
}

}  // namespace

void plan_linear_fp8(LinearFp8Params& p, int cus, int64_t* required, int64_t* workspace) {
    if (cus <= 0) cus = 256;
    *required = *workspace = p.y_scale != nullptr ? 4 * (int64_t)p.m * p.n : 0;
    const RowsForm f = rows_form(p, cus);
    const int64_t nb = p.m <= 16 ? 1 : 2;
    p.shape = f.groups * ((p.m + 16 * nb - 1) / (16 * nb)) * 64 * f.waves <= UINT32_MAX ? -1 : -2;  // work items of a launch
}

hipError_t launch_linear_fp8(const LinearFp8Params& p, int cus, hipStream_t stream) {
    if (cus <= 0) cus = 256;
    LinearFp8Params r = p;
    r.y32 = p.y_scale != nullptr ? (float*)p.ws : nullptr;
    hipError_t e;
    if (p.x_scale == nullptr)
        e = p.m <= 16 ? launch_rows<1, true>(r, cus, stream) : launch_rows<2, true>(r, cus, stream);
    else
        e = p.m <= 16 ? launch_rows<1, false>(r, cus, stream) : launch_rows<2, false>(r, cus, stream);
    if (e != hipSuccess || p.y_scale == nullptr) return e;
    return launch_result(r, stream);
}

}  // namespace h3a
