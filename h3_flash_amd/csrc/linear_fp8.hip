// Matrix product of 8-bit operands with bias, activation, gate and residual in its
// epilogue (gfx950): linear.hip's layers with e4m3 values and a power of two for each
// 128 values of K (fp8_util.h).
//
//   z[m, f] = sum_b xs[m, b] ws[f / 128, b] sum_{k in block b} x[m, k] * w[f, k]
// and then as in linear.hip, the result in bf16 or in 8 bits in groups of 128
// features. The matrix instructions take both scales with their operands
// (v_mfma_scale_f32_*_f8f6f4: one e8m0 for each row's 32 values of K), so a scaled
// sum accumulates as an unscaled one does, without a separate sum per block.
//
// Two forms, as there: tiles (linear_fp8_tile.h) from a few dozen tokens on, and a form
// that streams w once for fewer. bf16 rows are rounded to 8 bits by a launch of their
// own before the tiles, and as they come in by the other form.
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
// whole group. 1 x 1,024 x 1,024 from bf16: 4.2 us, launch and one round of loads.
constexpr int kRowsMaxTokens = 32;
// It serves small weights, where the call's latency counts. Larger ones come in faster
// by the tiles' deep rings of loads, also for one block of 16 tokens and a launch more
// that rounds bf16 rows (us, this form at its best / tiles: 16 x 5,376 x 5,376 12.4 /
// 14.7; 16 x 14,336 x 5,376 26.2 / 20.4; 16 x 5,376 x 32,256 37.2 / 31.5; 32 x 1,024 x
// 4,096 5.4 / 6.4; 32 x 5,376 x 5,376 16.8 / 15: the limits lie between those points).
constexpr int64_t kRowsMaxWeight[2] = {48 << 20, 16 << 20};  // bytes, up to 16 and 32 tokens
constexpr int kRowsForm = -1, kNoForm = -2;  // in place of a tile shape

template <int NA, int NB, bool kGated, bool kXBf16>
__global__ __launch_bounds__(NA == 1 ? 1024 : 512) void linear_fp8_rows_kernel(LinearFp8Params p) {
    constexpr int kS = kGated ? 2 : 1, NF = NA / kS;  // blocks of output features
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
    for (int c = wave; c < chunks; c += waves) {
        i32x4 w[2][NA], x[kX][NB];
        int sw[kS], sx[NB];
        bool in[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = c * kFp8Group + h * 64 + q * 16;
            in[h] = at < p.k;
            const int o = in[h] ? at : p.k - 16;
#pragma unroll
            for (int a = 0; a < NA; ++a) w[h][a] = *(const i32x4*)(wr[a] + o);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (kXBf16) {
                    x[2 * h][b] = *(const i32x4*)(xr[b] + 2 * o);
                    x[2 * h + 1][b] = *(const i32x4*)(xr[b] + 2 * o + 16);
                } else {
                    x[h][b] = *(const i32x4*)(xr[b] + o);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < kS; ++s) sw[s] = ws[s][c];
        if constexpr (!kXBf16) {
#pragma unroll
            for (int b = 0; b < NB; ++b) sx[b] = xs[b][c];
        }
        i32x8 xv[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (kXBf16) {
                float v[4][8];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const i32x4 raw = in[i / 2] ? x[i][b] : i32x4{};
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
                sx[b] = fp8_exponent(top);
                const float inv = fp8_inverse(sx[b]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    xv[b][2 * i] = fp8x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
                    xv[b][2 * i + 1] = fp8x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) xv[b][4 * h + e] = in[h] ? x[h][b][e] : 0;
            }
        }
#pragma unroll
        for (int a = 0; a < NA; ++a) {
            i32x8 wv;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) wv[4 * h + e] = in[h] ? w[h][a][e] : 0;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv[b], acc[a][b], 0, 0, 0, sw[a % kS], 0, sx[b]);
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
    f.na = blocks >= 4ll * cus ? 4 : blocks > cus || p.gated ? 2 : 1;
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

// ---------------------------------------------------------------- tiles

// The tile shapes, with the time of a K step of 128 with all CUs busy and a tile's
// fixed part (launch, first loads, epilogue). Fitted to graph replays of 26 sizes (16
// to 12,480 tokens, 2,048 to 32,256 features, k 1,552 to 14,336) in every shape and
// split; the choice by them takes 0.5% longer than the best of all, in the mean.
struct Shape {
    int tf, nt;
    float step_us, fixed_us;
    hipError_t (*launch)(const LinearFp8Params&, hipStream_t);
};
constexpr Shape kShapes[] = {
    {256, 16, 1.352f, 6.57f, launch_linear_fp8_tile<256, 16, 3, 2>}, {256, 12, 1.034f, 6.07f, launch_linear_fp8_tile<256, 12, 3, 2>},
    {256, 8, 0.795f, 5.18f, launch_linear_fp8_tile<256, 8, 3, 3>},   {128, 8, 0.472f, 4.78f, launch_linear_fp8_tile<128, 8, 5, 4>},
    {128, 6, 0.375f, 4.98f, launch_linear_fp8_tile<128, 6, 6, 4>},   {128, 4, 0.317f, 5.74f, launch_linear_fp8_tile<128, 4, 6, 5>},
    {128, 2, 0.295f, 2.95f, launch_linear_fp8_tile<128, 2, 8, 6>},
};
constexpr float kIdleGain = 0.29f;  // of a K step's time, saved as the CUs of a round go idle
// A second launch joins the pieces, over their sums at 0.24 us a MB.
constexpr float kJoinUs = 2.13f, kJoinUsPerByte = 0.24e-6f;
// The operands from memory; of this and the tiles' time the larger counts, and a tenth
// of the smaller.
constexpr float kMemoryUs = 7.2f, kMemoryUsPerByte = 1.0f / 7.52e6f;
constexpr int kSplits[] = {2, 3, 4, 6, kLinearFp8MaxSplit};
constexpr int kMinPieceSteps = 8;

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// x in 8 bits, for the tiles, at the start of the workspace.
struct RoundedX {
    int64_t scale_rs, scale_at, bytes;
};
RoundedX rounded_x(const LinearFp8Params& p) {
    const int64_t rs = ((p.k + kFp8Group - 1) / kFp8Group + 15) / 16 * 16, at = round256((int64_t)p.m * p.k);
    return RoundedX{rs, at, at + round256(p.m * rs)};
}

hipError_t launch_rounded_x(LinearFp8Params& p, hipStream_t stream) {
    const RoundedX r = rounded_x(p);
    QuantizeParams q{};
    q.x = p.x; q.q = p.ws; q.scale = (uint8_t*)p.ws + r.scale_at;
    q.x_rs = p.x_rs; q.q_rs = p.k; q.scale_rs = r.scale_rs;
    q.rows = p.m; q.part_rows = p.m; q.cols = p.k;
    p.x = q.q; p.x_rs = p.k; p.x_scale = q.scale; p.x_scale_rs = r.scale_rs;
    return launch_quantize(q, stream);
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
    *required = *workspace = 0;
    p.shape = kNoForm;
    const int64_t w_bytes = (p.gated ? 2 : 1) * (int64_t)p.n * p.k;
    if (p.m <= kRowsMaxTokens && w_bytes <= kRowsMaxWeight[p.m > 16]) {
        const RowsForm f = rows_form(p, cus);
        if (f.groups * 64 * f.waves <= UINT32_MAX) p.shape = kRowsForm;  // work items of a launch
        if (p.y_scale != nullptr) *required = *workspace = 4 * (int64_t)p.m * p.n;
        return;
    }
    if (p.x_scale == nullptr) {
        *required = rounded_x(p).bytes;
        if ((int64_t)p.m * ((p.k + kFp8Group - 1) / kFp8Group) > quantize_max_groups(false)) return;
    }
    const int steps = (p.k + kFp8Group - 1) / kFp8Group;
    const float memory_us = kMemoryUs + kMemoryUsPerByte * ((float)w_bytes + (float)p.m * (float)p.k + 2.f * (float)p.m * (float)p.n);
    float best_us = 0.f;
    for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
        const Shape& s = kShapes[i];
        const int to = p.gated ? s.tf / 2 : s.tf, tokens = 16 * s.nt;
        if (p.y_scale != nullptr && to % kFp8Group != 0) continue;  // a group in two tiles
        const int64_t n_tiles = (p.n + to - 1) / to, m_tiles = (p.m + tokens - 1) / tokens, tiles = n_tiles * m_tiles;
        if (tiles * 256 > UINT32_MAX) continue;  // work items of a launch
        // Whole: rounds of tiles over the CUs, the last one faster the fewer CUs it
        // keeps busy; past six rounds the tiles no longer run in step, and the
        // last round costs about half of one.
        const int64_t full = tiles / cus * cus, rest = tiles - full;
        const float tile_us = (float)steps * s.step_us + s.fixed_us, rounds = (float)tiles / (float)cus;
        auto last_us = [&](int n) {
            return (float)steps / (float)n * s.step_us * (1.f - kIdleGain * (1.f - (float)(rest * n) / (float)cus)) + s.fixed_us;
        };
        float us = rounds > 6.f ? (rounds + 0.5f) * tile_us : (float)(full / cus) * tile_us + (rest > 0 ? last_us(1) : 0.f);
        int split = 1;
        // The last round in pieces, at most one per CU (of the smallest tiles none: they
        // serve short reductions; nor with the result in 8 bits, whose groups the join's
        // workgroups, 32 tokens x 8 features a wave, do not hold: with few tiles over a long
        // reduction that costs up to four times a bf16 result's time, 64 x 14,336 x 1,024
        // gated 65.8 us against 15.1, 256 x 5,376 x 2,688 29.8 against 20.8).
        for (const int n : kSplits) {
            if (rest == 0 || rest * n > cus || steps / n < kMinPieceSteps || s.nt == 2 || p.y_scale != nullptr) break;
            const float cut = (float)(full / cus) * tile_us + last_us(n) + kJoinUs + (float)(rest * n * s.tf * tokens * 4) * kJoinUsPerByte;
            if (cut < us) {
                us = cut;
                split = n;
            }
        }
        us = us > memory_us ? us + 0.1f * memory_us : memory_us + 0.1f * us;
        if (p.shape >= 0 && us >= best_us) continue;
        best_us = us;
        p.shape = i;
        p.m_tiles = (int32_t)m_tiles;
        p.n_tiles = (int32_t)n_tiles;
        // Tokens of a group of the tile order, as in linear.hip.
        const int group_tokens = p.m <= 2048 ? 2048 : p.m <= 16384 ? 1536 : 768;
        p.group_m = (int32_t)(group_tokens / tokens < m_tiles ? group_tokens / tokens : m_tiles);
        p.split = split;
        p.n_full = (int32_t)(split > 1 ? full : tiles);
        *workspace = *required + (split > 1 ? rest * split * (int64_t)(s.tf * tokens * 4) : 0);
    }
}

hipError_t launch_linear_fp8(const LinearFp8Params& p, int cus, hipStream_t stream) {
    if (p.shape == kNoForm) return hipErrorInvalidConfiguration;
    if (cus <= 0) cus = 256;
    LinearFp8Params r = p;
    if (p.shape >= 0) {
        r.sums = p.ws;
        if (p.x_scale == nullptr) {
            r.sums = (char*)p.ws + rounded_x(p).bytes;
            const hipError_t e = launch_rounded_x(r, stream);
            if (e != hipSuccess) return e;
        }
        return kShapes[p.shape].launch(r, stream);
    }
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
