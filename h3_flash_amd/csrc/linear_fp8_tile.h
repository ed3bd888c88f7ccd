// The tile kernels of linear_fp8.hip (gfx950): gemm_fp8_tile.h's product with the
// epilogue of a linear layer. Each shape is compiled in one of the linear_fp8_*.hip
// files.
#pragma once

#include "fp8_util.h"
#include "gemm_fp8_tile.h"
#include "kernels.h"
#include "linear_util.h"

namespace h3a {
namespace {

typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef __attribute__((address_space(3))) int lds_i32;

// Maximum over aligned groups of 32 lanes; all lanes must be active.
__device__ __forceinline__ uint32_t group32_max(uint32_t v) {
    v = group16_max(v);
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

// Modulation-table row of token m (gate_row without its 64-bit division).
__device__ __forceinline__ int64_t gate_row32(const LinearFp8Params& p, int m) {
    const uint32_t i = (int64_t)m < p.n_index ? (uint32_t)m : (uint32_t)m % (uint32_t)p.n_index;
    int64_t t = p.index_i64 ? ((const int64_t*)p.index)[i] : (int64_t)((const int32_t*)p.index)[i];
    t = t < 0 ? 0 : t;
    return t >= p.table_rows ? p.table_rows - 1 : t;
}

// SiLU where nothing else is asked for. (-inf comes to its limit -0; NaN stays in s.)
__device__ __forceinline__ float silu(float z) {
    const float s = __builtin_amdgcn_rcpf(1.0f + fast_exp2(z * -1.44269504088896f));
    return fmaxf(z, -1e30f) * s;
}

// Bits of the largest magnitude of four values.
__device__ __forceinline__ uint32_t top4(const f32x4& y) {
    // (maximum keeps NaN, and takes magnitudes at no cost)
    const float a = __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(y[0]), fabsf(y[1])), fabsf(y[2]));
    return __float_as_uint(__builtin_elementwise_maximum(a, fabsf(y[3]))) & 0x7fffffffu;
}

// Epilogue of a tile: lane l holds, for token block b (token 32 (NB wm + b) + (l & 31)),
// row block a of w and group g, tile rows 32 (NA wn + a) + 8g + 4 (l >> 5) + e; gated,
// groups 0 and 1 of a block are its 16 values and 2 and 3 their gates. kPass blocks of
// tokens at a time go through LDS (the idle stages) in fp32, row r's 16-byte chunk c at
// c ^ (r & 7), and a thread then takes four features of a token at a time, kBatch
// tokens in flight. In 8 bits, 32 neighbouring threads hold a group of 128 features.
// Rows past m and features past n are outside the records of the result's (and the
// residual's) buffer, so that no branch breaks up a batch; without a bias, gate or
// residual, and with a bias alone, the loop has a form of its own. (With a branch per
// token for each of them, as linear.hip has it, the epilogue took 25,400 of the 129,500
// cycles of a 256 x 256 tile of k = 5,120, and 32,800 of 140,700 gated, in 8 bits, at
// k = 5,376; now 9,000 and 16,700.) The tokens' gate rows are looked up once, into LDS behind the rows.
template <typename T, bool kGated, bool kQuant>
__device__ __forceinline__ void linear_fp8_epilogue(const LinearFp8Params& p, int f0, int m0, const f32x16 (&acc)[T::NA][T::NB],
                                                    int wn, int wm, int tid, char* smem) {
    constexpr int kS = kGated ? 2 : 1, TO = T::kTF / kS, kRowBytes = T::kTF * 4;
    constexpr int kCols = TO / 4, kRows = kPThreads / kCols;  // threads of a row, rows at a time
    constexpr int kRowsPass = 32 * T::kPass, kIts = kRowsPass / kRows;  // of one wave row
    constexpr int kBatch = kIts % 8 == 0 ? 8 : kIts % 6 == 0 ? 6 : kIts;
    static_assert(kIts % kBatch == 0 && kBatch <= 8, "batches of a pass");
    static_assert(!kQuant || TO % kFp8Group == 0, "whole groups of features");
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int r0 = tid / kCols, c = tid % kCols, f = f0 + 4 * c;
    const bool in = f < p.n;
    const int fc = in ? f : 0, rows = min(T::kTokens, p.m - m0);
    constexpr uint32_t kOut = 0x80000000u;  // past any record
    f32x4 bias[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) bias[s] = p.bias != nullptr ? load4(p.bias, s * p.n + fc, p.bias_f32 != 0) : f32x4{};
    const auto y_rsrc = make_rsrc((char*)p.y + (int64_t)m0 * p.y_rs, (uint32_t)((rows - 1) * p.y_rs + (kQuant ? 1 : 2) * (int64_t)p.n));
    const uint32_t y_off = in ? (uint32_t)(r0 * p.y_rs + (kQuant ? 1 : 2) * f) : kOut;
    const auto s_rsrc = make_rsrc(kQuant ? p.y_scale + (int64_t)m0 * p.y_scale_rs : nullptr, kQuant ? (uint32_t)(rows * p.y_scale_rs) : 0u);
    const uint32_t s_off = in && (c & 31) == 0 ? (uint32_t)(r0 * p.y_scale_rs + f / kFp8Group) : kOut;
    const auto r_rsrc = make_rsrc((const char*)p.residual + (int64_t)m0 * p.res_rs,
                                  p.residual != nullptr ? (uint32_t)((rows - 1) * p.res_rs + 2 * (int64_t)p.n) : 0u);
    const uint32_t r_off = in ? (uint32_t)(r0 * p.res_rs + 2 * f) : kOut;
    lds_char* const buf = (lds_char*)smem;
    lds_i32* const gate_rows = (lds_i32*)(buf + T::kEpiRows);
    if (p.gate != nullptr && tid < T::kTokens) gate_rows[tid] = (int)gate_row32(p, min(m0 + tid, p.m - 1));  // (read after the pass's barrier)
    lds_char* const wr = buf + (wm * kRowsPass + (lane & 31)) * kRowBytes;
    const int sw = lane & 7;
    auto pass = [&](auto h_c) __attribute__((always_inline)) {
        constexpr int h = decltype(h_c)::value, b0 = h * T::kPass;
        if constexpr (h > 0) __syncthreads();  // the rows of the pass before have been read
#pragma unroll
        for (int b = 0; b < T::kPass; ++b)
#pragma unroll
            for (int a = 0; a < T::NA; ++a)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int x = T::NA * wn + a, e = 2 * (kGated ? g & 1 : g) + (lane >> 5);
                    const int chunk = kGated ? (g >> 1) * kCols + 4 * x + e : 8 * x + e;
                    const f32x16& v = acc[a][b0 + b];
                    *(lds_f32x4*)(wr + b * 32 * kRowBytes + ((chunk ^ sw) << 4)) = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                }
        __syncthreads();
        // Batch j: tokens t0 + r0 + kRows i, at rows l0 + r0 + kRows i of the buffer.
        constexpr int kPerWave = kIts / kBatch;
        auto first_token = [&](int j) __attribute__((always_inline)) {
            return (T::WM == 2 ? j / kPerWave : 0) * (32 * T::NB) + 32 * b0 + (T::WM == 2 ? j % kPerWave : j) * (kBatch * kRows);
        };
        // kMode 0: nothing but the activation; 1: a bias; 2: any of bias, gate, residual.
        auto loop = [&](auto act, auto mode_c) __attribute__((always_inline)) {
            constexpr int kMode = decltype(mode_c)::value;
            struct Batch {
                i32x2 res[kBatch];
                f32x4 gate[kBatch];
            };
            auto load_batch = [&](Batch& q, int j) __attribute__((always_inline)) {
                const int t0 = first_token(j);
                if (p.residual != nullptr) {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        q.res[i] = __builtin_amdgcn_raw_buffer_load_b64(r_rsrc, (int)r_off, (int)((t0 + kRows * i) * p.res_rs), 0);
                }
                if (p.gate != nullptr) {
                    const char* at[kBatch];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) at[i] = (const char*)p.gate + gate_rows[t0 + r0 + kRows * i] * p.gate_rs;
                    if (p.gate_f32) {
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) q.gate[i] = *(const f32x4*)(at[i] + 4 * fc);
                    } else {
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) q.gate[i] = unpack4(*(const i32x2*)(at[i] + 2 * fc));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) q.gate[i] = f32x4{1.f, 1.f, 1.f, 1.f};
                }
            };
            Batch cur;
            if constexpr (kMode == 2) load_batch(cur, 0);
#pragma unroll 1
            for (int j = 0; j < T::WM * kPerWave; ++j) {
                Batch next;
                if constexpr (kMode == 2)
                    if (j + 1 < T::WM * kPerWave) load_batch(next, j + 1);
                const int t0 = first_token(j), l0 = j * (kBatch * kRows) + r0;
                f32x4 z[kBatch][kS];
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
#pragma unroll
                    for (int s = 0; s < kS; ++s) {
                        const int r = l0 + kRows * i;
                        z[i][s] = *(const lds_f32x4*)(buf + r * kRowBytes + (((s * kCols + c) ^ (r & 7)) << 4));
                        if constexpr (kMode > 0) z[i][s] += bias[s];
                    }
                f32x4 y[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[i][e] = act(z[i][kS - 1][e]);
                        if constexpr (kGated) y[i][e] *= z[i][0][e];
                    }
                    if constexpr (kMode == 2) y[i] *= cur.gate[i];
                }
                if constexpr (kMode == 2) {
                    if (p.residual != nullptr) {
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) y[i] += unpack4(cur.res[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int row = t0 + kRows * i;
                    if constexpr (kQuant) {
                        const int s = fp8_exponent(group32_max(in ? top4(y[i]) : 0));
                        const float inv = fp8_inverse(s);
                        __builtin_amdgcn_raw_buffer_store_b32(fp8x4(y[i][0] * inv, y[i][1] * inv, y[i][2] * inv, y[i][3] * inv), y_rsrc,
                                                              (int)y_off, (int)(row * p.y_rs), 0);
                        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)s, s_rsrc, (int)s_off, (int)(row * p.y_scale_rs), 0);
                    } else {
                        __builtin_amdgcn_raw_buffer_store_b64(i32x2{(int)pack_bf16x2(y[i][0], y[i][1]), (int)pack_bf16x2(y[i][2], y[i][3])}, y_rsrc,
                                                              (int)y_off, (int)(row * p.y_rs), 0);
                    }
                }
                if constexpr (kMode == 2) cur = next;
            }
        };
        // One copy of the loop per activation (with gate or residual, two activations
        // share one): its code is what runs.
        auto with = [&](auto mode) __attribute__((always_inline)) {
            if (p.act == H3A_ACT_NONE)
                loop([](float z) { return z; }, mode);
            else if (p.act == H3A_ACT_RELU)
                loop([](float z) { return activate(z, H3A_ACT_RELU); }, mode);
            else if (p.act == H3A_ACT_GELU)
                loop([](float z) { return activate(z, H3A_ACT_GELU); }, mode);
            else if constexpr (decltype(mode)::value == 2)
                loop([&](float z) { return activate(z, p.act == H3A_ACT_SILU ? H3A_ACT_SILU : H3A_ACT_GELU_TANH); }, mode);
            else if (p.act == H3A_ACT_SILU)
                loop([](float z) { return silu(z); }, mode);
            else
                loop([](float z) { return activate(z, H3A_ACT_GELU_TANH); }, mode);
        };
        if (p.gate != nullptr || p.residual != nullptr)
            with(std::integral_constant<int, 2>{});
        else if (p.bias != nullptr)
            with(std::integral_constant<int, 1>{});
        else
            with(std::integral_constant<int, 0>{});
    };
    static_for<T::NB / T::kPass>(pass);
}

// Tile `tile` of groups of p.group_m token tiles x every feature tile, token
// tile fastest.
struct TileCoord {
    int f0, m0;
};
__device__ __forceinline__ TileCoord tile_coord(const LinearFp8Params& p, int tile, int to, int tokens) {
    const int in_group = p.group_m * p.n_tiles, first_m = (tile / in_group) * p.group_m;
    const int group_m = min(p.m_tiles - first_m, p.group_m);
    return TileCoord{(tile % in_group) / group_m * to, (first_m + (tile % in_group) % group_m) * tokens};
}

// Workgroups [0, n_full) run whole tiles, the others the tiles after them in `split`
// pieces along K, whose sums linear_fp8_join_kernel adds in order (linear.hip).
// Bound by power where the product is large: 256 x 256 tiles keep the matrix cores 69 to
// 72% busy at 1.9 to 2.1 GHz. In graph replays on seven cards 6,240 x 5,376 x 28,672 gated,
// into 8 bits, takes 717 to 782 us (2,460 to 2,680 TFLOP/s), 6,240 x 14,336 x 5,376 348 to
// 378, with its 13 last tiles in 8 pieces (whole: 433 to 449), 6,240 x 5,120 x 15,360 from
// 8-bit rows 376 to 398. Workgroups that stay for several tiles and load the next one's
// first stages during the epilogue took as long or up to 3% longer, with half the LDS for
// their epilogue.
template <int TF, int NT, int SW, int SX, bool kGated, bool kQuant>
__global__ __launch_bounds__(kPThreads, 1) void linear_fp8_kernel(LinearFp8Params p) {
    using T = Fp8Tile<TF, NT, SW, SX>;
    __shared__ __attribute__((aligned(1024))) char smem[T::kSmem];
    constexpr int TO = kGated ? TF / 2 : TF;  // output features of a tile
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave / T::WM, wm = wave % T::WM;

    const int bid = blockIdx.x;
    const bool whole = bid < p.n_full;
    const int rest = p.m_tiles * p.n_tiles - p.n_full;
    const int tile = whole ? xcd_tile(bid, p.n_full) : p.n_full + (bid - p.n_full) % rest;
    const int part = whole ? 0 : (bid - p.n_full) / rest;
    const TileCoord tc = tile_coord(p, tile, TO, T::kTokens);
    const int f0 = tc.f0, m0 = tc.m0;

    const int steps = (p.k + kP8K - 1) / kP8K;
    const int k0 = whole ? 0 : part * steps / p.split, k1 = whole ? steps : (part + 1) * steps / p.split;
    const int chunk = gemm_chunk(wave, lane);
    // Gated: of every 32 rows of the tile the first 16 are value rows, the
    // others the same features' gate rows: waves 0 and 1 load the former, 2 and
    // 3 the latter.
    const int half = kGated ? wave >> 1 : 0;
    const int w_row = (kGated ? 8 * (wave & 1) : 8 * wave) + (lane >> 3), x_row = 8 * wave + (lane >> 3);
    const uint32_t wl = (uint32_t)(w_row * p.w_rs + chunk), xl = (uint32_t)(x_row * p.x_rs + chunk);
    const int rows = min(T::kTokens, p.m - m0);
    // The blocks of w rows: gated the values' and the gates', else the tile's first and,
    // where it has one, second.
    const int first = f0 / kFp8Group;
    const int second = kGated ? p.w_blocks + first : min(first + (TO > kFp8Group ? 1 : 0), p.w_blocks - 1);
    const int w_block = kGated ? (lane >> 4) & 1 : 32 * T::NA * wn / kFp8Group;
    const uint32_t ws_rs = (uint32_t)p.w_scale_rs;
    f32x16 acc[T::NA][T::NB];
#pragma unroll
    for (int a = 0; a < T::NA; ++a)
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            acc[a][b] = f32x16{};
            if constexpr (T::NA * T::NB >= 8) asm volatile("" : "+a"(acc[a][b]));
        }
    // (All K steps at once, but for the tile whose lanes hold the scales of some.)
    constexpr int kMost = kHeldSegs * kSegSteps;
    for (int c0 = k0, c1; c0 < k1; c0 = c1) {
        c1 = T::kScaleRegs ? min(k1, c0 / kSegSteps * kSegSteps + kMost) : k1;
        const bool past = (c1 - 1) * kPRow + chunk >= p.k;
        const GemmRows w{make_rsrc_words((const char*)p.w + ((int64_t)half * p.n + f0) * p.w_rs + c0 * kPRow,
                                         (uint32_t)((min(TO, p.n - f0) - 1) * p.w_rs + p.k)),
                         wl, (uint32_t)((kGated ? 16 : 32) * p.w_rs), past ? 0x80000000u : wl};
        const GemmRows x{make_rsrc_words((const char*)p.x + (int64_t)m0 * p.x_rs + c0 * kPRow, (uint32_t)((rows - 1) * p.x_rs + p.k)),
                         xl, (uint32_t)(32 * p.x_rs), past ? 0x80000000u : xl};
        const GemmScales scales{make_rsrc_words(p.x_scale + (int64_t)m0 * p.x_scale_rs, (uint32_t)(rows * p.x_scale_rs)),
                                make_rsrc_words(p.w_scale, (uint32_t)(kGated ? 2 : 1) * (uint32_t)p.w_blocks * ws_rs),
                                (uint32_t)p.x_scale_rs, {(uint32_t)first * ws_rs, (uint32_t)second * ws_rs}, c0};
        gemm_fp8_k_loop<T, true>(w, x, scales, c1 - c0, smem, lane, wave, wn, wm, w_block, acc);
    }
    if (whole) {
        linear_fp8_epilogue<T, kGated, kQuant>(p, f0, m0, acc, wn, wm, tid, smem);
        return;
    }
    f32x4* const out = (f32x4*)p.sums + (int64_t)(bid - p.n_full) * (4 * T::NA * T::NB * kPThreads) + threadIdx.x;
#pragma unroll
    for (int a = 0; a < T::NA; ++a)
#pragma unroll
        for (int b = 0; b < T::NB; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x16& v = acc[a][b];
                out[((a * T::NB + b) * 4 + g) * kPThreads] = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            }
}

// Workgroup (i, a, 4 b + g or, gated, 2 b + g): group g of blocks (a, b) of every wave
// of split tile i.
template <int TF, int NT, int SW, int SX, bool kGated>
__global__ __launch_bounds__(kPThreads) void linear_fp8_join_kernel(LinearFp8Params p) {
    using T = Fp8Tile<TF, NT, SW, SX>;
    constexpr int kS = kGated ? 2 : 1, kG = 4 / kS, kPiece = 4 * T::NA * T::NB * kPThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave / T::WM, wm = wave % T::WM;
    const int a = blockIdx.y, b = blockIdx.z / kG, g = blockIdx.z % kG, rest = p.m_tiles * p.n_tiles - p.n_full;
    const TileCoord tc = tile_coord(p, p.n_full + (int)blockIdx.x, TF / kS, T::kTokens);
    const int f = tc.f0 + 32 / kS * (T::NA * wn + a) + 8 * g + 4 * (lane >> 5);
    const int m = tc.m0 + 32 * (T::NB * wm + b) + (lane & 31);
    if (f >= p.n || m >= p.m) return;
    const f32x4* const in = (const f32x4*)p.sums + (int64_t)blockIdx.x * kPiece + (a * T::NB + b) * 4 * kPThreads + tid;
    const int64_t step = (int64_t)rest * kPiece;
    f32x4 part[kLinearFp8MaxSplit][kS];
#pragma unroll
    for (int c = 0; c < kLinearFp8MaxSplit; ++c) {
        if (c >= p.split) break;
#pragma unroll
        for (int s = 0; s < kS; ++s) part[c][s] = in[c * step + (g + 2 * s) * kPThreads];
    }
    f32x4 z[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) z[s] = f32x4{};
#pragma unroll
    for (int c = 0; c < kLinearFp8MaxSplit; ++c) {
        if (c >= p.split) break;
#pragma unroll
        for (int s = 0; s < kS; ++s) z[s] += part[c][s];
    }
    finish4<kS>(p, z, m, f);
}

template <int TF, int NT, int SW, int SX, bool kGated, bool kQuant>
hipError_t launch_tile_t(const LinearFp8Params& p, hipStream_t stream) {
    using T = Fp8Tile<TF, NT, SW, SX>;
    const int rest = p.m_tiles * p.n_tiles - p.n_full;
    const dim3 grid((unsigned)(p.n_full + rest * p.split));
    hipLaunchKernelGGL((linear_fp8_kernel<TF, NT, SW, SX, kGated, kQuant>), grid, dim3(kPThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || rest == 0) return e;
    hipLaunchKernelGGL((linear_fp8_join_kernel<TF, NT, SW, SX, kGated>), dim3((unsigned)rest, T::NA, T::NB * (kGated ? 2 : 4)),
                       dim3(kPThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

template <int TF, int NT, int SW, int SX>
hipError_t launch_linear_fp8_tile(const LinearFp8Params& p, hipStream_t stream) {
    if (p.gated) {
        if constexpr (TF / 2 % kFp8Group == 0) {
            if (p.y_scale != nullptr) return launch_tile_t<TF, NT, SW, SX, true, true>(p, stream);
        }
        return launch_tile_t<TF, NT, SW, SX, true, false>(p, stream);
    }
    return p.y_scale != nullptr ? launch_tile_t<TF, NT, SW, SX, false, true>(p, stream) : launch_tile_t<TF, NT, SW, SX, false, false>(p, stream);
}

}  // namespace h3a
