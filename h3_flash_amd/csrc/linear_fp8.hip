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
// Two forms, as there: tiles (gemm_fp8_tile.h) from a few dozen tokens on, and a form
// that streams w once for fewer. bf16 rows are rounded to 8 bits by a launch of their
// own before the tiles, and as they come in by the other form.
#include "fp8_util.h"
#include "gemm_fp8_tile.h"
#include "kernels.h"
#include "linear_util.h"

namespace h3a {
namespace {

typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

// ---------------------------------------------------------------- few tokens

// linear.hip's row form on bytes: NA blocks of 16 rows of w x 16 NB tokens per
// workgroup, K split over its waves by chunks of 128 bytes, a scale's block each. Lane
// l holds of row l & 15 the 16-byte pieces l >> 4 and 4 + (l >> 4) of a chunk, of w and
// of x alike (which of the chunk's K they are does not matter to a sum over all).
// bf16 rows of x are rounded to 8 bits as they come in: the four lanes of a row hold a
// whole group.
constexpr int kRowsMaxTokens = 32;
constexpr int kRowsForm = -1, kNoForm = -2;  // in place of a tile shape

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

// ---------------------------------------------------------------- tiles

// Maximum over aligned groups of 32 lanes; all lanes must be active.
__device__ __forceinline__ uint32_t group32_max(uint32_t v) {
    v = group16_max(v);
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

// Epilogue of a tile, linear.hip's with this product's layout: lane l holds, for token
// block b (token 32 (NB wm + b) + (l & 31)), row block a of w and group g, tile rows
// 32 (NA wn + a) + 8g + 4 (l >> 5) + e; gated, groups 0 and 1 of a block are its 16
// values and 2 and 3 their gates. kPass blocks of tokens at a time go through LDS (the
// idle stages) in fp32, row r's 16-byte chunk c at c ^ (r & 7), and a thread then takes
// four features of a token at a time. In 8 bits, 32 neighbouring threads hold a group
// of 128 features.
template <typename T, bool kGated, bool kQuant>
__device__ __forceinline__ void linear_fp8_epilogue(const LinearFp8Params& p, int f0, int m0, const f32x16 (&acc)[T::NA][T::NB],
                                                    int wn, int wm, int tid, char* smem) {
    constexpr int kS = kGated ? 2 : 1, TO = T::kTF / kS, kRowBytes = T::kTF * 4;
    constexpr int kCols = TO / 4, kRows = kPThreads / kCols;  // threads of a row, rows at a time
    constexpr int kRowsPass = 32 * T::kPass, kIts = kRowsPass * T::WM / kRows;
    constexpr int kBatch = kIts % 8 == 0 ? 8 : kIts;
    static_assert(kIts % kBatch == 0 && kBatch <= 12, "batches of a pass");
    static_assert(!kQuant || TO % kFp8Group == 0, "whole groups of features");
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int r0 = tid / kCols, c = tid % kCols, f = f0 + 4 * c;
    const bool in = f < p.n;
    const int fc = in ? f : 0;  // (features past the end read the first ones' and store nothing)
    f32x4 bias[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) bias[s] = p.bias != nullptr ? load4(p.bias, s * p.n + fc, p.bias_f32 != 0) : f32x4{};
    lds_char* const buf = (lds_char*)smem;
    lds_char* const wr = buf + (wm * kRowsPass + (lane & 31)) * kRowBytes;
    const int sw = lane & 7;
    auto pass = [&](auto h_c) __attribute__((always_inline)) {
        constexpr int h = decltype(h_c)::value, b0 = h * T::kPass;
        // Token of row r of this pass (rows of the two wave rows side by side).
        auto token = [&](int i) __attribute__((always_inline)) {
            const int r = r0 + kRows * i, w = T::WM == 2 ? r / kRowsPass : 0;
            return r + w * (32 * T::NB - kRowsPass) + 32 * b0;
        };
        struct Batch {
            i32x2 res[kBatch];
            int64_t gate[kBatch];
        };
        auto load_batch = [&](Batch& q, int i0) __attribute__((always_inline)) {
            if (p.residual != nullptr) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    q.res[i] = *(const i32x2*)((const char*)p.residual + (int64_t)min(m0 + token(i0 + i), p.m - 1) * p.res_rs + 2 * fc);
            }
            if (p.gate != nullptr) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) q.gate[i] = gate_row(p, min(m0 + token(i0 + i), p.m - 1)) * p.gate_rs;
            }
        };
        Batch cur;
        load_batch(cur, 0);
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
        auto rows = [&](auto act) __attribute__((always_inline)) {
            for (int i0 = 0; i0 < kIts; i0 += kBatch) {
                Batch next;
                if (i0 + kBatch < kIts) load_batch(next, i0 + kBatch);
                f32x4 g[kBatch];
                if (p.gate != nullptr) {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) g[i] = load4((const char*)p.gate + cur.gate[i], fc, p.gate_f32 != 0);
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int t = token(i0 + i), r = r0 + kRows * (i0 + i);
                    f32x4 z[kS];
#pragma unroll
                    for (int s = 0; s < kS; ++s)
                        z[s] = *(const lds_f32x4*)(buf + r * kRowBytes + (((s * kCols + c) ^ (r & 7)) << 4)) + bias[s];
                    f32x4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = act(z[kS - 1][e]);
                        if constexpr (kGated) y[e] *= z[0][e];
                    }
                    if (p.gate != nullptr) y *= g[i];
                    if (p.residual != nullptr) y += unpack4(cur.res[i]);
                    const bool live = in && m0 + t < p.m;
                    if constexpr (kQuant) {
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
                        const int s = fp8_exponent(group32_max(in ? top : 0));
                        const float inv = fp8_inverse(s);
                        if (live) {
                            __builtin_nontemporal_store(fp8x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                                                        (int*)((char*)p.y + (int64_t)(m0 + t) * p.y_rs + f));
                            if ((c & 31) == 0) p.y_scale[(int64_t)(m0 + t) * p.y_scale_rs + f / kFp8Group] = (uint8_t)s;
                        }
                    } else if (live) {
                        __builtin_nontemporal_store(i32x2{(int)pack_bf16x2(y[0], y[1]), (int)pack_bf16x2(y[2], y[3])},
                                                    (i32x2*)((char*)p.y + (int64_t)(m0 + t) * p.y_rs + 2 * f));
                    }
                }
                cur = next;
            }
        };
        // One copy of the loop per activation: its code is what runs.
        if (p.act == H3A_ACT_NONE)
            rows([](float z) { return z; });
        else if (p.act == H3A_ACT_RELU)
            rows([](float z) { return activate(z, H3A_ACT_RELU); });
        else if (p.act == H3A_ACT_GELU)
            rows([](float z) { return activate(z, H3A_ACT_GELU); });
        else
            rows([&](float z) { return activate(z, p.act == H3A_ACT_SILU ? H3A_ACT_SILU : H3A_ACT_GELU_TANH); });
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
    const bool past = (k1 - 1) * kPRow + chunk >= p.k;
    // Gated: of every 32 rows of the tile the first 16 are value rows, the
    // others the same features' gate rows: waves 0 and 1 load the former, 2 and
    // 3 the latter.
    const int half = kGated ? wave >> 1 : 0;
    const int w_row = (kGated ? 8 * (wave & 1) : 8 * wave) + (lane >> 3), x_row = 8 * wave + (lane >> 3);
    const uint32_t wl = (uint32_t)(w_row * p.w_rs + chunk), xl = (uint32_t)(x_row * p.x_rs + chunk);
    const int rows = min(T::kTokens, p.m - m0);
    const GemmRows w{make_rsrc_words((const char*)p.w + ((int64_t)half * p.n + f0) * p.w_rs + k0 * kPRow,
                                     (uint32_t)((min(TO, p.n - f0) - 1) * p.w_rs + p.k)),
                     wl, (uint32_t)((kGated ? 16 : 32) * p.w_rs), past ? 0x80000000u : wl};
    const GemmRows x{make_rsrc_words((const char*)p.x + (int64_t)m0 * p.x_rs + k0 * kPRow, (uint32_t)((rows - 1) * p.x_rs + p.k)),
                     xl, (uint32_t)(32 * p.x_rs), past ? 0x80000000u : xl};
    // The blocks of w rows: gated the values' and the gates', else the tile's first and,
    // where it has one, second.
    const int first = f0 / kFp8Group;
    const int second = kGated ? p.w_blocks + first : min(first + (TO > kFp8Group ? 1 : 0), p.w_blocks - 1);
    const uint32_t ws_rs = (uint32_t)p.w_scale_rs;
    const GemmScales scales{make_rsrc_words(p.x_scale + (int64_t)m0 * p.x_scale_rs, (uint32_t)(rows * p.x_scale_rs)),
                            make_rsrc_words(p.w_scale, (uint32_t)(kGated ? 2 : 1) * (uint32_t)p.w_blocks * ws_rs),
                            (uint32_t)p.x_scale_rs, {(uint32_t)first * ws_rs, (uint32_t)second * ws_rs}, k0};
    const int w_block = kGated ? (lane >> 4) & 1 : 32 * T::NA * wn / kFp8Group;
    f32x16 acc[T::NA][T::NB];
    gemm_fp8_k_loop<T, true>(w, x, scales, k1 - k0, smem, lane, wave, wn, wm, w_block, acc);
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
constexpr int kMaxSplit = 8;

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
    f32x4 part[kMaxSplit][kS];
#pragma unroll
    for (int c = 0; c < kMaxSplit; ++c) {
        if (c >= p.split) break;
#pragma unroll
        for (int s = 0; s < kS; ++s) part[c][s] = in[c * step + (g + 2 * s) * kPThreads];
    }
    f32x4 z[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) z[s] = f32x4{};
#pragma unroll
    for (int c = 0; c < kMaxSplit; ++c) {
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

template <int TF, int NT, int SW, int SX>
hipError_t launch_tile(const LinearFp8Params& p, hipStream_t stream) {
    if (p.gated) {
        if constexpr (TF / 2 % kFp8Group == 0) {
            if (p.y_scale != nullptr) return launch_tile_t<TF, NT, SW, SX, true, true>(p, stream);
        }
        return launch_tile_t<TF, NT, SW, SX, true, false>(p, stream);
    }
    return p.y_scale != nullptr ? launch_tile_t<TF, NT, SW, SX, false, true>(p, stream) : launch_tile_t<TF, NT, SW, SX, false, false>(p, stream);
}

// The tile shapes, with the time of a K step of 128 with all CUs busy and a tile's
// fixed part (launch, first loads, epilogue).
struct Shape {
    int tf, nt;
    float step_us, fixed_us;
    hipError_t (*launch)(const LinearFp8Params&, hipStream_t);
};
constexpr Shape kShapes[] = {
    {256, 12, 1.05f, 11.8f, launch_tile<256, 12, 3, 2>}, {256, 8, 0.80f, 9.3f, launch_tile<256, 8, 3, 2>},
    {128, 8, 0.50f, 5.9f, launch_tile<128, 8, 5, 4>},    {128, 6, 0.40f, 5.9f, launch_tile<128, 6, 6, 4>},
    {128, 4, 0.34f, 5.3f, launch_tile<128, 4, 6, 5>},    {128, 2, 0.27f, 3.6f, launch_tile<128, 2, 8, 6>},
};
constexpr float kIdleGain = 0.36f;  // of a K step's time, saved as the CUs of a round go idle
// A second launch joins the pieces, over their sums at 0.32 us a MB.
constexpr float kJoinUs = 1.9f, kJoinUsPerByte = 0.32e-6f;
constexpr int kSplits[] = {2, 3, 4, 6, kMaxSplit};
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
    if (p.m <= kRowsMaxTokens) {
        const RowsForm f = rows_form(p, cus);
        if (f.groups * 64 * f.waves <= UINT32_MAX) p.shape = kRowsForm;  // work items of a launch
        if (p.y_scale != nullptr) *required = *workspace = 4 * (int64_t)p.m * p.n;
        return;
    }
    if (p.x_scale == nullptr) {
        *required = rounded_x(p).bytes;
        if ((int64_t)p.m * ((p.k + kFp8Group - 1) / kFp8Group) >= (int64_t)1 << 30) return;  // as h3a_quantize_fp8
    }
    const int steps = (p.k + kP8K - 1) / kP8K;
    float best_us = 0.f;
    for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
        const Shape& s = kShapes[i];
        const int to = p.gated ? s.tf / 2 : s.tf, tokens = 16 * s.nt;
        if (p.y_scale != nullptr && to % kFp8Group != 0) continue;  // a group in two tiles
        const int64_t n_tiles = (p.n + to - 1) / to, m_tiles = (p.m + tokens - 1) / tokens, tiles = n_tiles * m_tiles;
        if (tiles * kPThreads > UINT32_MAX) continue;  // work items of a launch
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
        // workgroups do not hold).
        for (const int n : kSplits) {
            if (rest == 0 || rest * n > cus || steps / n < kMinPieceSteps || s.nt == 2 || p.y_scale != nullptr) break;
            const float cut = (float)(full / cus) * tile_us + last_us(n) + kJoinUs + (float)(rest * n * s.tf * tokens * 4) * kJoinUsPerByte;
            if (cut < us) {
                us = cut;
                split = n;
            }
        }
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
