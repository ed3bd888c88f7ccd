// Matrix product with bias, activation, gate and residual in its epilogue
// (gfx950): the MLP and modulation projections of a DiT block.
//
//   z[m, f] = sum_k x[m, k] * w[f, k] (+ bias[f])
//   a[m, f] = act(z[m, f])                            f < n
//   a[m, f] = z[m, f] * act(z[m, n + f])              gated: w has 2 n rows
//   y[m, f] = residual[m, f] + gate[t(m), f] * a[m, f]
// with t(m) = index[m mod n_index], clamped to the table. x, w, residual and y
// are bf16, bias and gate bf16 or fp32; everything between the operands and y
// is fp32, rounded once.
//
// Two forms. From a few dozen tokens on the product is bound by the matrix
// cores and runs on the tiles of gemm_tile.h, whose accumulators the epilogue
// finishes where they lie. With fewer tokens it is bound by reading w once: the
// row form streams it from HBM straight into MFMA operands.
#include "gemm_tile.h"
#include "kernels.h"

namespace h3a {
namespace {

typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

// act(z). silu and the tanh form of GELU are both z * sigmoid(u): 0.5 (1 +
// tanh(v)) = sigmoid(2 v). GELU proper is z * Phi(z), Phi(z) = erfc(-z /
// sqrt 2) / 2, with erfc(x) = t exp(-x^2) 2^P(t), t = 1 / (1 + 0.38 x), x >= 0,
// P the degree-6 polynomial of least maximal error over 0 <= x <= 10 (a relative
// 1.3e-6): the tail of Phi keeps its relative precision, where 1 + erf cancels.
__device__ __forceinline__ float activate(float z, int act) {
    if (act == H3A_ACT_NONE) return z;
    if (act == H3A_ACT_RELU) return z < 0.f ? 0.f : z;  // (NaN stays)
    constexpr float kLog2e = 1.44269504088896f;
    if (act == H3A_ACT_GELU) {
        const float x = fabsf(z) * 0.70710678118654752f;
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.38f, x, 1.0f));
        float p = 0.3967597484588623f;
        p = __builtin_fmaf(p, t, -1.3749288320541382f);
        p = __builtin_fmaf(p, t, 1.3808318376541138f);
        p = __builtin_fmaf(p, t, -0.4088878929615021f);
        p = __builtin_fmaf(p, t, 0.8127332329750061f);
        p = __builtin_fmaf(p, t, 1.4133836030960083f);
        p = __builtin_fmaf(p, t, -2.2198920249938965f);
        const float h = 0.5f * t * fast_exp2(__builtin_fmaf(x * -kLog2e, x, p));
        // (z = -inf: the limit is -0, where the product would be NaN.)
        return z < 0.f ? fmaxf(z, -1e30f) * h : z * (1.0f - h);
    }
    // u = z for silu, 2 sqrt(2 / pi) (z + 0.044715 z^3) for the tanh form
    const float c0 = act == H3A_ACT_SILU ? kLog2e : 1.5957691216057308f * kLog2e;
    const float c1 = act == H3A_ACT_SILU ? 0.f : 0.044715f * 1.5957691216057308f * kLog2e;
    // (Far out the sigmoid is 0 or 1; the bounds keep u finite and -inf at its
    // limit -0. NaN stays.)
    const float zu = __builtin_amdgcn_fmed3f(z, -1e12f, 1e12f);
    const float u = zu * __builtin_fmaf(c1, zu * zu, c0);
    const float s = __builtin_amdgcn_rcpf(1.0f + fast_exp2(-u));
    return (z < -1e12f ? -1e12f : z) * s;
}

__device__ __forceinline__ f32x4 unpack4(const i32x2& raw) {
    return f32x4{__uint_as_float((uint32_t)raw.x << 16), __uint_as_float((uint32_t)raw.x & 0xffff0000u),
                 __uint_as_float((uint32_t)raw.y << 16), __uint_as_float((uint32_t)raw.y & 0xffff0000u)};
}

// Four consecutive values of a bf16 or fp32 row (16-byte aligned rows).
__device__ __forceinline__ f32x4 load4(const void* row, int col, bool f32) {
    if (f32) return *(const f32x4*)((const float*)row + col);
    return unpack4(*(const i32x2*)((const uint16_t*)row + col));
}

__device__ __forceinline__ int64_t gate_row(const LinearParams& p, int m) {
    const int64_t i = m % p.n_index;
    int64_t t = p.index_i64 ? ((const int64_t*)p.index)[i] : (int64_t)((const int32_t*)p.index)[i];
    t = t < 0 ? 0 : t;
    return t >= p.table_rows ? p.table_rows - 1 : t;
}

// y of token m, features f .. f+3, from their sums (gated: z[0] of the values,
// z[1] of the gates).
template <int kS>
__device__ __forceinline__ void finish4(const LinearParams& p, f32x4 (&z)[kS], int m, int f) {
    if (p.bias != nullptr) {
#pragma unroll
        for (int s = 0; s < kS; ++s) z[s] += load4(p.bias, s * p.n + f, p.bias_f32 != 0);
    }
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = activate(z[kS - 1][e], p.act);
        if constexpr (kS == 2) y[e] *= z[0][e];
    }
    if (p.gate != nullptr) y *= load4((const char*)p.gate + gate_row(p, m) * p.gate_rs, f, p.gate_f32 != 0);
    if (p.residual != nullptr) y += unpack4(*(const i32x2*)((const char*)p.residual + m * p.res_rs + 2 * f));
    *(i32x2*)((char*)p.y + m * p.y_rs + 2 * f) = i32x2{(int)pack_bf16x2(y[0], y[1]), (int)pack_bf16x2(y[2], y[3])};
}

// ---------------------------------------------------------------- tiles

// Epilogue of a tile, in two halves of its tokens. Lane l holds, for token block b
// (token 16 (NB wm + b) + (l & 15)) and row block a of w, tile rows 16 (NA wn + a)
// + 4 (l >> 4) + e; gated, block 2 a' is of the values and 2 a' + 1 of their gates.
// The sums of a half go through LDS (the idle stages) in fp32: row r of the half,
// its 16-byte chunk c at c ^ (r & 7), free of bank conflicts on both sides. Then a
// thread takes four features of a token at a time, neighbouring lanes along the
// row, so that residual, gate and result move in whole lines. A batch of tokens'
// residuals is loaded ahead of the one before it.
// (Finished in the accumulators' layout instead, every block with its own copy of
// the activations, a tile's code passes the instruction cache: 6,240 x 5,120 x
// 15,360 without an epilogue took 848 us, then 709 on the same card.)
template <typename T, bool kGated>
__device__ __forceinline__ void linear_epilogue(const LinearParams& p, int f0, int m0, const f32x4 (&acc)[T::NA][T::NB],
                                                int wn, int wm, int tid, char* smem) {
    constexpr int kS = kGated ? 2 : 1, NBh = T::NB / 2;
    constexpr int kWRows = 16 * T::NA * T::WN, TO = kWRows / kS, kRowBytes = kWRows * 4;
    constexpr int kCols = TO / 4, kRows = kPThreads / kCols;      // threads of a row, rows at a time
    constexpr int kIts = T::kTokens / 2 / kRows;                  // of a half
    constexpr int kBatch = kIts % 8 == 0 ? 8 : kIts;
    static_assert(T::NB % 2 == 0 && kIts % kBatch == 0 && kBatch <= 12, "batches of a half");
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int r0 = tid / kCols, c = tid % kCols, f = f0 + 4 * c;
    const bool in = f < p.n;
    const int fc = in ? f : 0;  // (features past the end read the first ones' and store nothing)
    f32x4 bias[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) bias[s] = p.bias != nullptr ? load4(p.bias, s * p.n + fc, p.bias_f32 != 0) : f32x4{};
    lds_char* const buf = (lds_char*)smem;
    // (Gated, the row is the values of its features, then their gates.)
    lds_char* const wr = buf + ((wm * NBh) * 16 + (lane & 15)) * kRowBytes;
    const int sw = lane & 7;
    auto half = [&](auto h_c) __attribute__((always_inline)) {
        constexpr int h = decltype(h_c)::value, b0 = h * NBh;
        // Token of row r of this half (rows of the two wave rows side by side).
        auto token = [&](int i) __attribute__((always_inline)) {
            const int r = r0 + kRows * i;
            return r + 16 * NBh * ((T::WM == 2 ? r / (16 * NBh) : 0) + h);
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
        if constexpr (h > 0) __syncthreads();  // the first half's rows have been read
#pragma unroll
        for (int b = 0; b < NBh; ++b)
#pragma unroll
            for (int a = 0; a < T::NA; ++a) {
                const int x = (T::NA / kS) * wn + a / kS, chunk = (kGated ? (a & 1) * kCols : 0) + 4 * x + (lane >> 4);
                *(lds_f32x4*)(wr + b * 16 * kRowBytes + ((chunk ^ sw) << 4)) = acc[a][b0 + b];
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
                    if (in && m0 + t < p.m)
                        __builtin_nontemporal_store(i32x2{(int)pack_bf16x2(y[0], y[1]), (int)pack_bf16x2(y[2], y[3])},
                                                    (i32x2*)((char*)p.y + (int64_t)(m0 + t) * p.y_rs + 2 * f));
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
    half(std::integral_constant<int, 0>{});
    half(std::integral_constant<int, 1>{});
}

// Tile `tile` of groups of p.group_m token tiles x every feature tile, token
// tile fastest.
struct TileCoord {
    int f0, m0;
};
__device__ __forceinline__ TileCoord tile_coord(const LinearParams& p, int tile, int to, int tokens) {
    const int in_group = p.group_m * p.n_tiles, first_m = (tile / in_group) * p.group_m;
    const int group_m = min(p.m_tiles - first_m, p.group_m);
    return TileCoord{(tile % in_group) / group_m * to, (first_m + (tile % in_group) % group_m) * tokens};
}

// Workgroups [0, n_full) run whole tiles. The others run the tiles after them in
// `split` pieces along K, for a last round that would leave most CUs idle; their
// sums, in fp32, go to the workspace as the lanes hold them, and
// linear_join_kernel adds a tile's pieces in order.
template <int TF, int NT, int SW, int SX, bool kGated>
__global__ __launch_bounds__(kPThreads, 1) void linear_kernel(LinearParams p) {
    using T = Tile<TF, NT, SW, SX>;
    __shared__ __attribute__((aligned(1024))) char smem[T::kStages > T::kOutBytes ? T::kStages : T::kOutBytes];
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

    // The last K step's lanes past the reduction hold an offset that no record
    // covers (records are under 2^31 bytes).
    const int steps = (p.k + kPK - 1) / kPK;
    const int k0 = whole ? 0 : part * steps / p.split, k1 = whole ? steps : (part + 1) * steps / p.split;
    const int chunk = gemm_chunk(wave, lane);
    const bool past = (k1 - 1) * kPRow + chunk >= p.k * 2;
    // Gated: of every 32 rows of the tile the first 16 are value rows, the
    // others the same features' gate rows: waves 0 and 1 load the former, 2 and
    // 3 the latter.
    const int half = kGated ? wave >> 1 : 0;
    const int w_row = (kGated ? 8 * (wave & 1) : 8 * wave) + (lane >> 3), x_row = 8 * wave + (lane >> 3);
    const uint32_t wl = (uint32_t)(w_row * p.w_rs + chunk), xl = (uint32_t)(x_row * p.x_rs + chunk);
    const GemmRows w{make_rsrc_words((const char*)p.w + ((int64_t)half * p.n + f0) * p.w_rs + k0 * kPRow,
                                     (uint32_t)((min(TO, p.n - f0) - 1) * p.w_rs + p.k * 2)),
                     wl, (uint32_t)((kGated ? 16 : 32) * p.w_rs), past ? 0x80000000u : wl};
    const GemmRows x{make_rsrc_words((const char*)p.x + (int64_t)m0 * p.x_rs + k0 * kPRow,
                                     (uint32_t)((min(T::kTokens, p.m - m0) - 1) * p.x_rs + p.k * 2)),
                     xl, (uint32_t)(32 * p.x_rs), past ? 0x80000000u : xl};
    f32x4 acc[T::NA][T::NB];
    gemm_k_loop<T, true>(w, x, k1 - k0, smem, lane, wave, wn, wm, acc);
    if (whole) {
        linear_epilogue<T, kGated>(p, f0, m0, acc, wn, wm, tid, smem);
        return;
    }
    f32x4* const out = (f32x4*)p.ws + (int64_t)(bid - p.n_full) * (T::NA * T::NB * kPThreads) + threadIdx.x;
#pragma unroll
    for (int a = 0; a < T::NA; ++a)
#pragma unroll
        for (int b = 0; b < T::NB; ++b) out[(a * T::NB + b) * kPThreads] = acc[a][b];
}

// Workgroup (i, a, b): blocks (a, b) of every wave of split tile i, the pieces' sums
// all in flight before they are added. (All token blocks in one workgroup: 24 us
// for 13 tiles of 256 x 256 in 8 pieces, now 7.)
constexpr int kMaxSplit = 8;

template <int TF, int NT, int SW, int SX, bool kGated>
__global__ __launch_bounds__(kPThreads) void linear_join_kernel(LinearParams p) {
    using T = Tile<TF, NT, SW, SX>;
    constexpr int kS = kGated ? 2 : 1, NF = T::NA / kS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave / T::WM, wm = wave % T::WM;
    const int a = blockIdx.y, rest = p.m_tiles * p.n_tiles - p.n_full;
    const TileCoord tc = tile_coord(p, p.n_full + (int)blockIdx.x, 16 * NF * T::WN, T::kTokens);
    const int f = tc.f0 + 16 * (NF * wn + a) + 4 * (lane >> 4);
    const f32x4* const in = (const f32x4*)p.ws + (int64_t)blockIdx.x * (T::NA * T::NB * kPThreads) + tid;
    const int64_t step = (int64_t)rest * (T::NA * T::NB * kPThreads);
    const int b = blockIdx.z, m = tc.m0 + 16 * (T::NB * wm + b) + (lane & 15);
    if (f >= p.n || m >= p.m) return;
    f32x4 part[kMaxSplit][kS];
#pragma unroll
    for (int c = 0; c < kMaxSplit; ++c) {
        if (c >= p.split) break;
#pragma unroll
        for (int s = 0; s < kS; ++s) part[c][s] = in[c * step + ((kS * a + s) * T::NB + b) * kPThreads];
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

template <int TF, int NT, int SW, int SX, bool kGated>
hipError_t launch_tile_t(const LinearParams& p, hipStream_t stream) {
    using T = Tile<TF, NT, SW, SX>;
    const int rest = p.m_tiles * p.n_tiles - p.n_full;
    const dim3 grid((unsigned)(p.n_full + rest * p.split));
    hipLaunchKernelGGL((linear_kernel<TF, NT, SW, SX, kGated>), grid, dim3(kPThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || rest == 0) return e;
    hipLaunchKernelGGL((linear_join_kernel<TF, NT, SW, SX, kGated>), dim3((unsigned)rest, T::NA / (kGated ? 2 : 1), T::NB),
                       dim3(kPThreads), 0, stream, p);
    return hipGetLastError();
}

template <int TF, int NT, int SW, int SX>
hipError_t launch_tile(const LinearParams& p, hipStream_t stream) {
    return p.gated ? launch_tile_t<TF, NT, SW, SX, true>(p, stream) : launch_tile_t<TF, NT, SW, SX, false>(p, stream);
}

// The tile shapes, with the time of a K step of 64 with all CUs busy and a tile's
// fixed part (launch, first loads, epilogue). Fitted to graph replays of 25 sizes
// (40 to 12,480 tokens, 1,024 to 32,256 features, k 1,024 to 14,336) in every shape
// and split; the choice by them takes 0.3% longer than the best of all, in the
// mean. (Up to 128 features a K step is bound by what the L2s deliver: 32 KB per
// CU at 128 x 128, 21 TB/s over the chip.)
struct Shape {
    int tf, nt;
    float step_us, fixed_us;
    hipError_t (*launch)(const LinearParams&, hipStream_t);
};
constexpr Shape kShapes[] = {
    {256, 16, 1.36f, 13.3f, launch_tile<256, 16, 3, 2>}, {256, 12, 1.05f, 11.8f, launch_tile<256, 12, 3, 2>},
    {256, 8, 0.80f, 9.3f, launch_tile<256, 8, 4, 2>},    {128, 8, 0.50f, 5.9f, launch_tile<128, 8, 6, 4>},
    {128, 6, 0.40f, 5.9f, launch_tile<128, 6, 7, 4>},    {128, 4, 0.34f, 5.3f, launch_tile<128, 4, 7, 5>},
    {128, 2, 0.27f, 3.6f, launch_tile<128, 2, 8, 6>},
};
constexpr float kIdleGain = 0.36f;  // of a K step's time, saved as the CUs of a round go idle
// A second launch joins the pieces, over their sums at 0.32 us a MB.
constexpr float kJoinUs = 1.9f, kJoinUsPerByte = 0.32e-6f;
constexpr int kSplits[] = {2, 3, 4, 6, kMaxSplit};
constexpr int kMinPieceSteps = 16;

// ---------------------------------------------------------------- few tokens

// NA blocks of 16 rows of w (gated: half of them the values' gates) x 16 NB
// tokens per workgroup, K split over its waves: wave v takes the 128-byte chunks
// v, v + waves, ... of every row, kU of them in flight, each lane loading the 16
// bytes that it holds of the MFMA operands. w comes from HBM, once; x, a few
// rows, from the caches, once per NA blocks. The waves' partial sums meet in
// LDS, in wave order.
constexpr int kRowsMaxTokens = 32;
constexpr int kRowsForm = -1, kNoForm = -2;  // in place of a tile shape

template <int NA, int NB, bool kGated>
__global__ __launch_bounds__(NA == 1 ? 1024 : 512) void linear_rows_kernel(LinearParams p) {
    constexpr int kS = kGated ? 2 : 1, NF = NA / kS;  // blocks of output features
    constexpr int kU = NA * NB >= 4 ? 1 : 4;
    extern __shared__ f32x4 part[];  // [wave][NA * NB][64]
    const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, l15 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)blockDim.x >> 6;
    const int f0 = (int)blockIdx.x * 16 * NF, m0 = (int)blockIdx.y * 16 * NB;
    const char* wr[NA];
#pragma unroll
    for (int a = 0; a < NA; ++a)
        wr[a] = (const char*)p.w + ((int64_t)(a % kS) * p.n + min(f0 + 16 * (a / kS) + l15, p.n - 1)) * p.w_rs;
    const char* xr[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) xr[b] = (const char*)p.x + (int64_t)min(m0 + 16 * b + l15, p.m - 1) * p.x_rs;
    f32x4 acc[NA][NB];
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{};
    const int bytes = p.k * 2, chunks = (bytes + 127) >> 7;
    for (int c0 = wave; c0 < chunks; c0 += waves * kU) {
        i32x4 w[kU][2][NA], x[kU][2][NB];
        bool in[kU][2];
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = (c0 + u * waves) * 128 + h * 64 + q * 16;
                in[u][h] = at < bytes;
                const int o = in[u][h] ? at : bytes - 16;
#pragma unroll
                for (int a = 0; a < NA; ++a) w[u][h][a] = *(const i32x4*)(wr[a] + o);
#pragma unroll
                for (int b = 0; b < NB; ++b) x[u][h][b] = *(const i32x4*)(xr[b] + o);
            }
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int a = 0; a < NA; ++a) {
                    const i32x4 wv = in[u][h] ? w[u][h][a] : i32x4{};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const i32x4 xv = in[u][h] ? x[u][h][b] : i32x4{};
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv),
                                                                            __builtin_bit_cast(bf16x8, xv), acc[a][b], 0, 0, 0);
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
        finish4<kS>(p, z, m, f);
    }
}

template <int NA, int NB, bool kGated>
hipError_t launch_rows_t(const LinearParams& p, int waves, hipStream_t stream) {
    constexpr int kFeatures = 16 * NA / (kGated ? 2 : 1);
    const dim3 grid((unsigned)((p.n + kFeatures - 1) / kFeatures), (unsigned)((p.m + 16 * NB - 1) / (16 * NB)));
    const size_t lds = (size_t)waves * NA * NB * 1024;
    hipLaunchKernelGGL((linear_rows_kernel<NA, NB, kGated>), grid, dim3(64 * waves), lds, stream, p);
    return hipGetLastError();
}

// Blocks of rows per workgroup: x is read once for each of them, and a launch
// wants a workgroup per CU (us, 1 / 2 / 4 blocks: 16 x 5,376 x 32,256 106 / 83
// / 72; 16 x 5,376 x 14,336 gated - / 78 / 67; 32 x 5,376 x 5,376 36 / 23 / 34;
// 4 x 14,336 x 5,376 46 / 42 / 74). Waves so that 16 per CU share a launch,
// each with a chunk at least.
struct RowsForm {
    int na, waves;
    int64_t groups;  // workgroups
};

RowsForm rows_form(const LinearParams& p, int cus) {
    const int64_t blocks = (int64_t)((p.n + 15) / 16) * (p.gated ? 2 : 1);  // (the tokens are one block of 16 NB)
    RowsForm f;
    f.na = blocks >= 4ll * cus ? 4 : blocks >= cus || p.gated ? 2 : 1;
    f.groups = (blocks + f.na - 1) / f.na;
    f.waves = 4;
    while (f.waves < (f.na == 1 ? 16 : 8) && f.groups * f.waves < 16ll * cus && f.waves * 128 < p.k * 2) f.waves *= 2;
    return f;
}

template <int NB>
hipError_t launch_rows(const LinearParams& p, int cus, hipStream_t stream) {
    const RowsForm f = rows_form(p, cus);
    if (p.gated) return f.na == 4 ? launch_rows_t<4, NB, true>(p, f.waves, stream) : launch_rows_t<2, NB, true>(p, f.waves, stream);
    return f.na == 4   ? launch_rows_t<4, NB, false>(p, f.waves, stream)
           : f.na == 2 ? launch_rows_t<2, NB, false>(p, f.waves, stream)
                       : launch_rows_t<1, NB, false>(p, f.waves, stream);
}

}  // namespace

void plan_linear(LinearParams& p, int cus, int64_t* workspace) {
    if (cus <= 0) cus = 256;
    *workspace = 0;
    p.shape = kNoForm;
    if (p.m <= kRowsMaxTokens) {
        const RowsForm f = rows_form(p, cus);
        if (f.groups * 64 * f.waves <= UINT32_MAX) p.shape = kRowsForm;  // work items of a launch
        return;
    }
    const int steps = (p.k + kPK - 1) / kPK;
    float best_us = 0.f;
    for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
        const Shape& s = kShapes[i];
        const int to = p.gated ? s.tf / 2 : s.tf, tokens = 16 * s.nt;
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
        // The last round in pieces, at most one per CU (of the smallest tiles none:
        // they serve short reductions).
        for (const int n : kSplits) {
            if (rest == 0 || rest * n > cus || steps / n < kMinPieceSteps || s.nt == 2) break;
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
        // Tokens of a group of the tile order: each group reads all of w from HBM
        // (us at 256 tokens a tile, groups of 2 / 4 / 6 / 8 / 12 / 25: 6,240 x 5,376 x
        // 28,672 1,461 / 1,397 / 1,361 / 1,379 / 1,374 / 1,407; 6,240 x 14,336 x
        // 5,376 720 / 712 / 711 / 711 / 713 / 737; of 2 / 3 / 4 / 6 / 8: 24,960 x
        // 5,120 x 15,360 2,826 / 2,799 / 2,838 / 2,986 / 2,997).
        const int group_tokens = p.m <= 2048 ? 2048 : p.m <= 16384 ? 1536 : 768;
        p.group_m = (int32_t)(group_tokens / tokens < m_tiles ? group_tokens / tokens : m_tiles);
        p.split = split;
        p.n_full = (int32_t)(split > 1 ? full : tiles);
        *workspace = split > 1 ? rest * split * (int64_t)(s.tf * tokens * 4) : 0;
    }
}

hipError_t launch_linear(const LinearParams& p, int cus, hipStream_t stream) {
    if (p.shape == kNoForm) return hipErrorInvalidConfiguration;
    if (p.shape >= 0) return kShapes[p.shape].launch(p, stream);
    if (p.m <= 16) return launch_rows<1>(p, cus, stream);
    return launch_rows<2>(p, cus, stream);
}

int linear_max_tile() { return 256; }

}  // namespace h3a
