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

// ---------------------------------------------------------------- tiles

// Epilogue of a tile: TO output features (TF, or gated TF / 2) x kTokens.
// Lane l holds, for token block b (token 16 (NB wm + b) + (l & 15)) and row
// block a of w, tile rows 16 (NA wn + a) + 4 (l >> 4) + e; gated, block 2 a' is
// of the values and 2 a' + 1 of their gates, so that both lie in one lane. The
// residual is read in that layout, all of it ahead of its use (one latency for
// the tile), the gate rows, shared by neighbouring tokens, a block ahead from
// cache. The rounded rows go through LDS (the idle stages): token t's 16-byte
// chunk c at c ^ (t & 7), which leaves both sides free of bank conflicts, and
// out in whole lines.
template <typename T, bool kGated>
__device__ __forceinline__ void linear_epilogue(const LinearParams& p, int f0, int m0, const f32x4 (&acc)[T::NA][T::NB],
                                                int wn, int wm, int tid, char* smem) {
    constexpr int kS = kGated ? 2 : 1, NF = T::NA / kS, TO = 16 * NF * T::WN, kRowBytes = TO * 2;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, q = lane >> 4, l15 = lane & 15;
    const int f_wave = 16 * NF * wn + 4 * q;  // first of the lane's features in the tile
    lds_char* const out = (lds_char*)smem;
    // Tokens and features past the end read the last token's and the first
    // features' values; their results are not stored.
    int m[T::NB];
#pragma unroll
    for (int b = 0; b < T::NB; ++b) m[b] = min(m0 + 16 * (T::NB * wm + b) + l15, p.m - 1);
    int f[NF];
#pragma unroll
    for (int a = 0; a < NF; ++a) f[a] = f0 + f_wave + 16 * a < p.n ? f0 + f_wave + 16 * a : 4 * (q & 1);
    i32x2 res[NF][T::NB];
    if (p.residual != nullptr) {
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            const uint16_t* const row = (const uint16_t*)((const char*)p.residual + m[b] * p.res_rs);
#pragma unroll
            for (int a = 0; a < NF; ++a) res[a][b] = __builtin_nontemporal_load((const i32x2*)(row + f[a]));
        }
    } else {
#pragma unroll
        for (int a = 0; a < NF; ++a)
#pragma unroll
            for (int b = 0; b < T::NB; ++b) res[a][b] = i32x2{(int)0x80008000, (int)0x80008000};  // -0: y = a as it is
    }
    const char* gate[T::NB];
    if (p.gate != nullptr) {
#pragma unroll
        for (int b = 0; b < T::NB; ++b) gate[b] = (const char*)p.gate + gate_row(p, m[b]) * p.gate_rs;
    }
    const bool bf = p.bias_f32 != 0, gf = p.gate_f32 != 0;
#pragma unroll
    for (int a = 0; a < NF; ++a) {
        f32x4 bias0{}, bias1{};
        if (p.bias != nullptr) {
            bias0 = load4(p.bias, f[a], bf);
            if constexpr (kGated) bias1 = load4(p.bias, p.n + f[a], bf);
        }
        f32x4 g[T::NB];
        if (p.gate != nullptr) {
#pragma unroll
            for (int b = 0; b < T::NB; ++b) g[b] = load4(gate[b], f[a], gf);
        } else {
#pragma unroll
            for (int b = 0; b < T::NB; ++b) g[b] = f32x4{1.f, 1.f, 1.f, 1.f};
        }
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            f32x4 z = acc[kS * a][b], r = unpack4(res[a][b]), y;
            if constexpr (kGated) {
                const f32x4 u = acc[2 * a + 1][b];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (z[e] + bias0[e]) * activate(u[e] + bias1[e], p.act);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = activate(z[e] + bias0[e], p.act);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(g[b][e], y[e], r[e]);
            const int t = 16 * (T::NB * wm + b) + l15, c = (f_wave + 16 * a) >> 3;
            *(lds_i32x2*)(out + t * kRowBytes + ((c ^ (t & 7)) << 4) + (q & 1) * 8) =
                i32x2{(int)pack_bf16x2(y[0], y[1]), (int)pack_bf16x2(y[2], y[3])};
        }
    }
    __syncthreads();
    constexpr int kChunks = TO / 8;  // 16-byte chunks of a row
    const int c = tid % kChunks, tokens = min(T::kTokens, p.m - m0);
    if (f0 + 8 * c >= p.n) return;
    char* const yb = (char*)p.y + (int64_t)m0 * p.y_rs + (int64_t)(f0 + 8 * c) * 2;
#pragma unroll 4
    for (int t = tid / kChunks; t < tokens; t += kPThreads / kChunks)
        __builtin_nontemporal_store(*(const lds_i32x4*)(out + t * kRowBytes + ((c ^ (t & 7)) << 4)), (i32x4*)(yb + t * p.y_rs));
}

template <int TF, int NT, int SW, int SX, bool kGated>
__global__ __launch_bounds__(kPThreads, 1) void linear_kernel(LinearParams p) {
    using T = Tile<TF, NT, SW, SX>;
    __shared__ __attribute__((aligned(1024))) char smem[T::kStages > T::kOutBytes ? T::kStages : T::kOutBytes];
    constexpr int TO = kGated ? TF / 2 : TF;  // output features of a tile
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave / T::WM, wm = wave % T::WM;

    // Groups of p.group_m token tiles x every feature tile, token tile fastest.
    const int tile = xcd_tile(blockIdx.x, p.m_tiles * p.n_tiles);
    const int in_group = p.group_m * p.n_tiles, first_m = (tile / in_group) * p.group_m;
    const int group_m = min(p.m_tiles - first_m, p.group_m);
    const int m0 = (first_m + (tile % in_group) % group_m) * T::kTokens, f0 = (tile % in_group) / group_m * TO;

    // The last K step's lanes past the reduction hold an offset that no record
    // covers (records are under 2^31 bytes).
    const int nk = (p.k + kPK - 1) / kPK;
    const int chunk = gemm_chunk(wave, lane);
    const bool past = (nk - 1) * kPRow + chunk >= p.k * 2;
    // Gated: of every 32 rows of the tile the first 16 are value rows, the
    // others the same features' gate rows: waves 0 and 1 load the former, 2 and
    // 3 the latter.
    const int part = kGated ? wave >> 1 : 0;
    const int w_row = (kGated ? 8 * (wave & 1) : 8 * wave) + (lane >> 3), x_row = 8 * wave + (lane >> 3);
    const uint32_t wl = (uint32_t)(w_row * p.w_rs + chunk), xl = (uint32_t)(x_row * p.x_rs + chunk);
    const GemmRows w{make_rsrc_words((const char*)p.w + ((int64_t)part * p.n + f0) * p.w_rs,
                                     (uint32_t)((min(TO, p.n - f0) - 1) * p.w_rs + p.k * 2)),
                     wl, (uint32_t)((kGated ? 16 : 32) * p.w_rs), past ? 0x80000000u : wl};
    const GemmRows x{make_rsrc_words((const char*)p.x + (int64_t)m0 * p.x_rs,
                                     (uint32_t)((min(T::kTokens, p.m - m0) - 1) * p.x_rs + p.k * 2)),
                     xl, (uint32_t)(32 * p.x_rs), past ? 0x80000000u : xl};
    f32x4 acc[T::NA][T::NB];
    gemm_k_loop<T, true>(w, x, nk, smem, lane, wave, wn, wm, acc);
    linear_epilogue<T, kGated>(p, f0, m0, acc, wn, wm, tid, smem);
}

template <int TF, int NT, int SW, int SX>
hipError_t launch_tile(LinearParams& p, hipStream_t stream) {
    const int to = p.gated ? TF / 2 : TF;
    p.m_tiles = (p.m + 16 * NT - 1) / (16 * NT);
    p.n_tiles = (p.n + to - 1) / to;
    const int group_tokens = p.m <= 2048 ? 2048 : p.m <= 16384 ? 1024 : 768;
    p.group_m = group_tokens / (16 * NT) < p.m_tiles ? group_tokens / (16 * NT) : p.m_tiles;
    const dim3 grid((unsigned)(p.m_tiles * p.n_tiles));
    if (p.gated)
        hipLaunchKernelGGL((linear_kernel<TF, NT, SW, SX, true>), grid, dim3(kPThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((linear_kernel<TF, NT, SW, SX, false>), grid, dim3(kPThreads), 0, stream, p);
    return hipGetLastError();
}

struct Shape {
    int tf, nt;
    float step_us;  // of a K step of 64 when most CUs run one
    hipError_t (*launch)(LinearParams&, hipStream_t);
};
constexpr Shape kShapes[] = {
    {256, 16, 1.33f, launch_tile<256, 16, 3, 2>}, {256, 12, 1.07f, launch_tile<256, 12, 3, 2>},
    {256, 8, 0.78f, launch_tile<256, 8, 4, 2>},   {128, 8, 0.49f, launch_tile<128, 8, 6, 4>},
    {128, 4, 0.33f, launch_tile<128, 4, 7, 5>},
};

const Shape* pick_shape(const LinearParams& p, int cus) {
    const Shape* best = nullptr;
    float best_us = 0.f;
    for (const Shape& s : kShapes) {
        const int to = p.gated ? s.tf / 2 : s.tf;
        const int64_t tiles = ((int64_t)(p.n + to - 1) / to) * ((p.m + 16 * s.nt - 1) / (16 * s.nt));
        if (tiles >= ((int64_t)1 << 31)) continue;
        const float r = (float)tiles / (float)cus;
        const float rounds = r > 3.f ? r + 0.5f : ceilf(r);
        const float us = rounds * ((float)((p.k + kPK - 1) / kPK) * s.step_us + 3.f + (float)(s.nt * s.tf) / 1024.f);
        if (best == nullptr || us < best_us) {
            best = &s;
            best_us = us;
        }
    }
    return best;
}

// ---------------------------------------------------------------- few tokens

// 16 features (gated: and their gate rows) x 16 NB tokens per workgroup, K split
// over its waves: wave w takes the 128-byte chunks w, w + waves, ... of every
// row, kU of them in flight, each lane loading the 16 bytes that it holds of the
// MFMA operand. w is read once, from HBM; x, a few rows, from the caches. The
// waves' partial sums meet in LDS, in wave order.
template <int NB, bool kGated>
__global__ __launch_bounds__(1024) void linear_rows_kernel(LinearParams p) {
    constexpr int kS = kGated ? 2 : 1, kU = NB + kS == 2 ? 8 : 4;
    extern __shared__ f32x4 part[];  // [wave][kS * NB][64]
    const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, l15 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)blockDim.x >> 6;
    const int f0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * NB;
    const char* wr[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) wr[s] = (const char*)p.w + ((int64_t)s * p.n + min(f0 + l15, p.n - 1)) * p.w_rs;
    const char* xr[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) xr[b] = (const char*)p.x + (int64_t)min(m0 + 16 * b + l15, p.m - 1) * p.x_rs;
    f32x4 acc[kS][NB];
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[s][b] = f32x4{};
    const int bytes = p.k * 2, chunks = (bytes + 127) >> 7;
    for (int c0 = wave; c0 < chunks; c0 += waves * kU) {
        i32x4 w[kU][2][kS], x[kU][2][NB];
        bool in[kU][2];
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = (c0 + u * waves) * 128 + h * 64 + q * 16;
                in[u][h] = at < bytes;
                const int o = in[u][h] ? at : bytes - 16;
#pragma unroll
                for (int s = 0; s < kS; ++s) w[u][h][s] = *(const i32x4*)(wr[s] + o);
#pragma unroll
                for (int b = 0; b < NB; ++b) x[u][h][b] = *(const i32x4*)(xr[b] + o);
            }
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int s = 0; s < kS; ++s) {
                    const i32x4 wv = in[u][h] ? w[u][h][s] : i32x4{};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const i32x4 xv = in[u][h] ? x[u][h][b] : i32x4{};
                        acc[s][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv),
                                                                            __builtin_bit_cast(bf16x8, xv), acc[s][b], 0, 0, 0);
                    }
                }
    }
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int b = 0; b < NB; ++b) part[(wave * kS * NB + s * NB + b) * 64 + lane] = acc[s][b];
    __syncthreads();
    // Wave b finishes token block b: lane l holds token l & 15, features 4 (l >> 4) + e.
    for (int b = wave; b < NB; b += waves) {
        f32x4 z[kS];
#pragma unroll
        for (int s = 0; s < kS; ++s) {
            z[s] = f32x4{};
            for (int v = 0; v < waves; ++v) z[s] += part[(v * kS * NB + s * NB + b) * 64 + lane];
        }
        const int m = m0 + 16 * b + l15, f = f0 + 4 * q;
        if (m >= p.m || f >= p.n) continue;
        f32x4 y;
        if (p.bias != nullptr) {
#pragma unroll
            for (int s = 0; s < kS; ++s) z[s] += load4(p.bias, s * p.n + f, p.bias_f32 != 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = activate(z[kS - 1][e], p.act);
            if constexpr (kGated) y[e] *= z[0][e];
        }
        if (p.gate != nullptr) y *= load4((const char*)p.gate + gate_row(p, m) * p.gate_rs, f, p.gate_f32 != 0);
        if (p.residual != nullptr) y += unpack4(*(const i32x2*)((const char*)p.residual + m * p.res_rs + 2 * f));
        *(i32x2*)((char*)p.y + m * p.y_rs + 2 * f) = i32x2{(int)pack_bf16x2(y[0], y[1]), (int)pack_bf16x2(y[2], y[3])};
    }
}

template <int NB>
hipError_t launch_rows(const LinearParams& p, int cus, hipStream_t stream) {
    const int kS = p.gated ? 2 : 1;
    const dim3 grid((unsigned)((p.n + 15) / 16), (unsigned)((p.m + 16 * NB - 1) / (16 * NB)));
    // Waves of a workgroup: enough for 16 per CU over the launch, each with a
    // chunk at least.
    const int64_t blocks = (int64_t)grid.x * grid.y;
    int waves = 4;
    while (waves < 16 && blocks * waves < 16ll * cus && waves * 128 < p.k * 2) waves *= 2;
    const size_t lds = (size_t)waves * kS * NB * 1024;
    if (p.gated)
        hipLaunchKernelGGL((linear_rows_kernel<NB, true>), grid, dim3(64 * waves), lds, stream, p);
    else
        hipLaunchKernelGGL((linear_rows_kernel<NB, false>), grid, dim3(64 * waves), lds, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_linear(LinearParams p, int cus, hipStream_t stream) {
    if (cus <= 0) cus = 256;
    if (p.m <= 16) return launch_rows<1>(p, cus, stream);
    if (p.m <= 32) return launch_rows<2>(p, cus, stream);
    const Shape* s = pick_shape(p, cus);
    return s == nullptr ? hipErrorInvalidConfiguration : s->launch(p, stream);
}

int linear_max_tile() { return 256; }

}  // namespace h3a
