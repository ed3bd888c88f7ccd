// Selection of key blocks by a cheap score (gfx950): per block of 256 query
// rows, the topk blocks of 64 keys whose mean key has the largest product with
// the mean query.
//
//   qm[i] = fp32(mean of the query rows of block i), km[j] of the key rows
//   s[i, j] = fp32(<qm[i], km[j]>)
// Blocks marked in `always` come before all others (by their index alone), NaN
// counts as -inf, equal scores are taken in ascending order of their index; the
// result is ascending.
//
// The means and products are summed in 64 bits and rounded to 32 once, so that
// the choice between nearly equal scores is that of the exact ones, whatever the
// order of the sums (a bf16 sum of 256 rows is exact in 64 bits but for extreme
// ranges). The first kernel reads q and k once (HBM-bound); the products are few
// (2 * 128 * nq * nk per head) and run on v_mfma_f64_16x16x4_f64; the third finds
// each row's threshold by bisection over the scores' bits.
#include <math.h>

#include "common.h"
#include "kernels.h"

namespace h3a {
namespace {

constexpr int kD = 128;
typedef double f64x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- means

// One workgroup per (block, head, batch): 16 lanes a row of 256 bytes, 16 rows
// at a time, 8 columns per lane.
__global__ __launch_bounds__(256) void block_mean_kernel(SelectParams p) {
    __shared__ double sums[16][kD];
    const int64_t nqb = (int64_t)p.nq * p.heads * p.batch;
    const bool is_q = (int64_t)blockIdx.x < nqb;
    const int64_t i = is_q ? blockIdx.x : (int64_t)blockIdx.x - nqb;
    // Heads fastest: the workgroups that run together read whole rows of a
    // (batch, seq, head) tensor.
    const int nb = is_q ? p.nq : p.nk;
    const int h = (int)(i % p.heads), blk = (int)(i / p.heads % nb), b = (int)(i / p.heads / nb);
    const int rows = is_q ? kSelectBlockQ : kSelectBlockK, len = is_q ? p.seqlen_q : p.seqlen_k;
    const int row0 = blk * rows, n = min(rows, len - row0);
    const int64_t rs = is_q ? p.q_rs : p.k_rs;
    const char* const base = is_q ? (const char*)p.q + 2 * (b * p.q_sb + h * p.q_sh) : (const char*)p.k + 2 * (b * p.k_sb + h * p.k_sh);
    const int g = threadIdx.x >> 4, j = threadIdx.x & 15;
    double acc[8] = {};
    for (int r0 = 0; r0 < n; r0 += 64) {
        i32x4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)  // rows past the block are read from its last one and dropped
            raw[u] = *(const i32x4*)(base + (int64_t)(row0 + min(r0 + 16 * u + g, n - 1)) * rs + 16 * j);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (r0 + 16 * u + g >= n) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = (uint32_t)raw[u][e];
                acc[2 * e] += (double)__uint_as_float(w << 16);
                acc[2 * e + 1] += (double)__uint_as_float(w & 0xffff0000u);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[g][8 * j + e] = acc[e];
    __syncthreads();
    if (threadIdx.x < kD) {
        double s = 0.0;
#pragma unroll
        for (int r = 0; r < 16; ++r) s += sums[r][threadIdx.x];
        float* const out = is_q ? p.qm : p.km;
        out[(((int64_t)b * p.heads + h) * nb + blk) * kD + threadIdx.x] = (float)(s / (double)n);
    }
}

// ---------------------------------------------------------------- scores

// One wave per 16 query blocks x 32 key blocks: two chains of products. Lane l
// holds, of row l & 15 of each operand, columns 16 i + 4 g .. +4 (g = l >> 4) for
// i = 0 .. 7, so that the four lanes of a row load 64 bytes side by side; MFMA
// step (i, e) multiplies column 16 i + 4 g + e of every lane group. The result:
// column l & 15, rows g + 4 i. (With 32 columns of a lane in one piece, 64 lines
// a load, 780 x 195 blocks at 5 heads took 13.5 us.)
constexpr int kKT = 2;

__global__ __launch_bounds__(256) void block_score_kernel(SelectParams p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t bh = blockIdx.y;
    const int groups = (p.nk + 16 * kKT * 4 - 1) / (16 * kKT * 4);  // of a workgroup's key blocks
    const int qt = (int)(blockIdx.x / groups), k0 = ((int)(blockIdx.x % groups) * 4 + wave) * 16 * kKT;
    if (k0 >= p.nk) return;
    const int l15 = lane & 15, g = lane >> 4;
    const float* const qr = p.qm + (bh * p.nq + min(qt * 16 + l15, p.nq - 1)) * kD + 4 * g;
    const float* kr[kKT];
#pragma unroll
    for (int t = 0; t < kKT; ++t) kr[t] = p.km + (bh * p.nk + min(k0 + 16 * t + l15, p.nk - 1)) * kD + 4 * g;
    f32x4 a[8], b[kKT][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] = *(const f32x4*)(qr + 16 * i);
#pragma unroll
        for (int t = 0; t < kKT; ++t) b[t][i] = *(const f32x4*)(kr[t] + 16 * i);
    }
    f64x4 acc[kKT] = {};
#pragma unroll
    for (int s = 0; s < 32; ++s)
#pragma unroll
        for (int t = 0; t < kKT; ++t)
            acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)a[s >> 2][s & 3], (double)b[t][s >> 2][s & 3], acc[t], 0, 0, 0);
#pragma unroll
    for (int t = 0; t < kKT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = qt * 16 + g + 4 * i, col = k0 + 16 * t + l15;
            if (row < p.nq && col < p.nk) p.score[(bh * p.nq + row) * p.nk + col] = (float)acc[t][i];
        }
}

// ---------------------------------------------------------------- choice

// Ascending in the score: NaN with -inf, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float s) {
    s = s != s ? -INFINITY : s + 0.0f;
    const uint32_t u = __float_as_uint(s);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One wave (kWaves == 1) or workgroup per row, kR keys per lane: block
// (r * kWaves + wave) * 64 + lane in register r. The threshold, the topk-th
// largest key, bit by bit from the top; then the blocks above it, and as many of
// those at it, in order of their index, as are left.
template <int kR, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void block_choose_kernel(SelectParams p) {
    __shared__ int counts[2][kWaves];
    const int lane = threadIdx.x & 63, wave = kWaves == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t row = blockIdx.x;
    const float* const score = p.score + row * p.nk;
    uint32_t key[kR];
    // Loads in groups, past the row from its last block: behind a branch each
    // would wait for the one before it.
    constexpr int kG = kR < 16 ? kR : 16;
#pragma unroll
    for (int r0 = 0; r0 < kR; r0 += kG) {
        float s[kG];
        uint32_t marked[kG];
#pragma unroll
        for (int r = 0; r < kG; ++r) s[r] = score[min(((r0 + r) * kWaves + wave) * 64 + lane, p.nk - 1)];
        if (p.always != nullptr) {
#pragma unroll
            for (int r = 0; r < kG; ++r) marked[r] = p.always[min(((r0 + r) * kWaves + wave) * 64 + lane, p.nk - 1)];
        } else {
#pragma unroll
            for (int r = 0; r < kG; ++r) marked[r] = 0;
        }
#pragma unroll
        for (int r = 0; r < kG; ++r) {
            const uint32_t k = marked[r] != 0 ? 0xffffffffu : order_key(s[r]);
            key[r0 + r] = ((r0 + r) * kWaves + wave) * 64 + lane < p.nk ? k : 0;  // past the row: below every score
        }
    }
    // Number of the row's keys at or above x.
    int turn = 0;
    auto at_least = [&](uint32_t x) {
        int n = 0;
#pragma unroll
        for (int r = 0; r < kR; ++r) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] >= x));
        if constexpr (kWaves > 1) {
            if (lane == 0) counts[turn][wave] = n;
            __syncthreads();
            n = 0;
            for (int w = 0; w < kWaves; ++w) n += counts[turn][w];
            turn ^= 1;  // the other buffer next: one barrier a step
            n = __builtin_amdgcn_readfirstlane(n);
        }
        return n;
    };
    uint32_t threshold = 0;
    int above = 0;  // keys above the threshold
    bool exact = false;
    for (int bit = 31; bit >= 0 && !exact; --bit) {
        const uint32_t x = threshold | (1u << bit);
        const int n = at_least(x);
        if (n >= p.topk) {
            threshold = x;
            exact = n == p.topk;  // every key from here on up, no more
        }
    }
    if (!exact) above = threshold == 0xffffffffu ? 0 : at_least(threshold + 1);
    int left = exact ? p.topk : p.topk - above;  // of the keys at the threshold
    int32_t* const out = p.index + row * p.topk;
    int at = 0;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        // (exact: all keys at or above count as "above".)
        const bool up = exact ? key[r] >= threshold : key[r] > threshold;
        const bool eq = !exact && key[r] == threshold;
        const uint64_t mu = __builtin_amdgcn_ballot_w64(up), me = __builtin_amdgcn_ballot_w64(eq);
        int eq_before = 0, eq_all = __builtin_popcountll(me), up_before = 0, up_all = __builtin_popcountll(mu);
        if constexpr (kWaves > 1) {
            __syncthreads();
            if (lane == 0) {
                counts[0][wave] = up_all;
                counts[1][wave] = eq_all;
            }
            __syncthreads();
            eq_all = up_all = 0;
            for (int w = 0; w < kWaves; ++w) {
                if (w == wave) {
                    up_before = up_all;
                    eq_before = eq_all;
                }
                up_all += counts[0][w];
                eq_all += counts[1][w];
            }
        }
        const uint64_t below = (1ull << lane) - 1;
        const int eq_rank = eq_before + __builtin_popcountll(me & below);
        const int up_rank = up_before + __builtin_popcountll(mu & below);
        const bool take = up || (eq && eq_rank < left);
        const int place = at + up_rank + min(eq_rank, left);
        const int j = (r * kWaves + wave) * 64 + lane;
        if (take) out[place] = j;
        at += up_all + min(eq_all, left);
        left -= min(eq_all, left);
    }
}

}  // namespace

int select_max_blocks() { return 32 * 64 * 16; }

hipError_t launch_block_select(const SelectParams& p, hipStream_t stream) {
    const int64_t bh = (int64_t)p.batch * p.heads;
    hipLaunchKernelGGL(block_mean_kernel, dim3((unsigned)(bh * (p.nq + p.nk))), dim3(256), 0, stream, p);
    const int64_t qtiles = (p.nq + 15) / 16, kgroups = (p.nk + 16 * kKT * 4 - 1) / (16 * kKT * 4);
    hipLaunchKernelGGL(block_score_kernel, dim3((unsigned)(qtiles * kgroups), (unsigned)bh), dim3(256), 0, stream, p);
    const dim3 rows((unsigned)(bh * p.nq));
    auto choose = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, rows, dim3(threads), 0, stream, p); };
    if (p.nk <= 64)
        choose(block_choose_kernel<1, 1>, 64);
    else if (p.nk <= 256)
        choose(block_choose_kernel<4, 1>, 64);
    else if (p.nk <= 1024)
        choose(block_choose_kernel<16, 1>, 64);
    else if (p.nk <= 4096)
        choose(block_choose_kernel<64, 1>, 64);
    else if (p.nk <= 16384)
        choose(block_choose_kernel<16, 16>, 1024);
    else
        choose(block_choose_kernel<32, 16>, 1024);
    return hipGetLastError();
}

}  // namespace h3a
