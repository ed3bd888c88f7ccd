// Attention over lists of key blocks (gfx950): the 64-key blocks that a list
// names for each block of 256 query rows.
//
//   O = softmax(scale * Q K_L^T) V_L,  LSE = log sum exp(scale * Q K_L^T)
// over the keys of the listed blocks, each as often as it is named. Entries past
// the row's count or outside the key blocks name nothing; a row without keys
// has O = 0 and LSE = -inf. As in the dense forward the weights are rounded to
// bf16 for the product with V, and nothing else before O (attn_tile.h).
//
// A listed block is one key tile of attn_tile (or two key blocks of attn_unit),
// so the tile's pipeline runs as in the dense forward with the list in place of
// the key range. Every workgroup first packs its list into LDS, without the
// entries that name nothing: no content of a list can address outside K or V.
#include <math.h>

#include "attn_tile.h"
#include "common.h"
#include "kernels.h"

namespace h3a {
namespace {

// Packs the list of a query block into `ids` and returns its length; `scratch`
// holds a word per wave. Ends on a barrier.
__device__ __forceinline__ int load_list(const SparseParams& p, int b, int h, int qt, int nblk, lds_int* ids, lds_int* scratch) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t* const list = p.list + b * p.list_sb + h * p.list_sh + qt * p.list_sq;
    int n = p.max_blocks;
    if (p.count != nullptr) n = min(max(p.count[b * p.count_sb + h * p.count_sh + qt * p.count_sq], 0), n);
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += kThreads) {
        const int id = i0 + tid < n ? list[i0 + tid] : -1;
        const bool in = (unsigned)id < (unsigned)nblk;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
        if (lane == 0) scratch[wave] = __builtin_popcountll(mask);
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int c = scratch[w];
            before += w < wave ? c : 0;
            all += c;
        }
        if (in) ids[total + before + __builtin_popcountll(mask & ((1ull << lane) - 1))] = id;
        total += all;
        __syncthreads();
    }
    return __builtin_amdgcn_readfirstlane(total);
}

// Workgroup -> query tile and part of its list: each XCD runs one contiguous
// range of (tile, piece), so that neighbouring query blocks of a head, whose
// lists share blocks, read them through one L2.
__device__ __forceinline__ int contiguous(int bid, int n) {
    const int xcd = bid & 7, per = n >> 3, rem = n & 7;
    return xcd * per + min(xcd, rem) + (bid >> 3);
}

__global__ __launch_bounds__(kThreads, 2) void attn_sparse_kernel(SparseParams p) {
    __shared__ int ids[kListMax + kListPad];
    __shared__ int scratch[kWaves];
    const int at = contiguous(blockIdx.x, (int)gridDim.x);
    const int tile = at / p.pieces, piece = at % p.pieces;
    const int qt = tile % p.n_qtiles, h = tile / p.n_qtiles % p.heads, b = tile / p.n_qtiles / p.heads;
    const int nblk = (p.seqlen_k + kBN - 1) / kBN;
    const int n = load_list(p, b, h, qt, nblk, (lds_int*)ids, (lds_int*)scratch);
    const int t0 = (int)((int64_t)n * piece / p.pieces), t1 = (int)((int64_t)n * (piece + 1) / p.pieces);
    if (threadIdx.x < kListPad) ids[t1 + threadIdx.x] = nblk;
    __syncthreads();
    // The tile reads the launch arguments afresh from the kernel-argument
    // segment (an opaque zero offset), rather than hold in scalar registers
    // what the list's loads above took of them.
    int zero;
    asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
    using Args = const __attribute__((address_space(4))) SparseParams;
    Args* const pk = (Args*)((const __attribute__((address_space(4))) char*)&p + zero);
    attn_tile<false, false, false, true, true>(*pk, tile, -1, 1, p.pieces > 1 ? piece * p.split_tiles + tile : -1, false, nullptr, false,
                                               -1, nullptr, nullptr, 0, KeyList{(const lds_int*)ids + t0, t1 - t0});
}

// Few query rows: units of 32 rows, the list's keys split over the waves.
__global__ __launch_bounds__(kThreads, 2) void attn_sparse_short_kernel(SparseParams p) {
    __shared__ int ids[kListMax + kListPad];
    __shared__ int scratch[kWaves];
    const int at = contiguous(blockIdx.x, (int)gridDim.x);
    const int m0 = at % p.n_units * kUnitRows, qt = m0 / kBM;
    const int h = at / p.n_units % p.heads, b = at / p.n_units / p.heads;
    const int nblk = (p.seqlen_k + kBN - 1) / kBN;
    const int n = load_list(p, b, h, qt, nblk, (lds_int*)ids, (lds_int*)scratch);
    attn_unit<true>(p, UnitView{(const char*)p.q + 2 * (b * p.q_sb + h * p.q_sh) + (int64_t)m0 * p.q_rs,
                                (const char*)p.k + 2 * (b * p.k_sb + h * p.k_sh), (const char*)p.v + 2 * (b * p.v_sb + h * p.v_sh),
                                (char*)p.o + 2 * (b * p.o_sb + h * p.o_sh) + (int64_t)m0 * p.o_rs,
                                p.lse == nullptr ? nullptr : p.lse + b * p.lse_sb + h * p.lse_sh + m0, p.seqlen_q - m0, p.seqlen_k},
                    KeyList{(const lds_int*)ids, n});
}

}  // namespace

// Expected time (us) of `jobs` tiles or pieces over kt listed blocks each: rounds
// over the CUs of a fixed part and the blocks, slower the more CUs are busy.
static double round_us(int64_t jobs, double kt, int cus) {
    const double busy = jobs < cus ? (double)jobs / (double)cus : 1.0;
    return (double)((jobs + cus - 1) / cus) * (9.7 + kt * (1.0 + 0.6 * busy));
}

// Units of 32 rows, whole tiles, or (for less than a round of tiles) tiles in
// pieces, by the expected time. A round of units: 5 us and 1.5 per 256 keys, a
// tenth more in practice; pieces: the merge, 3 us and 0.055 a piece (its fp32
// partial rows written and read). On 17 sizes of 1 to 24,960 rows, 4 to 40 heads
// and 3 to 150 blocks, each run as units, whole and in 2 to 8 pieces, this picks
// the fastest or one within 6% of it (us, units / whole / best in pieces: 4 heads
// of 4,095 x 16 blocks 26 / 28 / 31; 20 of 2,048 x 8 46 / 22 / 41; 20 of 512 x 32
// 35 / 45 / 29; 8 of 512 x 16 12 / 26 / 20; 5 of 256 x 150 55 / 172 / 38).
void plan_attn_sparse(SparseParams& p, int cus) {
    const int64_t tiles = (int64_t)p.n_qtiles * p.heads * p.n_groups;
    if (cus <= 0 || p.max_blocks == 0) return;
    const double n = (double)p.max_blocks;
    const int32_t per = (p.seqlen_q + kUnitRows - 1) / kUnitRows;
    const int64_t units = (int64_t)per * p.heads * p.n_groups;
    const double units_us = 1.15 * (double)((units + cus - 1) / cus) * (4.8 + 1.5 * ceil(n * kBN / 256.0));
    double best = round_us(tiles, n, cus);
    for (int c = 2; c <= 8 && c <= p.max_blocks && tiles < cus; ++c) {
        const double us = round_us(tiles * c, n / c, cus) + 3.0 + 0.055 * (double)(tiles * c);
        if (us < best) {
            best = us;
            p.pieces = c;
        }
    }
    if (units_us >= best) return;
    p.pieces = 1;
    p.n_units = per;
}

hipError_t launch_attn_sparse(const SparseParams& p, hipStream_t stream) {
    if (p.n_units > 0) {
        const int64_t units = (int64_t)p.n_units * p.heads * p.n_groups;
        hipLaunchKernelGGL(attn_sparse_short_kernel, dim3((unsigned)units), dim3(kThreads), 0, stream, p);
        return hipGetLastError();
    }
    const int64_t tiles = (int64_t)p.n_qtiles * p.heads * p.n_groups;
    hipLaunchKernelGGL(attn_sparse_kernel, dim3((unsigned)(tiles * p.pieces)), dim3(kThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.pieces < 2) return e;
    AttnParams m = p;
    m.n_full = 0;
    m.split_n = p.pieces;
    hipLaunchKernelGGL((attn_merge_kernel<8, true>), dim3((unsigned)(tiles * (kBM / kMergeRows))), dim3(256), 0, stream, m);
    return hipGetLastError();
}

}  // namespace h3a
