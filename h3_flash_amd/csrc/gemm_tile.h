// The matrix product of the GEMM kernels (gfx950): C^T = W X^T of one tile,
// over bf16 operands with K contiguous, accumulated in fp32 on
// v_mfma_f32_16x16x32_bf16. The W fragment is the A operand (16 features x
// 32 K) and the X fragment the B operand (32 K x 16 tokens), so every lane of
// the result holds one token and 4 consecutive features per 16-feature block.
//
// Tiling: one workgroup of 4 waves per CU computes TF features x 16*NT tokens,
// one wave per SIMD. Large tiles split the waves
// 2 x 2 (128 features x 8*NT tokens each), small ones 4 x 1 (TF/4 features x
// all tokens), whichever reads fewer LDS bytes per MFMA; the accumulators are
// held in the accumulation registers (256 per lane at TF = 256, NT = 16).
//
// K advances 64 at a time through rings of SW (W rows) and SX (X rows) LDS
// stages, as many as fit in 160 KB, filled HBM -> LDS by buffer_load ... lds (16 bytes per lane, no VGPR
// staging; each load covers whole 128-byte lines of 8 rows). LDS rows are 128
// bytes; the 16-byte chunk c of row r sits at c ^ ((r >> 1) & 7), so the 16
// rows a quarter-wave's fragment read touches hit 16 distinct bank groups.
// One barrier per K step of 64, in its middle (see the step below).
#pragma once

#include <math.h>

#include <type_traits>
#include <utility>

#include "common.h"

namespace h3a {
namespace {

constexpr int kPK = 64;                   // K per stage (two MFMA K steps of 32)
constexpr int kPWaves = 4;
constexpr int kPThreads = kPWaves * 64;
constexpr int kPRow = kPK * 2;            // LDS bytes per tile row

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// vmcnt(N) and lgkmcnt(0): the wave's own DMA loads beyond the newest N have
// landed and its LDS reads have completed.
template <int N>
__device__ __forceinline__ void wait_vm_lgkm() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
}

__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }

// acc += A B on v_mfma_f32_16x16x32_bf16 with the accumulator pinned to the
// accumulation registers: with the builtin, the 256 accumulators of a lane
// are split between VGPRs and AGPRs and copied around the loop back edge.
__device__ __forceinline__ void mfma_acc(f32x4& acc, const bf16x8& a, const bf16x8& b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// f(0), ..., f(N - 1) with compile-time indices.
template <int... I, typename F>
__device__ __forceinline__ void static_for_seq(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    static_for_seq(std::make_integer_sequence<int, N>{}, f);
}

// A tile shape: TF features x 16*NT tokens; SW stages of W rows, SX of X rows.
template <int TF, int NT, int SW, int SX>
struct Tile {
    static constexpr int kSW = SW, kSX = SX;
    static constexpr int kTokens = 16 * NT;
    // Waves over features x tokens. LDS reads per MFMA K step: 2 x 2 reads
    // 4 * (8 + NT/2) KB, 4 x 1 reads 4 * (TF/64 + NT) KB.
    static constexpr int WN = TF == 256 && NT >= 10 ? 2 : 4, WM = kPWaves / WN;
    static constexpr int NA = TF / 16 / WN, NB = NT / WM;  // 16 x 16 MFMA blocks of a wave
    static constexpr int kWBytes = TF * kPRow, kXBytes = kTokens * kPRow;
    static constexpr int kXBase = SW * kWBytes, kStages = kXBase + SX * kXBytes;  // X stages follow the W stages
    // DMA loads (1 KB: 8 rows) per wave and stage
    static constexpr int kLoadsW = TF / 8 / kPWaves, kLoadsX = kTokens / 8 / kPWaves;
    // Epilogue: the tile's bf16 output rows over the (then idle) stages, and
    // a row buffer per 16-lane group for RoPE partners across lanes.
    static constexpr int kOutRow = TF * 2;
    static constexpr int kOutBytes = kTokens * kOutRow;
    static constexpr int kPartner = any_r_row_bytes(16);
    static constexpr int kEpiBytes = kOutBytes + kPThreads / 16 * kPartner;
    static constexpr int kLds = kStages > kEpiBytes ? kStages : kEpiBytes;
    static_assert(NT % 2 == 0 && TF % 128 == 0, "DMA map: whole loads per wave");
    static_assert(NB * WM == NT && NA * NB >= 4, "wave map; an accumulator is next used 4 MFMAs later at the least");
    static_assert(SX >= 2 && SW > SX, "the waits below count loads in this order");
    static_assert(kLds <= 160 * 1024, "LDS of one workgroup");
};

// Workgroup b of `total` runs on XCD b mod 8 (round-robin dispatch) as that
// XCD's (b / 8)-th; each XCD owns one contiguous range of the tile order, so
// the ~32 tiles an XCD runs at a time are consecutive in it and share their X
// and W panels in the XCD's L2. (A persistent grid of one workgroup per CU
// looping over its XCD's range measured from 1% faster to 4% slower, and is
// not used.)
__device__ __forceinline__ int xcd_tile(int bid, int total) {
    const int xcd = bid & 7, local = bid >> 3;
    const int per = total >> 3, rem = total & 7;
    return xcd * per + min(xcd, rem) + local;
}

// One operand's rows as a wave loads them: the resource of the tile's first
// row (rows past the operand are outside its records and load as zeros), the
// lane's byte offset in it, the bytes from one load's rows to the next one's,
// and the lane's offset in the last K step (kTailK: lanes whose 16 bytes lie
// past the reduction hold an offset outside the records).
struct GemmRows {
    i32x4 rsrc;
    uint32_t lane, step, tail;
};

// The 16-byte chunk (a byte offset in the K step's 128) that a lane loads.
// DMA map: load i of wave w fills rows 8 (4i + w) .. +8 of an operand's
// stage; lane L writes LDS chunk (L & 7) of row r = 8 (4i + w) + (L >> 3),
// which holds the row's 16-byte chunk (L & 7) ^ ((r >> 1) & 7) =
// (L & 7) ^ (4 (w & 1) + (L >> 4)). Everything that depends on the lane is
// the same for every load; i and the K step go into the scalar offset.
__device__ __forceinline__ int gemm_chunk(int wave, int lane) { return ((lane & 7) ^ (4 * (wave & 1) + (lane >> 4))) << 4; }

// acc = W X^T over nk K steps; all waves of the workgroup call it. On return no
// load is in flight and no wave reads the stages any more. kTailK: the last K
// step is partial.
template <typename T, bool kTailK = false>
__device__ __forceinline__ void gemm_k_loop(const GemmRows& w_rows, const GemmRows& x_rows, const int nk, char* smem,
                                            int lane, int wave, int wn, int wm, f32x4 (&acc)[T::NA][T::NB]) {
    constexpr int SW = T::kSW, SX = T::kSX;
    i32x4 rw = w_rows.rsrc, rx = x_rows.rsrc;
    const uint32_t dw = w_rows.lane, dx = x_rows.lane;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char*)smem;
    const uint32_t lds_wave = lds0 + (uint32_t)wave * 1024u;
    // Load j of this wave's share of a K step's rows (32 j rows on from the
    // wave's first), into LDS at dst + 4096 j. buffer_load ... lds writes 16
    // bytes per lane to LDS address M0 + 16*lane; M0 needs one wait state
    // before the load reads it. The row offsets stay in scalar registers and
    // the resources' bases move along K: three instructions a load, which fit
    // between two MFMAs (offsets formed per load took six, and held up the
    // lone wave's MFMAs).
    auto dma1 = [&](const i32x4& rsrc, uint32_t voff, uint32_t soff, uint32_t dst, int j) __attribute__((always_inline)) {
        asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds"
                     :
                     : "s"(dst), "i"(j * 4096), "v"(voff), "s"(rsrc), "s"(soff)
                     : "memory", "scc");
    };
    uint32_t sow[T::kLoadsW], sox[T::kLoadsX];
#pragma unroll
    for (int j = 0; j < T::kLoadsW; ++j) sow[j] = (uint32_t)j * w_rows.step;
#pragma unroll
    for (int j = 0; j < T::kLoadsX; ++j) sox[j] = (uint32_t)j * x_rows.step;
    // (last: the load is of the last K step.)
    auto dma_w1 = [&](const i32x4& r, uint32_t stage, int j, bool last = false) __attribute__((always_inline)) {
        dma1(r, kTailK && last ? w_rows.tail : dw, sow[j], lds_wave + stage, j);
    };
    auto dma_x1 = [&](const i32x4& r, uint32_t stage, int j, bool last = false) __attribute__((always_inline)) {
        dma1(r, kTailK && last ? x_rows.tail : dx, sox[j], lds_wave + T::kXBase + stage, j);
    };
    // The resource one K step further along its rows. The records stay: a
    // lane's offset in its row is under 128 bytes and a row is at least the
    // reduction long, so the row after the last one is out of range at every
    // base.
    auto advance = [](i32x4& r) __attribute__((always_inline)) {
        const uint64_t base = ((uint64_t)(uint32_t)r.y << 32 | (uint32_t)r.x) + kPRow;
        r.x = (int)(uint32_t)base;
        r.y = (int)((uint32_t)(base >> 32) & 0xffffu);
    };

    // Fragment reads: lane l takes row (16*block + (l & 15)) of the wave's
    // operand rows and, for MFMA K step h of the stage, logical chunk
    // 4h + (l >> 4) (K 32h + 8*(l>>4) .. +8); swz(row) = ((l & 15) >> 1) & 7.
    const int sl = (lane >> 1) & 7;
    const int fo0 = (lane & 15) * kPRow + (((lane >> 4) ^ sl) << 4);
    const int fo1 = (lane & 15) * kPRow + (((4 + (lane >> 4)) ^ sl) << 4);
    const lds_char* const lds = (const lds_char*)smem;
    const lds_char* const wfr0 = lds + wn * 16 * T::NA * kPRow + fo0;
    const lds_char* const wfr1 = lds + wn * 16 * T::NA * kPRow + fo1;
    const lds_char* const xfr0 = lds + T::kXBase + wm * 16 * T::NB * kPRow + fo0;
    const lds_char* const xfr1 = lds + T::kXBase + wm * 16 * T::NB * kPRow + fo1;

    bf16x8 fw[2][T::NA], fx[2][T::NB];
    constexpr int kReads = T::NA + T::NB, kMfmas = T::NA * T::NB;

    // Fragment j of MFMA K step h of the stages at byte offsets sw, sx.
    auto read1 = [&](uint32_t sw, uint32_t sx, int h, int j) __attribute__((always_inline)) {
        const lds_char* const xf = (h ? xfr1 : xfr0) + sx;
        const lds_char* const wf = (h ? wfr1 : wfr0) + sw;
        if (j < T::NB)
            fx[h][j] = *(const lds_bf16x8*)(xf + j * 16 * kPRow);
        else
            fw[h][j - T::NB] = *(const lds_bf16x8*)(wf + (j - T::NB) * 16 * kPRow);
    };
    // The MFMAs of fragment set h, feature block major, token blocks snaking,
    // with `extra(t)` issued after MFMA t.
    auto mfmas = [&](int h, auto&& extra) __attribute__((always_inline)) {
        static_for<kMfmas>([&](auto tc_) __attribute__((always_inline)) {
            constexpr int t = decltype(tc_)::value, a = t / T::NB, r = t % T::NB, b = (a & 1) ? T::NB - 1 - r : r;
            mfma_acc(acc[a][b], fw[h][a], fx[h][b]);
            extra(tc_);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // n items spread over the first `over` MFMAs: those that follow MFMA t.
    auto spread = [](auto tc_, auto n_c, auto over_c, auto&& item) __attribute__((always_inline)) {
        constexpr int t = decltype(tc_)::value, n = decltype(n_c)::value, over = decltype(over_c)::value;
        constexpr int lo = t < over ? t * n / over : n, hi = t < over ? (t + 1) * n / over : n;
        static_for<hi - lo>([&](auto i) __attribute__((always_inline)) { item(lo + decltype(i)::value); });
    };
    using Reads = std::integral_constant<int, kReads>;
    using LoadsW = std::integral_constant<int, T::kLoadsW>;
    using LoadsX = std::integral_constant<int, T::kLoadsX>;
    using Most = std::integral_constant<int, kMfmas * 3 / 4>;
    using All = std::integral_constant<int, kMfmas>;

    // K step i of W is loaded in the first half of step i + 1 - SW, of X in the
    // second half of step i - SX. Those before step 0 come here, in that order
    // (steps past the end of a short reduction through an empty resource: they
    // load zeros, so that the waits count the same).
    const i32x4 none{0, 0, 0, kBufferWord3};
#pragma unroll
    for (int i = 0; i < SW - 1; ++i) {
        const int ix = i + 1 - SW + SX;
#pragma unroll
        for (int j = 0; j < T::kLoadsW; ++j) dma_w1(i < nk ? rw : none, (uint32_t)(i * T::kWBytes), j, i == nk - 1);
        advance(rw);
        if (ix < 0) continue;
#pragma unroll
        for (int j = 0; j < T::kLoadsX; ++j) dma_x1(ix < nk ? rx : none, (uint32_t)(ix * T::kXBytes), j, ix == nk - 1);
        advance(rx);
    }
#pragma unroll
    for (int a = 0; a < T::NA; ++a)
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            acc[a][b] = f32x4{};
            asm volatile("" : "+a"(acc[a][b]));
        }
    wait_vm_lgkm<(SX - 1) * (T::kLoadsW + T::kLoadsX)>();  // K step 0 (own loads) landed
    barrier();
#pragma unroll
    for (int j = 0; j < kReads; ++j) read1(0, 0, 0, j);

    // K step kt in the stages at `cw` and `cx`, its first-half fragments in set
    // 0. First half: MFMAs of set 0 while set 1 is read from the same stages,
    // and the W rows of step kt+SW-1 go into the W stage before `cw`. Then the
    // wave's own loads of step kt+1 are waited for (later ones stay in flight),
    // with its reads of the stages; after the barrier every wave's part of
    // step kt+1 is in LDS and step kt's stages are no longer read by anyone.
    // Second half: MFMAs of set 1 while step kt+1's first-half fragments are
    // read into set 0 and the X rows of step kt+SX go into `cx`. The loads of a
    // step are thus spread over it (the CU's address path takes 64 bytes a
    // clock, and a lone wave that finds it busy holds up its MFMAs), and W, the
    // operand that comes from HBM, has SW - 1 steps to land.
    // `left` K steps follow; the last steps run out of loads, the last one
    // reads nothing.
    uint32_t cw = 0, pw = (SW - 1) * T::kWBytes, cx = 0;
    int kt = 0;
    auto step = [&](auto left_c) __attribute__((always_inline)) {
        constexpr int left = decltype(left_c)::value;  // SW: that many or more
        constexpr int kAheadW = left - (SW - SX) < SX - 1 ? left - (SW - SX) : SX - 1;
        constexpr int kAheadX = left - 1 < SX - 2 ? left - 1 : SX - 2;
        const uint32_t nw = cw == (SW - 1) * T::kWBytes ? 0u : cw + T::kWBytes;
        const uint32_t nx = cx == (SX - 1) * T::kXBytes ? 0u : cx + T::kXBytes;
        mfmas(0, [&](auto t) __attribute__((always_inline)) {
            spread(t, Reads{}, Most{}, [&](int i) __attribute__((always_inline)) { read1(cw, cx, 1, i); });
            if constexpr (left >= SW - 1)
                spread(t, LoadsW{}, All{}, [&](int i) __attribute__((always_inline)) { dma_w1(rw, pw, i, left == SW - 1); });
        });
        wait_vm_lgkm<(kAheadW > 0 ? kAheadW : 0) * T::kLoadsW + (kAheadX > 0 ? kAheadX : 0) * T::kLoadsX>();
        barrier();
        mfmas(1, [&](auto t) __attribute__((always_inline)) {
            if constexpr (left > 0)
                spread(t, Reads{}, All{}, [&](int i) __attribute__((always_inline)) { read1(nw, nx, 0, i); });
            if constexpr (left >= SX)
                spread(t, LoadsX{}, Most{}, [&](int i) __attribute__((always_inline)) { dma_x1(rx, cx, i, left == SX); });
        });
        advance(rw);
        advance(rx);
        pw = cw;
        cw = nw;
        cx = nx;
        ++kt;
    };
    while (kt < nk - SW) step(std::integral_constant<int, SW>{});
    // The last min(SW, nk) steps.
    auto tail = [&](auto self, auto left_c) __attribute__((always_inline)) -> void {
        constexpr int left = decltype(left_c)::value;
        if (left < nk) step(left_c);
        if constexpr (left > 0) self(self, std::integral_constant<int, left - 1>{});
    };
    tail(tail, std::integral_constant<int, SW - 1>{});
    // No load is in flight and no wave reads the stages any more (the last
    // step's barrier followed every wave's last fragment read). The MFMAs are
    // inline asm, outside the compiler's hazard tracking: give the last ones
    // time to write their results before they are read.
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
}

}  // namespace
}  // namespace h3a
