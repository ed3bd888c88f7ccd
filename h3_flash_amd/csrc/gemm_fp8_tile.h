// The matrix product of the 8-bit GEMM kernels (gfx950): C^T = W X^T of one tile over
// e4m3 operands with K contiguous and a power of two for each 128 values of K,
// accumulated in fp32 on v_mfma_scale_f32_32x32x64_f8f6f4. A K step of 128 is a scale's
// block and the 128 bytes of a row that gemm_tile.h's K step of 64 bf16 is, so stages,
// loads, swizzle and waits are that file's; what differs:
//   - fragments are 32 rows x 64 K, 32 bytes a lane: lane l holds of row l & 31 the
//     16-byte chunks 4h + (l >> 5) and 4h + 2 + (l >> 5) of half h, of W and X alike;
//   - a lane of the result holds token l & 31 of its block and, in group g of four,
//     rows 8g + 4 (l >> 5) .. +3 of W;
//   - the scales of the tile's tokens and of its one or two blocks of W rows lie in a
//     ring of segments behind the stages: 16 K steps' bytes of each token, as they lie
//     in memory, loaded once. A lane reads the byte of its token for the K step ahead,
//     with the fragments. (Both operands' scales go into the instruction: the sums need
//     no multiplication of their own.)
#pragma once

#include "gemm_tile.h"

namespace h3a {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kP8K = 128;       // K of a step
constexpr int kSegSteps = 16;   // K steps of a segment of scales

template <int N>
__device__ __forceinline__ void mfma_fp8(f32x16& acc, const i32x8& w, const i32x8& x, int sw, int sx) {
    // Pinned to the accumulation registers where a lane holds many (gemm_tile.h).
    if constexpr (N >= 8)
        asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                     : "+a"(acc)
                     : "v"(w), "v"(x), "v"(sw), "v"(sx));
    else
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, acc, 0, 0, 0, sw, 0, sx);
}

// A tile shape: TF rows of W x 16 NT tokens; SW stages of W rows, SX of X rows.
template <int TF, int NT, int SW, int SX>
struct Fp8Tile {
    static constexpr int kSW = SW, kSX = SX, kTF = TF;
    static constexpr int kTokens = 16 * NT;
    static constexpr int WN = TF == 256 && NT >= 10 ? 2 : 4, WM = kPWaves / WN;
    static constexpr int NA = TF / 32 / WN, NB = NT / 2 / WM;  // 32 x 32 MFMA blocks of a wave
    static constexpr int kWBytes = TF * kPRow, kXBytes = kTokens * kPRow;
    static constexpr int kXBase = SW * kWBytes, kStages = kXBase + SX * kXBytes;
    static constexpr int kLoadsW = TF / 8 / kPWaves, kLoadsX = kTokens / 8 / kPWaves;
    // A segment: 16 bytes for each token, then for each of the two blocks of W rows.
    static constexpr int kSegLoads = (kTokens + 63) / 64, kSegW = kSegLoads * 1024, kSegBytes = kSegW + 64;
    static constexpr int kSegRoom = (160 * 1024 - kStages) / kSegBytes, kSegs = kSegRoom < 8 ? kSegRoom : 8;
    static constexpr int kLds = kStages + kSegs * kSegBytes;
    // Blocks of tokens of a wave that the epilogue takes at a time: all, or what fits.
    static constexpr int kPass = kTokens * TF * 4 <= 160 * 1024 ? NB : NB % 2 == 0 ? NB / 2 : 1;
    static constexpr int kEpiBytes = 32 * kPass * WM * TF * 4;
    static constexpr int kSmem = kLds > kEpiBytes ? kLds : kEpiBytes;
    static_assert(NT % 2 == 0 && TF % 128 == 0, "DMA map: whole loads per wave");
    static_assert(NA * WN * 32 == TF && 2 * NB * WM == NT && NB % kPass == 0, "wave map");
    static_assert(SX >= 2 && SW > SX, "the waits below count loads in this order");
    static_assert((kSegs - 2) * kSegSteps >= SW && kSmem <= 160 * 1024, "LDS of one workgroup");
};

// The rows' scales as a workgroup loads them: the tokens' (the resource of the tile's
// first row; rows past the operand load as zeros), and W's, with the offsets of the
// tile's two blocks of rows (the same one twice where it has one).
struct GemmScales {
    i32x4 x, w;
    uint32_t x_rs;  // bytes from a token's to the next one's
    uint32_t w_at[2];
    int first;      // the K range's first step
};

// acc = W X^T over nk K steps; all waves of the workgroup call it. On return no load is
// in flight and no wave reads the stages any more. kTailK: the last K step is partial.
// w_block: per lane, which of the two blocks of W rows its fragment row belongs to.
template <typename T, bool kTailK = false>
__device__ __forceinline__ void gemm_fp8_k_loop(const GemmRows& w_rows, const GemmRows& x_rows, const GemmScales& scales,
                                                const int nk, char* smem, int lane, int wave, int wn, int wm, int w_block,
                                                f32x16 (&acc)[T::NA][T::NB]) {
    constexpr int SW = T::kSW, SX = T::kSX;
    i32x4 rw = w_rows.rsrc, rx = x_rows.rsrc;
    const uint32_t dw = w_rows.lane, dx = x_rows.lane;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char*)smem;
    const uint32_t lds_wave = lds0 + (uint32_t)wave * 1024u;
    uint32_t sow[T::kLoadsW], sox[T::kLoadsX];
#pragma unroll
    for (int j = 0; j < T::kLoadsW; ++j) sow[j] = (uint32_t)j * w_rows.step;
#pragma unroll
    for (int j = 0; j < T::kLoadsX; ++j) sox[j] = (uint32_t)j * x_rows.step;
    auto dma_w1 = [&](const i32x4& r, uint32_t stage, int j, bool last = false) __attribute__((always_inline)) {
        gemm_dma(r, kTailK && last ? w_rows.tail : dw, sow[j], lds_wave + stage, j);
    };
    auto dma_x1 = [&](const i32x4& r, uint32_t stage, int j, bool last = false) __attribute__((always_inline)) {
        gemm_dma(r, kTailK && last ? x_rows.tail : dx, sox[j], lds_wave + T::kXBase + stage, j);
    };
    // Segment s of the scales into slot s mod kSegs, the work spread over the waves
    // (a wave's loads differ in number; they come before, or in the middle of, the
    // counted ones, which then are waited for a little early at worst).
    const int first_segment = scales.first / kSegSteps, segments = (scales.first + nk - 1) / kSegSteps - first_segment + 1;
    auto dma_segment = [&](int s) __attribute__((always_inline)) {
        const uint32_t to = lds0 + T::kStages + (uint32_t)(s % T::kSegs) * T::kSegBytes, from = (uint32_t)(first_segment + s) * kSegSteps;
#pragma unroll
        for (int i = 0; i < T::kSegLoads; ++i)
            if ((i & 3) == wave && 64 * i + lane < T::kTokens)
                gemm_dma(scales.x, (uint32_t)(64 * i + lane) * scales.x_rs, from, to + 1024 * i, 0);
        if (wave == 3 && lane == 0) {
            gemm_dma(scales.w, 0, scales.w_at[0] + from, to + T::kSegW, 0);
            gemm_dma(scales.w, 0, scales.w_at[1] + from, to + T::kSegW + 32, 0);
        }
    };

    const int sl = (lane >> 1) & 7, l31 = lane & 31, hi = lane >> 5;
    const lds_char* const lds = (const lds_char*)smem;
    const lds_char* const wfr = lds + wn * 32 * T::NA * kPRow + l31 * kPRow;
    const lds_char* const xfr = lds + T::kXBase + wm * 32 * T::NB * kPRow + l31 * kPRow;
    int fo[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) fo[h][i] = ((4 * h + 2 * i + hi) ^ sl) << 4;

    typedef __attribute__((address_space(3))) const uint8_t lds_u8;
    lds_u8* const xsc = (lds_u8*)(lds + T::kStages + (wm * 32 * T::NB + l31) * 16);
    lds_u8* const wsc = (lds_u8*)(lds + T::kStages + T::kSegW + w_block * 32);
    int sw = 0, sx[T::NB], sw_next = 0, sx_next[T::NB];

    i32x8 fw[2][T::NA], fx[2][T::NB];
    constexpr int kScales = T::NB + 1, kReads = 2 * (T::NA + T::NB), kMfmas = T::NA * T::NB;

    // 16-byte piece j of the fragments of half h of the stages at byte offsets cw, cx.
    auto read1 = [&](uint32_t cw, uint32_t cx, int h, int j) __attribute__((always_inline)) {
        const int i = j & 1, b = j >> 1;
        if (b < T::NB) {
            const i32x4 v = *(const lds_i32x4*)(xfr + cx + fo[h][i] + b * 32 * kPRow);
            if (i == 0) fx[h][b].lo = v; else fx[h][b].hi = v;
        } else {
            const i32x4 v = *(const lds_i32x4*)(wfr + cw + fo[h][i] + (b - T::NB) * 32 * kPRow);
            if (i == 0) fw[h][b - T::NB].lo = v; else fw[h][b - T::NB].hi = v;
        }
    };
    // Scale j of the K step whose byte lies at `at` in the ring.
    auto read_scale = [&](uint32_t at, int j) __attribute__((always_inline)) {
        if (j < T::NB)
            sx_next[j] = xsc[at + j * 32 * 16];
        else
            sw_next = wsc[at];
    };
    auto mfmas = [&](int h, auto&& extra) __attribute__((always_inline)) {
        static_for<kMfmas>([&](auto tc_) __attribute__((always_inline)) {
            constexpr int t = decltype(tc_)::value, a = t / T::NB, r = t % T::NB, b = (a & 1) ? T::NB - 1 - r : r;
            mfma_fp8<kMfmas>(acc[a][b], fw[h][a], fx[h][b], sw, sx[b]);
            extra(tc_);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto spread = [](auto tc_, auto n_c, auto over_c, auto&& item) __attribute__((always_inline)) {
        constexpr int t = decltype(tc_)::value, n = decltype(n_c)::value, over = decltype(over_c)::value;
        constexpr int lo = t < over ? t * n / over : n, hi = t < over ? (t + 1) * n / over : n;
        static_for<hi - lo>([&](auto i) __attribute__((always_inline)) { item(lo + decltype(i)::value); });
    };
    using Reads = std::integral_constant<int, kReads>;
    using ReadsAll = std::integral_constant<int, kReads + kScales>;
    using LoadsW = std::integral_constant<int, T::kLoadsW>;
    using LoadsX = std::integral_constant<int, T::kLoadsX>;
    using Most = std::integral_constant<int, (kMfmas * 3 + 3) / 4>;
    using All = std::integral_constant<int, kMfmas>;

    // As in gemm_k_loop, with the first segments of the scales ahead of all.
    for (int s = 0; s < min(segments, T::kSegs); ++s) dma_segment(s);
    const i32x4 none{0, 0, 0, kBufferWord3};
#pragma unroll
    for (int i = 0; i < SW - 1; ++i) {
        const int ix = i + 1 - SW + SX;
#pragma unroll
        for (int j = 0; j < T::kLoadsW; ++j) dma_w1(i < nk ? rw : none, (uint32_t)(i * T::kWBytes), j, i == nk - 1);
        gemm_advance(rw);
        if (ix < 0) continue;
#pragma unroll
        for (int j = 0; j < T::kLoadsX; ++j) dma_x1(ix < nk ? rx : none, (uint32_t)(ix * T::kXBytes), j, ix == nk - 1);
        gemm_advance(rx);
    }
#pragma unroll
    for (int a = 0; a < T::NA; ++a)
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            acc[a][b] = f32x16{};
            if constexpr (kMfmas >= 8) asm volatile("" : "+a"(acc[a][b]));
        }
    wait_vm_lgkm<(SX - 1) * (T::kLoadsW + T::kLoadsX)>();  // K step 0 and the scales (own loads) landed
    barrier();
#pragma unroll
    for (int j = 0; j < kReads; ++j) read1(0, 0, 0, j);
    // The next step's byte in the ring; `turn`: steps to the end of its segment.
    uint32_t at = (uint32_t)scales.first % kSegSteps;
    int turn = kSegSteps - (int)at, segment = 0;
#pragma unroll
    for (int j = 0; j < kScales; ++j) read_scale(at, j);

    uint32_t cw = 0, pw = (SW - 1) * T::kWBytes, cx = 0;
    int kt = 0;
    auto step = [&](auto left_c) __attribute__((always_inline)) {
        constexpr int left = decltype(left_c)::value;  // SW: that many or more
        constexpr int kAheadW = left - (SW - SX) < SX - 1 ? left - (SW - SX) : SX - 1;
        constexpr int kAheadX = left - 1 < SX - 2 ? left - 1 : SX - 2;
        const uint32_t nw = cw == (SW - 1) * T::kWBytes ? 0u : cw + T::kWBytes;
        const uint32_t nx = cx == (SX - 1) * T::kXBytes ? 0u : cx + T::kXBytes;
        sw = sw_next;
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            sx[b] = sx_next[b];
            asm volatile("" : "+v"(sx[b]));
        }
        // (Two wait states between a VALU write and an MFMA that reads the register;
        // the compiler does not see that inline asm is one.)
        asm volatile("s_nop 1" : "+v"(sw), "+v"(sx[0]), "+v"(sx[T::NB - 1]));
        // The next step's scales: on in the segment, or at the start of the next one.
        // Then the segment before it is read no more (after this step's barrier), and
        // the one a ring ahead of it is loaded there.
        bool fresh = false;
        ++at;
        if (--turn == 0) {
            turn = kSegSteps;
            ++segment;
            at = segment % T::kSegs == 0 ? 0 : at + (T::kSegBytes - kSegSteps);
            fresh = true;
        }
        mfmas(0, [&](auto t) __attribute__((always_inline)) {
            spread(t, Reads{}, Most{}, [&](int i) __attribute__((always_inline)) { read1(cw, cx, 1, i); });
            if constexpr (left >= SW - 1)
                spread(t, LoadsW{}, All{}, [&](int i) __attribute__((always_inline)) { dma_w1(rw, pw, i, left == SW - 1); });
        });
        wait_vm_lgkm<(kAheadW > 0 ? kAheadW : 0) * T::kLoadsW + (kAheadX > 0 ? kAheadX : 0) * T::kLoadsX>();
        barrier();
        // (In the last steps none is left to load: it would be read a ring later.)
        if constexpr (left >= SW)
            if (fresh && segment + T::kSegs - 1 < segments) dma_segment(segment + T::kSegs - 1);
        mfmas(1, [&](auto t) __attribute__((always_inline)) {
            if constexpr (left > 0)
                spread(t, ReadsAll{}, All{}, [&](int i) __attribute__((always_inline)) {
                    if (i < kReads)
                        read1(nw, nx, 0, i);
                    else
                        read_scale(at, i - kReads);
                });
            if constexpr (left >= SX)
                spread(t, LoadsX{}, Most{}, [&](int i) __attribute__((always_inline)) { dma_x1(rx, cx, i, left == SX); });
        });
        gemm_advance(rw);
        gemm_advance(rx);
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
    // The last MFMAs write their results before they are read (gemm_tile.h).
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
}

}  // namespace
}  // namespace h3a
