// The matrix product of the 8-bit GEMM kernels (gfx950): C^T = W X^T of one tile over
// e4m3 operands with K contiguous and a power of two for each 128 values of K,
// accumulated in fp32 on v_mfma_scale_f32_32x32x64_f8f6f4. A K step of 128 is a scale's
// block and the 128 bytes of a row that gemm_tile.h's K step of 64 bf16 is, so stages,
// loads and swizzle are that file's; what differs:
//   - fragments are 32 rows x 64 K, 32 bytes a lane: lane l holds of row l & 31 the
//     16-byte chunks 4h + (l >> 5) and 4h + 2 + (l >> 5) of half h, of W and X alike;
//   - a lane of the result holds token l & 31 of its block and, in group g of four,
//     rows 8g + 4 (l >> 5) .. +3 of W;
//   - the scales of the tile's tokens and of its one or two blocks of W rows lie in a
//     ring of segments behind the stages: 16 K steps' bytes of each token, as they lie
//     in memory, loaded once. A lane reads the byte of its token for the K step ahead,
//     with the fragments. (Both operands' scales go into the instruction: the sums need
//     no multiplication of their own.) The largest tile's stages leave no LDS for a
//     ring: there a lane holds its rows' bytes of up to 48 K steps in registers.
//   - the large tiles read all fragments of an X stage half a K step earlier (kEarlyX).
// A K step of a 256 x 256 tile takes 2,400 cycles where its MFMAs take 2,048; the others
// are gaps between MFMAs on end, the barriers, and MFMAs held up by the fragments' reads,
// the scales and the loads, which overlap. It writes 64 KB to LDS and reads 128: at 128
// bytes a cycle 1,536 cycles, three quarters of the MFMAs' and 64% of the step's. A wave
// per SIMD with 128 x 128 of the result is what keeps it there.
#pragma once

#include "gemm_tile.h"

namespace h3a {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kP8K = 128;       // K of a step
constexpr int kSegSteps = 16;   // K steps of a segment of scales
constexpr int kHeldSegs = 3;    // segments that a lane holds in registers

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
    // Waves over features and tokens: the smaller side of what they read of LDS per MFMA.
    // (128 x 128: 2 x 2, 22.2 us at 390 x 5,376 x 5,376, 22.8 by 4 x 1.)
    static constexpr int WN = (TF == 256 && NT >= 10) || (TF == 128 && NT == 8) ? 2 : 4, WM = kPWaves / WN;
    static constexpr int NA = TF / 32 / WN, NB = NT / 2 / WM;  // 32 x 32 MFMA blocks of a wave
    static constexpr int kWBytes = TF * kPRow, kXBytes = kTokens * kPRow;
    static constexpr int kXBase = SW * kWBytes, kStages = kXBase + SX * kXBytes;
    static constexpr int kLoadsW = TF / 8 / kPWaves, kLoadsX = kTokens / 8 / kPWaves;
    // A segment: 16 bytes for each token, then for each of the two blocks of W rows.
    static constexpr int kSegLoads = (kTokens + 63) / 64, kSegW = kSegLoads * 1024, kSegBytes = kSegW + 64;
    static constexpr int kSegRoom = (160 * 1024 - kStages) / kSegBytes, kSegs = kSegRoom < 8 ? kSegRoom : 8;
    static constexpr bool kScaleRegs = kSegs == 0;
    static constexpr int kFirstSeg = kScaleRegs ? (SW - 1) * kWBytes : kStages;  // (a stage that is loaded last)
    // The product at twice bf16's rate needs a stage of X 1.2 us ahead, of which two
    // stages that are held until their K step's middle give half to one step (1.06 us
    // at 256 x 256). So a step's X fragments are all read in the half step before it,
    // those of its second half as the current ones are used up, and the stage is
    // loaded again from the step's start on, after a barrier of its own.
    static constexpr bool kEarlyX = TF == 256;
    static constexpr int kLds = kStages + kSegs * kSegBytes;
    // Blocks of tokens of a wave that the epilogue takes at a time: all, or what fits.
    static constexpr int kPass = kTokens * (TF + 1) * 4 <= 160 * 1024 ? NB : NB % 2 == 0 ? NB / 2 : 1;
    static constexpr int kEpiRows = 32 * kPass * WM * TF * 4, kEpiBytes = kEpiRows + kTokens * 4;
    static constexpr int kSmem = kLds > kEpiBytes ? kLds : kEpiBytes;
    static_assert(NT % 2 == 0 && TF % 128 == 0, "DMA map: whole loads per wave");
    static_assert(NA * WN * 32 == TF && 2 * NB * WM == NT && NB % kPass == 0, "wave map");
    static_assert(SX >= 2 && (kEarlyX ? SW >= SX : SW > SX), "the waits below count loads in this order");
    static_assert((kScaleRegs ? kHeldSegs * kSegBytes <= kWBytes && kEarlyX : (kSegs - 2) * kSegSteps >= SW) && kSmem <= 160 * 1024,
                  "LDS of one workgroup");

    // Loads of one wave that may be in flight in the middle of a K step with `left`
    // steps behind it, the next step's having landed. kEarlyX: stage X[i] is loaded in
    // the first half of step i - SX, W[i] in the second half of step i - SW; else W[i]
    // in the first half of step i + 1 - SW and X[i] in the second half of step i - SX.
    static constexpr int in_flight(int left) {
        // (half steps, the present one's second half being 1)
        const int w1 = kEarlyX ? 2 * (1 - SW) + 1 : 2 * (2 - SW), x1 = kEarlyX ? 2 * (1 - SX) : 2 * (1 - SX) + 1;
        const int newest = w1 > x1 ? w1 : x1;
        int n = 0;
        for (int i = 2; i <= left; ++i) {
            const int w = w1 + 2 * (i - 1), x = x1 + 2 * (i - 1);
            n += (w > newest && w < 1 ? kLoadsW : 0) + (x > newest && x < 1 ? kLoadsX : 0);
        }
        return n;
    }
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

// acc += W X^T over nk K steps (kScaleRegs: in at most kHeldSegs segments); all waves of
// the workgroup call it. On return no load is in flight and no wave reads the stages any
// more. kTailK: the last K step is partial. w_block: per lane, which of the two blocks of
// W rows its fragment row belongs to.
template <typename T, bool kTailK = false>
__device__ __forceinline__ void gemm_fp8_k_loop(const GemmRows& w_rows, const GemmRows& x_rows, const GemmScales& scales,
                                                const int nk, char* smem, int lane, int wave, int wn, int wm, int w_block,
                                                f32x16 (&acc)[T::NA][T::NB]) {
    constexpr int SW = T::kSW, SX = T::kSX;
    constexpr bool kEarlyX = T::kEarlyX, kScaleRegs = T::kScaleRegs;
    i32x4 rw = w_rows.rsrc, rx = x_rows.rsrc;
    const uint32_t dw = w_rows.lane, dx = x_rows.lane;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char*)smem;
    const uint32_t lds_wave = lds0 + (uint32_t)wave * 1024u;
    uint32_t sow[T::kLoadsW], sox[T::kLoadsX];
#pragma unroll
    for (int j = 0; j < T::kLoadsW; ++j) sow[j] = (uint32_t)j * w_rows.step;
#pragma unroll
    for (int j = 0; j < T::kLoadsX; ++j) sox[j] = (uint32_t)j * x_rows.step;
    auto dma_w1 = [&](uint32_t stage, int j, bool last = false) __attribute__((always_inline)) {
        gemm_dma(rw, kTailK && last ? w_rows.tail : dw, sow[j], lds_wave + stage, j);
    };
    auto dma_x1 = [&](uint32_t stage, int j, bool last = false) __attribute__((always_inline)) {
        gemm_dma(rx, kTailK && last ? x_rows.tail : dx, sox[j], lds_wave + T::kXBase + stage, j);
    };
    // Segment s of the scales into slot s of the ring, the work spread over the waves
    // (a wave's loads differ in number; they come before, or in the middle of, the
    // counted ones, which then are waited for a little early at worst).
    constexpr int kSlots = kScaleRegs ? kHeldSegs : T::kSegs;
    const int first_segment = scales.first / kSegSteps, segments = (scales.first + nk - 1) / kSegSteps - first_segment + 1;
    auto dma_segment = [&](int s) __attribute__((always_inline)) {
        const uint32_t to = lds0 + T::kFirstSeg + (uint32_t)(s % kSlots) * T::kSegBytes, from = (uint32_t)(first_segment + s) * kSegSteps;
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
    const lds_char* const xsc = lds + T::kFirstSeg + (wm * 32 * T::NB + l31) * 16;
    const lds_char* const wsc = lds + T::kFirstSeg + T::kSegW + w_block * 32;
    int sw = 0, sx[T::NB], sw_next = 0, sx_next[T::NB];
    // kScaleRegs: the bytes of the next step and those after it, W's last.
    constexpr int kScales = T::NB + 1;
    uint32_t held[kScaleRegs ? kScales : 1][4 * kHeldSegs];

    i32x8 fw[2][T::NA], fx[2][T::NB];
    constexpr int kMfmas = T::NA * T::NB;

    // 16-byte piece i of the fragment of block b of half h of a stage at byte offset c.
    auto read_x = [&](uint32_t c, int h, int b, int i) __attribute__((always_inline)) {
        const i32x4 v = *(const lds_i32x4*)(xfr + c + fo[h][i] + b * 32 * kPRow);
        if (i == 0) fx[h][b].lo = v; else fx[h][b].hi = v;
    };
    auto read_w = [&](uint32_t c, int h, int a, int i) __attribute__((always_inline)) {
        const i32x4 v = *(const lds_i32x4*)(wfr + c + fo[h][i] + a * 32 * kPRow);
        if (i == 0) fw[h][a].lo = v; else fw[h][a].hi = v;
    };
    // Both operands' pieces of half h, X's first.
    constexpr int kReads = 2 * (T::NA + T::NB);
    auto read1 = [&](uint32_t cw, uint32_t cx, int h, int j) __attribute__((always_inline)) {
        if (j < 2 * T::NB)
            read_x(cx, h, j >> 1, j & 1);
        else
            read_w(cw, h, (j >> 1) - T::NB, j & 1);
    };
    // Scale j of the next K step, whose byte lies at `at` in the ring.
    auto read_scale = [&](uint32_t at, int j) __attribute__((always_inline)) {
        if constexpr (kScaleRegs) {
            // (a new dword's first byte is in place)
            const uint32_t by = (at & 3) == 0 ? 0 : 8;
            asm volatile("v_lshrrev_b32 %0, %1, %0" : "+v"(held[j][0]) : "s"(by));
        } else if (j < T::NB)
            sx_next[j] = *(lds_u8*)(xsc + at + j * 32 * 16);
        else
            sw_next = *(lds_u8*)(wsc + at);
    };
    // The next dword of the segment to the front, or (at its end) the next segment. (In
    // place by asm: the compiler would keep both sides of the branch around it in
    // registers of their own and move all to one at its end.)
    auto move_held = [&](int j, int to, int from) __attribute__((always_inline)) {
        asm volatile("v_mov_b32 %0, %1" : "+v"(held[j][to]) : "v"(held[j][from]));
    };
    auto next_dword = [&](uint32_t at) __attribute__((always_inline)) {
        if (at % kSegSteps != 0) {
#pragma unroll
            for (int j = 0; j < (kScaleRegs ? kScales : 0); ++j)
#pragma unroll
                for (int e = 0; e < 3; ++e) move_held(j, e, e + 1);
        } else {
#pragma unroll
            for (int j = 0; j < (kScaleRegs ? kScales : 0); ++j)
#pragma unroll
                for (int e = 0; e < 4 * (kHeldSegs - 1); ++e) move_held(j, e, e + 4);
        }
    };
    // The MFMAs of half h, with `extra(t)` issued after MFMA t: feature block major,
    // token blocks snaking, or (kByToken) the other way round.
    auto mfmas = [&](int h, auto by_token, auto&& extra) __attribute__((always_inline)) {
        static_for<kMfmas>([&](auto tc_) __attribute__((always_inline)) {
            constexpr int t = decltype(tc_)::value;
            constexpr bool kByToken = decltype(by_token)::value;
            constexpr int kInner = kByToken ? T::NA : T::NB, o = t / kInner, r = t % kInner, i = (o & 1) ? kInner - 1 - r : r;
            constexpr int a = kByToken ? i : o, b = kByToken ? o : i;
            mfma_fp8<kMfmas>(acc[a][b], fw[h][a], fx[h][b], sw, sx[b]);
            extra(tc_);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // n items spread over MFMAs from .. to - 1: those that follow MFMA t.
    auto spread = [](auto tc_, auto n_c, auto from_c, auto to_c, auto&& item) __attribute__((always_inline)) {
        constexpr int n = decltype(n_c)::value, from = decltype(from_c)::value, over = decltype(to_c)::value - from;
        constexpr int t = decltype(tc_)::value - from;
        constexpr int lo = t < 0 ? 0 : t < over ? t * n / over : n, hi = t < 0 ? 0 : t < over ? (t + 1) * n / over : n;
        static_for<hi - lo>([&](auto i) __attribute__((always_inline)) { item(lo + decltype(i)::value); });
    };
#define H3A_C(n) std::integral_constant<int, (n)>{}

    // The first segments of the scales, then the stages in the order of the loop below
    // (those before step 0; of steps past the end of a short reduction the lanes' offsets
    // are outside the records: they load zeros, so that the waits count the same).
    for (int s = 0; s < min(segments, kSlots); ++s) dma_segment(s);
    auto lane_at = [&](int i, uint32_t lane_off, uint32_t tail) __attribute__((always_inline)) {
        return i < nk - 1 ? lane_off : i == nk - 1 ? (kTailK ? tail : lane_off) : 0x80000000u;
    };
    auto load_x = [&](int i) __attribute__((always_inline)) {
        const uint32_t off = lane_at(i, dx, x_rows.tail);
#pragma unroll
        for (int j = 0; j < T::kLoadsX; ++j) gemm_dma(rx, off, sox[j], lds_wave + T::kXBase + (uint32_t)(i * T::kXBytes), j);
        gemm_advance(rx);
    };
    auto load_w = [&](int i) __attribute__((always_inline)) {
        const uint32_t off = lane_at(i, dw, w_rows.tail);
#pragma unroll
        for (int j = 0; j < T::kLoadsW; ++j) gemm_dma(rw, off, sow[j], lds_wave + (uint32_t)(i * T::kWBytes), j);
        gemm_advance(rw);
    };
    if constexpr (kEarlyX) {
#pragma unroll
        for (int j = -SW; j < 0; ++j) {
            if (j + SX >= 0) load_x(j + SX);
            if (!kScaleRegs || j < -1) load_w(j + SW);
        }
        // K step 0 and the scales (own loads) landed
        if constexpr (SW > SX)
            wait_vm_lgkm<(kScaleRegs ? SX - 1 : SX) * T::kLoadsW + (SX - 1) * T::kLoadsX>();
        else
            wait_vm_lgkm<(SX - 1) * (T::kLoadsW + T::kLoadsX)>();
    } else {
#pragma unroll
        for (int j = 1 - SW; j < 0; ++j) {
            load_w(j + SW - 1);
            if (j + SX >= 0) load_x(j + SX);
        }
        wait_vm_lgkm<(SX - 1) * (T::kLoadsW + T::kLoadsX)>();
    }
    barrier();
    uint32_t at = (uint32_t)scales.first % kSegSteps;  // the next step's byte in the ring
    int turn = kSegSteps - (int)at, segment = 0;       // steps to the end of its segment
    if constexpr (kScaleRegs) {
#pragma unroll
        for (int j = 0; j < kScales; ++j)
#pragma unroll
            for (int s = 0; s < kHeldSegs; ++s) {
                const i32x4 v = *(const lds_i32x4*)((j < T::NB ? xsc + j * 32 * 16 : wsc) + s * T::kSegBytes);
#pragma unroll
                for (int e = 0; e < 4; ++e) held[j][4 * s + e] = (uint32_t)v[e];
            }
#pragma unroll
        for (int j = 0; j < kScales; ++j)
#pragma unroll
            for (int e = 0; e < 4 * kHeldSegs; ++e) asm volatile("" : "+v"(held[j][e]));
        barrier();  // every wave has read the stage's place
        load_w(SW - 1);
        for (uint32_t i = 1; i <= at / 4; ++i) next_dword(4 * i);
#pragma unroll
        for (int j = 0; j < kScales; ++j) held[j][0] >>= 8 * (at & 3);
    } else {
#pragma unroll
        for (int j = 0; j < kScales; ++j) read_scale(at, j);
    }
#pragma unroll
    for (int j = 0; j < kReads; ++j) read1(0, 0, 0, j);
    if constexpr (kEarlyX) {
#pragma unroll
        for (int j = 0; j < 2 * (T::NB - 1); ++j) read_x(0, 1, j >> 1, j & 1);
    }

    // K step kt in the stages at `cw` and `cx`, its first-half fragments in set 0.
    // First half: the MFMAs of set 0, while set 1 is read from the same stages. Then the
    // wave's own loads of step kt + 1 are waited for (later ones stay in flight), with
    // its reads of the stages; after the barrier every wave's part of step kt + 1 is in
    // LDS, and step kt's stages are read no more. Second half: the MFMAs of set 1, while
    // step kt + 1's fragments are read into set 0, its scales too. W goes into the stage
    // before `cw` in the first half, X into `cx` in the second.
    // kEarlyX: X's set 1 has been read with set 0, block by block behind the MFMAs that
    // use the one before it, but for the last block, which comes first here; after a
    // barrier the step's X stage is loaded again in the first half, its W stage in the
    // second.
    // (The last reads of a half go out a few MFMAs before its end, which waits for them.)
    // `left` K steps follow; the last steps run out of loads, the last one reads nothing.
    uint32_t cw = 0, pw = (SW - 1) * T::kWBytes, cx = 0;
    int kt = 0;
    constexpr int kXAt = kMfmas >= 8 ? kMfmas / 4 : 1;  // MFMAs before the barrier of the X stage
    auto step = [&](auto left_c) __attribute__((always_inline)) {
        constexpr int left = decltype(left_c)::value;  // the largest: that many or more
        const uint32_t nw = cw == (SW - 1) * T::kWBytes ? 0u : cw + T::kWBytes;
        const uint32_t nx = cx == (SX - 1) * T::kXBytes ? 0u : cx + T::kXBytes;
        sw = kScaleRegs ? (int)held[kScaleRegs ? T::NB : 0][0] : sw_next;
#pragma unroll
        for (int b = 0; b < T::NB; ++b) {
            sx[b] = kScaleRegs ? (int)held[kScaleRegs ? b : 0][0] : sx_next[b];
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
        if constexpr (!kScaleRegs) {
            if (--turn == 0) {
                turn = kSegSteps;
                ++segment;
                at = segment % kSlots == 0 ? 0 : at + (T::kSegBytes - kSegSteps);
                fresh = true;
            }
        }
        mfmas(0, std::false_type{}, [&](auto t) __attribute__((always_inline)) {
            if constexpr (kEarlyX) {
                if constexpr (decltype(t)::value == 0) {
                    read_x(cx, 1, T::NB - 1, 0);
                    read_x(cx, 1, T::NB - 1, 1);
                }
                if constexpr (decltype(t)::value == kXAt - 1 && left >= SX) {
                    asm volatile("" : "+v"(fx[1][T::NB - 1]));  // (read)
                    barrier();
                }
                spread(t, H3A_C(2 * T::NA), H3A_C(kXAt), H3A_C(kMfmas - 3), [&](int i) __attribute__((always_inline)) { read_w(cw, 1, i >> 1, i & 1); });
                if constexpr (left >= SX)
                    spread(t, H3A_C(T::kLoadsX), H3A_C(kXAt), H3A_C(kMfmas), [&](int i) __attribute__((always_inline)) { dma_x1(cx, i, left == SX); });
            } else {
                spread(t, H3A_C(kReads), H3A_C(0), H3A_C((kMfmas * 3 + 3) / 4), [&](int i) __attribute__((always_inline)) { read1(cw, cx, 1, i); });
                if constexpr (left >= SW - 1)
                    spread(t, H3A_C(T::kLoadsW), H3A_C(0), H3A_C(kMfmas), [&](int i) __attribute__((always_inline)) { dma_w1(pw, i, left == SW - 1); });
            }
        });
        wait_vm_lgkm<T::in_flight(left)>();
        barrier();
        // (In the last steps none is left to load: it would be read a ring later.)
        if constexpr (left >= SW && !kScaleRegs)
            if (fresh && segment + kSlots - 1 < segments) dma_segment(segment + kSlots - 1);
        if constexpr (kScaleRegs) {
            if ((at & 3) == 0) next_dword(at);
        }
        mfmas(1, std::integral_constant<bool, kEarlyX>{}, [&](auto t) __attribute__((always_inline)) {
            // (The scales first: the next step's first MFMA needs them all.)
            constexpr int kFirst = kScales;
            if constexpr (left > 0) {
                spread(t, H3A_C(kReads + kFirst), H3A_C(0), H3A_C(kEarlyX ? kMfmas - 2 : kMfmas), [&](int i) __attribute__((always_inline)) {
                    if (i >= kFirst)
                        read1(nw, nx, 0, i - kFirst);
                    else
                        read_scale(at, i);
                });
                constexpr int tv = decltype(t)::value, done = tv / T::NA - 1;
                if constexpr (kEarlyX && tv % T::NA == 0 && done >= 0) {
                    read_x(nx, 1, done, 0);
                    read_x(nx, 1, done, 1);
                }
            }
            if constexpr (kEarlyX) {
                if constexpr (left >= SW)
                    spread(t, H3A_C(T::kLoadsW), H3A_C(0), H3A_C(kMfmas), [&](int i) __attribute__((always_inline)) { dma_w1(cw, i, left == SW); });
            } else if constexpr (left >= SX) {
                spread(t, H3A_C(T::kLoadsX), H3A_C(0), H3A_C((kMfmas * 3 + 3) / 4), [&](int i) __attribute__((always_inline)) { dma_x1(cx, i, left == SX); });
            }
        });
        gemm_advance(rw);
        gemm_advance(rx);
        pw = cw;
        cw = nw;
        cx = nx;
        ++kt;
    };
#undef H3A_C
    // (From kMost on, a step's loads are all wanted and none is the last.)
    constexpr int kMost = kEarlyX ? SW + 1 : SW;
    while (kt < nk - kMost) step(std::integral_constant<int, kMost>{});
    // The last min(kMost, nk) steps.
    auto tail = [&](auto self, auto left_c) __attribute__((always_inline)) -> void {
        constexpr int left = decltype(left_c)::value;
        if (left < nk) step(left_c);
        if constexpr (left > 0) self(self, std::integral_constant<int, left - 1>{});
    };
    tail(tail, std::integral_constant<int, kMost - 1>{});
    // The last MFMAs write their results before they are read (gemm_tile.h).
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
}

}  // namespace
}  // namespace h3a
