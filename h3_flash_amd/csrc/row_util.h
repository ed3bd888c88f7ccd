// Helpers of the row kernels (gfx950): rows of bf16 held 16 bytes per lane and
// vector, weights and modulation tables in bf16 or fp32, sums over a row.
#pragma once

#include "common.h"

namespace h3a {
namespace {

constexpr int kThreads = 256;  // one row per workgroup in the norm kernels
constexpr int kWaves = kThreads / 64;

__device__ __forceinline__ void unpack8(i32x4 raw, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)raw[i];
        f[2 * i] = __uint_as_float(w << 16);
        f[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
}

__device__ __forceinline__ i32x4 pack8(const float* f) {
    i32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (int)pack_bf16x2(f[2 * i], f[2 * i + 1]);
    return r;
}

__device__ __forceinline__ float load1(const void* base, int64_t idx, bool f32) {
    return f32 ? ((const float*)base)[idx] : bf16_to_f32(((const uint16_t*)base)[idx]);
}

// Modulation-table row of a token: index[row mod n_index], clamped to the table.
template <typename Params>
__device__ __forceinline__ int64_t table_row(const Params& p, int64_t row) {
    const int64_t i = row % p.n_index;
    int64_t t = p.index_i64 ? ((const int64_t*)p.index)[i] : (int64_t)((const int32_t*)p.index)[i];
    t = t < 0 ? 0 : t;
    return t >= p.table_rows ? p.table_rows - 1 : t;
}

// Sum of v over the workgroup (fixed order: lanes, then waves in order).
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += lds[w];
    return s;
}

// Eight consecutive bf16 (16 bytes) or fp32 (32 bytes) values as loaded,
// unpacked only when used, so that many loads can be in flight at once.
template <bool kF32>
struct Raw8 {
    i32x4 a;
    i32x4 b;  // second half of fp32 values; unused for bf16
};

template <bool kF32>
__device__ __forceinline__ Raw8<kF32> fetch8(const void* base, int64_t idx) {
    Raw8<kF32> r;
    if constexpr (kF32) {
        r.a = *(const i32x4*)((const float*)base + idx);
        r.b = *(const i32x4*)((const float*)base + idx + 4);
    } else {
        r.a = *(const i32x4*)((const uint16_t*)base + idx);
    }
    return r;
}

template <bool kF32>
__device__ __forceinline__ void unpack_raw8(const Raw8<kF32>& r, float* out) {
    if constexpr (kF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[i] = __int_as_float(r.a[i]);
            out[4 + i] = __int_as_float(r.b[i]);
        }
    } else {
        unpack8(r.a, out);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Eight values at byte offset `off` (of the bf16 column) of a row that starts
// at `base`: a uniform base and a 32-bit lane offset, one address register.
template <bool kF32>
__device__ __forceinline__ Raw8<kF32> fetch8o(const char* base, uint32_t off) {
    Raw8<kF32> r;
    if constexpr (kF32) {
        r.a = *(const i32x4*)(base + 2 * off);
        r.b = *(const i32x4*)(base + 2 * off + 16);
    } else {
        r.a = *(const i32x4*)(base + off);
    }
    return r;
}

}  // namespace
}  // namespace h3a
