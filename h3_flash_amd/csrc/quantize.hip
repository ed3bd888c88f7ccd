// Rounding to 8 bits (gfx950): rows of activations in groups of 128 columns, weights
// in blocks of 128 x 128, each with a power of two (fp8_util.h holds the arithmetic).
// Bound by HBM: 2 (bf16) or 4 (fp32) bytes read and 1 written a value, each once; a
// value stays in registers between its group's maximum and its rounding. Rows of 6,240 x
// 5,120: 17 to 19 us for 97 MB, 5.1 to 5.6 TB/s (a copy: 5.2); a weight of 28,672 x
// 5,376: 71 us for 463 MB, 6.5 TB/s (two thirds of it are reads).
#include "fp8_util.h"
#include "kernels.h"
#include "row_util.h"

namespace h3a {
namespace {

// Bits of the largest magnitude of eight values.
template <bool kF32>
__device__ __forceinline__ uint32_t top8(const Raw8<kF32>& r) {
    float v[8];
    unpack_raw8<kF32>(r, v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    return top;
}

template <bool kF32>
__device__ __forceinline__ i32x2 rounded8(const Raw8<kF32>& r, float inv) {
    float v[8];
    unpack_raw8<kF32>(r, v);
    return i32x2{fp8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), fp8x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
}

template <bool kF32>
__device__ __forceinline__ Raw8<kF32> fetch8nt(const char* at) {
    Raw8<kF32> r;
    r.a = __builtin_nontemporal_load((const i32x4*)at);
    if constexpr (kF32) r.b = __builtin_nontemporal_load((const i32x4*)(at + 16));
    return r;
}

// 16 lanes per group, 8 columns a lane; U groups a lane, all loaded before the first
// is rounded. Lanes past a row's end load its last columns, count for no group and
// store nothing.
template <bool kF32, int U>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(QuantizeParams p) {
    const uint32_t kb = (uint32_t)(p.cols + kFp8Group - 1) / kFp8Group, groups = (uint32_t)p.rows * kb;
    const uint32_t first = blockIdx.x * (U * kThreads / 16) + (threadIdx.x >> 4);
    const int lane = threadIdx.x & 15;
    Raw8<kF32> raw[U];
    uint32_t row[U], block[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t g = min(first + u * (kThreads / 16), groups - 1);
        row[u] = g / kb;
        block[u] = g - row[u] * kb;
        const int c = min((int)block[u] * kFp8Group + lane * 8, p.cols - 8);
        raw[u] = fetch8nt<kF32>((const char*)p.x + (int64_t)row[u] * p.x_rs + (int64_t)c * (kF32 ? 4 : 2));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = (int)block[u] * kFp8Group + lane * 8;
        const bool in = c < p.cols;
        const int s = fp8_exponent(group16_max(in ? top8<kF32>(raw[u]) : 0));
        if (!in || first + u * (kThreads / 16) >= groups) continue;
        *(i32x2*)((char*)p.q + (int64_t)row[u] * p.q_rs + c) = rounded8<kF32>(raw[u], fp8_inverse(s));
        if (lane == 0) p.scale[(int64_t)row[u] * p.scale_rs + block[u]] = (uint8_t)s;
    }
}

// A workgroup per block: 16 lanes a row, 16 rows at a time. Workgroup b: column
// block b mod kb, row block b / kb (those of the parts after one another).
template <bool kF32>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(QuantizeParams p) {
    constexpr int kIts = kFp8Group / (kThreads / 16);
    __shared__ uint32_t red[kWaves];
    const uint32_t kb = (uint32_t)(p.cols + kFp8Group - 1) / kFp8Group;
    const uint32_t rb = blockIdx.x / kb, block = blockIdx.x - rb * kb;
    const uint32_t per_part = (uint32_t)((p.part_rows + kFp8Group - 1) / kFp8Group), part = rb / per_part;
    const int64_t row0 = part * p.part_rows + (int64_t)(rb - part * per_part) * kFp8Group;
    const int rows = (int)min((int64_t)kFp8Group, (part + 1) * p.part_rows - row0);
    const int c = (int)block * kFp8Group + (threadIdx.x & 15) * 8, r = threadIdx.x >> 4;
    const bool in = c < p.cols;
    const char* const x = (const char*)p.x + (int64_t)min(c, p.cols - 8) * (kF32 ? 4 : 2);
    Raw8<kF32> raw[kIts];
#pragma unroll
    for (int i = 0; i < kIts; ++i) raw[i] = fetch8nt<kF32>(x + (row0 + min(r + 16 * i, rows - 1)) * p.x_rs);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kIts; ++i) top = max(top, top8<kF32>(raw[i]));
    // (A clamped row or column is one of the block's own: it counts twice.)
    top = group16_max(top);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = max(top, red[w]);
    const int s = fp8_exponent(top);
    const float inv = fp8_inverse(s);
    if (threadIdx.x == 0) p.scale[(int64_t)rb * p.scale_rs + block] = (uint8_t)s;
    if (!in) return;
#pragma unroll
    for (int i = 0; i < kIts; ++i)
        if (r + 16 * i < rows) *(i32x2*)((char*)p.q + (row0 + r + 16 * i) * p.q_rs + c) = rounded8<kF32>(raw[i], inv);
}

constexpr int kRowGroups = 4;  // groups a lane, but for small launches

template <bool kF32>
void launch_t(const QuantizeParams& p, hipStream_t stream) {
    const int64_t kb = (p.cols + kFp8Group - 1) / kFp8Group;
    if (p.blocks) {
        const int64_t n = p.rows / p.part_rows * ((p.part_rows + kFp8Group - 1) / kFp8Group) * kb;
        hipLaunchKernelGGL((quantize_blocks_kernel<kF32>), dim3((unsigned)n), dim3(kThreads), 0, stream, p);
        return;
    }
    const int64_t groups = p.rows * kb;
    auto grid = [&](int u) { return dim3((unsigned)((groups + u * (kThreads / 16) - 1) / (u * (kThreads / 16)))); };
    if (groups >= 1 << 16)
        hipLaunchKernelGGL((quantize_rows_kernel<kF32, kRowGroups>), grid(kRowGroups), dim3(kThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((quantize_rows_kernel<kF32, 1>), grid(1), dim3(kThreads), 0, stream, p);
}

}  // namespace

// A launch has at most 2^32 - 1 work items, in workgroups of 256: one for each block, or
// for 64 groups of rows (fewer in the last).
int64_t quantize_max_groups(bool blocks) { return (int64_t)(UINT32_MAX / kThreads) * (blocks ? 1 : kRowGroups * kThreads / 16); }

hipError_t launch_quantize(const QuantizeParams& p, hipStream_t stream) {
    if (p.rows == 0) return hipSuccess;
    p.x_f32 ? launch_t<true>(p, stream) : launch_t<false>(p, stream);
    return hipGetLastError();
}

}  // namespace h3a
