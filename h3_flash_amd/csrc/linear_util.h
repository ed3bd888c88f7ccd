// What follows a linear layer's product (gfx950), for the kernels that finish it:
// bias, activation or gated activation, modulation gate and residual.
#pragma once

#include "common.h"
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

// y of token m, features f .. f+3, from their sums (gated: z[0] of the values,
// z[1] of the gates).
template <int kS>
__device__ __forceinline__ f32x4 finished4(const LinearParams& p, f32x4 (&z)[kS], int m, int f) {
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
    return y;
}

template <int kS>
__device__ __forceinline__ void finish4(const LinearParams& p, f32x4 (&z)[kS], int m, int f) {
    const f32x4 y = finished4<kS>(p, z, m, f);
    *(i32x2*)((char*)p.y + m * p.y_rs + 2 * f) = i32x2{(int)pack_bf16x2(y[0], y[1]), (int)pack_bf16x2(y[2], y[3])};
}

}  // namespace
}  // namespace h3a
