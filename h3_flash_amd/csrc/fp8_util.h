// Rounding to 8 bits (gfx950): groups of 128 values (or blocks of 128 x 128) as e4m3
// with one power of two s, held as e8m0 (the byte e of 2^(e - 127), 255 for NaN).
//   s = the smallest power of two, 2^-126 at the least, by which no value of the
//       group passes e4m3's largest, 448: max |x| <= 448 s
//   q = e4m3(x / s), to nearest, ties to even
// A group with a value that is not finite is NaN throughout, scale and values.
#pragma once

#include "common.h"

namespace h3a {
namespace {

constexpr int kFp8Group = 128;

// e of a group from the bits of its largest magnitude (as integers, magnitudes keep
// their order, and NaN lies above all). 448 = 1.75 2^8: a mantissa over 1.75 takes
// the next power.
__device__ __forceinline__ int fp8_exponent(uint32_t top) {
    const int e = max((int)((top + 0x1fffffu) >> 23) - 8, 1);
    return top >= 0x7f800000u ? 255 : e;
}

// 1 / s, exact; NaN for e = 255.
__device__ __forceinline__ float fp8_inverse(int e) { return __uint_as_float(e == 255 ? 0x7fc00000u : (uint32_t)(254 - e) << 23); }

// Four values as e4m3, the first in the lowest byte (v_cvt_pk_fp8_f32 rounds to
// nearest even; none passes 448 but NaN).
__device__ __forceinline__ int fp8x4(float a, float b, float c, float d) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// Maximum over aligned groups of 16 lanes; all lanes must be active.
__device__ __forceinline__ uint32_t group16_max(uint32_t v) {
    v = max(v, (uint32_t)dpp<kDppXor1>((int)v));
    v = max(v, (uint32_t)dpp<kDppXor2>((int)v));
    v = max(v, (uint32_t)dpp<kDppHalfMirror>((int)v));
    return max(v, (uint32_t)dpp<kDppMirror>((int)v));
}

}  // namespace
}  // namespace h3a
