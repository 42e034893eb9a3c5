// 4-bit floating point (e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) in
// blocks of 32 values that share a power-of-two scale.
//
// A block's scale is 2^e with the least e >= -127 for which its largest magnitude
// over 2^e is no larger than 6 (e = 0 for a block of zeros), kept as the byte e +
// 127: nothing is cut off at 6, which would cost the largest value up to a quarter.
// A value divided by a power of two is exact (but where it underflows), so a code
// has one rounding, to the nearest, ties to even.  A block with an infinity or a
// NaN has the scale NaN (0xff) and codes of zero: whatever is computed from it is
// NaN.
//
// Codes lie two a byte, the earlier one low, rows padded with zero codes to 256
// values (128 bytes).  Scales lie by blocks of 128 values, a row's four bytes in a
// word: [K / 128][rows][4], so that what a product reads of them for a step along K
// is adjacent.
#pragma once

#include "gdn_common.hpp"

namespace {

constexpr int kFp4Row = 256;  // values a code row is padded to

// Scale byte of a block whose largest magnitude has the bits `amax`.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax) {
    if (amax >= 0x7f800000u) return 0xffu;
    if (amax == 0) return 127u;
    // amax = m 2^E, 1 <= m < 2: e = E - 2 where m <= 1.5, else one more; numbers
    // below 2^-126 lie under the least scale's range.
    const int b = static_cast<int>(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x400000u ? 1 : 0);
    return static_cast<uint32_t>(b < 0 ? 0 : b);
}
// 2^-e of a scale byte (of a finite block: 253 at most).
__device__ __forceinline__ float fp4_inverse(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }

// Codes of eight values times inv (a scale's inverse), the first one lowest; zeros where bad.
__device__ __forceinline__ uint32_t fp4_codes8(const float* f, float inv, bool bad) {
    uint32_t v = 0;
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, f[0] * inv, f[1] * inv, 1.f, 0);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, f[2] * inv, f[3] * inv, 1.f, 1);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, f[4] * inv, f[5] * inv, 1.f, 2);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, f[6] * inv, f[7] * inv, 1.f, 3);
    return bad ? 0u : v;
}
// Four values' codes in the low 16 bits.
__device__ __forceinline__ uint32_t fp4_codes4(float a, float b, float c, float d, float inv, bool bad) {
    uint32_t v = 0;
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, a * inv, b * inv, 1.f, 0);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, c * inv, d * inv, 1.f, 1);
    return bad ? 0u : v;
}

// Eight codes times a power of two as bf16, exactly (an e8m0 byte s as the fp32 bits
// s << 23, of which the instruction reads the exponent alone: 0 is 2^-127 and 255
// NaN).  The smallest, 2^-128, is a subnormal that the bf16 MFMA keeps; beyond
// bf16's largest (6 2^126) lies infinity.
__device__ __forceinline__ gdn::bf16x8 fp4_to_bf16(uint32_t codes, uint32_t scale_byte) {
    const float s = __uint_as_float(scale_byte << 23);
    union {
        gdn::bf16x2 p[4];
        gdn::bf16x8 v;
    } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
    return u.v;
}

}  // namespace
