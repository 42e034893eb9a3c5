// 8-bit floating point in blocks of 128 values that share a power-of-two scale.
//
// Formats: e4m3 (largest 448 = 1.75 * 2^8) and e5m2 (57344 = 1.75 * 2^15).  A
// block's scale is 2^e with the least e >= -127 for which its largest magnitude
// over 2^e is no larger than the format's largest number (e = 0 for a block of
// zeros), kept as the byte e + 127.  A value divided by a power of two is exact
// (but where it underflows), so a code has one rounding, to the nearest, ties
// to even.  A block with an infinity or a NaN has the scale NaN (0xff) and codes
// NaN (0x7f): whatever is computed from it is NaN.
#pragma once

#include "gdn_common.hpp"

namespace {

constexpr int kBlk = 128;

template <int FMT>  // GDN_E4M3 or GDN_E5M2
struct Fp8 {
    static constexpr int top = FMT == GDN_E4M3 ? 8 : 15;
    // Scale byte of a block whose largest magnitude has the bits `amax`.
    __device__ __forceinline__ static uint32_t scale_byte(uint32_t amax) {
        if (amax >= 0x7f800000u) return 0xffu;
        if (amax == 0) return 127u;
        // amax = m 2^E, 1 <= m < 2: e = E - top where m <= 1.75, else one more;
        // numbers below 2^-126 lie under the least scale's range.
        const int b = static_cast<int>(amax >> 23) - top + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
        return static_cast<uint32_t>(b < 0 ? 0 : b);
    }
    // 2^-e of a scale byte.
    __device__ __forceinline__ static float inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
    // Codes of four values times inv (a scale's inverse), all NaN where bad.
    __device__ __forceinline__ static uint32_t codes4(float a, float b, float c, float d, float inv, bool bad) {
        int v = 0;
        if constexpr (FMT == GDN_E4M3) {
            v = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, v, false);
            v = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, v, true);
        } else {
            v = __builtin_amdgcn_cvt_pk_bf8_f32(a * inv, b * inv, v, false);
            v = __builtin_amdgcn_cvt_pk_bf8_f32(c * inv, d * inv, v, true);
        }
        return bad ? 0x7f7f7f7fu : static_cast<uint32_t>(v);
    }
    __device__ __forceinline__ static gdn::u32x2 codes8(const float* f, float inv, bool bad) {
        return gdn::u32x2{codes4(f[0], f[1], f[2], f[3], inv, bad), codes4(f[4], f[5], f[6], f[7], inv, bad)};
    }
};

// The largest magnitude's bits among eight values (as whole numbers infinities
// and NaN rank above every finite one).
__device__ __forceinline__ uint32_t amax8(const float* f) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
// Maximum over each 16 lanes (the lanes of a block of 128), in every lane.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, dpp_u<0xB1>(v));   // quad_perm [1,0,3,2]
    v = max(v, dpp_u<0x4E>(v));   // quad_perm [2,3,0,1]
    v = max(v, dpp_u<0x141>(v));  // row_half_mirror
    return max(v, dpp_u<0x140>(v));  // row_mirror
}

}  // namespace
