// Parameter block and launches of the fp8 block-scaled product (fp8_matmul.hip
// holds its entry point and the rule that picks its kernel; fp8_tiles.hpp the
// tiled kernel, instantiated for each pair of formats in fp8_mm_*.hip).
#pragma once

#include "gdn_common.hpp"

namespace gdn_fp8 {

struct MatmulParams {
    const uint8_t *a, *b;        // codes [M, lda], [N, ldb]
    const uint8_t* a_scale;      // e8m0 [K / 128][lda_s]
    const void* b_scale;         // see Scales
    void* out;                   // [M, ldo] bf16 or fp32
    long long lda, ldb, lda_s, ldb_s, ldo;
    int M, N, K;
};

// b's scales: e8m0 or fp32, one a 128 x 128 block [ceil(N / 128)][ldb_s >= K / 128]
// or one a row and block of 128, [K / 128][ldb_s >= N].
enum Scales { kE8Block = 0, kE8Row = 1, kF32Block = 2, kF32Row = 3 };

// Tiles of the tiled kernel (columns x tokens), largest first; those before
// k128x128 for bf16 results alone.
enum Tile { k256x256 = 0, k256x192, k256x160, k256x128, k128x192, k128x128, k64x128, k64x64, k64x32, k32x32, k16x16Alone, k16x16 };

// Defined in fp8_mm_*.hip for each pair of formats (of a, of b).  f32: out is
// fp32 (and the products are summed in full, see fp8_tiles.hpp), else bf16.
template <int FA, int FB>
int launch_tile(int tile, int scales, bool f32, const MatmulParams& p, hipStream_t stream);

}  // namespace gdn_fp8

namespace {

using namespace gdn;

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 join(const u32x4 lo, const u32x4 hi) {
    return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
                 static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

// MFMA 16x16x128 of fp8 operands with fp32 sums: tokens (format FX) as the A
// operand, rows of W (format FW) as the B operand, so a lane's accumulator is
// one column (lane % 16) of four tokens (4 (lane / 16) + i), and neighbouring
// lanes store neighbouring columns.  Lane l supplies row l % 16 of its operand
// and 32 of the 128 k values, which 32 is free as long as both agree (one scale
// covers all 128).  SX, SW: byte of `sx`, `sw` that is the lane's row's e8m0
// scale; 127 is 1.
//
// The instruction lines a block's products up with the largest and drops what
// lies below about 2^-17 of that (measured: 2^-1 next to 1.75 * 2^16 is lost),
// 1.4e-5 of a sum over normal values: nothing beside a bf16 result's 2^-8 unless
// large products cancel, too much for an fp32 one.
template <int FX, int FW, int SX, int SW>
__device__ __forceinline__ f32x4 mfma_fp8(const i32x8 x, const i32x8 w, const f32x4 c, int sx, int sw) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, w, c, FX, FW, SX, sx, SW, sw);
}

// An fp32 scale as a power of two, which the instruction takes together with the
// other operand's scale (a product of the two alone may leave fp32's range where the
// result does not), and the rest, 1 to 2 in magnitude (0, infinite or NaN as the
// scale is).
__device__ __forceinline__ uint32_t scale_byte_of(uint32_t bits) { return min(bits >> 23 & 0xffu, 254u); }
__device__ __forceinline__ float scale_rest(uint32_t bits, uint32_t byte) {
    return __builtin_amdgcn_ldexpf(__uint_as_float(bits), 127 - static_cast<int>(byte));
}

// codes_to_bf16 is exact while code times scale lies in bf16's normal range: for
// e8m0 bytes 64 to 191 in any case (`near`, in bit 7 of each byte of a word).  Others
// are converted with a byte nearby, 96 to 159, with which a block's sum is in fp32's
// range whatever the codes, and the powers of two that this leaves, `s - nearby(s)`,
// are applied to the sum.
__device__ __forceinline__ uint32_t near_bits(uint32_t bytes) { return bytes ^ bytes << 1; }
__device__ __forceinline__ int nearby(int s) { return s == 255 ? 255 : min(max(s, 96), 159); }

// Eight codes times a power of two as bf16: an e8m0 scale byte s as the fp32 bits
// s << 23, 255 giving NaN.  Their products are exact in fp32 and the bf16 MFMA sums
// them in fp32.
template <int F>
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t lo, uint32_t hi, uint32_t scale_byte) {
    const float s = __uint_as_float(scale_byte << 23);
    union {
        bf16x2 p[4];
        bf16x8 v;
    } u;
    if constexpr (F == GDN_E4M3) {
        u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
        u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
        u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
        u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    } else {
        u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, s, false);
        u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, s, true);
        u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, s, false);
        u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, s, true);
    }
    return u.v;
}

// Writes NC neighbouring columns from col on of row `row`, in one store where
// they fit.
template <bool F32, int NC>
__device__ __forceinline__ void store_cols(const gdn_fp8::MatmulParams& p, long long row, int col, const float (&v)[NC]) {
    using T = std::conditional_t<F32, float, bf16>;
    typedef T vec __attribute__((ext_vector_type(NC)));
    T* const o = static_cast<T*>(p.out) + static_cast<size_t>(row) * p.ldo + col;
    if (col + NC <= p.N) {
        vec w;
#pragma unroll
        for (int i = 0; i < NC; ++i) w[i] = static_cast<T>(v[i]);
        __builtin_memcpy(o, &w, sizeof(w));  // at any address: odd rows too leave in whole stores
        return;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (col + i < p.N) o[i] = static_cast<T>(v[i]);
}

}  // namespace
