// Parameter block, launches and operand helpers of the product with 4-bit weights
// (fp4_matmul.hip holds its entry point, the rule that picks its kernel and the
// kernel for one token or two; fp4_tiles.hpp and fp4_phased.hpp the tiled kernels and
// fp4_launch.hpp their launches, instantiated for each format of the activations in
// fp4_mm_*.hip).
#pragma once

#include "fp4_blocks.hpp"
#include "fp8_matmul.hpp"

namespace gdn_fp4 {

struct MatmulParams {
    const uint8_t *a, *b;  // codes [M, lda bytes], [N, ldb bytes]; b's two a byte, rows padded to 256 values
    const uint8_t* a_scale;  // 4-bit codes: words of four bytes [K / 128][lda_s]; 8-bit ones: bytes [K / 128][lda_s]
    const uint32_t* b_scale;  // words of four bytes [K / 128][ldb_s]
    void* out;             // [M, ldo] bf16 or fp32
    long long lda, ldb, lda_s, ldb_s, ldo;
    int M, N, K;           // K: a multiple of 128, of 256 where a's codes are 4-bit too
};

// Tiles of the tiled kernels (columns x tokens), largest first: 128 x 128 and 64 x 128 for
// 4-bit codes of a alone, 256 x 128 and 16 x 16 alone on a CU for 8-bit ones.
enum Tile { k256x256 = 0, k256x128, k128x128, k128x64, k64x128, k64x64, k64x32, k32x32, k16x16Alone, k16x16 };

// Defined in fp4_mm_*.hip for each format of a.  f32: out is fp32, else bf16.
template <int FA>
int launch_tile(int tile, bool f32, const MatmulParams& p, hipStream_t stream);

}  // namespace gdn_fp4

namespace {

__device__ __forceinline__ i32x8 codes4(const u32x4 v) {  // 32 4-bit codes: half of an operand's registers
    return i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}

// MFMA 16x16x128 of a's codes (format FA: tokens, the A operand) and 4-bit ones (rows
// of W, the B operand) with fp32 sums; a lane's accumulator is column lane % 16 of
// tokens 4 (lane / 16) + i.  Lane l supplies row l % 16: of 4-bit codes values 32 (l /
// 16) .. + 31 (16 bytes), of 8-bit ones values 16 (l / 16) .. + 15 and 64 on from
// there; byte SX of sx and SW of sw is the scale of the 4-bit codes that the lane
// supplies (of 8-bit ones all four lanes of a row have the same).  127 is 1.
//
// The sum of a block of 32 products of 4-bit codes is exact, and four blocks and the
// accumulator are added with an error of at most 2^-21 of the largest of the products, the
// four sums, the accumulator and the result (measured: 2^-22.2 over 10^7 results, scales up
// to 2^78 apart, terms that cancel or do not; a sum of 129 terms in fp32 may be off by 2^-17
// of its largest partial sum), so fp32 results are summed here too.  Of products with 8-bit
// codes the instruction drops what lies below about 2^-17 of the largest: good for bf16
// results alone.
template <int FA, int SX, int SW>
__device__ __forceinline__ f32x4 mfma_fp4(const i32x8 x, const i32x8 w, const f32x4 c, uint32_t sx, uint32_t sw) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, w, c, FA == GDN_E2M1 ? 4 : FA, 4, SX, static_cast<int>(sx), SW,
                                                            static_cast<int>(sw));
}

// fp32 results of 8-bit codes run on the bf16 instruction, a block of 128 at a time:
// a's codes without their scale, b's with theirs over the largest of the block's four,
// so that both lie in bf16's range whatever the scales are; the powers of two that
// this leaves (a's scale and b's largest) are applied to the block's sum.
__device__ __forceinline__ uint32_t largest_byte(uint32_t w) { return max(max(w & 0xffu, w >> 8 & 0xffu), max(w >> 16 & 0xffu, w >> 24)); }
// The byte of a block whose scale is `byte`, over `most`; NaN where one of the four is.
__device__ __forceinline__ uint32_t byte_over(uint32_t byte, uint32_t most) {
    return most == 255u ? 255u : static_cast<uint32_t>(max(static_cast<int>(byte) - static_cast<int>(most) + 127, 0));
}
// sum times 2^(sx + most - 254); a scale of 255 is NaN.
__device__ __forceinline__ float scaled_sum(float sum, uint32_t sx, uint32_t most) {
    const float v = __builtin_amdgcn_ldexpf(sum, static_cast<int>(sx + most) - 254);
    return sx == 255u ? __uint_as_float(0x7fc00000u) : v;
}

// Writes NC neighbouring columns from col on of row `row`, in one store where they fit.
template <bool F32, int NC>
__device__ __forceinline__ void store_cols(const gdn_fp4::MatmulParams& p, long long row, int col, const float (&v)[NC]) {
    gdn_fp8::MatmulParams q = {};
    q.out = p.out, q.ldo = p.ldo, q.N = p.N;
    store_cols<F32>(q, row, col, v);
}

}  // namespace
