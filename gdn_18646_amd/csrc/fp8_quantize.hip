// Quantisation to 8-bit floating point in blocks of 128 (fp8_blocks.hpp), along
// the rows of x [M, K], along its columns (the codes of x^T, for a product that
// sums over x's rows), or both from one read; a block is 1 x 128 values along
// the codes' own rows, or 128 x 128 of x.
//
// One workgroup a 128 x 128 tile: a thread holds 4 x 8 of it in registers, a
// row's maximum meets over 16 lanes by DPP, a column's over LDS, and the
// transposed codes pass through LDS so that both layouts leave in whole
// 128-byte lines.  What bounds it: HBM (2 bytes read, 1 or 2 written a value)
// above some 1000 tiles, below that a tile's chain of loads, maxima and stores,
// which is why eight waves share one (8224 x 2048 by blocks both ways: 11.6 us,
// 5.7 TB/s, 14.1 with four waves and conflicting transposition; 1500 x 2048 along
// its rows: 3.7 us).
#include "block_norm.hpp"
#include "fp8_blocks.hpp"

namespace {

struct QuantParams {
    const void* x;
    long long ldx;
    uint8_t *codes, *scales, *codes_t, *scales_t;  // codes [M, ldc], codes_t [K, ldt]; null: not wanted
    long long ldc, lds, ldt, ldst;
    int M, K, kb;  // kb: tiles along K
    int vec;       // 16-byte loads fit
};

template <class TX, int FMT, bool BLOCK>
__global__ __launch_bounds__(512) void gdn_fp8_quantize_kernel(QuantParams p) {
    constexpr int RT = 4;  // rows of a thread
    __shared__ __attribute__((aligned(16))) unsigned char tile[128 * 128];
    __shared__ __attribute__((aligned(16))) uint32_t most[32][132];
    __shared__ __attribute__((aligned(16))) uint32_t bytes[128];
    const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4;
    const int k0 = static_cast<int>(blockIdx.x % p.kb) * kBlk, m0 = static_cast<int>(blockIdx.x / p.kb) * kBlk;
    const int c = k0 + 8 * cg, r0 = m0 + RT * rg;

    Oct<TX> o[RT];
    if (p.vec) {
#pragma unroll
        for (int i = 0; i < RT; ++i) o[i] = Oct<TX>::template load<true>(p.x, min(r0 + i, p.M - 1) * p.ldx, c, p.K);
    } else {
#pragma unroll
        for (int i = 0; i < RT; ++i) o[i] = Oct<TX>::template load<false>(p.x, min(r0 + i, p.M - 1) * p.ldx, c, p.K);
    }
    float f[RT][8];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        o[i].get(f[i]);
        if (!p.vec) to_natural(f[i], c - vector_at(c, p.K), p.K);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = r0 + i < p.M && c + j < p.K ? f[i][j] : 0.f;
    }

    uint32_t rowb[RT];  // scale bytes of the thread's rows
    if constexpr (BLOCK) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < RT; ++i) m = max(m, amax8(f[i]));
        m = max16(m);
        if (cg == 0) bytes[rg] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max(m, bytes[i]);
#pragma unroll
        for (int i = 0; i < RT; ++i) rowb[i] = Fp8<FMT>::scale_byte(m);
        if (tid == 0) {
            const int kt = k0 / kBlk, mt = m0 / kBlk;
            if (p.codes) p.scales[mt * p.lds + kt] = static_cast<uint8_t>(rowb[0]);
            if (p.codes_t) p.scales_t[kt * p.ldst + mt] = static_cast<uint8_t>(rowb[0]);
        }
    } else if (p.codes) {
#pragma unroll
        for (int i = 0; i < RT; ++i) rowb[i] = Fp8<FMT>::scale_byte(max16(amax8(f[i])));
        if (cg == 0) {
            uint8_t* const at = p.scales + static_cast<long long>(k0 / kBlk) * p.lds + r0;
            if (r0 + RT <= p.M) {
                *reinterpret_cast<uint32_t*>(at) = rowb[0] | rowb[1] << 8 | rowb[2] << 16 | rowb[3] << 24;
            } else {  // what lies past the last row is the caller's
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    if (r0 + i < p.M) at[i] = static_cast<uint8_t>(rowb[i]);
            }
        }
    }
    if (p.codes) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const u32x2 w = Fp8<FMT>::codes8(f[i], Fp8<FMT>::inverse(rowb[i]), rowb[i] == 0xffu);
            if (r0 + i < p.M) *reinterpret_cast<u32x2*>(p.codes + static_cast<long long>(r0 + i) * p.ldc + c) = w;
        }
    }
    if (!p.codes_t) return;

    uint32_t colb[8];
    if constexpr (BLOCK) {
#pragma unroll
        for (int j = 0; j < 8; ++j) colb[j] = rowb[0];
    } else {
        u32x4 w[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < RT; ++i) m = max(m, __float_as_uint(f[i][j]) & 0x7fffffffu);
            w[j / 4][j % 4] = m;
        }
        *reinterpret_cast<u32x4*>(&most[rg][8 * cg]) = w[0];
        *reinterpret_cast<u32x4*>(&most[rg][8 * cg + 4]) = w[1];
        __syncthreads();
        if (tid < 128) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) m = max(m, most[i][tid]);
            const uint32_t b = Fp8<FMT>::scale_byte(m);
            bytes[tid] = b;
            if (k0 + tid < p.K) p.scales_t[static_cast<long long>(m0 / kBlk) * p.ldst + k0 + tid] = static_cast<uint8_t>(b);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) colb[j] = bytes[8 * cg + j];
    }
    // Row k of the transposed tile holds its 4-byte piece q (rows m0 + 4 q ..) at
    // slot q ^ 4 (k / 8 % 8): the 16 lanes of a row group write to different
    // banks, and 16 bytes stay together.
#pragma unroll
    for (int j = 0; j < 8; ++j)
        *reinterpret_cast<uint32_t*>(tile + (8 * cg + j) * 128 + 4 * (rg ^ (4 * (cg & 7)))) =
            Fp8<FMT>::codes4(f[0][j], f[1][j], f[2][j], f[3][j], Fp8<FMT>::inverse(colb[j]), colb[j] == 0xffu);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int k = 64 * i + tid / 8;
        if (k0 + k < p.K)
            *reinterpret_cast<u32x4*>(p.codes_t + static_cast<long long>(k0 + k) * p.ldt + m0 + 16 * (tid & 7)) =
                *reinterpret_cast<const u32x4*>(tile + k * 128 + 16 * ((tid & 7) ^ (k / 8 & 7)));
    }
}

}  // namespace

extern "C" int gdn_fp8_quantize_hip(const void* x, int64_t ldx, int type_x, int64_t M, int64_t K, int block_rows, int format,
                                    uint8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, uint8_t* codes_t, int64_t ldt,
                                    uint8_t* scales_t, int64_t ldst, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (M < 0 || K < 0) return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_quantize: M=%lld K=%lld", (long long)M, (long long)K);
    if (block_rows != 1 && block_rows != kBlk) return fail(GDN_ERR_UNSUPPORTED, "fp8_quantize: blocks of %d x 128, 1 or 128 rows are supported", block_rows);
    if (type_x != GDN_BF16 && type_x != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp8_quantize: type %d of x", type_x);
    if (format != GDN_E4M3 && format != GDN_E5M2) return fail(GDN_ERR_UNSUPPORTED, "fp8_quantize: format %d", format);
    const int64_t MB = (M + kBlk - 1) / kBlk, KB = (K + kBlk - 1) / kBlk;
    if (M > 0x7fffffffLL - kBlk || K > 0x7fffffffLL - kBlk || MB * KB > 0x7fffffffLL || !gdn_host::grid_fits(MB * KB, 512))
        return fail(GDN_ERR_UNSUPPORTED, "fp8_quantize: problem too large");
    if (!codes && !codes_t) return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_quantize: no output");
    if (M == 0 || K == 0) return GDN_OK;
    if (!x || !aligned(x, type_bytes(type_x)) || ldx < K) return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_quantize: x null, unaligned or ldx < K");
    const bool block = block_rows == kBlk;
    if (codes && (!scales || !aligned(codes, 16) || ldc % 16 != 0 || ldc < KB * kBlk ||
                  (block ? lds < KB : lds < M || lds % 16 != 0 || !aligned(scales, 16))))
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_quantize: codes [M, ldc >= K padded to 128] with 16-byte rows, scales of lds >= %lld",
                    (long long)(block ? KB : M));
    if (codes_t && (!scales_t || !aligned(codes_t, 16) || ldt % 16 != 0 || ldt < MB * kBlk || ldst < (block ? MB : K)))
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_quantize: codes_t [K, ldt >= M padded to 128] with 16-byte rows, scales_t of ldst >= %lld",
                    (long long)(block ? MB : K));
    QuantParams p = {};
    p.x = x, p.ldx = ldx, p.M = static_cast<int>(M), p.K = static_cast<int>(K), p.kb = static_cast<int>(KB);
    p.codes = codes, p.scales = scales, p.ldc = ldc, p.lds = lds;
    p.codes_t = codes_t, p.scales_t = scales_t, p.ldt = ldt, p.ldst = ldst;
    p.vec = K % 8 == 0 && vec_rows(x, ldx, type_x);
    const auto launch = [&](auto tx, auto fmt, auto blk) {
        hipLaunchKernelGGL((gdn_fp8_quantize_kernel<decltype(tx), decltype(fmt)::value, decltype(blk)::value>),
                           dim3(static_cast<unsigned>(MB * KB)), dim3(512), 0, static_cast<hipStream_t>(stream), p);
        return gdn_host::check_launch("gdn_fp8_quantize_kernel");
    };
    const auto of_format = [&](auto tx, auto blk) {
        return format == GDN_E4M3 ? launch(tx, std::integral_constant<int, GDN_E4M3>{}, blk)
                                  : launch(tx, std::integral_constant<int, GDN_E5M2>{}, blk);
    };
    const auto of_type = [&](auto blk) { return type_x == GDN_F32 ? of_format(0.f, blk) : of_format(bf16(), blk); };
    return block ? of_type(std::true_type{}) : of_type(std::false_type{});
}
