// Quantisation to 4-bit floating point in blocks of 32 (fp4_blocks.hpp), along the
// rows of x [M, K], along its columns (the codes of x^T, for a product that sums
// over x's rows), or both from one read; a block is 1 x 32 values along the codes'
// own rows, or 32 x 32 of x, whose codes are the same ones both ways.  Or along its rows
// in 4 bits and along its columns in 8 (e4m3, blocks of 1 x 128, fp8_blocks.hpp): what a
// training step with 4-bit activations takes of them, from one read.  And back.
//
// Quantisation: one workgroup a 128 x 128 tile, as for 8 bits: a thread holds 4 x 8
// of it in registers, a row's maximum meets over 4 lanes by DPP, a column's over
// LDS, and the transposed codes pass through LDS.  Bound by memory where there are tiles
// enough: 8224 x 2048 bf16 both ways (52 MB) 12.9 us, 4.0 TB/s; 8192 x 4096 along the rows
// (85 MB) 15.9, 5.4, and with 8-bit columns (118 MB) 24.1, 4.9 (two kernels 33.3); one row of 2048 3.3 us, a launch, a load and a store.
//
// Back: 8224 x 2048 to bf16 (43 MB) 9.2 us, 4.6 TB/s.
#include <algorithm>

#include "block_norm.hpp"
#include "fp4_blocks.hpp"
#include "fp8_blocks.hpp"

namespace {

constexpr int kTile = 128;

struct Quant4Params {
    const void* x;
    long long ldx;
    uint8_t *codes, *codes_t;      // [M, ldc bytes], [K, ldt bytes]; null: not wanted
    uint32_t *scales, *scales_t;   // words of four bytes: [K / 128][lds], [M / 128][ldst] (8-bit columns: bytes)
    long long ldc, lds, ldt, ldst;
    int M, K, kb;                  // kb: tiles along K (256-value rows: an even number)
    int vec;                       // 16-byte loads fit
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp4(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
// Maximum over each 4 lanes (the lanes of a row's block of 32), in every lane.
__device__ __forceinline__ uint32_t max4(uint32_t v) {
    v = max(v, dpp4<0xB1>(v));      // quad_perm [1,0,3,2]
    return max(v, dpp4<0x4E>(v));   // quad_perm [2,3,0,1]
}
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// T8: the columns' codes are 8-bit ones.
template <class TX, bool BLOCK, bool T8>
__global__ __launch_bounds__(512) void gdn_fp4_quantize_kernel(Quant4Params p) {
    constexpr int RT = 4, PITCH = T8 ? 128 : 68;  // rows of a thread; bytes of a transposed row in LDS (17 words: 16 lanes' columns on 8 banks)
    static_assert(!(BLOCK && T8), "8-bit columns are blocks of 1 x 128");
    __shared__ __attribute__((aligned(16))) unsigned char tile[128 * PITCH];
    __shared__ __attribute__((aligned(16))) uint32_t most[32][BLOCK ? 4 : 132];
    __shared__ __attribute__((aligned(16))) uint32_t bytes[4][132];
    const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4;
    const int kt = static_cast<int>(blockIdx.x % p.kb), mt = static_cast<int>(blockIdx.x / p.kb);
    const int k0 = kt * kTile, m0 = mt * kTile;
    const int c = k0 + 8 * cg, r0 = m0 + RT * rg;

    float f[RT][8];
    {
        Oct<TX> o[RT];
        const bool inside = k0 < p.K && m0 < p.M;  // not a tile of padding
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (!inside) continue;
            const long long row = min(r0 + i, p.M - 1) * p.ldx;
            o[i] = p.vec ? Oct<TX>::template load<true>(p.x, row, c, p.K) : Oct<TX>::template load<false>(p.x, row, c, p.K);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (inside) {
                o[i].get(f[i]);
                if (!p.vec) to_natural(f[i], c - vector_at(c, p.K), p.K);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = r0 + i < p.M && c + j < p.K ? f[i][j] : 0.f;
        }
    }

    uint32_t rowb[RT];  // scale bytes of the thread's rows
    if constexpr (BLOCK) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, magnitude(f[i][j]));
        m = max4(m);
        if ((cg & 3) == 0) most[rg][cg >> 2] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, most[(rg & 24) + i][cg >> 2]);
#pragma unroll
        for (int i = 0; i < RT; ++i) rowb[i] = fp4_scale_byte(m);
    } else {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, magnitude(f[i][j]));
            rowb[i] = fp4_scale_byte(max4(m));
        }
    }
    if (p.codes) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uint32_t w = fp4_codes8(f[i], fp4_inverse(rowb[i]), rowb[i] == 0xffu);
            if (r0 + i < p.M) {
                *reinterpret_cast<uint32_t*>(p.codes + (r0 + i) * p.ldc + c / 2) = w;
                if ((cg & 3) == 0) reinterpret_cast<uint8_t*>(p.scales + kt * p.lds + r0 + i)[cg >> 2] = static_cast<uint8_t>(rowb[i]);
            }
        }
    }
    if (!p.codes_t) return;

    uint32_t colb[8];
    if constexpr (BLOCK) {
        if ((rg & 7) == 0 && (cg & 3) == 0) bytes[rg >> 3][cg >> 2] = rowb[0];
#pragma unroll
        for (int j = 0; j < 8; ++j) colb[j] = rowb[0];
        __syncthreads();
        if (tid < 128 && k0 + tid < p.K)
            p.scales_t[mt * p.ldst + k0 + tid] = bytes[0][tid >> 5] | bytes[1][tid >> 5] << 8 | bytes[2][tid >> 5] << 16 | bytes[3][tid >> 5] << 24;
    } else {
        u32x4 w[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < RT; ++i) m = max(m, magnitude(f[i][j]));
            w[j / 4][j % 4] = m;
        }
        *reinterpret_cast<u32x4*>(&most[rg][8 * cg]) = w[0];
        *reinterpret_cast<u32x4*>(&most[rg][8 * cg + 4]) = w[1];
        __syncthreads();
        if constexpr (T8) {
            if (tid < 128) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) m = max(m, most[i][tid]);
                m = Fp8<GDN_E4M3>::scale_byte(m);
                bytes[0][tid] = m;
                if (k0 + tid < p.K) reinterpret_cast<uint8_t*>(p.scales_t)[mt * p.ldst + k0 + tid] = static_cast<uint8_t>(m);
            }
        } else {
            const int col = tid & 127, q = tid >> 7;
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, most[8 * q + i][col]);
            bytes[q][col] = fp4_scale_byte(m);
        }
        __syncthreads();
        if (!T8 && tid < 128 && k0 + tid < p.K)
            p.scales_t[mt * p.ldst + k0 + tid] = bytes[0][tid] | bytes[1][tid] << 8 | bytes[2][tid] << 16 | bytes[3][tid] << 24;
#pragma unroll
        for (int j = 0; j < 8; ++j) colb[j] = bytes[T8 ? 0 : rg >> 3][8 * cg + j];
    }
    if constexpr (T8) {
        // Row k of the transposed tile holds its 4-byte piece q (rows m0 + 4 q ..) at slot
        // q ^ 4 (k / 8 % 8): the 16 lanes of a row group write to different banks, and 16
        // bytes stay together.
#pragma unroll
        for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint32_t*>(tile + (8 * cg + j) * PITCH + 4 * (rg ^ (4 * (cg & 7)))) =
                Fp8<GDN_E4M3>::codes4(f[0][j], f[1][j], f[2][j], f[3][j], Fp8<GDN_E4M3>::inverse(colb[j]), colb[j] == 0xffu);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = 64 * i + tid / 8;
            if (k0 + k < p.K)
                *reinterpret_cast<u32x4*>(p.codes_t + (k0 + k) * p.ldt + m0 + 16 * (tid & 7)) =
                    *reinterpret_cast<const u32x4*>(tile + k * PITCH + 16 * ((tid & 7) ^ (k / 8 & 7)));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        *reinterpret_cast<uint16_t*>(tile + (8 * cg + j) * PITCH + 2 * rg) =
            static_cast<uint16_t>(fp4_codes4(f[0][j], f[1][j], f[2][j], f[3][j], fp4_inverse(colb[j]), colb[j] == 0xffu));
    __syncthreads();
    const int k = tid >> 2;
    if (k0 + k < p.K) {
        const uint32_t* const at = reinterpret_cast<const uint32_t*>(tile + k * PITCH + 16 * (tid & 3));
        *reinterpret_cast<u32x4*>(p.codes_t + (k0 + k) * p.ldt + m0 / 2 + 16 * (tid & 3)) = u32x4{at[0], at[1], at[2], at[3]};
    }
}

struct Dequant4Params {
    const uint8_t* codes;
    const uint32_t* scales;
    void* out;
    long long ldc, lds, ldo;
    int M, K, units;  // units of 8 values in a row
    long long total;  // units
};

// A lane takes 8 codes (a word) to 8 values: a wave's loads and stores are adjacent.
template <class T>
__global__ __launch_bounds__(256) void gdn_fp4_dequantize_kernel(Dequant4Params p) {
    const long long step = static_cast<long long>(gridDim.x) * 256;
    for (long long u = blockIdx.x * 256LL + threadIdx.x; u < p.total; u += step) {
        const long long row = u / p.units;
        const int c = 8 * static_cast<int>(u - row * p.units);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p.codes + row * p.ldc + c / 2);
        const uint32_t s = p.scales[(c >> 7) * p.lds + row] >> (c >> 5 & 3) * 8 & 0xffu;
        const u32x4 v = as_u32x4(fp4_to_bf16(w, s));
        T* const o = static_cast<T*>(p.out) + row * p.ldo + c;
        if constexpr (sizeof(T) == 2) {
            if (c + 8 <= p.K) {
                __builtin_memcpy(o, &v, 16);  // whole stores at any address
            } else {
                for (int i = 0; i < p.K - c; ++i) reinterpret_cast<uint16_t*>(o)[i] = static_cast<uint16_t>(v[i / 2] >> 16 * (i % 2));
            }
        } else {
            float f[8];
            unpack8(v, f);
            if (c + 8 <= p.K) {
                __builtin_memcpy(o, f, 32);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < p.K) o[i] = f[i];
            }
        }
    }
}

}  // namespace

extern "C" int gdn_fp4_quantize_hip(const void* x, int64_t ldx, int type_x, int64_t M, int64_t K, int block_rows, uint8_t* codes,
                                    int64_t ldc, uint8_t* scales, int64_t lds, uint8_t* codes_t, int64_t ldt, uint8_t* scales_t,
                                    int64_t ldst, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (M < 0 || K < 0) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_quantize: M=%lld K=%lld", (long long)M, (long long)K);
    if (block_rows != 1 && block_rows != 32) return fail(GDN_ERR_UNSUPPORTED, "fp4_quantize: blocks of %d x 32, 1 or 32 rows are supported", block_rows);
    if (type_x != GDN_BF16 && type_x != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp4_quantize: type %d of x", type_x);
    // tiles of 128 x 128, in pairs along the codes' rows
    const int64_t MB = (M + kTile - 1) / kTile, KB = (K + kFp4Row - 1) / kFp4Row * 2, MT = (M + kFp4Row - 1) / kFp4Row * 2;
    const int64_t tiles_m = codes_t ? MT : MB;
    if (M > 0x7fffffffLL - kFp4Row || K > 0x7fffffffLL - kFp4Row || tiles_m * KB > 0x7fffffffLL || !gdn_host::grid_fits(tiles_m * KB, 512))
        return fail(GDN_ERR_UNSUPPORTED, "fp4_quantize: problem too large");
    if (!codes && !codes_t) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_quantize: no output");
    if (M == 0 || K == 0) return GDN_OK;
    if (!x || !aligned(x, type_bytes(type_x)) || ldx < K) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_quantize: x null, unaligned or ldx < K");
    if (codes && (!scales || !aligned(codes, 16) || ldc % 16 != 0 || ldc < KB * kTile / 2 || !aligned(scales, 4) || lds < M))
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_quantize: codes [M, ldc >= %lld bytes] with 16-byte rows, scales [%lld, lds >= %lld, 4] at 4 bytes",
                    (long long)(KB * kTile / 2), (long long)KB, (long long)M);
    if (codes_t && (!scales_t || !aligned(codes_t, 16) || ldt % 16 != 0 || ldt < MT * kTile / 2 || !aligned(scales_t, 4) || ldst < K))
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_quantize: codes_t [K, ldt >= %lld bytes] with 16-byte rows, scales_t [%lld, ldst >= %lld, 4] at 4 bytes",
                    (long long)(MT * kTile / 2), (long long)MT, (long long)K);
    Quant4Params p = {};
    p.x = x, p.ldx = ldx, p.M = static_cast<int>(M), p.K = static_cast<int>(K), p.kb = static_cast<int>(KB);
    p.codes = codes, p.scales = reinterpret_cast<uint32_t*>(scales), p.ldc = ldc, p.lds = lds;
    p.codes_t = codes_t, p.scales_t = reinterpret_cast<uint32_t*>(scales_t), p.ldt = ldt, p.ldst = ldst;
    p.vec = K % 8 == 0 && vec_rows(x, ldx, type_x);
    const auto launch = [&](auto tx, auto blk) {
        hipLaunchKernelGGL((gdn_fp4_quantize_kernel<decltype(tx), decltype(blk)::value, false>), dim3(static_cast<unsigned>(tiles_m * KB)),
                           dim3(512), 0, static_cast<hipStream_t>(stream), p);
        return gdn_host::check_launch("gdn_fp4_quantize_kernel");
    };
    const auto of_type = [&](auto blk) { return type_x == GDN_F32 ? launch(0.f, blk) : launch(bf16(), blk); };
    return block_rows == 32 ? of_type(std::true_type{}) : of_type(std::false_type{});
}

extern "C" int gdn_fp4_fp8_quantize_hip(const void* x, int64_t ldx, int type_x, int64_t M, int64_t K, uint8_t* codes, int64_t ldc, uint8_t* scales,
                                        int64_t lds, uint8_t* codes_t, int64_t ldt, uint8_t* scales_t, int64_t ldst, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (M < 0 || K < 0) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_fp8_quantize: M=%lld K=%lld", (long long)M, (long long)K);
    if (type_x != GDN_BF16 && type_x != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp4_fp8_quantize: type %d of x", type_x);
    const int64_t MB = (M + kTile - 1) / kTile, KB = (K + kFp4Row - 1) / kFp4Row * 2;
    if (M > 0x7fffffffLL - kFp4Row || K > 0x7fffffffLL - kFp4Row || MB * KB > 0x7fffffffLL || !gdn_host::grid_fits(MB * KB, 512))
        return fail(GDN_ERR_UNSUPPORTED, "fp4_fp8_quantize: problem too large");
    if (M == 0 || K == 0) return GDN_OK;
    if (!x || !aligned(x, type_bytes(type_x)) || ldx < K) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_fp8_quantize: x null, unaligned or ldx < K");
    if (!codes || !scales || !aligned(codes, 16) || ldc % 16 != 0 || ldc < KB * kTile / 2 || !aligned(scales, 4) || lds < M)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_fp8_quantize: codes [M, ldc >= %lld bytes] with 16-byte rows, scales [%lld, lds >= %lld, 4] at 4 bytes",
                    (long long)(KB * kTile / 2), (long long)KB, (long long)M);
    if (!codes_t || !scales_t || !aligned(codes_t, 16) || ldt % 16 != 0 || ldt < MB * kTile || ldst < K)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_fp8_quantize: codes_t [K, ldt >= %lld] with 16-byte rows, scales_t [%lld, ldst >= %lld]",
                    (long long)(MB * kTile), (long long)MB, (long long)K);
    Quant4Params p = {};
    p.x = x, p.ldx = ldx, p.M = static_cast<int>(M), p.K = static_cast<int>(K), p.kb = static_cast<int>(KB);
    p.codes = codes, p.scales = reinterpret_cast<uint32_t*>(scales), p.ldc = ldc, p.lds = lds;
    p.codes_t = codes_t, p.scales_t = reinterpret_cast<uint32_t*>(scales_t), p.ldt = ldt, p.ldst = ldst;
    p.vec = K % 8 == 0 && vec_rows(x, ldx, type_x);
    const dim3 grid(static_cast<unsigned>(MB * KB));
    if (type_x == GDN_F32)
        hipLaunchKernelGGL((gdn_fp4_quantize_kernel<float, false, true>), grid, dim3(512), 0, static_cast<hipStream_t>(stream), p);
    else
        hipLaunchKernelGGL((gdn_fp4_quantize_kernel<bf16, false, true>), grid, dim3(512), 0, static_cast<hipStream_t>(stream), p);
    return gdn_host::check_launch("gdn_fp4_quantize_kernel");
}

extern "C" int gdn_fp4_dequantize_hip(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, void* out, int64_t ldo,
                                      int type_out, int64_t M, int64_t K, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (M < 0 || K < 0) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_dequantize: M=%lld K=%lld", (long long)M, (long long)K);
    if (type_out != GDN_BF16 && type_out != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp4_dequantize: type %d of out", type_out);
    if (M > 0x7fffffffLL || K > 0x7fffffffLL - 8) return fail(GDN_ERR_UNSUPPORTED, "fp4_dequantize: problem too large");
    if (M == 0 || K == 0) return GDN_OK;
    if (!codes || !aligned(codes, 4) || ldc % 4 != 0 || ldc < (K + 7) / 8 * 4)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_dequantize: codes null or not in 4-byte rows of at least K / 2 bytes");
    if (!scales || !aligned(scales, 4) || lds < M) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_dequantize: scales [K / 128, lds >= M, 4] null or unaligned");
    if (!out || !aligned(out, type_bytes(type_out)) || ldo < K) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_dequantize: out null, unaligned or ldo < K");
    Dequant4Params p = {};
    p.codes = codes, p.scales = reinterpret_cast<const uint32_t*>(scales), p.out = out;
    p.ldc = ldc, p.lds = lds, p.ldo = ldo, p.M = static_cast<int>(M), p.K = static_cast<int>(K), p.units = static_cast<int>((K + 7) / 8);
    p.total = M * p.units;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((p.total + 255) / 256, 4096)));
    if (type_out == GDN_F32)
        hipLaunchKernelGGL(gdn_fp4_dequantize_kernel<float>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), p);
    else
        hipLaunchKernelGGL(gdn_fp4_dequantize_kernel<bf16>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return gdn_host::check_launch("gdn_fp4_dequantize_kernel");
}
