// Entry point of the product with 4-bit weights, the rule that picks its kernel, and
// the kernel for one token or two.
//
// gdn_fp4_few_kernel (a decode step's token): what counts is the weights' bytes. A
// workgroup owns 16 columns; each of its waves takes every WAVES-th 256 values of K
// straight from memory into MFMA fragments (no LDS: nothing is used twice), and
// the waves' sums meet in LDS.  The workgroups of an XCD begin at different
// places: 16 rows at a stride of a power of two lie in one or two of its L2's
// channels, and in step they would all wait for the same ones.  A token by 8224 x 2048
// takes 4.0 us with 4-bit codes and 4.3-4.5 with 8-bit ones, by 65536 x 2048 (71 MB) 13.4,
// 5.3 TB/s, and 17.4; the 16 x 16 tile of fp4_tiles.hpp, which takes three tokens and more,
// 4.4, 4.3 (level), 20.8 and 23.1, and fp32 results of 8-bit codes 5-30% longer than here.
#include "fp4_matmul.hpp"

namespace {

template <int FA, bool OUT32, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void gdn_fp4_few_kernel(gdn_fp4::MatmulParams p, int rot_mask) {
    constexpr bool kFp4X = FA == GDN_E2M1, kBf16 = OUT32 && !kFp4X;
    __shared__ f32x4 sums[WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    const int n0 = blockIdx.x * 16, nblocks = p.K / 128, nslices = (nblocks + 1) / 2;
    const int row = min(n0 + r16, p.N - 1), tok = min(r16, p.M - 1);
    const uint8_t* const w = p.b + static_cast<size_t>(row) * p.ldb;
    const uint8_t* const x = p.a + static_cast<size_t>(tok) * p.lda;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const int rot = static_cast<int>(blockIdx.x >> 3) & rot_mask;
    for (int i = wave; i < nslices; i += WAVES) {
        const int slice = i + rot < nslices ? i + rot : i + rot - nslices;
        const u32x4* const wp = reinterpret_cast<const u32x4*>(w + static_cast<size_t>(slice) * 128) + g4;
        const u32x4 wc[2] = {wp[0], wp[4]};
        u32x4 xc[2][2];
        uint32_t sw[2], sx[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sw[h] = p.b_scale[(2 * slice + h) * p.ldb_s + row];
            if constexpr (kFp4X) {
                xc[h][0] = reinterpret_cast<const u32x4*>(x + static_cast<size_t>(slice) * 128)[4 * h + g4];
                sx[h] = reinterpret_cast<const uint32_t*>(p.a_scale)[(2 * slice + h) * p.lda_s + tok] >> (8 * g4);
            } else {
                const int kb = min(2 * slice + h, nblocks - 1);
                const u32x4* const xp = reinterpret_cast<const u32x4*>(x + static_cast<size_t>(kb) * 128);
                xc[h][0] = xp[kBf16 ? 2 * g4 : g4];
                xc[h][1] = xp[kBf16 ? 2 * g4 + 1 : 4 + g4];
                sx[h] = p.a_scale[kb * p.lda_s + tok];
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!kFp4X && 2 * slice + h >= nblocks) break;
            if constexpr (!kBf16) {
                i32x8 xv;
                if constexpr (kFp4X)
                    xv = codes4(xc[h][0]);
                else
                    xv = join(xc[h][0], xc[h][1]);
                acc = mfma_fp4<FA, 0, 0>(xv, codes4(wc[h]), acc, sx[h], sw[h] >> (8 * g4));
            } else {
                const uint32_t most = largest_byte(sw[h]), own = byte_over(sw[h] >> (8 * g4) & 0xffu, most);
                f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    t = mfma16x16x32(codes_to_bf16<FA>(xc[h][q / 2][2 * (q % 2)], xc[h][q / 2][2 * (q % 2) + 1], 127u), fp4_to_bf16(wc[h][q], own), t);
                // the tokens of accumulators 0 and 1; there are no others
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2)
                    acc[t2] += scaled_sum(t[t2], static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(sx[h]), t2)), most);
            }
        }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 1; i < WAVES; ++i) acc += sums[i][lane];
    if (n0 + r16 >= p.N) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v[1] = {acc[i]};
        if (4 * g4 + i < p.M) store_cols<OUT32>(p, 4 * g4 + i, n0 + r16, v);
    }
}

// What a call on a tile takes, us: c + rounds (a + b slices of 256 of K), a round being
// 256 workgroups, or, where a CU holds per_cu of them, up to per_cu times 256,
// with a and b between a1, b1 (one a CU) and a2, b2 (per_cu).
struct TileCost {
    int tile, cols, toks, per_cu;
    float c, a1, b1, a2, b2;  // per_cu above 1: alone (1) and with per_cu on each CU (2)
    int least_k = 0;          // shorter rows go to other tiles: what is stored then takes longer than the products
};
// Fitted to 320 products each, 3 to 8192 tokens, N 64 to 8224, K 256 to 8192, kernels
// back to back on operands that the L2s do not hold: the tile that the fit picks takes
// 1.016 times the best one's time on average (1.35 at most; 8-bit codes 1.011 and 1.17,
// fp32 results of those 1.007 and 1.09).  Up to ten tiles were timed; those here are the
// ones whose absence costs.
constexpr TileCost kCost4[] = {
    {gdn_fp4::k256x256, 256, 256, 1, 0.00f, 6.66f, 1.887f, 0.f, 0.f},
    {gdn_fp4::k128x128, 128, 128, 2, 3.36f, 1.26f, 0.937f, 3.47f, 1.181f},
    {gdn_fp4::k128x64, 128, 64, 2, 1.51f, 1.83f, 0.573f, 2.78f, 0.801f},
    {gdn_fp4::k64x128, 64, 128, 1, 0.82f, 2.98f, 0.450f, 0.f, 0.f},
    {gdn_fp4::k64x64, 64, 64, 1, 1.07f, 2.39f, 0.322f, 0.f, 0.f},
    {gdn_fp4::k64x32, 64, 32, 1, 1.40f, 2.21f, 0.177f, 0.f, 0.f},
    {gdn_fp4::k32x32, 32, 32, 1, 1.88f, 1.72f, 0.119f, 0.f, 0.f},
    {gdn_fp4::k16x16, 16, 16, 3, 2.71f, 1.20f, 0.027f, 0.86f, 0.145f},
};
constexpr TileCost kCost8[] = {  // 8-bit codes of a, bf16 results
    {gdn_fp4::k256x256, 256, 256, 1, 0.00f, 8.65f, 2.482f, 0.f, 0.f, 1280},
    {gdn_fp4::k256x128, 256, 128, 1, 0.00f, 5.08f, 1.661f, 0.f, 0.f},
    {gdn_fp4::k128x64, 128, 64, 2, 3.42f, 0.33f, 0.908f, 1.43f, 1.108f},
    {gdn_fp4::k64x64, 64, 64, 1, 0.77f, 2.62f, 0.413f, 0.f, 0.f},
    {gdn_fp4::k64x32, 64, 32, 1, 1.08f, 2.36f, 0.234f, 0.f, 0.f},
    {gdn_fp4::k32x32, 32, 32, 1, 1.53f, 1.81f, 0.186f, 0.f, 0.f},
    {gdn_fp4::k16x16Alone, 16, 16, 1, 2.09f, 1.47f, 0.066f, 0.f, 0.f},
    {gdn_fp4::k16x16, 16, 16, 3, 2.51f, 1.04f, 0.076f, 0.94f, 0.197f},
};
constexpr TileCost kCost32[] = {  // the same, fp32 results
    {gdn_fp4::k128x64, 128, 64, 2, 2.76f, 0.44f, 1.889f, 3.29f, 2.653f},
    {gdn_fp4::k64x64, 64, 64, 1, 0.56f, 2.79f, 1.011f, 0.f, 0.f},
    {gdn_fp4::k64x32, 64, 32, 1, 0.95f, 2.64f, 0.542f, 0.f, 0.f},
    {gdn_fp4::k32x32, 32, 32, 1, 1.33f, 2.08f, 0.333f, 0.f, 0.f},
    {gdn_fp4::k16x16Alone, 16, 16, 1, 1.80f, 1.83f, 0.116f, 0.f, 0.f},
    {gdn_fp4::k16x16, 16, 16, 3, 2.64f, 0.97f, 0.120f, 1.04f, 0.278f},
};

struct Choice {
    int tile;
    float us;
};
template <size_t N>
Choice choose_tile(const TileCost (&table)[N], long long M, long long cols, int K) {
    constexpr long long kCUs = 256;
    const float nk = static_cast<float>((K + 255) / 256);
    Choice best = {0, 0.f};
    for (size_t i = 0; i < N; ++i) {
        const TileCost& t = table[i];
        if (K < t.least_k) continue;
        const long long tiles = (M + t.toks - 1) / t.toks * ((cols + t.cols - 1) / t.cols);
        const float alone = t.a1 + t.b1 * nk, full = t.a2 + t.b2 * nk;
        float us = t.c;
        if (t.per_cu == 1) {
            us += static_cast<float>((tiles + kCUs - 1) / kCUs) * alone;
        } else {
            const long long round = kCUs * t.per_cu, each = (tiles % round + kCUs - 1) / kCUs;  // workgroups a CU in the last one
            us += static_cast<float>(tiles / round) * full;
            if (each > 0) us += alone + static_cast<float>(each - 1) / static_cast<float>(t.per_cu - 1) * (full - alone);
        }
        if (best.us == 0.f || us < best.us) best = {t.tile, us};
    }
    return best;
}

template <int FA>
int launch(const gdn_fp4::MatmulParams& p, bool f32, hipStream_t stream) {
    if (p.M <= 2) {
        int mask = 1;
        while (2 * mask <= (p.K + 255) / 256) mask *= 2;
        const auto few = [&](auto out32, auto waves) {
            constexpr int W = decltype(waves)::value;
            if (!gdn_host::grid_fits((p.N + 15) / 16, 64 * W))
                return gdn_host::fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: M=%d N=%d are too large for a launch", p.M, p.N);
            hipLaunchKernelGGL((gdn_fp4_few_kernel<FA, decltype(out32)::value, W>), dim3((p.N + 15) / 16), dim3(64 * W), 0, stream, p, mask - 1);
            return gdn_host::check_launch("gdn_fp4_few_kernel");
        };
        // The CUs hold 512 workgroups of eight waves or 1024 of four.  Eight read more at a
        // time, which wins where they fit one round (a token in 8-bit codes by 8192 x 4096 7.3
        // us with four and 6.4 with eight, by 2048 x 4096 5.5 and 3.9).  Past it they need a
        // second one and four do not (8224 x 4096 7.7 and 8.2, 9216 8.1 and 8.8, 12288 8.8 and
        // 9.3), until that one is full: level just below 1024 workgroups (16368 x 4096 10.5 and
        // 10.4), eight ahead there (16384 10.5 and 10.3) and beyond, where four need more than
        // one round too (16400 11.3 and 10.9, 24576 15.8 and 14.4, 65536 x 2048 17.9 and 17.4).
        // 4-bit codes rank alike, closer together.
        const auto of_n = [&](auto out32) {
            return p.N > 8192 && p.N < 16384 ? few(out32, std::integral_constant<int, 4>{}) : few(out32, std::integral_constant<int, 8>{});
        };
        return f32 ? of_n(std::true_type{}) : of_n(std::false_type{});
    }
    const auto choose = [&](long long cols) {
        if constexpr (FA == GDN_E2M1) return choose_tile(kCost4, p.M, cols, p.K);
        return f32 ? choose_tile(kCost32, p.M, cols, p.K) : choose_tile(kCost8, p.M, cols, p.K);
    };
    // The last columns past a multiple of 256 in a launch of their own, on a tile
    // of their size, where the fit says that this is faster than a column of
    // large tiles for them.
    const Choice whole = choose(p.N);
    const int rest = p.N % 256, main = p.N - rest;
    if (rest > 0 && main > 0) {
        const Choice left = choose(main), right = choose(rest);
        if (left.us + right.us < whole.us) {
            gdn_fp4::MatmulParams q = p;
            q.N = main;
            const int st = gdn_fp4::launch_tile<FA>(left.tile, f32, q, stream);
            if (st != GDN_OK) return st;
            q.N = rest;
            q.b = p.b + static_cast<size_t>(main) * p.ldb;
            q.b_scale = p.b_scale + main;
            q.out = static_cast<uint8_t*>(p.out) + static_cast<size_t>(main) * (f32 ? 4 : 2);
            return gdn_fp4::launch_tile<FA>(right.tile, f32, q, stream);
        }
    }
    return gdn_fp4::launch_tile<FA>(whole.tile, f32, p, stream);
}

}  // namespace

extern "C" int gdn_fp4_matmul_hip(const uint8_t* a, int64_t lda, int format_a, const uint8_t* a_scale, int64_t lda_s, const uint8_t* b,
                                  int64_t ldb, const uint8_t* b_scale, int64_t ldb_s, void* out, int64_t ldo, int type_out, int64_t M,
                                  int64_t N, int64_t K, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (M < 0 || N < 0 || K <= 0) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_matmul: M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
    if (format_a != GDN_E4M3 && format_a != GDN_E5M2 && format_a != GDN_E2M1) return fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: format %d of a", format_a);
    const bool fp4 = format_a == GDN_E2M1;
    if (K % (fp4 ? 256 : 128) != 0)
        return fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: K=%lld must be a multiple of %d (pad with zero codes)", (long long)K, fp4 ? 256 : 128);
    if (type_out != GDN_BF16 && type_out != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: type %d of out", type_out);
    // 32-bit copy offsets within a tile and a row of scales
    constexpr int64_t kMost = int64_t{1} << 22, kRows = int64_t{1} << 28, kScales = int64_t{1} << 29;
    if (K > kMost || lda > kMost || ldb > kMost || M > kRows || N > kRows || lda_s > kScales || ldb_s > kScales || (M + 15) / 16 * ((N + 15) / 16) > 0x7fffffffLL)
        return fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: problem too large (rows of at most 2^22 bytes, 2^28 of them)");
    if (M == 0 || N == 0) return GDN_OK;
    if (!a || !a_scale || !b || !b_scale || !out) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_matmul: null pointer argument");
    const int64_t row_a = fp4 ? K / 2 : K, row_b = (K + 255) / 256 * 128;
    if (!aligned(a, 16) || !aligned(b, 16) || lda % 16 != 0 || ldb % 16 != 0 || lda < row_a || ldb < row_b)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_matmul: codes need 16-byte aligned rows of at least %lld (a) and %lld (b) bytes", (long long)row_a, (long long)row_b);
    const int64_t whole = fp4 ? 4 : 16;
    if (!aligned(a_scale, 16) || lda_s % whole != 0 || lda_s < M)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_matmul: a's scales [K / 128, lda_s%s] need 16-byte aligned rows of at least M", fp4 ? ", 4" : "");
    if (!aligned(b_scale, 16) || ldb_s % 4 != 0 || ldb_s < N)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_matmul: b's scales [K / 128, ldb_s, 4] need 16-byte aligned rows of at least N");
    if (!aligned(out, type_out == GDN_F32 ? 4 : 2) || ldo < N) return fail(GDN_ERR_INVALID_ARGUMENT, "fp4_matmul: out unaligned or ldo < N");
    gdn_fp4::MatmulParams p = {};
    p.a = a, p.b = b, p.a_scale = a_scale, p.b_scale = reinterpret_cast<const uint32_t*>(b_scale), p.out = out;
    p.lda = lda, p.ldb = ldb, p.lda_s = lda_s, p.ldb_s = ldb_s, p.ldo = ldo;
    p.M = static_cast<int>(M), p.N = static_cast<int>(N), p.K = static_cast<int>(K);
    const auto s = static_cast<hipStream_t>(stream);
    const bool f32 = type_out == GDN_F32;
    return fp4 ? launch<GDN_E2M1>(p, f32, s) : format_a == GDN_E4M3 ? launch<GDN_E4M3>(p, f32, s) : launch<GDN_E5M2>(p, f32, s);
}
