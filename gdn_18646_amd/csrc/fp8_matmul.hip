// Entry point of the fp8 block-scaled product, the rule that picks its kernel, and
// the kernel for one token or two.
//
// gdn_fp8_few_kernel (a decode step's token): what counts is the weights' bytes. A
// workgroup owns 16 columns; each of its waves takes every WAVES-th block of K
// straight from memory into MFMA fragments (no LDS: nothing is used twice), and
// the waves' sums meet in LDS.  The workgroups of an XCD begin at different
// blocks: 16 rows at a stride of a power of two lie in one or two of its L2's
// channels, and in step they would all wait for the same ones (one token, 4096 x
// 4096: 5.0 us against 6.2).  One token: 2048 x 2048 4.0 us (launch bound), 8224 x
// 2048 5.5, 8192 x 8192 11.6 (5.8 TB/s of weights).  More loads under way a wave
// (four blocks' at once, 110 registers) made it slower: 2048 x 8192 7.0 -> 7.7.
#include "fp8_matmul.hpp"

namespace {

template <int FA, int FB, bool OUT32, bool F32, int WAVES>  // F32: b's scales are fp32
__global__ __launch_bounds__(64 * WAVES) void gdn_fp8_few_kernel(gdn_fp8::MatmulParams p, int scales, int rot_mask) {
    __shared__ f32x4 sums[WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    const int n0 = blockIdx.x * 16, nslices = p.K / 128;
    const int row = min(n0 + r16, p.N - 1), tok = min(r16, p.M - 1);
    const uint8_t* const w = p.b + static_cast<size_t>(row) * p.ldb + 16 * g4;
    const uint8_t* const x = p.a + static_cast<size_t>(tok) * p.lda + 16 * g4;
    const bool rows = scales == gdn_fp8::kE8Row || scales == gdn_fp8::kF32Row;
    // the scale of the lane's row of b, its accumulator's column
    const size_t sstep = rows ? p.ldb_s : 1, sat = rows ? row : static_cast<size_t>(row / 128) * p.ldb_s;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const int rot = static_cast<int>(blockIdx.x >> 3) & rot_mask;
#pragma unroll 4
    for (int i = wave; i < nslices; i += WAVES) {
        const int kb = i + rot < nslices ? i + rot : i + rot - nslices;
        const u32x4* const wp = reinterpret_cast<const u32x4*>(w + static_cast<size_t>(kb) * 128);
        const u32x4* const xp = reinterpret_cast<const u32x4*>(x + static_cast<size_t>(kb) * 128);
        const int sx = p.a_scale[kb * p.lda_s + tok];
        uint32_t sw;  // b's scale as a power of two, and what is left of an fp32 one
        float fw = 1.f;
        if constexpr (F32) {
            const uint32_t bits = static_cast<const uint32_t*>(p.b_scale)[sat + kb * sstep];
            sw = scale_byte_of(bits);
            fw = scale_rest(bits, sw);
        } else {
            sw = static_cast<const uint8_t*>(p.b_scale)[sat + kb * sstep];
        }
        const i32x8 wc = join(wp[0], wp[4]), xc = join(xp[0], xp[4]);
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
        if constexpr (OUT32) {
            const int cx = nearby(sx), cw = nearby(static_cast<int>(sw));
#pragma unroll
            for (int q = 0; q < 4; ++q)
                t = mfma16x16x32(codes_to_bf16<FA>(xc[2 * q], xc[2 * q + 1], cx), codes_to_bf16<FB>(wc[2 * q], wc[2 * q + 1], cw), t);
            // the tokens of accumulators 0 and 1; there are no others
            const int left = sx - cx, left0 = __builtin_amdgcn_readlane(left, 0), left1 = __builtin_amdgcn_readlane(left, 1);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                acc[i] = fmaf(fw, __builtin_amdgcn_ldexpf(t[i], (i == 0 ? left0 : left1) + static_cast<int>(sw) - cw), acc[i]);
        } else {
            t = mfma_fp8<FA, FB, 0, 0>(xc, wc, t, sx, static_cast<int>(sw));
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(fw, t[i], acc[i]);
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

// What a call on a tile takes, us: c + rounds (a + b blocks of K), a round being
// 256 workgroups, or, where a CU holds per_cu of them, up to per_cu times 256,
// with a and b between a1, b1 (one a CU) and a2, b2 (per_cu).  Fitted to 336
// products (fp32 results: 336), 1 to 8192 tokens, N 200 to 8224, K 512 to 8192,
// kernels back to back on operands that the L2s do not hold: the tile that the fit
// picks takes at most 1.12 times the best one's time (fp32 1.05) and 1.003 times on
// average; 39 tiles were timed, those here are the ones whose absence costs.
// Small products take some 3.3 us whatever their K (c + a), and then what a CU needs
// to take in its rows: by b, 58 GB/s with one 256 x 256 tile, 76 to 78 with one of
// 16 x 16 or 64 x 128, 110 with three of 16 x 16.  So the small tiles spread the rows
// over the CUs, split K over groups of waves and keep several stages under way: 16 x
// 2048 x 8192 takes 6.8 us on 16 x 16 with eight groups and four stages (a workgroup
// a CU), 8.6 with two stages, 10.5 on 32 x 32; 16 x 8224 x 2048 6.2 on 16 x 16 with
// three a CU, 6.8 on 64 x 32.  256 x 160 and 128 x 192 are up to 9% faster where they
// make one round of what others make two of or a half (1500 x 6176 x 2048: 22.7 us on
// 256 x 160, 24.3 on 256 x 192).
struct TileCost {
    int tile, cols, toks, per_cu;
    float c, a1, b1, a2, b2;  // per_cu above 1: alone (1) and with per_cu on each CU (2)
};
constexpr TileCost kBf16[] = {
    {gdn_fp8::k256x256, 256, 256, 1, 0.f, 6.75f, 1.135f, 0.f, 0.f},
    {gdn_fp8::k256x192, 256, 192, 1, 0.f, 6.22f, 1.012f, 0.f, 0.f},
    {gdn_fp8::k256x160, 256, 160, 1, 0.f, 5.75f, 0.904f, 0.f, 0.f},
    {gdn_fp8::k256x128, 256, 128, 1, 0.f, 5.56f, 0.725f, 0.f, 0.f},
    {gdn_fp8::k128x192, 128, 192, 1, 0.f, 4.78f, 0.688f, 0.f, 0.f},
    {gdn_fp8::k128x128, 128, 128, 1, 0.f, 4.28f, 0.511f, 0.f, 0.f},
    {gdn_fp8::k64x128, 64, 128, 1, 0.40f, 4.22f, 0.315f, 0.f, 0.f},
    {gdn_fp8::k64x64, 64, 64, 1, 0.92f, 3.20f, 0.222f, 0.f, 0.f},
    {gdn_fp8::k64x32, 64, 32, 1, 1.26f, 2.73f, 0.144f, 0.f, 0.f},
    {gdn_fp8::k32x32, 32, 32, 1, 1.48f, 2.16f, 0.106f, 0.f, 0.f},
    {gdn_fp8::k16x16Alone, 16, 16, 1, 1.64f, 1.78f, 0.054f, 0.f, 0.f},
    {gdn_fp8::k16x16, 16, 16, 3, 2.60f, 0.70f, 0.064f, 1.37f, 0.112f},
};
constexpr TileCost kF32[] = {
    {gdn_fp8::k128x128, 128, 128, 2, 1.01f, 3.08f, 0.915f, 8.07f, 1.556f},
    {gdn_fp8::k64x128, 64, 128, 1, 0.11f, 4.40f, 0.525f, 0.f, 0.f},
    {gdn_fp8::k64x64, 64, 64, 1, 0.76f, 3.32f, 0.346f, 0.f, 0.f},
    {gdn_fp8::k64x32, 64, 32, 1, 1.09f, 3.09f, 0.200f, 0.f, 0.f},
    {gdn_fp8::k32x32, 32, 32, 1, 1.34f, 2.25f, 0.150f, 0.f, 0.f},
    {gdn_fp8::k16x16Alone, 16, 16, 1, 1.63f, 1.84f, 0.064f, 0.f, 0.f},
    {gdn_fp8::k16x16, 16, 16, 3, 2.61f, 0.70f, 0.081f, 1.53f, 0.123f},
};

struct Choice {
    int tile;
    float us;
};
Choice choose_tile(long long M, long long N, int K, bool f32) {
    constexpr long long kCUs = 256;
    const TileCost* const table = f32 ? kF32 : kBf16;
    const int n = static_cast<int>(f32 ? sizeof(kF32) / sizeof(kF32[0]) : sizeof(kBf16) / sizeof(kBf16[0]));
    const float nk = static_cast<float>(K / 128);
    Choice best = {0, 0.f};
    for (int i = 0; i < n; ++i) {
        const TileCost& t = table[i];
        const long long tiles = (M + t.toks - 1) / t.toks * ((N + t.cols - 1) / t.cols);
        const float alone = t.a1 + t.b1 * nk, full = t.a2 + t.b2 * nk;
        float us = t.c;
        if (t.per_cu == 1) {
            us += static_cast<float>((tiles + kCUs - 1) / kCUs) * alone;
        } else {
            const long long round = kCUs * t.per_cu, each = (tiles % round + kCUs - 1) / kCUs;  // workgroups a CU in the last one
            us += static_cast<float>(tiles / round) * full;
            if (each > 0) us += alone + static_cast<float>(each - 1) / static_cast<float>(t.per_cu - 1) * (full - alone);
        }
        if (i == 0 || us < best.us) best = {t.tile, us};
    }
    return best;
}

template <int FA, int FB>
int launch(const gdn_fp8::MatmulParams& p, int scales, bool f32, hipStream_t stream) {
    // One token, us here and on tiles: 4096 x 4096 5.0 and 5.8, 4096 x 8192 7.1 and
    // 8.0, 8224 x 2048 5.6 and 6.0, but 2048 x 8192 7.0 and 6.4, 6176 x 4096 7.0 and
    // 6.6; three tokens: 8224 x 2048 6.0 and 6.1, 6176 x 4096 7.5 and 6.8.  Eight
    // waves share a sum up to a workgroup a CU (2048 x 4096: 4.8 us, 5.9 with four),
    // above that four (8224 x 2048: 5.6, 5.8 with eight).
    if (p.M <= 2) {
        int mask = 1;
        while (2 * mask <= p.K / 128) mask *= 2;
        const auto few = [&](auto out32, auto f32_scales, auto waves) {
            constexpr int W = decltype(waves)::value;
            if (!gdn_host::grid_fits((p.N + 15) / 16, 64 * W)) return gdn_host::fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: N=%d is too large for a launch", p.N);
            hipLaunchKernelGGL((gdn_fp8_few_kernel<FA, FB, decltype(out32)::value, decltype(f32_scales)::value, W>), dim3((p.N + 15) / 16), dim3(64 * W), 0, stream, p,
                               scales, mask - 1);
            return gdn_host::check_launch("gdn_fp8_few_kernel");
        };
        const auto of_n = [&](auto out32, auto f32_scales) {
            return p.N <= 4096 ? few(out32, f32_scales, std::integral_constant<int, 8>{}) : few(out32, f32_scales, std::integral_constant<int, 4>{});
        };
        const auto of_scales = [&](auto out32) {
            return scales == gdn_fp8::kF32Block || scales == gdn_fp8::kF32Row ? of_n(out32, std::true_type{}) : of_n(out32, std::false_type{});
        };
        return f32 ? of_scales(std::true_type{}) : of_scales(std::false_type{});
    }
    // The last columns past a multiple of 256 in a launch of their own, on a tile
    // of their size, where the fit says that this is faster than a column of
    // large tiles for them: 16384 x 6176 x 2048, 32 columns past 6144, 209 us in
    // one launch.
    const Choice whole = choose_tile(p.M, p.N, p.K, f32);
    const int rest = p.N % 256, main = p.N - rest;
    if (rest > 0 && main > 0) {
        const Choice left = choose_tile(p.M, main, p.K, f32), right = choose_tile(p.M, rest, p.K, f32);
        if (left.us + right.us < whole.us) {
            gdn_fp8::MatmulParams q = p;
            q.N = main;
            const int st = gdn_fp8::launch_tile<FA, FB>(left.tile, scales, f32, q, stream);
            if (st != GDN_OK) return st;
            const bool rows = scales == gdn_fp8::kE8Row || scales == gdn_fp8::kF32Row;
            const size_t at = rows ? main : static_cast<size_t>(main / 128) * p.ldb_s;
            q.N = rest;
            q.b = p.b + static_cast<size_t>(main) * p.ldb;
            q.b_scale = static_cast<const uint8_t*>(p.b_scale) + at * (scales == gdn_fp8::kF32Block || scales == gdn_fp8::kF32Row ? 4 : 1);
            q.out = static_cast<uint8_t*>(p.out) + static_cast<size_t>(main) * (f32 ? 4 : 2);
            return gdn_fp8::launch_tile<FA, FB>(right.tile, scales, f32, q, stream);
        }
    }
    return gdn_fp8::launch_tile<FA, FB>(whole.tile, scales, f32, p, stream);
}

}  // namespace

extern "C" int gdn_fp8_matmul_hip(const uint8_t* a, int64_t lda, int format_a, const uint8_t* a_scale, int64_t lda_s,
                                  const uint8_t* b, int64_t ldb, int format_b, const void* b_scale, int64_t ldb_s,
                                  int b_block_rows, int type_b_scale, void* out, int64_t ldo, int type_out, int64_t M,
                                  int64_t N, int64_t K, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (M < 0 || N < 0 || K <= 0) return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_matmul: M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
    if (K % 128 != 0) return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: K=%lld must be a multiple of 128 (pad with zero codes)", (long long)K);
    if ((format_a != GDN_E4M3 && format_a != GDN_E5M2) || (format_b != GDN_E4M3 && format_b != GDN_E5M2))
        return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: formats %d, %d", format_a, format_b);
    if (b_block_rows != 1 && b_block_rows != 128) return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: b's blocks of %d x 128, 1 or 128 rows are supported", b_block_rows);
    if (type_b_scale != GDN_E8M0 && type_b_scale != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: type %d of b's scales", type_b_scale);
    if (type_out != GDN_BF16 && type_out != GDN_F32) return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: type %d of out", type_out);
    // 32-bit copy offsets within a tile, 32-bit tile numbers
    constexpr int64_t kMost = int64_t{1} << 22, kRows = 0x7fffff00LL;
    if (lda > kMost || ldb > kMost || M > kRows || N > kRows || (M + 31) / 32 * ((N + 31) / 32) > 0x7fffffffLL)
        return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: problem too large (rows of at most 2^22 codes)");
    if (b_block_rows == 1 && type_b_scale == GDN_F32 && N > int64_t{1} << 30)  // 32-bit byte offsets within a row of scales
        return fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: problem too large (at most 2^30 columns with an fp32 scale each)");
    if (M == 0 || N == 0) return GDN_OK;
    if (!a || !a_scale || !b || !b_scale || !out) return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_matmul: null pointer argument");
    if (!aligned(a, 16) || !aligned(b, 16) || lda % 16 != 0 || ldb % 16 != 0 || lda < K || ldb < K)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_matmul: codes need 16-byte aligned rows of at least K");
    if (!aligned(a_scale, 16) || lda_s % 16 != 0 || lda_s < M)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_matmul: a's scales [K / 128, lda_s] need 16-byte aligned rows of at least M");
    const size_t bs = type_b_scale == GDN_F32 ? 4 : 1, bo = type_out == GDN_F32 ? 4 : 2;
    if (b_block_rows == 1 ? !aligned(b_scale, 16) || ldb_s % 16 != 0 || ldb_s < N : !aligned(b_scale, bs) || ldb_s < K / 128)
        return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_matmul: b's scales: rows of at least N, 16-byte aligned ([K / 128, ldb_s]), or of K / 128 (128 x 128 blocks)");
    if (!aligned(out, bo) || ldo < N) return fail(GDN_ERR_INVALID_ARGUMENT, "fp8_matmul: out unaligned or ldo < N");
    gdn_fp8::MatmulParams p = {};
    p.a = a, p.b = b, p.a_scale = a_scale, p.b_scale = b_scale, p.out = out;
    p.lda = lda, p.ldb = ldb, p.lda_s = lda_s, p.ldb_s = ldb_s, p.ldo = ldo;
    p.M = static_cast<int>(M), p.N = static_cast<int>(N), p.K = static_cast<int>(K);
    const int scales = type_b_scale == GDN_F32 ? (b_block_rows == 1 ? gdn_fp8::kF32Row : gdn_fp8::kF32Block)
                                               : (b_block_rows == 1 ? gdn_fp8::kE8Row : gdn_fp8::kE8Block);
    const auto s = static_cast<hipStream_t>(stream);
    if (format_a == GDN_E4M3) return format_b == GDN_E4M3 ? launch<GDN_E4M3, GDN_E4M3>(p, scales, type_out == GDN_F32, s) : launch<GDN_E4M3, GDN_E5M2>(p, scales, type_out == GDN_F32, s);
    return format_b == GDN_E4M3 ? launch<GDN_E5M2, GDN_E4M3>(p, scales, type_out == GDN_F32, s) : launch<GDN_E5M2, GDN_E5M2>(p, scales, type_out == GDN_F32, s);
}
