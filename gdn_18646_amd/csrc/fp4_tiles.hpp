// The tiled kernel of the product with 4-bit weights
//   out[m, n] = sum over k of a[m, k] a_scale[m, block of k] b[n, k] b_scale[n, block of k]
// with fp32 sums, one rounding where out is written.  b's codes are 4-bit, a's 4-bit
// (blocks of 32) or 8-bit (blocks of 128).
//
// In tiles of columns x tokens (W = b, x = a).  A stage is 256 values of K: rows of
// 128 bytes of W and of 4-bit x, two of 128 bytes of 8-bit x (one after the other for
// all tokens).  They reach LDS by DMA in a ring, every 8 lanes of a copy one whole
// line, placed with an XOR swizzle that keeps the fragment reads at linear-read speed,
// and the scales with them.  A 4-bit row's four scales of 128 values are a word, of
// which a lane of the product needs one byte, that of its own 32 values: a few byte
// permutations a stage gather those of up to four tiles into one register, from which
// the instruction picks.  fp32 results of 8-bit codes: see fp4_matmul.hpp.
#pragma once

#include "fp4_matmul.hpp"

namespace {

constexpr int kRowB = 128;  // bytes of a staged row

// CW x TW waves, each WMT 16-column x WNT 16-token MFMA tiles, NS stages in LDS,
// PER_CU workgroups on a CU; KS groups of such waves, each on its own 256 values of a
// stage of KS times as many, summed at the end.  PHASED: the two-group main loop
// (eight waves, one workgroup on a CU).  XH: staged rows of a token (1: 4-bit, 2: 8-bit).
template <int XH_, int CW_, int TW_, int WMT_, int WNT_, int NS_, int PER_CU_, int KS_ = 1, bool PHASED_ = false>
struct Fp4Tile {
    static constexpr int XH = XH_, CW = CW_, TW = TW_, WMT = WMT_, WNT = WNT_, NS = NS_, PER_CU = PER_CU_, KS = KS_;
    static constexpr bool PHASED = PHASED_;
    static constexpr int cols = 16 * CW * WMT, toks = 16 * TW * WNT, rows = cols + XH * toks;
    static constexpr int gwaves = CW * TW, waves = gwaves * KS;
    static constexpr int dma = rows / 8 / gwaves;  // 1 KiB copies (8 rows) a wave and slice
    static_assert(PHASED || rows % (8 * gwaves) == 0, "copies split evenly");
    // PHASED: a stage is staged, and its buffer freed, region by region: the
    // first and second part of every wave's tokens (X0, X1) and columns (W0,
    // W1), in the order X0 and the scales, W0, W1, X1.  A region of `groups`
    // 4-row pieces is split over the waves, each taking whole copies of 8 rows
    // and, where 8 pieces are left, one of 4 rows by half its lanes.
    static constexpr int M0n = WMT / 2, M1n = WMT - M0n, X0n = (WNT + 1) / 2, X1n = WNT - X0n;
    static constexpr int groups(int r) { return 4 * (r == 0 ? XH * TW * X0n : r == 1 ? CW * M0n : r == 2 ? CW * M1n : XH * TW * X1n); }
    static constexpr int full(int r) { return groups(r) / 16; }
    static constexpr int piece(int r) { return groups(r) % 16 / 8; }
    static constexpr int ncopy(int r) { return full(r) + piece(r); }
    static constexpr int first(int r) { return r == 0 ? 0 : first(r - 1) + ncopy(r - 1); }
    static constexpr int row_copies = PHASED ? first(4) : dma;
    static_assert(!PHASED || (waves == 8 && PER_CU == 1 && KS == 1 && groups(0) % 8 == 0 && groups(1) % 8 == 0 && groups(2) % 8 == 0 &&
                              groups(3) % 8 == 0 && M0n > 0 && X1n > 0),
                  "phased tile");
    // A slice's bytes: rows, W's scales [2][cols] words, x's [2][toks] words or bytes.
    static constexpr int xsb = XH == 1 ? 4 : 1;  // bytes of a token's scales of 128 values
    static constexpr int off_ws = rows * kRowB, off_xs = off_ws + 8 * cols;
    static constexpr int slice_b = (off_xs + 2 * xsb * toks + 127) / 128 * 128, stage_b = KS * slice_b, lds_b = NS * stage_b;
    static constexpr int copies = row_copies + 2;  // a wave issues, for a slice
    static_assert(lds_b * PER_CU <= 160 * 1024, "LDS");
    static_assert((KS - 1) * gwaves * WMT * WNT * 1024 <= lds_b, "the groups' sums fit the dead stages");
};

__device__ __forceinline__ int swz(int r) { return r & 7; }

// Workgroup barrier alone (no LDS access of this wave is outstanding); no
// memory access moves across it.
__device__ __forceinline__ void wave_barrier() { asm volatile("s_barrier" ::: "memory"); }

template <class TL, int FA, bool OUT32>
__global__ __launch_bounds__(TL::waves * 64)
    __attribute__((amdgpu_waves_per_eu(TL::PER_CU * TL::waves / 4, TL::PER_CU * TL::waves / 4))) void gdn_fp4_matmul_kernel(
        gdn_fp4::MatmulParams p, int n_tok, int n_col) {
    constexpr int WMT = TL::WMT, WNT = TL::WNT, NS = TL::NS, KS = TL::KS, XH = TL::XH;
    constexpr bool kFp4X = FA == GDN_E2M1, kBf16 = OUT32 && !kFp4X;  // kBf16: products on the bf16 instruction
    static_assert((XH == 1) == kFp4X, "rows of x");
    __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[TL::lds_b];
    lds_u8* const smem = (lds_u8*)&smem_raw[0];

    // Workgroup -> tiles: each XCD gets a contiguous range of tiles, in bands of 4
    // column tiles with the token tile slowest, so that the workgroups of one XCD
    // share rows in its L2; a workgroup takes every step-th tile of its XCD's (one
    // tile where there is a workgroup for each).
    const int ntiles = n_tok * n_col, xcd = blockIdx.x & 7, per = ntiles >> 3, rest = ntiles & 7;
    const int begin = xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per, count = per + (xcd < rest ? 1 : 0);
    const int step = (static_cast<int>(gridDim.x) - xcd + 7) >> 3;
    auto tile_at = [&](int j, int& f, int& c) {
        const int lin = begin + j, band = lin / (4 * n_tok), base = 4 * band, gs = min(n_col - base, 4);
        const int within = lin - band * 4 * n_tok;
        f = within / gs * TL::toks;
        c = (base + within % gs) * TL::cols;
    };
    int f0, c0;  // the tile's first token and column
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = KS > 1 ? wave / TL::gwaves : 0, gw = KS > 1 ? wave % TL::gwaves : wave;
    const int wm = gw / TL::TW, wn = gw % TL::TW;
    const int r16 = lane & 15, g4 = lane >> 4;
    const int nblocks = p.K / 128, nslices = (nblocks + 1) / 2;  // blocks of 128, slices of 256

    // Copy sources.  Staged rows 0 .. cols - 1 are rows of b, the others rows of
    // a, in an order that gives a lane of the product WMT neighbouring columns and
    // lets it supply WNT neighbouring tokens, whose scales are neighbours
    // (accumulator (mt, nt)[i]: column WMT r16 + mt, token WNT (4 g4 + i) + nt of
    // the wave's).  Rows past the end repeat the last one; what they give is not
    // stored.
    const uint8_t *wsrc, *xsrc;
    auto src_off = [&](int srow, int lane) {
        const uint32_t chunk = 16u * ((lane & 7) ^ swz(srow));
        if (srow < TL::cols) {
            const int w = srow / (16 * WMT), s = srow % (16 * WMT);
            const int col = 16 * WMT * w + WMT * (s & 15) + (s >> 4);
            return static_cast<uint32_t>(min(c0 + col, p.N - 1) - c0) * static_cast<uint32_t>(p.ldb) + chunk;
        }
        const int t = (srow - TL::cols) % TL::toks, w = t / (16 * WNT), s = t % (16 * WNT);
        const int tok = 16 * WNT * w + WNT * (s & 15) + (s >> 4);
        return static_cast<uint32_t>(min(f0 + tok, p.M - 1) - f0) * static_cast<uint32_t>(p.lda) + chunk;
    };
    // Copy j of region r in the phased loop: the first staged row, the same for
    // the wave.
    auto copy_row = [&](int r, int j) {
        int g = j < TL::full(r) ? 2 * (wave + 8 * j) : 16 * TL::full(r) + wave;                          // in 4-row pieces
        const int per = 4 * (r == 0 ? TL::X0n : r == 1 ? TL::M0n : r == 2 ? TL::M1n : TL::X1n);  // pieces of one wave's part
        const bool x = r == 0 || r == 3;
        int base = 0;
        if (x) {
            const int h = g / (TL::TW * per);  // which 128 bytes of the tokens
            g -= h * TL::TW * per;
            base = TL::cols + h * TL::toks;
        }
        const int w = g / per, within = 4 * (g % per);
        return x ? base + 16 * WNT * w + (r == 3 ? 16 * TL::X0n : 0) + within : 16 * WMT * w + (r == 2 ? 16 * TL::M0n : 0) + within;
    };
    uint32_t voff[TL::row_copies], xs_off, ws_off;
    int crow[TL::row_copies];  // staged row of the copy's first lane (wave-uniform)
    if constexpr (TL::PHASED) {
        static_for<0, 4>([&](auto R) {
            constexpr int r = decltype(R)::value;
            static_for<0, TL::ncopy(r)>([&](auto J) { crow[TL::first(r) + decltype(J)::value] = __builtin_amdgcn_readfirstlane(copy_row(r, decltype(J)::value)); });
        });
    } else {
#pragma unroll
        for (int j = 0; j < TL::row_copies; ++j) crow[j] = 8 * (gw + TL::gwaves * j);
    }
    // The scales' copies: the waves of a group share 16-byte pieces out, each
    // wave one copy of at least one piece (the last waves may repeat pieces).
    // Pieces go by 128 values first, then by rows.
    constexpr int kWPieces = TL::cols / 2, kWLanes = (kWPieces + TL::gwaves - 1) / TL::gwaves;            // 4 rows each
    constexpr int kXPieces = 2 * TL::toks * TL::xsb / 16, kXLanes = (kXPieces + TL::gwaves - 1) / TL::gwaves;  // 4 tokens each, or 16
    static_assert(kWLanes <= 64 && kXLanes <= 64, "a copy has 64 lanes");
    const int wp = min(gw * kWLanes, kWPieces - kWLanes), xp = min(gw * kXLanes, kXPieces - kXLanes);
    auto set_tile = [&](int j) {
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));  // computed anew for each tile: kept over the loop, its parts would fill registers
        tile_at(j, f0, c0);
        wsrc = p.b + static_cast<size_t>(c0) * p.ldb;
        xsrc = p.a + static_cast<size_t>(f0) * p.lda;
        if constexpr (TL::PHASED) {
            static_for<0, 4>([&](auto R) {
                constexpr int r = decltype(R)::value;
                static_for<0, TL::ncopy(r)>([&](auto J) {
                    constexpr int i = decltype(J)::value, c = TL::first(r) + i;
                    voff[c] = src_off(crow[c] + (i < TL::full(r) ? lane >> 3 : (lane >> 3) & 3), lane);
                });
            });
        } else {
#pragma unroll
            for (int i = 0; i < TL::row_copies; ++i) voff[i] = src_off(crow[i] + (lane >> 3), lane);
        }
        const int wq = wp + lane, xq = xp + lane;
        constexpr int per_w = TL::cols / 4, per_x = kXPieces / 2, xrows = 16 / TL::xsb;
        ws_off = static_cast<uint32_t>(wq / per_w) * 4u * static_cast<uint32_t>(p.ldb_s) + 4u * min(c0 + 4 * (wq % per_w), (p.N - 1) / 4 * 4);
        xs_off = static_cast<uint32_t>(xq / per_x) * TL::xsb * static_cast<uint32_t>(p.lda_s) + TL::xsb * min(f0 + xrows * (xq % per_x), (p.M - 1) / xrows * xrows);
    };
    // Offset of a token's staged row `h` of slice `slice` (8-bit x: of its block, the last one where there is none).
    auto x_at = [&](int h, int slice) {
        return static_cast<size_t>(kFp4X ? slice : __builtin_amdgcn_readfirstlane(min(2 * slice + h, nblocks - 1))) * kRowB;
    };
    auto issue_row = [&](int c, bool x, int stage, int slice) {
        const int h = XH == 2 && crow[c] >= TL::cols + TL::toks ? 1 : 0;
        const uint8_t* const src = x ? xsrc + x_at(h, slice) : wsrc + static_cast<size_t>(slice) * kRowB;
        dma16(src, voff[c], smem + stage * TL::stage_b + ks * TL::slice_b + crow[c] * kRowB);
    };
    auto issue_rows = [&](int stage, int slice) {
#pragma unroll
        for (int j = 0; j < TL::row_copies; ++j) issue_row(j, crow[j] >= TL::cols, stage, slice);
    };
    auto issue_scales = [&](int stage, int slice) {
        lds_u8* const dst = smem + stage * TL::stage_b + ks * TL::slice_b;
        if (lane < kXLanes) {
            const size_t at = static_cast<size_t>(2 * slice) * TL::xsb * p.lda_s;
            uint32_t off = xs_off;
            // of 8-bit x there may be no second block: its pieces repeat the first's
            if (!kFp4X && 2 * slice + 1 >= nblocks && xp + lane >= kXPieces / 2) off -= static_cast<uint32_t>(p.lda_s);
            dma16(p.a_scale + at, off, dst + TL::off_xs + 16 * xp);
        }
        if (lane < kWLanes)
            dma16(reinterpret_cast<const uint8_t*>(p.b_scale) + static_cast<size_t>(2 * slice) * 4 * p.ldb_s, ws_off, dst + TL::off_ws + 16 * wp);
    };
    // Region r of a stage (phased loop); the scales come with the first.
    auto issue_region = [&](auto R, int stage, int slice) {
        constexpr int r = decltype(R)::value;
        static_for<0, TL::ncopy(r)>([&](auto J) {
            constexpr int j = decltype(J)::value, c = TL::first(r) + j;
            if (j < TL::full(r) || lane < 32) issue_row(c, r == 0 || r == 3, stage, slice);
        });
        if constexpr (r == 0) issue_scales(stage, slice);
    };
    // The slice of stage kk that this wave's group takes (the last stage's
    // groups past the end repeat the last slice and do not multiply it).
    auto slice_of = [&](int kk) { return KS > 1 ? min(kk * KS + ks, nslices - 1) : kk; };

    uint32_t rd[2];  // 16-byte pieces g4 and 4 + g4 of row r16
#pragma unroll
    for (int h = 0; h < 2; ++h) rd[h] = r16 * kRowB + 16u * ((4 * h + g4) ^ swz(r16));

    f32x4 acc[WMT][WNT];
    auto clear = [&]() {
#pragma unroll
        for (int mt = 0; mt < WMT; ++mt)
#pragma unroll
            for (int nt = 0; nt < WNT; ++nt) acc[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    // The tile's results: f, c its first token and column.
    auto store_tile = [&](int f, int c) {
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int R0 = f + 16 * WNT * wn + WNT * 4 * (lane >> 4), C0 = c + 16 * WMT * wm + WMT * (lane & 15);
        if (C0 >= p.N) return;
        static_for<0, 4 * WNT>([&](auto J) {
            constexpr int i = decltype(J)::value / WNT, nt = decltype(J)::value % WNT;
            if (R0 + WNT * i + nt >= p.M) return;
            float v[WMT];
#pragma unroll
            for (int mt = 0; mt < WMT; ++mt) v[mt] = acc[mt][nt][i];
            store_cols<OUT32>(p, R0 + WNT * i + nt, C0, v);
        });
    };

    auto half = [&](const lds_u8* at, int h) { return *reinterpret_cast<const lds_u32x4*>(at + rd[h]); };
    // N words of neighbouring rows' scales.
    auto read_words = [&](const lds_u8* at, auto N, uint32_t* w) {
        constexpr int n = decltype(N)::value;
        if constexpr (n % 4 == 0) {
#pragma unroll
            for (int i = 0; i < n; i += 4) {
                const u32x4 v = *reinterpret_cast<const lds_u32x4*>(at + 4 * i);
                w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2], w[i + 3] = v[3];
            }
        } else if constexpr (n % 2 == 0) {
#pragma unroll
            for (int i = 0; i < n; i += 2) {
                const u32x2 v = *reinterpret_cast<const lds_u32x2*>(at + 4 * i);
                w[i] = v[0], w[i + 1] = v[1];
            }
        } else {
#pragma unroll
            for (int i = 0; i < n; ++i) w[i] = reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at)[i];
        }
    };
    // Byte g4 of each of N words, four to a register.
    const uint32_t pick = static_cast<uint32_t>(g4) | static_cast<uint32_t>(4 + g4) << 8;
    auto gather = [&](const uint32_t* w, auto N, uint32_t* s) {
        constexpr int n = decltype(N)::value;
        static_for<0, (n + 3) / 4>([&](auto I) {
            constexpr int i = 4 * decltype(I)::value;
            if constexpr (i + 1 == n) {
                s[i / 4] = w[i] >> (8 * g4);
            } else {
                s[i / 4] = __builtin_amdgcn_perm(w[i + 1], w[i], pick);
                if constexpr (i + 3 == n)
                    s[i / 4] = __builtin_amdgcn_perm(w[i + 2] >> (8 * g4), s[i / 4], 0x07040100u);
                else if constexpr (i + 4 <= n)
                    s[i / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[i + 3], w[i + 2], pick), s[i / 4], 0x05040100u);
            }
        });
    };
    // W's scales of a staged slice: of each 128 values the bytes of the wave's columns that the lane supplies.
    auto read_sw = [&](const lds_u8* st, uint32_t (&sw)[2]) {
        static_for<0, 2>([&](auto H) {
            uint32_t w[WMT];
            read_words(st + TL::off_ws + 4 * (decltype(H)::value * TL::cols + 16 * WMT * wm + WMT * r16), std::integral_constant<int, WMT>{}, w);
            gather(w, std::integral_constant<int, WMT>{}, &sw[decltype(H)::value]);
        });
    };
    // x's: the same, or of 8-bit codes the tokens' bytes.
    constexpr bool kWords = kFp4X || (WNT & (WNT - 1)) == 0;  // four tokens to a register (of 8-bit codes not where their bytes lie askew)
    constexpr int NSX = kWords ? (WNT + 3) / 4 : WNT;
    auto read_sx = [&](const lds_u8* st, uint32_t (&sx)[2][NSX]) {
        static_for<0, 2>([&](auto H) {
            constexpr int h = decltype(H)::value;
            if constexpr (kFp4X) {
                uint32_t w[WNT];
                read_words(st + TL::off_xs + 4 * (h * TL::toks + 16 * WNT * wn + WNT * r16), std::integral_constant<int, WNT>{}, w);
                gather(w, std::integral_constant<int, WNT>{}, sx[h]);
            } else {
                const lds_u8* const at = st + TL::off_xs + h * TL::toks + 16 * WNT * wn + WNT * r16;
                if constexpr (WNT == 4) {
                    sx[h][0] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at);
                } else if constexpr (WNT == 2) {
                    sx[h][0] = *reinterpret_cast<const lds_u16*>(at);
                } else {
                    static_assert(WNT == 1 || !kWords, "tokens of a wave");
#pragma unroll
                    for (int nt = 0; nt < WNT; ++nt) sx[h][nt] = at[nt];
                }
            }
        });
    };

    // A tile's operand of a slice: W's 32 codes of each 128 values, x's 32 codes of each.
    struct W2 {
        u32x4 h[2];
    };
    struct X2 {
        u32x4 h[2][kFp4X ? 1 : 2];
    };
    auto frag_w = [&](const lds_u8* at) { return W2{{half(at, 0), half(at, 1)}}; };
    auto frag_x = [&](const lds_u8* at) {
        X2 x;
        if constexpr (kFp4X) {
            x.h[0][0] = half(at, 0);
            x.h[1][0] = half(at, 1);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x.h[h][0] = half(at + h * TL::toks * kRowB, 0);
                x.h[h][1] = half(at + h * TL::toks * kRowB, 1);
            }
        }
        return x;
    };
    // 128 values' product of operands mt and nt into the accumulator.
    auto multiply = [&](auto H, auto MT, auto NT, const X2& x, const W2& w, const uint32_t (&sx)[2][NSX], const uint32_t (&sw)[2]) {
        constexpr int h = decltype(H)::value, mt = decltype(MT)::value, nt = decltype(NT)::value, bx = kWords ? nt % 4 : 0;
        i32x8 xv;
        if constexpr (kFp4X)
            xv = codes4(x.h[h][0]);
        else
            xv = join(x.h[h][0], x.h[h][1]);
        acc[mt][nt] = mfma_fp4<FA, bx, mt>(xv, codes4(w.h[h]), acc[mt][nt], sx[h][kWords ? nt / 4 : nt], sw[h]);
    };

    const int nk = (nslices + KS - 1) / KS;
    int tile = static_cast<int>(blockIdx.x) >> 3;
    set_tile(tile);

    if constexpr (TL::PHASED) {
        // Two groups of four waves, one wave of each on every SIMD, take turns:
        // while one multiplies, the other reads its next fragments and issues its
        // copies.  A stage is four phases, each a part of the wave's tile (first
        // or second half of its columns x of its tokens) over the whole slice:
        // (W0, X0), (W1, X0), (W1, X1), (W0, X1).  Phase 0 reads W0, X0 and the
        // scales, phase 1 W1, phase 2 X1, phase 3 nothing.  A region's buffer is
        // free once both groups have read it, so stage kt + NS's X0, W0 and W1 go
        // out in phases 1, 2 and 3 of stage kt and its X1 in phase 0 of the next.
        // The waits count the copies issued after the region that the next phase
        // reads; T >= 0: T stages are left after this one and no new ones are
        // issued.
        static_assert(!kBf16, "fp32 results of 8-bit codes run on the ring");
        W2 w0[TL::M0n], w1[TL::M1n];
        X2 xf[TL::X0n];
        uint32_t sx[2][NSX], sw[2];
        constexpr int cX0 = TL::ncopy(0) + 2, cW1 = TL::ncopy(2), cX1 = TL::ncopy(3), cAll = TL::copies;
        auto next_buf = [](int b, int n) {
            b += n;
            return b >= NS ? b - NS : b;
        };
        auto stage = [&](int kt, int rs, auto Tc) {
            constexpr int T = decltype(Tc)::value;
            constexpr bool steady = T < 0;
            const lds_u8* st = smem + rs * TL::stage_b;
            const lds_u8* stx = st + (TL::cols + 16 * WNT * wn) * kRowB;
            const lds_u8* stw = st + 16 * WMT * wm * kRowB;
            const bool both = kFp4X || T != 0 || 2 * kt + 1 < nblocks;  // whether a has the slice's second 128 values
            static_for<0, 4>([&](auto Pc) {
                constexpr int ph = decltype(Pc)::value;
                if constexpr (ph == 0) {
                    static_for<0, TL::M0n>([&](auto I) { w0[decltype(I)::value] = frag_w(stw + 16 * decltype(I)::value * kRowB); });
                    static_for<0, TL::X0n>([&](auto I) { xf[decltype(I)::value] = frag_x(stx + 16 * decltype(I)::value * kRowB); });
                    read_sx(st, sx);
                    read_sw(st, sw);
                } else if constexpr (ph == 1) {
                    static_for<0, TL::M1n>([&](auto I) { w1[decltype(I)::value] = frag_w(stw + 16 * (TL::M0n + decltype(I)::value) * kRowB); });
                } else if constexpr (ph == 2) {
                    static_for<0, TL::X1n>([&](auto I) { xf[decltype(I)::value] = frag_x(stx + 16 * (TL::X0n + decltype(I)::value) * kRowB); });
                }
                if constexpr (ph == 0 && (steady || T == NS - 1))
                    issue_region(std::integral_constant<int, 3>{}, next_buf(rs, NS - 1), kt + NS - 1);
                else if constexpr (ph > 0 && steady)
                    issue_region(std::integral_constant<int, ph - 1>{}, rs, kt + NS);
                if constexpr (ph == 0)
                    wait_vm<cX1 + (steady ? NS - 1 : T) * cAll>();
                else if constexpr (ph == 1)
                    wait_vm<steady ? cX0 + (NS - 1) * cAll : T * cAll>();
                else if constexpr (ph == 3 && T != 0)
                    wait_vm<cW1 + (steady ? (NS - 1) * cAll : cX1 + (T - 1) * cAll)>();
                lds_barrier();  // this group's fragments are here, the other's multiplications issued
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
                constexpr int m0 = ph == 0 || ph == 3 ? 0 : TL::M0n, mn = ph == 0 || ph == 3 ? TL::M0n : TL::M1n;
                constexpr int n0 = ph < 2 ? 0 : TL::X0n, nn = ph < 2 ? TL::X0n : TL::X1n;
                static_for<0, 2>([&](auto H) {
                    if (decltype(H)::value == 1 && !both) return;
                    static_for<0, nn>([&](auto NT) {
                        constexpr int nt = n0 + decltype(NT)::value;
                        static_for<0, mn>([&](auto MT) {
                            constexpr int mt = m0 + decltype(MT)::value;
                            multiply(H, std::integral_constant<int, mt>{}, std::integral_constant<int, nt>{}, xf[nt - n0],
                                     m0 == 0 ? w0[mt - m0] : w1[mt - m0], sx, sw);
                        });
                    });
                });
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                wave_barrier();
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        // Fill the ring as the phases would have.
        auto fill = [&]() {
            static_for<0, NS>([&](auto S) {
                constexpr int s = decltype(S)::value;
                if (s < nk) static_for<0, s + 1 < NS ? 4 : 3>([&](auto R) { issue_region(R, s, s); });
            });
        };
        fill();
        // One tile after the other: the next one's first stages are copied while
        // this one's results are stored.  The stores are younger than those
        // copies and older than later ones, so the waits above hold as they are
        // (vector memory operations retire in order).
        for (;;) {
            const bool more = tile + step < count;
            clear();
            if (nk >= NS)
                wait_vm<cW1 + (NS - 1) * cAll>();  // X0, the scales and W0 of stage 0
            else
                wait_vm<0>();
            wave_barrier();
            const bool second = wave >= 4;
            if (second) wave_barrier();
            int kt = 0, rs = 0;
            for (; kt + NS < nk; ++kt) {
                stage(kt, rs, std::integral_constant<int, -1>{});
                rs = next_buf(rs, 1);
            }
            static_for<0, NS>([&](auto I) {
                constexpr int T = NS - 1 - decltype(I)::value;
                if (T < nk) {
                    stage(kt, rs, std::integral_constant<int, T>{});
                    ++kt;
                    rs = next_buf(rs, 1);
                }
            });
            if (!second) wave_barrier();
            const int f = f0, c = c0;
            if (more) {
                tile += step;
                set_tile(tile);
                fill();
            }
            store_tile(f, c);
            if (!more) return;
        }
    } else {
        clear();
        // Ring of NS stages: stage kt + NS - 1 is issued while stage kt is
        // multiplied, into the buffer that stage kt - 1 was read from.
#pragma unroll
        for (int st = 0; st < NS - 1; ++st)
            if (st < nk) {
                issue_rows(st, slice_of(st));
                issue_scales(st, slice_of(st));
            }
        int rs = 0, ws = NS - 1;  // buffers of stage kt and of stage kt + NS - 1
        for (int kt = 0; kt < nk; ++kt) {
            const bool next = kt + NS - 1 < nk;
            // Stage kt has landed (later ones may be in flight; the last NS - 1
            // stages wait for every copy).
            if (NS > 2 && next)
                wait_vm<(NS - 2) * TL::copies>();
            else
                wait_vm<0>();
            lds_barrier();  // for every wave; the buffer of stage kt - 1 is fully read
            const int slice = kt * KS + ks;
            if (next) {
                issue_rows(ws, slice_of(kt + NS - 1));
                issue_scales(ws, slice_of(kt + NS - 1));
            }
            if (KS == 1 || slice < nslices) {
                const lds_u8* const st = smem + rs * TL::stage_b + ks * TL::slice_b;
                const lds_u8* const stx = st + (TL::cols + 16 * WNT * wn) * kRowB;
                const lds_u8* const stw = st + 16 * WMT * wm * kRowB;
                const bool both = kFp4X || 2 * slice + 1 < nblocks;
                if constexpr (!kBf16) {
                    uint32_t sx[2][NSX], sw[2];
                    read_sx(st, sx);
                    read_sw(st, sw);
                    X2 x[WNT];
                    static_for<0, WNT>([&](auto NT) { x[decltype(NT)::value] = frag_x(stx + 16 * decltype(NT)::value * kRowB); });
                    W2 w[WMT];
                    static_for<0, WMT>([&](auto MT) { w[decltype(MT)::value] = frag_w(stw + 16 * decltype(MT)::value * kRowB); });
                    static_for<0, 2>([&](auto H) {
                        if (decltype(H)::value == 1 && !both) return;
                        static_for<0, WMT>([&](auto MT) {
                            static_for<0, WNT>([&](auto NT) { multiply(H, MT, NT, x[decltype(NT)::value], w[decltype(MT)::value], sx, sw); });
                        });
                    });
                } else {
                    static_for<0, 2>([&](auto H) {
                        constexpr int h = decltype(H)::value;
                        if (h == 1 && !both) return;
                        // W's scales over the block's largest of its column, and that one
                        uint32_t words[WMT], own[WMT], most[WMT];
                        read_words(st + TL::off_ws + 4 * (h * TL::cols + 16 * WMT * wm + WMT * r16), std::integral_constant<int, WMT>{}, words);
#pragma unroll
                        for (int mt = 0; mt < WMT; ++mt) {
                            most[mt] = largest_byte(words[mt]);
                            own[mt] = byte_over(words[mt] >> (8 * g4) & 0xffu, most[mt]);
                        }
                        f32x4 block[WMT][WNT];
                        u32x4 wc[WMT];
#pragma unroll
                        for (int mt = 0; mt < WMT; ++mt) {
                            wc[mt] = half(stw + 16 * mt * kRowB, h);
#pragma unroll
                            for (int nt = 0; nt < WNT; ++nt) block[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
                        }
                        // values 32 g4 .. + 31 of the row: 16-byte pieces 2 g4 and 2 g4 + 1
                        static_for<0, 2>([&](auto P) {
                            u32x4 xc[WNT];
#pragma unroll
                            for (int nt = 0; nt < WNT; ++nt)
                                xc[nt] = *reinterpret_cast<const lds_u32x4*>(stx + (h * TL::toks + 16 * nt + r16) * kRowB + 16 * ((2 * g4 + decltype(P)::value) ^ swz(r16)));
                            static_for<0, 2>([&](auto Q) {
                                constexpr int q = decltype(Q)::value;
                                bf16x8 x[WNT];
                                static_for<0, WNT>([&](auto NT) { x[decltype(NT)::value] = codes_to_bf16<FA>(xc[decltype(NT)::value][2 * q], xc[decltype(NT)::value][2 * q + 1], 127u); });
                                static_for<0, WMT>([&](auto MT) {
                                    constexpr int mt = decltype(MT)::value;
                                    const bf16x8 w = fp4_to_bf16(wc[mt][2 * decltype(P)::value + q], own[mt]);
                                    static_for<0, WNT>([&](auto NT) { block[mt][decltype(NT)::value] = mfma16x16x32(x[decltype(NT)::value], w, block[mt][decltype(NT)::value]); });
                                });
                            });
                        });
                        static_for<0, WNT>([&](auto NT) {
                            constexpr int nt = decltype(NT)::value;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t s = st[TL::off_xs + h * TL::toks + 16 * WNT * wn + WNT * (4 * g4 + i) + nt];
#pragma unroll
                                for (int mt = 0; mt < WMT; ++mt) acc[mt][nt][i] += scaled_sum(block[mt][nt][i], s, most[mt]);
                            }
                        });
                    });
                }
            }
            rs = rs + 1 == NS ? 0 : rs + 1;
            ws = ws + 1 == NS ? 0 : ws + 1;
        }
        if constexpr (KS > 1) {
            const auto part = [&](int k, int i) {
                return reinterpret_cast<lds_f32x4*>(smem + (((k - 1) * TL::gwaves + gw) * WMT * WNT + i) * 1024 + 16 * lane);
            };
            lds_barrier();  // every wave is past its last stage read
            if (ks > 0) {
#pragma unroll
                for (int i = 0; i < WMT * WNT; ++i) *part(ks, i) = acc[i / WNT][i % WNT];
            }
            lds_barrier();
            if (ks > 0) return;
#pragma unroll
            for (int k = 1; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < WMT * WNT; ++i) acc[i / WNT][i % WNT] += *part(k, i);
        }
        store_tile(f0, c0);
    }
}

}  // namespace

namespace gdn_fp4 {

template <class TL, int FA, bool OUT32>
int launch_tiled(const MatmulParams& p, hipStream_t stream) {
    const int n_tok = (p.M + TL::toks - 1) / TL::toks, n_col = (p.N + TL::cols - 1) / TL::cols;
    const unsigned tiles = static_cast<unsigned>(n_tok) * n_col;
    const dim3 grid(TL::PHASED && tiles > 256 ? 256 : tiles);  // phased: a workgroup a CU
    if (!gdn_host::grid_fits(grid.x, TL::waves * 64))
        return gdn_host::fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: M=%d N=%d are too large for a launch", p.M, p.N);
    hipLaunchKernelGGL((gdn_fp4_matmul_kernel<TL, FA, OUT32>), grid, dim3(TL::waves * 64), 0, stream, p, n_tok, n_col);
    return gdn_host::check_launch("gdn_fp4_matmul_kernel");
}

// columns x tokens; where 8-bit rows of x need the room, with fewer stages or groups
template <int FA, bool OUT32>
int launch_out(int tile, const MatmulParams& p, hipStream_t stream) {
    constexpr int XH = FA == GDN_E2M1 ? 1 : 2;
    if constexpr (XH == 1) {
        switch (tile) {
            case k256x256: return launch_tiled<Fp4Tile<XH, 4, 2, 4, 8, 2, 1, 1, true>, FA, OUT32>(p, stream);
            case k256x192: return launch_tiled<Fp4Tile<XH, 4, 2, 4, 6, 2, 1, 1, true>, FA, OUT32>(p, stream);
        }
    }
    if constexpr (XH == 1 || !OUT32) {
        switch (tile) {
            case k256x160: return launch_tiled<Fp4Tile<XH, 4, 2, 4, 5, 2, 1, 1, true>, FA, OUT32>(p, stream);
            case k256x128: return launch_tiled<Fp4Tile<XH, 4, 2, 4, 4, XH == 1 ? 3 : 2, 1, 1, true>, FA, OUT32>(p, stream);
            case k128x192: return launch_tiled<Fp4Tile<XH, 2, 4, 4, 3, XH == 1 ? 3 : 2, 1, 1, true>, FA, OUT32>(p, stream);
        }
    }
    switch (tile) {
        case k64x128: return launch_tiled<Fp4Tile<XH, 1, 4, 4, 2, 3, 1, XH == 1 ? 2 : 1>, FA, OUT32>(p, stream);
        case k64x64: return launch_tiled<Fp4Tile<XH, 2, 2, 2, 2, 3, 1, 2>, FA, OUT32>(p, stream);
        case k64x32: return launch_tiled<Fp4Tile<XH, 1, 2, 4, 1, XH == 1 ? 3 : 2, 1, 4>, FA, OUT32>(p, stream);
        case k32x32: return launch_tiled<Fp4Tile<XH, 1, 2, 2, 1, XH == 1 ? 3 : 2, 1, 4>, FA, OUT32>(p, stream);
        case k16x16Alone: return launch_tiled<Fp4Tile<XH, 1, 1, 1, 1, XH == 1 ? 4 : 3, 1, 8>, FA, OUT32>(p, stream);
        case k16x16: return launch_tiled<Fp4Tile<XH, 1, 1, 1, 1, XH == 1 ? 3 : 2, 3, 4>, FA, OUT32>(p, stream);
        default: return launch_tiled<Fp4Tile<XH, 2, 4, 4, 2, XH == 1 ? 4 : 3, 1>, FA, OUT32>(p, stream);
    }
}

template <int FA>
int launch_tile(int tile, bool f32, const MatmulParams& p, hipStream_t stream) {
    return f32 ? launch_out<FA, true>(tile, p, stream) : launch_out<FA, false>(tile, p, stream);
}

}  // namespace gdn_fp4
