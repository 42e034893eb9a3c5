// The tiled kernel of the fp8 block-scaled product
//   out[m, n] = sum over blocks kb of a_scale[m, kb] b_scale[n, kb] sum_k a[m, k] b[n, k]
// with fp32 sums, one rounding where out is written.
//
// In tiles of columns x tokens (W = b, x = a).  A stage is one block of 128 k:
// 128-byte rows, which reach LDS by DMA in a ring, every 8 lanes of a copy one
// whole line, placed with an XOR swizzle that keeps the fragment reads at
// linear-read speed; the stage's scales come with it.  bf16 results: one MFMA
// 16x16x128 takes a block: e8m0 scales are its own scale operands and cost nothing;
// of fp32 scales it takes the powers of two so, and the rest multiplies its result
// on the VALU, into the accumulator.  fp32 results: codes become bf16 in registers,
// times their e8m0 scale, and the block takes four MFMA 16x16x32, whose sums keep
// every bit that fp32 has.  Codes times scales far from 1 leave bf16's range: a
// workgroup that met one computes its tile again, block after block, for the rows
// and columns that have such scales (2048 x 2048 x 2688 27.3 us, 27.5 with the
// question; asking it before each block's product made the block wait for its
// scales, 30.4 us).
//
// What bounds it: the matrix cores for large products, and there the card's
// power: 8192 x 8192 x 8192 takes 413 us (2.66 PFLOP/s) with random codes and 345
// with zeros.  Waves of 128 x 128 (half the LDS reads a product) changed nothing
// for that reason.  A 256 x 256 tile takes 1.2-1.5 us a block of K and some 6.6
// to begin, fill the ring and store, of which a persistent workgroup hides the
// filling behind the stores before it: 16384 x 6176 x 2048, 193 us.  Running the
// stages on over tile borders (8192 x 8192 x 8192: 420 us), non-temporal stores
// (213 against 185 us at 16384 x 6144 x 2048) and staggered starts were slower or
// no faster.  Products of one round of tiles are bound by how many of the 256 CUs
// have one (1500 x 8224 x 2048: 198 tiles, 28 us, 1.8 PFLOP/s), small ones by
// how fast a CU takes in its rows, which more, smaller tiles with K over groups of
// waves spread over the CUs (fp8_matmul.hip has the figures).
#pragma once

#include "fp8_matmul.hpp"

namespace {

constexpr int kRowB = 128;  // bytes of a staged row: one block

// CW x TW waves, each WMT 16-column x WNT 16-token MFMA tiles, NS stages in LDS,
// PER_CU workgroups on a CU; KS groups of such waves, each on its own block of a
// stage of KS blocks, summed at the end.  PHASED: the two-group main loop (eight
// waves, one workgroup on a CU).
template <int CW_, int TW_, int WMT_, int WNT_, int NS_, int PER_CU_, int KS_ = 1, bool PHASED_ = false>
struct Fp8Tile {
    static constexpr int CW = CW_, TW = TW_, WMT = WMT_, WNT = WNT_, NS = NS_, PER_CU = PER_CU_, KS = KS_;
    static constexpr bool PHASED = PHASED_;
    static constexpr int cols = 16 * CW * WMT, toks = 16 * TW * WNT;
    static constexpr int gwaves = CW * TW, waves = gwaves * KS;
    static constexpr int dma = (cols + toks) / 8 / gwaves;  // 1 KiB copies (8 rows) a wave and block
    static_assert(PHASED || (cols + toks) % (8 * gwaves) == 0, "copies split evenly");
    static_assert(128 % (16 * WMT) == 0, "a wave's columns share a 128-column block");
    // PHASED: a stage is staged, and its buffer freed, region by region: the
    // first and second part of every wave's tokens (X0, X1) and columns (W0,
    // W1), in the order X0 and the scales, W0, W1, X1.  A region of `groups`
    // 4-row pieces is split over the waves, each taking whole copies of 8 rows
    // and, where 8 pieces are left, one of 4 rows by half its lanes.
    static constexpr int M0n = WMT / 2, M1n = WMT - M0n, X0n = (WNT + 1) / 2, X1n = WNT - X0n;
    static constexpr int groups(int r) { return 4 * (r == 0 ? TW * X0n : r == 1 ? CW * M0n : r == 2 ? CW * M1n : TW * X1n); }
    static constexpr int full(int r) { return groups(r) / 16; }
    static constexpr int piece(int r) { return groups(r) % 16 / 8; }
    static constexpr int ncopy(int r) { return full(r) + piece(r); }
    static constexpr int first(int r) { return r == 0 ? 0 : first(r - 1) + ncopy(r - 1); }
    static constexpr int copies = PHASED ? first(4) : dma;
    static_assert(!PHASED || (waves == 8 && PER_CU == 1 && KS == 1 && groups(0) % 8 == 0 && groups(1) % 8 == 0 && groups(2) % 8 == 0 &&
                              groups(3) % 8 == 0 && M0n > 0 && X1n > 0),
                  "phased tile");
};

// A stage's bytes with b's scales as SB says: rows, x scales, W scales.
template <class TL, int SB>
struct Fp8Stage {
    static constexpr int off_xs = (TL::cols + TL::toks) * kRowB;
    static constexpr int off_ws = off_xs + TL::toks;
    static constexpr int wsb = SB == gdn_fp8::kE8Row ? TL::cols : SB == gdn_fp8::kF32Row ? 4 * TL::cols : 0;
    static constexpr int slice_b = (off_ws + wsb + 127) / 128 * 128;
    static constexpr int stage_b = TL::KS * slice_b;
    static constexpr int scale_copies = 1 + (wsb > 0 ? 1 : 0);  // a wave issues, for a block
    static constexpr int copies = TL::copies + scale_copies;
    static constexpr int lds_b = TL::NS * stage_b;
    static_assert(lds_b * TL::PER_CU <= 160 * 1024, "LDS");
    static_assert((TL::KS - 1) * TL::gwaves * TL::WMT * TL::WNT * 1024 <= lds_b, "the groups' sums fit the dead stages");
};

__device__ __forceinline__ int swz(int r) { return r & 7; }

// Workgroup barrier alone (no LDS access of this wave is outstanding); no
// memory access moves across it.
__device__ __forceinline__ void wave_barrier() { asm volatile("s_barrier" ::: "memory"); }

template <class TL, int FA, int FB, int SB, bool OUT32>
__global__ __launch_bounds__(TL::waves * 64)
    __attribute__((amdgpu_waves_per_eu(TL::PER_CU * TL::waves / 4, TL::PER_CU * TL::waves / 4))) void gdn_fp8_matmul_kernel(
        gdn_fp8::MatmulParams p, int n_tok, int n_col) {
    using ST = Fp8Stage<TL, SB>;
    constexpr int WMT = TL::WMT, WNT = TL::WNT, NS = TL::NS, KS = TL::KS;
    constexpr bool kRow = SB == gdn_fp8::kE8Row || SB == gdn_fp8::kF32Row;
    constexpr bool kF32 = SB == gdn_fp8::kF32Block || SB == gdn_fp8::kF32Row;
    __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[ST::lds_b];
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
    const int nslices = p.K / kRowB;

    // Copy sources.  Staged rows 0 .. cols - 1 are rows of b, the others rows of
    // a, in an order that gives a lane of the product WMT neighbouring columns and
    // lets it supply WNT neighbouring tokens, whose scales are neighbouring bytes
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
        const int w = (srow - TL::cols) / (16 * WNT), s = (srow - TL::cols) % (16 * WNT);
        const int tok = 16 * WNT * w + WNT * (s & 15) + (s >> 4);
        return static_cast<uint32_t>(min(f0 + tok, p.M - 1) - f0) * static_cast<uint32_t>(p.lda) + chunk;
    };
    // Copy j of region r in the phased loop: the first staged row, the same for
    // the wave.
    auto copy_row = [&](int r, int j) {
        const int g = j < TL::full(r) ? 2 * (wave + 8 * j) : 16 * TL::full(r) + wave;                   // in 4-row pieces
        const int per = 4 * (r == 0 ? TL::X0n : r == 1 ? TL::M0n : r == 2 ? TL::M1n : TL::X1n);  // pieces of one wave's part
        const int w = g / per, within = 4 * (g % per);
        return r == 0 || r == 3 ? TL::cols + 16 * WNT * w + (r == 3 ? 16 * TL::X0n : 0) + within
                                : 16 * WMT * w + (r == 2 ? 16 * TL::M0n : 0) + within;
    };
    uint32_t voff[TL::copies], xs_off, ws_off;
    int crow[TL::copies];  // staged row of the copy's first lane (wave-uniform)
    if constexpr (TL::PHASED) {
        static_for<0, 4>([&](auto R) {
            constexpr int r = decltype(R)::value;
            static_for<0, TL::ncopy(r)>([&](auto J) { crow[TL::first(r) + decltype(J)::value] = __builtin_amdgcn_readfirstlane(copy_row(r, decltype(J)::value)); });
        });
    } else {
#pragma unroll
        for (int j = 0; j < TL::copies; ++j) crow[j] = 8 * (gw + TL::gwaves * j);
    }
    // The scales' copies: the waves of a group share 16-byte pieces out, each
    // wave one copy of at least one piece (the last waves may repeat pieces).
    constexpr int kXPieces = TL::toks / 16, kXLanes = (kXPieces + TL::gwaves - 1) / TL::gwaves;
    constexpr int kWPieces = ST::wsb / 16, kWLanes = (kWPieces + TL::gwaves - 1) / TL::gwaves;
    constexpr int kElem = kF32 ? 4 : 1;
    const int xp = min(gw * kXLanes, kXPieces - kXLanes), wp = min(gw * kWLanes, kWPieces - kWLanes);
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
            for (int i = 0; i < TL::copies; ++i) voff[i] = src_off(crow[i] + (lane >> 3), lane);
        }
        xs_off = static_cast<uint32_t>(min(f0 + 16 * (xp + lane), (p.M - 1) / 16 * 16));
        ws_off = static_cast<uint32_t>(min(c0 + 16 / kElem * (wp + lane), (p.N - 1) / 16 * 16 + 16 - 16 / kElem)) * kElem;
    };
    auto issue_rows = [&](int stage, int slice) {
        lds_u8* const dst = smem + stage * ST::stage_b + ks * ST::slice_b;
#pragma unroll
        for (int j = 0; j < TL::copies; ++j)
            dma16((crow[j] < TL::cols ? wsrc : xsrc) + static_cast<size_t>(slice) * kRowB, voff[j], dst + crow[j] * kRowB);
    };
    auto issue_scales = [&](int stage, int slice) {
        lds_u8* const dst = smem + stage * ST::stage_b + ks * ST::slice_b;
        if (lane < kXLanes) dma16(p.a_scale + slice * p.lda_s, xs_off, dst + ST::off_xs + 16 * xp);
        if constexpr (kRow) {
            if (lane < kWLanes)
                dma16(static_cast<const uint8_t*>(p.b_scale) + slice * p.ldb_s * kElem, ws_off, dst + ST::off_ws + 16 * wp);
        }
    };
    // Region r of a stage (phased loop); the scales come with the first.
    auto issue_region = [&](auto R, int stage, int slice) {
        constexpr int r = decltype(R)::value;
        const uint8_t* const src = (r == 0 || r == 3 ? xsrc : wsrc) + static_cast<size_t>(slice) * kRowB;
        static_for<0, TL::ncopy(r)>([&](auto J) {
            constexpr int j = decltype(J)::value, c = TL::first(r) + j;
            if (j < TL::full(r) || lane < 32) dma16(src, voff[c], smem + stage * ST::stage_b + crow[c] * kRowB);
        });
        if constexpr (r == 0) issue_scales(stage, slice);
    };
    // The block of stage kk that this wave's group takes (the last stage's
    // groups past the end repeat the last block and do not multiply it).
    auto slice_of = [&](int kk) { return KS > 1 ? min(kk * KS + ks, nslices - 1) : kk; };

    // Block scales of b: lane l holds that of block 64 w + l, w the window of 64
    // blocks the loop is in, and a stage reads its own into a scalar.
    uint32_t wscale = 127u;
    auto block_scales = [&](int c, int slice) -> uint32_t {  // of the wave's columns in the tile at column c
        if constexpr (kRow) return 127u;
        const int nb = min(c + 16 * WMT * wm, p.N - 1) / kRowB;
        const size_t at = static_cast<size_t>(nb) * p.ldb_s + min(slice / 64 * 64 + lane, nslices - 1);
        return kF32 ? static_cast<const uint32_t*>(p.b_scale)[at] : static_cast<const uint8_t*>(p.b_scale)[at];
    };
    // Landed here: no wait of the compiler's falls between the copies' own.
    auto landed = [](uint32_t& v) { asm volatile("" : "+v"(v)); };
    auto load_block_scales = [&](int slice) {
        wscale = block_scales(c0, slice);
        landed(wscale);
    };

    uint32_t rd[2];
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
    // W's scales of a staged block: WMT bytes of neighbouring columns in a word, the
    // block's byte in each, or WMT floats, whose powers of two the fp8 instruction
    // takes as bytes (split_w; the bf16 instruction's sums are in range without).
    auto read_sw = [&](const lds_u8* st, int slice, uint32_t (&sw)[WMT], float (&fw)[WMT]) {
        if constexpr (kF32) {
            const __attribute__((address_space(3))) float* const at = reinterpret_cast<const lds_f32*>(st + ST::off_ws) + 16 * WMT * wm + WMT * r16;
#pragma unroll
            for (int mt = 0; mt < WMT; ++mt) {
                sw[mt] = 127u;
                if constexpr (SB == gdn_fp8::kF32Row)
                    fw[mt] = at[mt];
                else
                    fw[mt] = __int_as_float(__builtin_amdgcn_readlane(static_cast<int>(wscale), slice & 63));
            }
        } else if constexpr (SB == gdn_fp8::kE8Block) {
            sw[0] = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wscale), slice & 63)) * 0x01010101u;
        } else {
            const lds_u8* const at = st + ST::off_ws + 16 * WMT * wm + WMT * r16;
            if constexpr (WMT == 4)
                sw[0] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at);
            else if constexpr (WMT == 2)
                sw[0] = *reinterpret_cast<const lds_u16*>(at);
            else
                sw[0] = *at;
        }
    };
    auto split_w = [&](auto MT, uint32_t (&sw)[WMT], float (&fw)[WMT]) {
        constexpr int mt = decltype(MT)::value;
        if constexpr (kF32) {
            const uint32_t bits = __float_as_uint(fw[mt]);
            sw[mt] = scale_byte_of(bits);
            fw[mt] = scale_rest(bits, sw[mt]);
        }
    };
    // Column mt's byte.
    auto byte_w = [&](int mt, const uint32_t (&sw)[WMT]) { return kF32 ? sw[mt] : sw[0] >> (8 * mt) & 0xffu; };
    // x's scales of a staged block, WNT bytes of neighbouring tokens: in words
    // where WNT is a power of two, else a register each.
    constexpr bool kWords = (WNT & (WNT - 1)) == 0;
    constexpr int NSX = kWords ? (WNT + 3) / 4 : WNT;
    auto read_sx = [&](const lds_u8* st, uint32_t (&sx)[NSX]) {
        const lds_u8* at = st + ST::off_xs + 16 * WNT * wn + WNT * r16;
        if constexpr (WNT == 8) {
            const u32x2 v = *reinterpret_cast<const lds_u32x2*>(at);
            sx[0] = v[0];
            sx[1] = v[1];
        } else if constexpr (WNT == 4) {
            sx[0] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at);
        } else if constexpr (WNT == 2) {
            sx[0] = *reinterpret_cast<const lds_u16*>(at);
        } else {
#pragma unroll
            for (int nt = 0; nt < WNT; ++nt) sx[nt] = at[nt];
        }
    };

    // One block's product of operands mt and nt into the accumulator.
    auto multiply = [&](auto MT, auto NT, const i32x8& x, const i32x8& w, const uint32_t (&sx)[NSX], const uint32_t (&sw)[WMT], const float (&fw)[WMT]) {
        constexpr int mt = decltype(MT)::value, nt = decltype(NT)::value, bx = kWords ? nt % 4 : 0;
        const int s = static_cast<int>(sx[kWords ? nt / 4 : nt]);
        if constexpr (kF32) {
            const f32x4 t = mfma_fp8<FA, FB, bx, 0>(x, w, f32x4{0.f, 0.f, 0.f, 0.f}, s, static_cast<int>(sw[mt]));
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[mt][nt][i] = fmaf(fw[mt], t[i], acc[mt][nt][i]);
        } else {
            acc[mt][nt] = mfma_fp8<FA, FB, bx, mt>(x, w, acc[mt][nt], s, static_cast<int>(sw[0]));
        }
    };

    const int nk = (nslices + KS - 1) / KS;
    int tile = static_cast<int>(blockIdx.x) >> 3;
    set_tile(tile);
    load_block_scales(0);
    uint32_t x_near = ~0u, w_near = ~0u;  // the AND of the near_bits of the scales that the lane met

    if constexpr (TL::PHASED) {
        // Two groups of four waves, one wave of each on every SIMD, take turns:
        // while one multiplies, the other reads its next fragments and issues its
        // copies.  A stage is four phases, each a part of the wave's tile (first
        // or second half of its columns x of its tokens) over the whole block:
        // (W0, X0), (W1, X0), (W1, X1), (W0, X1).  Phase 0 reads W0, X0 and the
        // scales, phase 1 W1, phase 2 X1, phase 3 nothing.  A region's buffer is
        // free once both groups have read it, so stage kt + NS's X0, W0 and W1 go
        // out in phases 1, 2 and 3 of stage kt and its X1 in phase 0 of the next.
        // The waits count the copies issued after the region that the next phase
        // reads; T >= 0: T stages are left after this one and no new ones are
        // issued.
        static_assert(!OUT32, "fp32 results run on the ring");
        i32x8 w0[TL::M0n], w1[TL::M1n], xf[TL::X0n];
        uint32_t sx[NSX];
        uint32_t sw[WMT];
        float fw[WMT];
        constexpr int cX0 = TL::ncopy(0) + ST::scale_copies, cW1 = TL::ncopy(2), cX1 = TL::ncopy(3), cAll = ST::copies;
        auto frag = [&](const lds_u8* at) { return join(half(at, 0), half(at, 1)); };
        auto next_buf = [](int b, int n) {
            b += n;
            return b >= NS ? b - NS : b;
        };
        auto stage = [&](int kt, int rs, auto Tc) {
            constexpr int T = decltype(Tc)::value;
            constexpr bool steady = T < 0;
            const lds_u8* st = smem + rs * ST::stage_b;
            const lds_u8* stx = st + (TL::cols + 16 * WNT * wn) * kRowB;
            const lds_u8* stw = st + 16 * WMT * wm * kRowB;
            static_for<0, 4>([&](auto Pc) {
                constexpr int ph = decltype(Pc)::value;
                if constexpr (ph == 0) {
                    static_for<0, TL::M0n>([&](auto I) { w0[decltype(I)::value] = frag(stw + 16 * decltype(I)::value * kRowB); });
                    static_for<0, TL::X0n>([&](auto I) { xf[decltype(I)::value] = frag(stx + 16 * decltype(I)::value * kRowB); });
                    read_sx(st, sx);
                    read_sw(st, kt, sw, fw);
                    static_for<0, TL::M0n>([&](auto I) { split_w(I, sw, fw); });
                } else if constexpr (ph == 1) {
                    static_for<TL::M0n, WMT>([&](auto I) { split_w(I, sw, fw); });
                    static_for<0, TL::M1n>([&](auto I) { w1[decltype(I)::value] = frag(stw + 16 * (TL::M0n + decltype(I)::value) * kRowB); });
                } else if constexpr (ph == 2) {
                    static_for<0, TL::X1n>([&](auto I) { xf[decltype(I)::value] = frag(stx + 16 * (TL::X0n + decltype(I)::value) * kRowB); });
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
                static_for<0, nn>([&](auto NT) {
                    constexpr int nt = n0 + decltype(NT)::value;
                    static_for<0, mn>([&](auto MT) {
                        constexpr int mt = m0 + decltype(MT)::value;
                        const i32x8 w = m0 == 0 ? w0[mt - m0] : w1[mt - m0];
                        multiply(std::integral_constant<int, mt>{}, std::integral_constant<int, nt>{}, xf[nt - n0], w, sx, sw, fw);
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
            uint32_t wnext = wscale;
            if (more) {
                int f, c;
                tile_at(tile + step, f, c);
                wnext = block_scales(c, 0);
            }
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
                if (!kRow && kt > 0 && kt % 64 == 0) load_block_scales(kt);
                stage(kt, rs, std::integral_constant<int, -1>{});
                rs = next_buf(rs, 1);
            }
            static_for<0, NS>([&](auto I) {
                constexpr int T = NS - 1 - decltype(I)::value;
                if (T < nk) {
                    if (!kRow && kt > 0 && kt % 64 == 0) load_block_scales(kt);
                    stage(kt, rs, std::integral_constant<int, T>{});
                    ++kt;
                    rs = next_buf(rs, 1);
                }
            });
            if (!second) wave_barrier();
            landed(wnext);
            const int f = f0, c = c0;
            if (more) {
                tile += step;
                set_tile(tile);
                wscale = wnext;
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
                wait_vm<(NS - 2) * ST::copies>();
            else
                wait_vm<0>();
            lds_barrier();  // for every wave; the buffer of stage kt - 1 is fully read
            const int slice = kt * KS + ks;
            if (!kRow && kt > 0 && kt * KS % 64 == 0) load_block_scales(min(slice, nslices - 1));
            if (next) {
                issue_rows(ws, slice_of(kt + NS - 1));
                issue_scales(ws, slice_of(kt + NS - 1));
            }
            if (KS == 1 || slice < nslices) {
                const lds_u8* const st = smem + rs * ST::stage_b + ks * ST::slice_b;
                const lds_u8* const stx = st + (TL::cols + 16 * WNT * wn) * kRowB;
                const lds_u8* const stw = st + 16 * WMT * wm * kRowB;
                uint32_t sx[NSX];
                read_sx(st, sx);
                uint32_t sw[WMT];
                float fw[WMT];
                read_sw(st, slice, sw, fw);
                if constexpr (!OUT32) {
                    static_for<0, WMT>([&](auto MT) { split_w(MT, sw, fw); });
                    i32x8 x[WNT];
                    static_for<0, WNT>([&](auto NT) {
                        constexpr int nt = decltype(NT)::value;
                        x[nt] = join(half(stx + 16 * nt * kRowB, 0), half(stx + 16 * nt * kRowB, 1));
                    });
                    static_for<0, WMT>([&](auto MT) {
                        constexpr int mt = decltype(MT)::value;
                        const i32x8 w = join(half(stw + 16 * mt * kRowB, 0), half(stw + 16 * mt * kRowB, 1));
                        static_for<0, WNT>([&](auto NT) { multiply(MT, NT, x[decltype(NT)::value], w, sx, sw, fw); });
                    });
                } else {
                    x_near &= near_bits(sx[0]);
                    if constexpr (!kF32) w_near &= near_bits(sw[0]);
                    f32x4 block[kF32 ? WMT : 1][kF32 ? WNT : 1];  // fp32 scales: this block's sums
                    if constexpr (kF32) {
#pragma unroll
                        for (int mt = 0; mt < WMT; ++mt)
#pragma unroll
                            for (int nt = 0; nt < WNT; ++nt) block[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
                    }
                    static_for<0, 2>([&](auto H) {
                        constexpr int h = decltype(H)::value;
                        u32x4 xc[WNT], wc[WMT];
#pragma unroll
                        for (int nt = 0; nt < WNT; ++nt) xc[nt] = half(stx + 16 * nt * kRowB, h);
#pragma unroll
                        for (int mt = 0; mt < WMT; ++mt) wc[mt] = half(stw + 16 * mt * kRowB, h);
                        static_for<0, 2>([&](auto Q) {
                            constexpr int q = decltype(Q)::value;
                            bf16x8 x[WNT];
                            static_for<0, WNT>([&](auto NT) {
                                constexpr int nt = decltype(NT)::value;
                                x[nt] = codes_to_bf16<FA>(xc[nt][2 * q], xc[nt][2 * q + 1], kWords ? sx[nt / 4] >> (8 * (nt % 4)) & 0xffu : sx[nt]);
                            });
                            static_for<0, WMT>([&](auto MT) {
                                constexpr int mt = decltype(MT)::value;
                                const bf16x8 w = codes_to_bf16<FB>(wc[mt][2 * q], wc[mt][2 * q + 1], byte_w(mt, sw));
                                static_for<0, WNT>([&](auto NT) {
                                    constexpr int nt = decltype(NT)::value;
                                    f32x4& c = kF32 ? block[kF32 ? mt : 0][kF32 ? nt : 0] : acc[mt][nt];
                                    c = mfma16x16x32(x[nt], w, c);
                                });
                            });
                        });
                    });
                    if constexpr (kF32) {
#pragma unroll
                        for (int mt = 0; mt < WMT; ++mt)
#pragma unroll
                            for (int nt = 0; nt < WNT; ++nt)
#pragma unroll
                                for (int i = 0; i < 4; ++i) acc[mt][nt][i] = fmaf(fw[mt], block[kF32 ? mt : 0][kF32 ? nt : 0][i], acc[mt][nt][i]);
                    }
                }
            }
            rs = rs + 1 == NS ? 0 : rs + 1;
            ws = ws + 1 == NS ? 0 : ws + 1;
        }
    }

    // fp32 results: whether a wave met a scale that is not near, in any row but those
    // past the last one, which may have any.
    __shared__ uint32_t met_far[TL::waves];
    if constexpr (OUT32) {
        constexpr uint32_t x_top = 0x80808080u >> (8 * (4 - WNT)), w_top = 0x80808080u >> (8 * (4 - WMT));
#pragma unroll
        for (int nt = 0; nt < WNT; ++nt)
            if (f0 + 16 * WNT * wn + WNT * r16 + nt >= p.M) x_near |= 0x80u << (8 * nt);
        if constexpr (kRow) {
#pragma unroll
            for (int mt = 0; mt < WMT; ++mt)
                if (c0 + 16 * WMT * wm + WMT * r16 + mt >= p.N) w_near |= 0x80u << (8 * mt);
        }
        met_far[wave] = __builtin_amdgcn_ballot_w64((~x_near & x_top) != 0 || (~w_near & w_top) != 0) != 0;
    }
    if constexpr (KS > 1 || OUT32) lds_barrier();  // every wave is past its last stage read
    auto any_far = [&]() {
        if constexpr (OUT32) return __builtin_amdgcn_ballot_w64(met_far[lane % TL::waves] != 0) != 0;
        return false;
    };
    const auto part = [&](int k, int i) {
        return reinterpret_cast<lds_f32x4*>(smem + (((k - 1) * TL::gwaves + gw) * WMT * WNT + i) * 1024 + 16 * lane);
    };
    if constexpr (KS > 1) {
        if (ks > 0) {
#pragma unroll
            for (int i = 0; i < WMT * WNT; ++i) *part(ks, i) = acc[i / WNT][i % WNT];
        }
        lds_barrier();
        if (ks > 0 && !any_far()) return;
    }
    if (KS == 1 || ks == 0) {
        if constexpr (KS > 1) {
#pragma unroll
            for (int k = 1; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < WMT * WNT; ++i) acc[i / WNT][i % WNT] += *part(k, i);
        }
        store_tile(f0, c0);
    }
    if constexpr (OUT32) {
        if ((KS == 1 || ks == 0) && !any_far()) return;
        // The tile once more, block after block, for the rows and columns that have a
        // scale which is not near: with scales nearby, and the powers of two that are
        // left on each block's sums.  Results of other rows and columns stay as they
        // are, so that they do not depend on their neighbours.  K's first group of waves
        // does it, the others keep to the barriers.
        clear();
        uint32_t far_tok = 0, far_col = 0;  // bit 4 nt + i: of accumulator (., nt)[i]'s token; bit mt: of (mt, .)'s column
        for (int slice = 0; slice < nslices; ++slice) {
            int lane = tid & 63;
            asm volatile("" : "+v"(lane));  // nothing of this is kept over the loop above
            const int r16 = lane & 15, g4 = lane >> 4;
            lds_barrier();  // the last block's rows, or the groups' sums, are read
            if (!kRow && slice % 64 == 0) load_block_scales(slice);
            if (KS == 1 || ks == 0) {
                issue_rows(0, slice);
                issue_scales(0, slice);
            }
            wait_vm<0>();
            lds_barrier();
            if (KS > 1 && ks > 0) continue;
            const lds_u8* const stx = smem + (TL::cols + 16 * WNT * wn) * kRowB;
            const lds_u8* const stw = smem + 16 * WMT * wm * kRowB;
            uint32_t sx[NSX], sw[WMT];
            float fw[WMT];
            read_sx(smem, sx);
            read_sw(smem, slice, sw, fw);
            static_for<0, WNT>([&](auto NT) {
                constexpr int nt = decltype(NT)::value;
                const int x = static_cast<int>(sx[0] >> (8 * nt) & 0xffu);
                int s[4];  // the accumulators' tokens' scales
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[i] = smem[ST::off_xs + 16 * WNT * wn + WNT * (4 * g4 + i) + nt];
                    far_tok |= (~near_bits(s[i]) >> 7 & 1u) << (4 * nt + i);
                }
                static_for<0, WMT>([&](auto MT) {
                    constexpr int mt = decltype(MT)::value;
                    const int w = static_cast<int>(byte_w(mt, sw));
                    if (nt == 0) far_col |= (~near_bits(w) >> 7 & 1u) << mt;
                    f32x4 sums = {0.f, 0.f, 0.f, 0.f};
                    static_for<0, 2>([&](auto H) {
                        const u32x4 xc = half(stx + 16 * nt * kRowB, decltype(H)::value), wc = half(stw + 16 * mt * kRowB, decltype(H)::value);
                        __builtin_amdgcn_sched_barrier(0);  // one after the other, in few registers
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            sums = mfma16x16x32(codes_to_bf16<FA>(xc[2 * q], xc[2 * q + 1], nearby(x)),
                                                codes_to_bf16<FB>(wc[2 * q], wc[2 * q + 1], nearby(w)), sums);
                    });
                    int left = w - nearby(w);
                    float rest = 1.f;
                    if constexpr (kF32) {
                        const uint32_t bits = __float_as_uint(fw[mt]), byte = scale_byte_of(bits);
                        left = static_cast<int>(byte) - 127;
                        rest = scale_rest(bits, byte);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[mt][nt][i] = fmaf(rest, __builtin_amdgcn_ldexpf(sums[i], s[i] - nearby(s[i]) + left), acc[mt][nt][i]);
                    __builtin_amdgcn_sched_barrier(0);
                });
            });
        }
        if (KS > 1 && ks > 0) return;
        static_for<0, 4 * WNT>([&](auto J) {
            constexpr int i = decltype(J)::value / WNT, nt = decltype(J)::value % WNT;
            const int row = f0 + 16 * WNT * wn + WNT * (4 * g4 + i) + nt, col = c0 + 16 * WMT * wm + WMT * r16;
#pragma unroll
            for (int mt = 0; mt < WMT; ++mt) {
                const float v[1] = {acc[mt][nt][i]};
                if (row < p.M && col + mt < p.N && ((far_tok >> (4 * nt + i) | far_col >> mt) & 1u)) store_cols<OUT32>(p, row, col + mt, v);
            }
        });
    }
}

}  // namespace

namespace gdn_fp8 {

using Tile256x256 = Fp8Tile<4, 2, 4, 8, 2, 1, 1, true>;
using Tile256x192 = Fp8Tile<4, 2, 4, 6, 2, 1, 1, true>;
using Tile256x160 = Fp8Tile<4, 2, 4, 5, 2, 1, 1, true>;
using Tile256x128 = Fp8Tile<4, 2, 4, 4, 3, 1, 1, true>;
using Tile128x192 = Fp8Tile<2, 4, 4, 3, 3, 1, 1, true>;
using Tile128x128 = Fp8Tile<2, 4, 4, 2, 4, 1>;
using Tile128x128Pair = Fp8Tile<2, 4, 4, 2, 2, 2>;  // fp32 results: two workgroups a CU, one converts while the other multiplies
using Tile64x128 = Fp8Tile<1, 4, 4, 2, 3, 1, 2>;
using Tile64x64 = Fp8Tile<2, 2, 2, 2, 3, 1, 2>;
using Tile64x32 = Fp8Tile<1, 2, 4, 1, 3, 1, 4>;
using Tile32x32 = Fp8Tile<1, 2, 2, 1, 3, 1, 4>;
using Tile16x16Alone = Fp8Tile<1, 1, 1, 1, 4, 1, 8>;
using Tile16x16 = Fp8Tile<1, 1, 1, 1, 3, 3, 4>;

template <class TL, int FA, int FB, int SB, bool OUT32>
int launch_scaled(const MatmulParams& p, hipStream_t stream) {
    const int n_tok = (p.M + TL::toks - 1) / TL::toks, n_col = (p.N + TL::cols - 1) / TL::cols;
    const unsigned tiles = static_cast<unsigned>(n_tok) * n_col;
    const dim3 grid(TL::PHASED && tiles > 256 ? 256 : tiles);  // phased: a workgroup a CU
    if (!gdn_host::grid_fits(grid.x, TL::waves * 64))
        return gdn_host::fail(GDN_ERR_UNSUPPORTED, "fp8_matmul: M=%d N=%d are too large for a launch", p.M, p.N);
    hipLaunchKernelGGL((gdn_fp8_matmul_kernel<TL, FA, FB, SB, OUT32>), grid, dim3(TL::waves * 64), 0, stream, p, n_tok, n_col);
    return gdn_host::check_launch("gdn_fp8_matmul_kernel");
}

template <class TL, int FA, int FB, bool OUT32>
int launch_tiled(int scales, const MatmulParams& p, hipStream_t stream) {
    switch (scales) {
        case kE8Row: return launch_scaled<TL, FA, FB, kE8Row, OUT32>(p, stream);
        case kF32Block: return launch_scaled<TL, FA, FB, kF32Block, OUT32>(p, stream);
        case kF32Row: return launch_scaled<TL, FA, FB, kF32Row, OUT32>(p, stream);
        default: return launch_scaled<TL, FA, FB, kE8Block, OUT32>(p, stream);
    }
}

template <int FA, int FB>
int launch_tile(int tile, int scales, bool f32, const MatmulParams& p, hipStream_t stream) {
    const auto small = [&](auto out32) {
        constexpr bool O = decltype(out32)::value;
        switch (tile) {
            case k64x128: return launch_tiled<Tile64x128, FA, FB, O>(scales, p, stream);
            case k64x64: return launch_tiled<Tile64x64, FA, FB, O>(scales, p, stream);
            case k64x32: return launch_tiled<Tile64x32, FA, FB, O>(scales, p, stream);
            case k32x32: return launch_tiled<Tile32x32, FA, FB, O>(scales, p, stream);
            case k16x16Alone: return launch_tiled<Tile16x16Alone, FA, FB, O>(scales, p, stream);
            case k16x16: return launch_tiled<Tile16x16, FA, FB, O>(scales, p, stream);
            default: return launch_tiled<std::conditional_t<O, Tile128x128Pair, Tile128x128>, FA, FB, O>(scales, p, stream);
        }
    };
    if (f32) return small(std::true_type{});
    switch (tile) {
        case k256x256: return launch_tiled<Tile256x256, FA, FB, false>(scales, p, stream);
        case k256x192: return launch_tiled<Tile256x192, FA, FB, false>(scales, p, stream);
        case k256x160: return launch_tiled<Tile256x160, FA, FB, false>(scales, p, stream);
        case k256x128: return launch_tiled<Tile256x128, FA, FB, false>(scales, p, stream);
        case k128x192: return launch_tiled<Tile128x192, FA, FB, false>(scales, p, stream);
        default: return small(std::false_type{});
    }
}

}  // namespace gdn_fp8
