// The kernel of the product of 8-bit activations with 4-bit weights for many tokens
// (bf16 results), in tiles of columns x tokens like those of fp4_tiles.hpp.
//
// A stage is 128 values of K: rows of 128 bytes of x, of 64 of W (half lines, but x's
// whole ones are most of the copies), and their scales; every 8 or 4 lanes of a copy take
// one row, placed with an XOR swizzle that keeps the fragment reads at linear-read speed.
// Two groups of four waves, one wave of each on every SIMD, take turns: while one
// multiplies, the other reads its next fragments and issues its copies.  A stage is four
// phases, each a part of the wave's tile (first or second half of its columns x of its
// tokens): (W0, X0), (W1, X0), (W1, X1), (W0, X1).
//
// Against the 256 x 128 tile of fp4_tiles.hpp, where both fill the CUs: 8192 x 8192 x 8192
// 420 us (2.6 PFLOP/s) instead of 470, 16384 x 6144 x 2048 166 and 183, 1500 x 8224 x 2048
// (198 tiles, one round) 30 and 35.  A block of K takes 1.2-1.3 us, of which the matrix
// cores need 0.9; tiles of 160 and 192 tokens and of 128 columns were slower than the
// 256 x 128 one or within 3% of it.
#pragma once

#include "fp4_tiles.hpp"

namespace {

// 4 x 2 waves, each 4 16-column x 8 16-token MFMA tiles; NS stages in LDS.
//
// A stage is copied, and its buffer freed, region by region: the first and second part of
// every wave's tokens (X0, X1) and columns (W0, W1), in the order X0 and the scales, W0,
// W1, X1.  A copy is 1 KiB: 8 rows of x, 16 of W; each wave takes as many of a region's.
struct Phased {
    static constexpr int CW = 4, TW = 2, WMT = 4, WNT = 8, NS = 3;
    static constexpr int cols = 16 * CW * WMT, toks = 16 * TW * WNT, waves = CW * TW;
    static constexpr int Mn = WMT / 2, Xn = WNT / 2;                                    // MFMA tiles of a wave's part
    static constexpr int cW = CW * Mn / waves, cX = 2 * TW * Xn / waves;                // copies of a region a wave issues
    static constexpr int rows_copies = 2 * (cW + cX), copies = rows_copies + 2;         // of a stage
    static_assert(CW * Mn % waves == 0 && 2 * TW * Xn % waves == 0, "copies split evenly");
    static constexpr int row_w = 64, row_x = 128;  // bytes
    static constexpr int off_x = cols * row_w, off_ws = off_x + toks * row_x, off_xs = off_ws + 4 * cols, stage_b = off_xs + toks;
    static_assert(stage_b % 128 == 0 && NS * stage_b <= 160 * 1024, "LDS");
    static_assert(NS * copies < 64, "copies that a wait counts");
};

// Workgroup barrier alone (no LDS access of this wave is outstanding); no memory access
// moves across it.
__device__ __forceinline__ void wave_barrier() { asm volatile("s_barrier" ::: "memory"); }

template <int FA>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void gdn_fp4_phased_kernel(gdn_fp4::MatmulParams p, int n_tok, int n_col) {
    using TL = Phased;
    constexpr int WMT = TL::WMT, WNT = TL::WNT, NS = TL::NS, Mn = TL::Mn, Xn = TL::Xn;
    __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[NS * TL::stage_b];
    lds_u8* const smem = (lds_u8*)&smem_raw[0];
    const Tiles tiles(n_tok, n_col);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / TL::TW, wn = wave % TL::TW, r16 = lane & 15, g4 = lane >> 4;
    const int nk = p.K / 128;

    // Copy sources: rows in the order of fp4_tiles.hpp (a lane of the product has
    // neighbouring columns and supplies neighbouring tokens); rows past the end repeat
    // the last one.
    int f0, c0;
    const uint8_t *wsrc, *xsrc;
    // Copy j of region r: the first row of W's or x's in the tile, the same for the wave.
    auto copy_row = [&](int r, int j) {
        const int h = wave + TL::waves * j;
        if (r == 0 || r == 3) return 16 * WNT * (h / (2 * Xn)) + (r == 3 ? 16 * Xn : 0) + 8 * (h % (2 * Xn));
        return 16 * WMT * (h / Mn) + (r == 2 ? 16 * Mn : 0) + 16 * (h % Mn);
    };
    constexpr auto count_of = [](int r) { return r == 0 || r == 3 ? TL::cX : TL::cW; };
    constexpr auto first_of = [](int r) { return r == 0 ? 0 : TL::cX + (r - 1) * TL::cW; };
    uint32_t voff[TL::rows_copies], xs_off, ws_off;
    int crow[TL::rows_copies];
    static_for<0, 4>([&](auto R) {
        constexpr int r = decltype(R)::value;
        static_for<0, count_of(r)>([&](auto J) { crow[first_of(r) + decltype(J)::value] = __builtin_amdgcn_readfirstlane(copy_row(r, decltype(J)::value)); });
    });
    constexpr int kXLanes = TL::toks / 16 / TL::waves, kWLanes = TL::cols / 4 / TL::waves;  // of the scales' copies: 16 bytes each
    const int xp = wave * kXLanes, wp = wave * kWLanes;
    auto set_tile = [&](int j) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));  // computed anew for each tile: kept over the loop, its parts would fill registers
        tiles.at<TL>(j, f0, c0);
        wsrc = p.b + static_cast<size_t>(c0) * p.ldb;
        xsrc = p.a + static_cast<size_t>(f0) * p.lda;
        static_for<0, 4>([&](auto R) {
            constexpr int r = decltype(R)::value;
            static_for<0, count_of(r)>([&](auto J) {
                constexpr int c = first_of(r) + decltype(J)::value;
                if constexpr (r == 0 || r == 3) {
                    const int row = crow[c] + (lane >> 3), w = row / (16 * WNT), s = row % (16 * WNT);
                    const int tok = 16 * WNT * w + WNT * (s & 15) + (s >> 4);
                    voff[c] = static_cast<uint32_t>(min(f0 + tok, p.M - 1) - f0) * static_cast<uint32_t>(p.lda) + 16u * ((lane & 7) ^ (row & 7));
                } else {
                    const int row = crow[c] + (lane >> 2), w = row / (16 * WMT), s = row % (16 * WMT);
                    const int col = 16 * WMT * w + WMT * (s & 15) + (s >> 4);
                    voff[c] = static_cast<uint32_t>(min(c0 + col, p.N - 1) - c0) * static_cast<uint32_t>(p.ldb) + 16u * ((lane & 3) ^ (row >> 2 & 3));
                }
            });
        });
        xs_off = static_cast<uint32_t>(min(f0 + 16 * (xp + lane), (p.M - 1) / 16 * 16));
        ws_off = 4u * static_cast<uint32_t>(min(c0 + 4 * (wp + lane), (p.N - 1) / 4 * 4));
    };
    // Region r of a stage; the scales come with the first.
    auto issue = [&](auto R, int stage, int block) {
        constexpr int r = decltype(R)::value;
        constexpr bool x = r == 0 || r == 3;
        lds_u8* const to = smem + stage * TL::stage_b;
        const uint8_t* const from = x ? xsrc + static_cast<size_t>(block) * TL::row_x : wsrc + static_cast<size_t>(block) * TL::row_w;
        static_for<0, count_of(r)>([&](auto J) {
            constexpr int c = first_of(r) + decltype(J)::value;
            dma16(from, voff[c], to + (x ? TL::off_x + crow[c] * TL::row_x : crow[c] * TL::row_w));
        });
        if constexpr (r == 0) {
            int k = block;
            asm volatile("" : "+s"(k));  // computed here: within a lane's branch it would go to vector registers
            if (lane < kXLanes) dma16(p.a_scale + static_cast<size_t>(k) * p.lda_s, xs_off, to + TL::off_xs + 16 * xp);
            if (lane < kWLanes) dma16(reinterpret_cast<const uint8_t*>(p.b_scale) + static_cast<size_t>(k) * 4 * p.ldb_s, ws_off, to + TL::off_ws + 16 * wp);
        }
    };

    const uint32_t rdw = r16 * TL::row_w + 16u * (g4 ^ (r16 >> 2 & 3));
    uint32_t rdx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) rdx[h] = r16 * TL::row_x + 16u * ((4 * h + g4) ^ swz(r16));
    const uint32_t sel32 = g4 < 2 ? 0x05040100u : 0x07060302u, sel16 = g4 % 2 == 0 ? 0x06020400u : 0x07030501u;
    f32x4 acc[WMT][WNT];

    // Phase 0 reads W0, X0 and the scales, phase 1 W1, phase 2 X1, phase 3 nothing.  A
    // region's buffer is free once both groups have read it, so stage kt + NS's X0, W0 and
    // W1 go out in phases 1, 2 and 3 of stage kt and its X1 in phase 0 of the next.  The
    // waits count the copies issued after the region that the next phase reads; T >= 0: T
    // stages are left after this one and no new ones are issued.
    u32x4 w0[Mn], w1[Mn];
    i32x8 xf[Xn];
    u32x2 sx = {0, 0};  // bytes of eight neighbouring tokens
    uint32_t sw = 0;    // of the lane's 32 values of the four column tiles
    constexpr int cX0 = TL::cX + 2, cW1 = TL::cW, cX1 = TL::cX, cAll = TL::copies;
    auto next_buf = [](int b, int n) { return b + n >= NS ? b + n - NS : b + n; };
    auto stage = [&](int kt, int rs, auto Tc) {
        constexpr int T = decltype(Tc)::value;
        constexpr bool steady = T < 0;
        const lds_u8* const st = smem + rs * TL::stage_b;
        const lds_u8* const stx = st + TL::off_x + 16 * WNT * wn * TL::row_x;
        const lds_u8* const stw = st + 16 * WMT * wm * TL::row_w + rdw;
        const auto frag_x = [&](int nt) {
            const lds_u8* const at = stx + 16 * nt * TL::row_x;
            return join(*reinterpret_cast<const lds_u32x4*>(at + rdx[0]), *reinterpret_cast<const lds_u32x4*>(at + rdx[1]));
        };
        static_for<0, 4>([&](auto Pc) {
            constexpr int ph = decltype(Pc)::value;
            if constexpr (ph == 0) {
                static_for<0, Mn>([&](auto I) { w0[decltype(I)::value] = *reinterpret_cast<const lds_u32x4*>(stw + 16 * decltype(I)::value * TL::row_w); });
                static_for<0, Xn>([&](auto I) { xf[decltype(I)::value] = frag_x(decltype(I)::value); });
                // the word of the row's tile g4: the four lanes of a row exchange bytes below
                sw = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(st + TL::off_ws + 4 * (16 * WMT * wm + WMT * r16 + g4));
                sx = *reinterpret_cast<const lds_u32x2*>(st + TL::off_xs + 16 * WNT * wn + WNT * r16);
            } else if constexpr (ph == 1) {
                static_for<0, Mn>([&](auto I) { w1[decltype(I)::value] = *reinterpret_cast<const lds_u32x4*>(stw + 16 * (Mn + decltype(I)::value) * TL::row_w); });
            } else if constexpr (ph == 2) {
                static_for<0, Xn>([&](auto I) { xf[decltype(I)::value] = frag_x(Xn + decltype(I)::value); });
            }
            if constexpr (ph == 0 && (steady || T == NS - 1))
                issue(std::integral_constant<int, 3>{}, next_buf(rs, NS - 1), kt + NS - 1);
            else if constexpr (ph > 0 && steady)
                issue(std::integral_constant<int, ph - 1>{}, rs, kt + NS);
            if constexpr (ph == 0)
                wait_vm<cX1 + (steady ? NS - 1 : T) * cAll>();
            else if constexpr (ph == 1)
                wait_vm<steady ? cX0 + (NS - 1) * cAll : T * cAll>();
            else if constexpr (ph == 3 && T != 0)
                wait_vm<cW1 + (steady ? (NS - 1) * cAll : cX1 + (T - 1) * cAll)>();
            lds_barrier();  // this group's fragments are here, the other's multiplications issued
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            if constexpr (ph == 0) sw = exchange_bytes(sw, sel32, sel16);
            constexpr int m0 = ph == 0 || ph == 3 ? 0 : Mn, n0 = ph < 2 ? 0 : Xn;
            static_for<n0, n0 + Xn>([&](auto NT) {
                constexpr int nt = decltype(NT)::value;
                static_for<m0, m0 + Mn>([&](auto MT) {
                    constexpr int mt = decltype(MT)::value;
                    acc[mt][nt] = mfma_fp4<FA, nt % 4, mt>(xf[nt - n0], codes4(m0 == 0 ? w0[mt - m0] : w1[mt - m0]), acc[mt][nt], sx[nt / 4], sw);
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
            if (s < nk) static_for<0, s + 1 < NS ? 4 : 3>([&](auto R) { issue(R, s, s); });
        });
    };
    int tile = static_cast<int>(blockIdx.x) >> 3;
    set_tile(tile);
    fill();
    // One tile after the other: the next one's first stages are copied while this one's
    // results are stored.  The stores are younger than those copies and older than later
    // ones, so the waits above hold as they are (vector memory operations retire in order).
    for (;;) {
        const bool more = tile + tiles.step < tiles.count;
        clear<TL>(acc);
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
            tile += tiles.step;
            set_tile(tile);
            fill();
        }
        int l = threadIdx.x & 63;
        asm volatile("" : "+v"(l));
        const int R0 = f + 16 * WNT * wn + WNT * 4 * (l >> 4), C0 = c + 16 * WMT * wm + WMT * (l & 15);
        if (f + TL::toks <= p.M && c + TL::cols <= p.N)
            store_inside<TL, false>(p, acc, R0, C0);
        else
            store<TL, false>(p, acc, R0, C0);
        if (!more) return;
    }
}

}  // namespace
