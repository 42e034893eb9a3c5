// The tiled kernel of the fp8 block-scaled product
//   out[m, n] = sum over blocks kb of a_scale[m, kb] b_scale[n, kb] sum_k a[m, k] b[n, k]
// with fp32 sums, one rounding where out is written.
//
// It computes the transposed product W x^T (W = b, x = a) in tiles of columns x
// tokens.  A stage is one block of 128 k: 128-byte rows, which reach LDS by DMA
// in a ring, every 8 lanes of a copy one whole line, placed with an XOR swizzle
// that keeps the fragment reads at linear-read speed; the stage's scales come
// with it.  bf16 results: one MFMA 16x16x128 takes a block: e8m0 scales are its
// own scale operands and cost nothing; fp32 scales multiply its result on the
// VALU, into the accumulator.  fp32 results: codes become bf16 in registers,
// times their e8m0 scale, and the block takes four MFMA 16x16x32, whose sums
// keep every bit that fp32 has.
#pragma once

#include "fp8_matmul.hpp"

namespace {

constexpr int kRowB = 128;  // bytes of a staged row: one block

// CW x TW waves, each WMT 16-column x WNT 16-token MFMA tiles, NS stages in LDS,
// PER_CU workgroups on a CU; KS groups of such waves, each on its own block of a
// stage of KS blocks, summed at the end.
template <int CW_, int TW_, int WMT_, int WNT_, int NS_, int PER_CU_, int KS_ = 1>
struct Fp8Tile {
    static constexpr int CW = CW_, TW = TW_, WMT = WMT_, WNT = WNT_, NS = NS_, PER_CU = PER_CU_, KS = KS_;
    static constexpr int cols = 16 * CW * WMT, toks = 16 * TW * WNT;
    static constexpr int gwaves = CW * TW, waves = gwaves * KS;
    static constexpr int dma = (cols + toks) / 8 / gwaves;  // 1 KiB copies (8 rows) a wave and block
    static_assert((cols + toks) % (8 * gwaves) == 0, "copies split evenly");
    static_assert(128 % (16 * WMT) == 0, "a wave's columns share a 128-column block");
};

// A stage's bytes with b's scales as SB says: rows, x scales, W scales.
template <class TL, int SB>
struct Fp8Stage {
    static constexpr int off_xs = (TL::cols + TL::toks) * kRowB;
    static constexpr int off_ws = off_xs + TL::toks;
    static constexpr int wsb = SB == gdn_fp8::kE8Row ? TL::cols : SB == gdn_fp8::kF32Row ? 4 * TL::cols : 0;
    static constexpr int slice_b = (off_ws + wsb + 127) / 128 * 128;
    static constexpr int stage_b = TL::KS * slice_b;
    static constexpr int copies = TL::dma + 1 + (wsb > 0 ? 1 : 0);  // a wave issues, for a block
    static constexpr int lds_b = TL::NS * stage_b;
    static_assert(lds_b * TL::PER_CU <= 160 * 1024, "LDS");
    static_assert((TL::KS - 1) * TL::gwaves * TL::WMT * TL::WNT * 1024 <= lds_b, "the groups' sums fit the dead stages");
};

__device__ __forceinline__ int swz(int r) { return r & 7; }

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

    // Workgroup -> tile: each XCD gets a contiguous range of tiles, in bands of
    // 4 column tiles with the token tile slowest, so that the workgroups of one
    // XCD share rows in its L2.
    const int ntiles = n_tok * n_col;
    int lin;
    {
        const int id = blockIdx.x, xcd = id & 7, j = id >> 3, q = ntiles >> 3, r = ntiles & 7;
        lin = xcd < r ? xcd * (q + 1) + j : r * (q + 1) + (xcd - r) * q + j;
        const int band = lin / (4 * n_tok), base = 4 * band, gs = min(n_col - base, 4);
        const int within = lin - band * 4 * n_tok;
        lin = (within / gs) * n_col + base + within % gs;
    }
    const int f0 = lin / n_col * TL::toks, c0 = lin % n_col * TL::cols;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = KS > 1 ? wave / TL::gwaves : 0, gw = KS > 1 ? wave % TL::gwaves : wave;
    const int wm = gw / TL::TW, wn = gw % TL::TW;
    const int r16 = lane & 15, g4 = lane >> 4;
    const int nslices = p.K / kRowB;

    // Copy sources.  Staged rows 0 .. cols - 1 are rows of b, the others rows of
    // a, in an order that gives a lane of the product WNT neighbouring tokens and
    // 4 WMT neighbouring columns (its accumulator (mt, nt): token WNT r16 + nt of
    // the wave's, columns 4 WMT g4 + 4 mt .. + 3).  Rows past the end repeat the
    // last one; what they give is not stored.
    const uint8_t* const wsrc = p.b + static_cast<size_t>(c0) * p.ldb;
    const uint8_t* const xsrc = p.a + static_cast<size_t>(f0) * p.lda;
    uint32_t voff[TL::dma];
#pragma unroll
    for (int j = 0; j < TL::dma; ++j) {
        const int srow = 8 * (gw + TL::gwaves * j) + (lane >> 3);
        const uint32_t chunk = 16u * ((lane & 7) ^ swz(srow));
        if (srow < TL::cols) {
            const int w = srow / (16 * WMT), s = srow % (16 * WMT);
            const int col = 16 * WMT * w + 4 * WMT * ((s & 15) >> 2) + 4 * (s >> 4) + (s & 3);
            voff[j] = static_cast<uint32_t>(min(c0 + col, p.N - 1) - c0) * static_cast<uint32_t>(p.ldb) + chunk;
        } else {
            const int w = (srow - TL::cols) / (16 * WNT), s = (srow - TL::cols) % (16 * WNT);
            const int tok = 16 * WNT * w + WNT * (s & 15) + (s >> 4);
            voff[j] = static_cast<uint32_t>(min(f0 + tok, p.M - 1) - f0) * static_cast<uint32_t>(p.lda) + chunk;
        }
    }
    // The scales' copies: the waves of a group share 16-byte pieces out, each
    // wave one copy of at least one piece (waves past the last piece repeat one).
    constexpr int kXPieces = TL::toks / 16, kXLanes = kXPieces > TL::gwaves ? kXPieces / TL::gwaves : 1;
    constexpr int kWPieces = ST::wsb / 16, kWLanes = kWPieces > TL::gwaves ? kWPieces / TL::gwaves : 1;
    constexpr int kElem = kF32 ? 4 : 1;
    const int xp = gw * kXLanes % kXPieces, wp = kWPieces > 0 ? gw * kWLanes % (kWPieces > 0 ? kWPieces : 1) : 0;
    const uint32_t xs_off = static_cast<uint32_t>(min(f0 + 16 * (xp + lane), (p.M - 1) / 16 * 16));
    const uint32_t ws_off = static_cast<uint32_t>(min(c0 + 16 / kElem * (wp + lane), (p.N - 1) / 16 * 16 + 16 - 16 / kElem)) * kElem;
    auto issue_rows = [&](int stage, int slice, int j0, int j1) {
        lds_u8* const dst = smem + stage * ST::stage_b + ks * ST::slice_b;
#pragma unroll
        for (int j = 0; j < TL::dma; ++j) {
            if (j < j0 || j >= j1) continue;
            const int row = 8 * (gw + TL::gwaves * j);
            dma16((row < TL::cols ? wsrc : xsrc) + static_cast<size_t>(slice) * kRowB, voff[j], dst + row * kRowB);
        }
    };
    auto issue_scales = [&](int stage, int slice) {
        lds_u8* const dst = smem + stage * ST::stage_b + ks * ST::slice_b;
        if (lane < kXLanes) dma16(p.a_scale + slice * p.lda_s, xs_off, dst + ST::off_xs + 16 * xp);
        if constexpr (kRow) {
            if (lane < kWLanes)
                dma16(static_cast<const uint8_t*>(p.b_scale) + slice * p.ldb_s * kElem, ws_off, dst + ST::off_ws + 16 * wp);
        }
    };
    // The block of stage kk that this wave's group takes (the last stage's
    // groups past the end repeat the last block and do not multiply it).
    auto slice_of = [&](int kk) { return KS > 1 ? min(kk * KS + ks, nslices - 1) : kk; };

    // Block scales of b: lane l holds that of block 64 w + l, w the window of 64
    // blocks the loop is in, and a stage reads its own into a scalar.
    const int nb = min(c0 + 16 * WMT * wm, p.N - 1) / kRowB;
    uint32_t wscale = 127u;
    auto load_block_scales = [&](int slice) {
        if constexpr (!kRow) {
            const size_t at = static_cast<size_t>(nb) * p.ldb_s + min(slice / 64 * 64 + lane, nslices - 1);
            if constexpr (kF32)
                wscale = static_cast<const uint32_t*>(p.b_scale)[at];
            else
                wscale = static_cast<const uint8_t*>(p.b_scale)[at];
            asm volatile("" : "+v"(wscale));  // landed here: no wait for it falls between the copies' own
        }
    };

    uint32_t rd[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) rd[h] = r16 * kRowB + 16u * ((4 * h + g4) ^ swz(r16));

    f32x4 acc[WMT][WNT];
#pragma unroll
    for (int mt = 0; mt < WMT; ++mt)
#pragma unroll
        for (int nt = 0; nt < WNT; ++nt) acc[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto half = [&](const lds_u8* at, int h) { return *reinterpret_cast<const lds_u32x4*>(at + rd[h]); };
    // W's scale of a staged block: of the lane's row of operand mt (e8m0), of the
    // accumulator's four columns (fp32).
    auto w_byte = [&](const lds_u8* st, int slice, int mt) -> int {
        if constexpr (SB == gdn_fp8::kE8Block)
            return __builtin_amdgcn_readlane(static_cast<int>(wscale), slice & 63);
        else if constexpr (SB == gdn_fp8::kE8Row)
            return st[ST::off_ws + 16 * WMT * wm + 4 * WMT * (r16 >> 2) + 4 * mt + (r16 & 3)];
        else
            return 127;
    };
    auto w_float = [&](const lds_u8* st, int slice, int mt) -> f32x4 {
        if constexpr (SB == gdn_fp8::kF32Row) {
            return *reinterpret_cast<const lds_f32x4*>(st + ST::off_ws + 4 * (16 * WMT * wm + 4 * WMT * g4 + 4 * mt));
        } else {
            const float s = __int_as_float(__builtin_amdgcn_readlane(static_cast<int>(wscale), slice & 63));
            return f32x4{s, s, s, s};
        }
    };
    // x's scales of a staged block: WNT bytes of neighbouring tokens.
    auto read_sx = [&](const lds_u8* st, uint32_t (&sx)[2]) {
        const lds_u8* at = st + ST::off_xs + 16 * WNT * wn + WNT * r16;
        sx[0] = sx[1] = 0u;
        if constexpr (WNT == 8) {
            const u32x2 v = *reinterpret_cast<const lds_u32x2*>(at);
            sx[0] = v[0];
            sx[1] = v[1];
        } else if constexpr (WNT == 4) {
            sx[0] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at);
        } else if constexpr (WNT == 2) {
            sx[0] = *reinterpret_cast<const lds_u16*>(at);
        } else {
            sx[0] = *at;
        }
    };

    const int nk = (nslices + KS - 1) / KS;
    load_block_scales(0);
#pragma unroll
    for (int st = 0; st < NS - 1; ++st)
        if (st < nk) {
            issue_rows(st, slice_of(st), 0, TL::dma);
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
            issue_rows(ws, slice_of(kt + NS - 1), 0, TL::dma);
            issue_scales(ws, slice_of(kt + NS - 1));
        }
        if (KS == 1 || slice < nslices) {
            const lds_u8* const st = smem + rs * ST::stage_b + ks * ST::slice_b;
            const lds_u8* const stx = st + (TL::cols + 16 * WNT * wn) * kRowB;
            const lds_u8* const stw = st + 16 * WMT * wm * kRowB;
            uint32_t sx[2];
            read_sx(st, sx);
            if constexpr (!OUT32) {
                i32x8 x[WNT];
                static_for<0, WNT>([&](auto NT) {
                    constexpr int nt = decltype(NT)::value;
                    x[nt] = join(half(stx + 16 * nt * kRowB, 0), half(stx + 16 * nt * kRowB, 1));
                });
                static_for<0, WMT>([&](auto MT) {
                    constexpr int mt = decltype(MT)::value;
                    const i32x8 w = join(half(stw + 16 * mt * kRowB, 0), half(stw + 16 * mt * kRowB, 1));
                    const int sw = w_byte(st, slice, mt);
                    static_for<0, WNT>([&](auto NT) {
                        constexpr int nt = decltype(NT)::value;
                        const int s = static_cast<int>(sx[nt / 4]);
                        if constexpr (kF32) {
                            const f32x4 t = mfma_fp8<FB, FA, 0, nt % 4>(w, x[nt], f32x4{0.f, 0.f, 0.f, 0.f}, sw, s);
                            const f32x4 fw = w_float(st, slice, mt);
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[mt][nt][i] = fmaf(fw[i], t[i], acc[mt][nt][i]);
                        } else {
                            acc[mt][nt] = mfma_fp8<FB, FA, 0, nt % 4>(w, x[nt], acc[mt][nt], sw, s);
                        }
                    });
                });
            } else {
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
                            x[nt] = codes_to_bf16<FA>(xc[nt][2 * q], xc[nt][2 * q + 1], sx[nt / 4] >> (8 * (nt % 4)) & 0xffu);
                        });
                        static_for<0, WMT>([&](auto MT) {
                            constexpr int mt = decltype(MT)::value;
                            const bf16x8 w = codes_to_bf16<FB>(wc[mt][2 * q], wc[mt][2 * q + 1], w_byte(st, slice, mt));
                            static_for<0, WNT>([&](auto NT) {
                                constexpr int nt = decltype(NT)::value;
                                if constexpr (kF32)
                                    block[mt][nt] = mfma16x16x32(w, x[nt], block[mt][nt]);
                                else
                                    acc[mt][nt] = mfma16x16x32(w, x[nt], acc[mt][nt]);
                            });
                        });
                    });
                });
                if constexpr (kF32) {
                    static_for<0, WMT>([&](auto MT) {
                        constexpr int mt = decltype(MT)::value;
                        const f32x4 fw = w_float(st, slice, mt);
#pragma unroll
                        for (int nt = 0; nt < WNT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[mt][nt][i] = fmaf(fw[i], block[mt][nt][i], acc[mt][nt][i]);
                    });
                }
            }
        }
        rs = rs + 1 == NS ? 0 : rs + 1;
        ws = ws + 1 == NS ? 0 : ws + 1;
    }

    if constexpr (KS > 1) {
        lds_barrier();  // every wave is past its last stage read
        const auto part = [&](int k, int i) {
            return reinterpret_cast<lds_f32x4*>(smem + (((k - 1) * TL::gwaves + gw) * WMT * WNT + i) * 1024 + 16 * lane);
        };
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

    const int R0 = f0 + 16 * WNT * wn + WNT * r16, C0 = c0 + 16 * WMT * wm + 4 * WMT * g4;
    static_for<0, WNT>([&](auto NT) {
        constexpr int nt = decltype(NT)::value;
        if (R0 + nt >= p.M) return;
        static_for<0, WMT>([&](auto MT) {
            constexpr int mt = decltype(MT)::value;
            if (C0 + 4 * mt < p.N) store4<OUT32>(p, R0 + nt, C0 + 4 * mt, acc[mt][nt]);
        });
    });
}

}  // namespace

namespace gdn_fp8 {

using Tile256x256 = Fp8Tile<4, 2, 4, 8, 2, 1>;
using Tile128x128 = Fp8Tile<4, 2, 2, 4, 4, 1>;
using Tile64x64 = Fp8Tile<2, 2, 2, 2, 2, 2, 2>;
using Tile32x32 = Fp8Tile<2, 2, 1, 1, 3, 1, 4>;

template <class TL, int FA, int FB, int SB, bool OUT32>
int launch_scaled(const MatmulParams& p, hipStream_t stream) {
    const int n_tok = (p.M + TL::toks - 1) / TL::toks, n_col = (p.N + TL::cols - 1) / TL::cols;
    hipLaunchKernelGGL((gdn_fp8_matmul_kernel<TL, FA, FB, SB, OUT32>), dim3(static_cast<unsigned>(n_tok) * n_col), dim3(TL::waves * 64),
                       0, stream, p, n_tok, n_col);
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
    const auto launch = [&](auto out32) {
        constexpr bool O = decltype(out32)::value;
        switch (tile) {
            case k128x128: return launch_tiled<Tile128x128, FA, FB, O>(scales, p, stream);
            case k64x64: return launch_tiled<Tile64x64, FA, FB, O>(scales, p, stream);
            case k32x32: return launch_tiled<Tile32x32, FA, FB, O>(scales, p, stream);
            default: break;
        }
        // Two sets of accumulators (fp32 scales, fp32 results) do not fit the largest tile.
        if constexpr (O) {
            if (scales == kF32Row) return launch_scaled<Tile128x128, FA, FB, kF32Row, true>(p, stream);
            if (scales == kF32Block) return launch_scaled<Tile128x128, FA, FB, kF32Block, true>(p, stream);
            return scales == kE8Row ? launch_scaled<Tile256x256, FA, FB, kE8Row, true>(p, stream)
                                    : launch_scaled<Tile256x256, FA, FB, kE8Block, true>(p, stream);
        } else {
            return launch_tiled<Tile256x256, FA, FB, false>(scales, p, stream);
        }
    };
    return f32 ? launch(std::true_type{}) : launch(std::false_type{});
}

}  // namespace gdn_fp8
