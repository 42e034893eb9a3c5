// The tiled kernels of the product with 4-bit weights
//   out[m, n] = sum over k of a[m, k] a_scale[m, block of k] b[n, k] b_scale[n, block of k]
// with fp32 sums, one rounding where out is written.  b's codes are 4-bit, a's 4-bit
// (blocks of 32) or 8-bit (blocks of 128).
//
// In tiles of columns x tokens (W = b, x = a).  A slice is 256 values of K: rows of
// 128 bytes of W and of 4-bit x, two of 128 bytes of 8-bit x (one after the other for
// all tokens).  They reach LDS by DMA, every 8 lanes of a copy one whole line (half
// lines took twice the requests for the same bytes: 8192 x 8192 x 8192 350 us), placed
// with an XOR swizzle that keeps the fragment reads at linear-read speed, and the scales
// with them.  The four scales of a 4-bit row's 128 values are a word, of which a lane of
// the product needs one byte, that of its own 32 values, for each of its tiles: the four
// lanes of a row read the words of a quarter of the tiles each and exchange bytes across
// the wave (two swaps and two permutations for four tiles).
//
// gdn_fp4_stream_kernel, for many tokens: one workgroup of eight waves a CU (or two of
// four) walks its tiles, and its stages run on over the borders between them.  A wave
// multiplies half a slice (128 values) at a time, and each operand's registers take the
// next half's codes from LDS as soon as they are free, so that LDS and the matrix cores
// work at the same time.  A stage's W is copied over once every wave has read it, x half a
// slice later.
//
// What bounds it, by leaving parts out (256 x 256 tiles, us a slice): products and LDS reads
// without copies 1.3 with codes of zero and 1.6 with random ones (the card's power; the
// products alone 1.1), copies alone 1.1, all of it 1.7 and 2.2: the copies' writes and the
// waves' reads meet in LDS.  And 6.7 us a tile on every CU for its results: 256 x 128 KiB of
// bf16 take 6 to HBM, but a later stage's wait also has all of a tile's stores, issued in
// one piece, retire first; the two were not told apart (fp32 results take 15 to 18 more).
// 16384 x 6144 x 2048 110-117 us (3.5-3.7 PFLOP/s; after a hundred calls: an idle card's
// first ones take 120 to 150, until its power has settled), fp32 results 228; 8192 x 8192 x
// 8192 250-303 (3.6-4.4) and 312.  Slower were, for the former in bf16 at 111, two groups of
// waves in turn with barriers around each quarter of a slice (124), four waves of 128 x 128
// (237: half the accumulators move between register files), and lines fetched into the L2
// two stages ahead (126: the fetches take the copies' time); workgroups that start in 2 to 8
// classes, 0.5 to 3.2 us apart, gained nothing (117-125 against 120, in the middle of a
// run).
//
// Of 8-bit x the same loop runs 256 x 128 tiles; the whole of 256 x 256 does not fit its
// stages (fp4_phased.hpp has another loop for them).
//
// gdn_fp4_ring_kernel, for few: small tiles with K over groups of waves and several
// stages under way.  It also takes fp32 results of 8-bit codes, see fp4_matmul.hpp.
#pragma once

#include "fp4_matmul.hpp"

namespace {

constexpr int kRowB = 128;  // bytes of a staged row

// CW x TW waves, each WMT 16-column x WNT 16-token MFMA tiles, NS stages in LDS,
// PER_CU workgroups on a CU; KS groups of such waves, each on its own slice of a
// stage of KS slices, summed at the end.  X8: x's codes are 8-bit.
template <bool X8_, int CW_, int TW_, int WMT_, int WNT_, int NS_, int PER_CU_, int KS_ = 1>
struct Fp4Tile {
    static constexpr bool X8 = X8_;
    static constexpr int XH = X8 ? 2 : 1;  // staged rows of a token
    static constexpr int CW = CW_, TW = TW_, WMT = WMT_, WNT = WNT_, NS = NS_, PER_CU = PER_CU_, KS = KS_;
    static constexpr int cols = 16 * CW * WMT, toks = 16 * TW * WNT, rows = cols + XH * toks;
    static constexpr int gwaves = CW * TW, waves = gwaves * KS;
    static constexpr int w_copies = cols / 8 / gwaves, x_copies = XH * toks / 8 / gwaves;  // 1 KiB copies (8 rows) a wave and slice
    static_assert(cols % (8 * gwaves) == 0 && toks % (8 * gwaves) == 0, "copies split evenly");
    // A slice's bytes: rows, W's scales [2][cols] words, x's [2][toks] words or bytes.
    static constexpr int xsb = X8 ? 1 : 4;  // bytes of a token's scales of 128 values
    static constexpr int off_ws = rows * kRowB, off_xs = off_ws + 8 * cols;
    static constexpr int slice_b = (off_xs + 2 * xsb * toks + 127) / 128 * 128, stage_b = KS * slice_b, lds_b = NS * stage_b;
    static constexpr int copies = w_copies + x_copies + 2;  // a wave issues, for a slice
    static_assert(lds_b * PER_CU <= 160 * 1024, "LDS");
    static_assert((KS - 1) * gwaves * WMT * WNT * 1024 <= lds_b, "the groups' sums fit the dead stages");
    static_assert(NS >= 2 && (NS - 2) * copies < 64, "copies that a wait counts");
};

__device__ __forceinline__ int swz(int r) { return r & 7; }

// Lane group g (lanes 16 g .. + 15) holds word g of four: gives it byte g of each word,
// word t's in byte t.
__device__ __forceinline__ uint32_t exchange_bytes(uint32_t w, uint32_t sel32, uint32_t sel16) {
    const auto a = __builtin_amdgcn_permlane32_swap(w, w, false, false);  // words of the lower, of the upper half of the wave
    const uint32_t v = __builtin_amdgcn_perm(a[1], a[0], sel32);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // of even, of odd rows of 16 lanes
    return __builtin_amdgcn_perm(b[1], b[0], sel16);
}

// Workgroup -> tiles: each XCD gets a contiguous range of tiles, in bands of 4
// column tiles with the token tile slowest, so that the workgroups of one XCD
// share rows in its L2; a workgroup takes every step-th tile of its XCD's.
struct Tiles {
    int begin, count, step, n_tok, n_col;
    __device__ Tiles(int n_tok_, int n_col_) : n_tok(n_tok_), n_col(n_col_) {
        const int ntiles = n_tok * n_col, xcd = blockIdx.x & 7, per = ntiles >> 3, rest = ntiles & 7;
        begin = xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per;
        count = per + (xcd < rest ? 1 : 0);
        step = (static_cast<int>(gridDim.x) - xcd + 7) >> 3;
    }
    // First token and column of the workgroup's tile j (blockIdx.x / 8, and on from there by step).
    template <class TL>
    __device__ __forceinline__ void at(int j, int& f, int& c) const {
        const int lin = begin + j, band = lin / (4 * n_tok), within = lin - band * 4 * n_tok, gs = min(n_col - 4 * band, 4);
        f = __builtin_amdgcn_readfirstlane(within / gs * TL::toks);
        c = __builtin_amdgcn_readfirstlane((4 * band + within % gs) * TL::cols);
    }
};

// A wave's part of a slice's copies into LDS.
//
// Staged rows 0 .. cols - 1 are rows of b, the others rows of a, in an order that gives
// a lane of the product WMT neighbouring columns and lets it supply WNT neighbouring
// tokens, whose scales are neighbours (accumulator (mt, nt)[i]: column WMT r16 + mt,
// token WNT (4 g4 + i) + nt of the wave's).  Rows past the end repeat the last one; what
// they give is not stored.
template <class TL>
struct Source {
    const uint8_t *w, *x;
    int f0, c0;
    bool inside;  // no rows past the end: a copy's are a fixed step from the first one's
    uint32_t w0, x0, ws_off, xs_off;

    // Rows of a copy j, from the first one's: whole waves' parts, then within one (its rows go by tiles first).
    template <int TILES>
    __device__ __forceinline__ static constexpr int step(int j) {
        const int r = 8 * TL::gwaves * j;
        return r / (16 * TILES) * (16 * TILES) + r % (16 * TILES) / 16;
    }
    static_assert(TL::gwaves % 2 == 0 || (TL::w_copies <= 2 && TL::WMT == 1 && TL::WNT == 1), "steps of 16 staged rows");

    // The scales: the waves share 16-byte pieces out, each wave one copy of at least one
    // piece (the last waves may repeat pieces).  Pieces go by 128 values first, then by rows.
    static constexpr int w_pieces = TL::cols / 2, w_lanes = (w_pieces + TL::gwaves - 1) / TL::gwaves;              // 4 rows each
    static constexpr int x_rows = 16 / TL::xsb, x_pieces = 2 * TL::toks / x_rows, x_lanes = (x_pieces + TL::gwaves - 1) / TL::gwaves;  // 4 tokens each, or 16
    static_assert(w_lanes <= 64 && x_lanes <= 64, "a copy has 64 lanes");
    __device__ __forceinline__ static int w_first(int gw) { return min(gw * w_lanes, w_pieces - w_lanes); }
    __device__ __forceinline__ static int x_first(int gw) { return min(gw * x_lanes, x_pieces - x_lanes); }

    __device__ __forceinline__ void set(const gdn_fp4::MatmulParams& p, int f, int c, int gw, int lane) {
        f0 = f, c0 = c;
        w = p.b + static_cast<size_t>(c) * p.ldb;
        x = p.a + static_cast<size_t>(f) * p.lda;
        inside = TL::gwaves % 2 == 0 && f + TL::toks <= p.M && c + TL::cols <= p.N;
        w0 = row_of_w(p, c, gw, 0, lane);
        x0 = row_of_x(p, f, gw, 0, lane);
        ws_off = scales_of_w(p, c, gw, lane);
        xs_off = scales_of_x(p, f, gw, lane);
    }
    // What the lane's offsets are: of copy j, of the scales.
    __device__ __forceinline__ static uint32_t row_of_w(const gdn_fp4::MatmulParams& p, int c0, int gw, int j, int lane) {
        const int r = 8 * (gw + TL::gwaves * j) + (lane >> 3), wave = r / (16 * TL::WMT), s = r % (16 * TL::WMT);
        const int col = 16 * TL::WMT * wave + TL::WMT * (s & 15) + (s >> 4);
        return static_cast<uint32_t>(min(c0 + col, p.N - 1) - c0) * static_cast<uint32_t>(p.ldb) + 16u * ((lane & 7) ^ swz(r));
    }
    __device__ __forceinline__ static uint32_t row_of_x(const gdn_fp4::MatmulParams& p, int f0, int gw, int j, int lane) {
        const int r = 8 * (gw + TL::gwaves * j) + (lane >> 3), wave = r / (16 * TL::WNT), s = r % (16 * TL::WNT);
        const int tok = 16 * TL::WNT * wave + TL::WNT * (s & 15) + (s >> 4);
        return static_cast<uint32_t>(min(f0 + tok, p.M - 1) - f0) * static_cast<uint32_t>(p.lda) + 16u * ((lane & 7) ^ swz(r));
    }
    __device__ __forceinline__ static uint32_t scales_of_w(const gdn_fp4::MatmulParams& p, int c0, int gw, int lane) {
        const int q = w_first(gw) + lane, half = w_pieces / 2;
        return static_cast<uint32_t>(q / half) * 4u * static_cast<uint32_t>(p.ldb_s) + 4u * min(c0 + 4 * (q % half), (p.N - 1) / 4 * 4);
    }
    __device__ __forceinline__ static uint32_t scales_of_x(const gdn_fp4::MatmulParams& p, int f0, int gw, int lane) {
        const int q = x_first(gw) + lane, half = x_pieces / 2;
        return static_cast<uint32_t>(q / half) * TL::xsb * static_cast<uint32_t>(p.lda_s) + TL::xsb * min(f0 + x_rows * (q % half), (p.M - 1) / x_rows * x_rows);
    }
    // W's rows and all scales; x's rows.
    __device__ __forceinline__ void issue_w(const gdn_fp4::MatmulParams& p, int slice, lds_u8* dst, int gw, int lane) const {
        const uint8_t* const from = w + static_cast<size_t>(slice) * kRowB;
        if (inside) {
#pragma unroll
            for (int j = 0; j < TL::w_copies; ++j) dma16(from + step<TL::WMT>(j) * p.ldb, w0, dst + 8 * (gw + TL::gwaves * j) * kRowB);
        } else {
#pragma unroll
            for (int j = 0; j < TL::w_copies; ++j) dma16(from, row_of_w(p, c0, gw, j, lane), dst + 8 * (gw + TL::gwaves * j) * kRowB);
        }
        int block = 2 * slice;
        asm volatile("" : "+s"(block));  // computed here: within a lane's branch it would go to vector registers
        if (lane < x_lanes) {
            // of 8-bit x there may be no second block: its scales (and rows) then repeat the first's
            uint32_t second = TL::X8 && x_first(gw) + lane >= x_pieces / 2 ? ~0u : 0u;
            asm volatile("" : "+v"(second));  // a number: as a branch it would draw the slice into vector registers
            const uint32_t none = TL::X8 && 2 * slice + 1 >= p.K / 128 ? static_cast<uint32_t>(p.lda_s) : 0u;
            dma16(p.a_scale + static_cast<size_t>(2 * slice) * TL::xsb * p.lda_s, xs_off - (none & second), dst + TL::off_xs + 16 * x_first(gw));
        }
        if (lane < w_lanes)
            dma16(reinterpret_cast<const uint8_t*>(p.b_scale) + static_cast<size_t>(block) * 4 * p.ldb_s, ws_off, dst + TL::off_ws + 16 * w_first(gw));
    }
    __device__ __forceinline__ void issue_x(const gdn_fp4::MatmulParams& p, int slice, lds_u8* dst, int gw, int lane) const {
#pragma unroll
        for (int h = 0; h < TL::XH; ++h) {
            const int at = TL::X8 ? __builtin_amdgcn_readfirstlane(min(2 * slice + h, p.K / 128 - 1)) : slice;
            const uint8_t* const from = x + static_cast<size_t>(at) * kRowB;
            if (inside) {
#pragma unroll
                for (int j = 0; j < TL::x_copies / TL::XH; ++j) dma16(from + step<TL::WNT>(j) * p.lda, x0, dst + (TL::cols + h * TL::toks + 8 * (gw + TL::gwaves * j)) * kRowB);
            } else {
#pragma unroll
                for (int j = 0; j < TL::x_copies / TL::XH; ++j)
                    dma16(from, row_of_x(p, f0, gw, j, lane), dst + (TL::cols + h * TL::toks + 8 * (gw + TL::gwaves * j)) * kRowB);
            }
        }
    }
};

// The operands and scales that a wave holds of one half (128 values) of a slice, and of
// W the next half's too.
template <class TL, int FA>
struct Operands {
    static constexpr int WMT = TL::WMT, WNT = TL::WNT, RW = (WMT + 3) / 4, RX = (WNT + 3) / 4;
    static_assert(WMT <= 8 && WNT <= 8, "tiles of a wave");
    u32x4 w[2][WMT], x[WNT][TL::XH];
    uint32_t next_sw[RW], next_sx[RX];  // as read
    uint32_t sw[RW], sx[RX];            // tile t's in byte t / R of register t % R (8-bit x: byte t % 4 of t / 4)

    // Words of N tiles' rows, of the lane's own tiles.
    template <int N>
    __device__ __forceinline__ static void read_words(const lds_u8* at, int r16, int g4, uint32_t* s) {
        static_assert(N == 1 || N == 2 || N == 4 || N == 8, "tiles of a wave");
        at += 4 * N * r16;
        if constexpr (N == 8) {
            const u32x2 v = *reinterpret_cast<const lds_u32x2*>(at + 8 * g4);
            s[0] = v[0], s[1] = v[1];
        } else {
            s[0] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at + 4 * (g4 % N));
        }
    }
    // 16-byte piece of row r16 that holds the lane's 4-bit codes of half h; of 8-bit ones both.
    __device__ __forceinline__ static uint32_t piece(int h, int r16, int g4) { return 16u * ((4 * h + g4) ^ swz(r16)); }

    // W and all scales of half h of a staged slice, for the step after this one.
    template <int H>
    __device__ __forceinline__ void read_w(const lds_u8* st, int wm, int wn, int r16, int g4) {
        read_words<WMT>(st + TL::off_ws + 4 * (H * TL::cols + 16 * WMT * wm), r16, g4, next_sw);
        if constexpr (!TL::X8) {
            read_words<WNT>(st + TL::off_xs + 4 * (H * TL::toks + 16 * WNT * wn), r16, g4, next_sx);
        } else {
            const lds_u8* const at = st + TL::off_xs + H * TL::toks + 16 * WNT * wn + WNT * r16;
            if constexpr (WNT == 8) {
                const u32x2 v = *reinterpret_cast<const lds_u32x2*>(at);
                next_sx[0] = v[0], next_sx[1] = v[1];
            } else if constexpr (WNT == 4) {
                next_sx[0] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(at);
            } else if constexpr (WNT == 2) {
                next_sx[0] = *reinterpret_cast<const lds_u16*>(at);
            } else {
                next_sx[0] = *at;
            }
        }
        const lds_u8* const at = st + (16 * WMT * wm + r16) * kRowB + piece(H, r16, g4);
#pragma unroll
        for (int mt = 0; mt < WMT; ++mt) w[H][mt] = *reinterpret_cast<const lds_u32x4*>(at + 16 * mt * kRowB);
    }
    // Token tile nt's codes of half h.
    template <int H, int NT>
    __device__ __forceinline__ void read_x(const lds_u8* st, int wn, int r16, int g4) {
        const lds_u8* const at = st + (TL::cols + 16 * WNT * wn + r16 + (TL::X8 ? H * TL::toks : 0) + 16 * NT) * kRowB;
        if constexpr (TL::X8) {
            x[NT][0] = *reinterpret_cast<const lds_u32x4*>(at + piece(0, r16, g4));
            x[NT][1] = *reinterpret_cast<const lds_u32x4*>(at + piece(1, r16, g4));
        } else {
            x[NT][0] = *reinterpret_cast<const lds_u32x4*>(at + piece(H, r16, g4));
        }
    }
    // The next half's scales become this one's.
    __device__ __forceinline__ void turn(int g4) {
        const uint32_t sel32 = g4 < 2 ? 0x05040100u : 0x07060302u, sel16 = g4 % 2 == 0 ? 0x06020400u : 0x07030501u;
#pragma unroll
        for (int i = 0; i < RW; ++i) sw[i] = WMT == 1 ? next_sw[i] >> (8 * g4) : exchange_bytes(next_sw[i], sel32, sel16);
#pragma unroll
        for (int i = 0; i < RX; ++i) sx[i] = TL::X8 ? next_sx[i] : WNT == 1 ? next_sx[i] >> (8 * g4) : exchange_bytes(next_sx[i], sel32, sel16);
    }
    // Half h's products of token tile nt with all column tiles.
    template <int H, int NT>
    __device__ __forceinline__ void multiply(f32x4 (&acc)[WMT][WNT]) const {
        i32x8 v;
        if constexpr (TL::X8)
            v = join(x[NT][0], x[NT][1]);
        else
            v = codes4(x[NT][0]);
        static_for<0, WMT>([&](auto MT) {
            constexpr int mt = decltype(MT)::value;
            acc[mt][NT] = mfma_fp4<FA, TL::X8 ? NT % 4 : NT / RX, mt / RW>(v, codes4(w[H][mt]), acc[mt][NT], sx[TL::X8 ? NT / 4 : NT % RX], sw[mt % RW]);
        });
        // Issued here: products that are not used before the next slice would move past the barriers.
        static_for<0, WMT>([&](auto MT) {
            f32x4& a = acc[decltype(MT)::value][NT];
            asm volatile("" : "+v"(a));
        });
    }
};

template <class TL>
__device__ __forceinline__ void clear(f32x4 (&acc)[TL::WMT][TL::WNT]) {
#pragma unroll
    for (int mt = 0; mt < TL::WMT; ++mt)
#pragma unroll
        for (int nt = 0; nt < TL::WNT; ++nt) acc[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// A wave's results: R0, C0 the first token and column of its lane.
template <class TL, bool OUT32>
__device__ __forceinline__ void store(const gdn_fp4::MatmulParams& p, const f32x4 (&acc)[TL::WMT][TL::WNT], int R0, int C0) {
    if (C0 >= p.N) return;
    static_for<0, 4 * TL::WNT>([&](auto J) {
        constexpr int i = decltype(J)::value / TL::WNT, nt = decltype(J)::value % TL::WNT;
        if (R0 + TL::WNT * i + nt >= p.M) return;
        constexpr int NC = TL::WMT < 4 ? TL::WMT : 4;
#pragma unroll
        for (int m = 0; m < TL::WMT; m += NC) {
            float v[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) v[c] = acc[m + c][nt][i];
            store_cols<OUT32>(p, R0 + TL::WNT * i + nt, C0 + m, v);
        }
    });
}
// The same of a tile inside the result: at least TL::WNT * 4 stores, whatever the lane.
// They go past the caches, which the operands need: a training step of 8192 x 2048 x 4096
// (three products among quantisations) takes 219 us, with ordinary stores 230.
template <class TL, bool OUT32>
__device__ __forceinline__ void store_inside(const gdn_fp4::MatmulParams& p, const f32x4 (&acc)[TL::WMT][TL::WNT], int R0, int C0) {
    using T = std::conditional_t<OUT32, float, bf16>;
    constexpr int NC = TL::WMT * sizeof(T) > 16 ? 16 / sizeof(T) : TL::WMT;  // columns of a store
    typedef T vec __attribute__((ext_vector_type(NC), aligned(sizeof(T))));  // whole stores at any address
    T* const o = static_cast<T*>(p.out) + static_cast<size_t>(R0) * p.ldo + C0;
    static_for<0, 4 * TL::WNT>([&](auto J) {
        constexpr int i = decltype(J)::value / TL::WNT, nt = decltype(J)::value % TL::WNT;
#pragma unroll
        for (int m = 0; m < TL::WMT; m += NC) {
            vec v;
#pragma unroll
            for (int c = 0; c < NC; ++c) v[c] = static_cast<T>(acc[m + c][nt][i]);
            __builtin_nontemporal_store(v, reinterpret_cast<vec*>(o + (TL::WNT * i + nt) * p.ldo + m));
        }
        __builtin_amdgcn_sched_barrier(0);  // one after the other, in few registers
    });
}

template <class TL, int FA, bool OUT32>
__global__ __launch_bounds__(TL::waves * 64)
    __attribute__((amdgpu_waves_per_eu(TL::PER_CU * TL::waves / 4, TL::PER_CU * TL::waves / 4))) void gdn_fp4_stream_kernel(
        gdn_fp4::MatmulParams p, int n_tok, int n_col) {
    static_assert(TL::NS == 2 && TL::KS == 1 && TL::X8 == (FA != GDN_E2M1) && TL::WMT % 2 == 0, "a stream tile");
    static_assert(!(TL::X8 && OUT32), "fp32 results of 8-bit codes run on the ring");
    __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[TL::lds_b];
    lds_u8* const smem = (lds_u8*)&smem_raw[0];
    const Tiles tiles(n_tok, n_col);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / TL::TW, wn = wave % TL::TW, r16 = lane & 15, g4 = lane >> 4;
    const int nblocks = p.K / 128, nslices = (nblocks + 1) / 2;
    constexpr int kStores = 4 * TL::WNT;  // of a wave, for a tile inside the result
    constexpr int kFirst = TL::WNT / 4, kSecond = TL::WNT / 8;  // the token tiles after which W, and x, have arrived
    constexpr int cW = TL::w_copies + 2, cX = TL::x_copies;

    // The copies run two stages ahead, over tile borders: stage s + 2's W goes out once
    // every wave has read stage s's, in its first half, x's in its second.
    int tile = static_cast<int>(blockIdx.x) >> 3, f0, c0;  // the tile in hand
    int next_tile = tile, next_slice = 0;                  // what is copied next
    const int stages = (tiles.count - tile + tiles.step - 1) / tiles.step * nslices;
    Source<TL> source;
    tiles.at<TL>(tile, f0, c0);
    source.set(p, f0, c0, wave, lane);
    auto issue_w = [&](int buf) { source.issue_w(p, next_slice, smem + buf * TL::stage_b, wave, lane); };
    auto issue_x = [&](int buf) {
        source.issue_x(p, next_slice, smem + buf * TL::stage_b, wave, lane);
        if (++next_slice < nslices) return;
        next_slice = 0;
        next_tile += tiles.step;
        if (next_tile >= tiles.count) return;
        int f, c, l = threadIdx.x & 63;
        asm volatile("" : "+v"(l));  // computed anew for each tile: kept over the loop, its parts would fill registers
        tiles.at<TL>(next_tile, f, c);
        source.set(p, f, c, wave, l);
    };
    Operands<TL, FA> op;
    f32x4 acc[TL::WMT][TL::WNT];
    clear<TL>(acc);
    issue_w(0);
    issue_x(0);
    if (stages > 1) {
        issue_w(1);
        issue_x(1);
    }
    if (stages > 1)
        wait_vm<cW + cX>();  // the first stage
    else
        wait_vm<0>();
    lds_barrier();
    op.template read_w<0>(smem, wm, wn, r16, g4);
    static_for<0, TL::WNT>([&](auto NT) { op.template read_x<0, decltype(NT)::value>(smem, wn, r16, g4); });

    int slice = 0, buf = 0;
    bool stored = false;  // kStores stores have been issued since the next stage's copies
    for (int s = 0;; ++s) {
        const bool last = slice + 1 == nslices, ahead = s + 2 < stages;
        const bool both = !TL::X8 || 2 * slice + 1 < nblocks;  // whether a has the slice's second 128 values
        const lds_u8* const here = smem + buf * TL::stage_b;
        const lds_u8* const there = smem + (buf ^ 1) * TL::stage_b;
        // First half.  A token tile's registers take the second half's codes as soon as
        // its products are issued.
        op.turn(g4);
        op.template read_w<1>(here, wm, wn, r16, g4);
        static_for<0, TL::WNT>([&](auto NT) {
            constexpr int nt = decltype(NT)::value;
            __builtin_amdgcn_sched_barrier(0);
            op.template multiply<0, nt>(acc);
            __builtin_amdgcn_sched_barrier(0);
            op.template read_x<1, nt>(here, wn, r16, g4);
            if constexpr (nt == kFirst) {
                // W and the scales have arrived (LDS answers in order; x's later reads are
                // under way), in every wave
                lds_barrier_but<(kFirst + 1) * TL::XH>();
                if (ahead) issue_w(buf);
            }
        });
        op.turn(g4);
        // Second half, and the next stage's first (after the last stage: whatever is there).
        static_for<0, TL::WNT>([&](auto NT) {
            constexpr int nt = decltype(NT)::value;
            __builtin_amdgcn_sched_barrier(0);
            if (both) op.template multiply<1, nt>(acc);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (nt == kSecond) {
                // the next stage has landed: all but the stores and W that are younger
                if (!ahead)
                    wait_vm<0>();
                else if (stored)
                    wait_vm<kStores + cW>();
                else
                    wait_vm<cW>();
                lds_barrier();  // for every wave, and every wave has read x
                if (ahead) issue_x(buf);
                op.template read_w<0>(there, wm, wn, r16, g4);
                static_for<0, kSecond>([&](auto I) { op.template read_x<0, decltype(I)::value>(there, wn, r16, g4); });
            }
            if constexpr (nt >= kSecond) op.template read_x<0, nt>(there, wn, r16, g4);
        });
        __builtin_amdgcn_sched_barrier(0);
        stored = false;
        if (last) {
            const int R0 = f0 + 16 * TL::WNT * wn + TL::WNT * 4 * g4, C0 = c0 + 16 * TL::WMT * wm + TL::WMT * r16;
            stored = f0 + TL::toks <= p.M && c0 + TL::cols <= p.N;
            if (stored)
                store_inside<TL, OUT32>(p, acc, R0, C0);
            else
                store<TL, OUT32>(p, acc, R0, C0);
            if (s + 1 == stages) return;
            clear<TL>(acc);
            tile += tiles.step;
            tiles.at<TL>(tile, f0, c0);
        }
        slice = last ? 0 : slice + 1;
        buf ^= 1;
    }
}

template <class TL, int FA, bool OUT32>
__global__ __launch_bounds__(TL::waves * 64)
    __attribute__((amdgpu_waves_per_eu((TL::PER_CU * TL::waves + 3) / 4, (TL::PER_CU * TL::waves + 3) / 4))) void gdn_fp4_ring_kernel(
        gdn_fp4::MatmulParams p, int n_tok, int n_col) {
    constexpr int WMT = TL::WMT, WNT = TL::WNT, NS = TL::NS, KS = TL::KS;
    constexpr bool kBf16 = OUT32 && TL::X8;  // products on the bf16 instruction
    static_assert(TL::X8 == (FA != GDN_E2M1), "rows of x");
    __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[TL::lds_b];
    lds_u8* const smem = (lds_u8*)&smem_raw[0];
    int f0, c0;  // the tile's first token and column
    Tiles(n_tok, n_col).at<TL>(static_cast<int>(blockIdx.x) >> 3, f0, c0);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = KS > 1 ? wave / TL::gwaves : 0, gw = KS > 1 ? wave % TL::gwaves : wave;
    const int wm = gw / TL::TW, wn = gw % TL::TW, r16 = lane & 15, g4 = lane >> 4;
    const int nblocks = p.K / 128, nslices = (nblocks + 1) / 2;
    Source<TL> source;
    source.set(p, f0, c0, gw, lane);
    // The slice of stage kk that this wave's group takes (the last stage's
    // groups past the end repeat the last slice and do not multiply it).
    auto issue = [&](int buf, int kk) {
        const int slice = __builtin_amdgcn_readfirstlane(KS > 1 ? min(kk * KS + ks, nslices - 1) : kk);
        source.issue_w(p, slice, smem + buf * TL::stage_b + ks * TL::slice_b, gw, lane);
        source.issue_x(p, slice, smem + buf * TL::stage_b + ks * TL::slice_b, gw, lane);
    };
    f32x4 acc[WMT][WNT];
    clear<TL>(acc);

    // Ring of NS stages: stage kt + NS - 1 is issued while stage kt is
    // multiplied, into the buffer that stage kt - 1 was read from.
    const int nk = (nslices + KS - 1) / KS;
#pragma unroll
    for (int st = 0; st < NS - 1; ++st)
        if (st < nk) issue(st, st);
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
        if (next) issue(ws, kt + NS - 1);
        if (KS == 1 || slice < nslices) {
            const lds_u8* const st = smem + rs * TL::stage_b + ks * TL::slice_b;
            const bool both = !TL::X8 || 2 * slice + 1 < nblocks;
            if constexpr (!kBf16) {
                Operands<TL, FA> op;
                static_for<0, 2>([&](auto H) {
                    constexpr int h = decltype(H)::value;
                    if (h == 1 && !both) return;
                    op.template read_w<h>(st, wm, wn, r16, g4);
                    op.turn(g4);
                    static_for<0, WNT>([&](auto NT) { op.template read_x<h, decltype(NT)::value>(st, wn, r16, g4); });
                    static_for<0, WNT>([&](auto NT) { op.template multiply<h, decltype(NT)::value>(acc); });
                });
            } else {
                static_for<0, 2>([&](auto H) {
                    constexpr int h = decltype(H)::value;
                    if (h == 1 && !both) return;
                    const lds_u8* const stw = st + (16 * WMT * wm + r16) * kRowB;
                    const lds_u8* const stx = st + (TL::cols + h * TL::toks + 16 * WNT * wn + r16) * kRowB;
                    // W's scales over the block's largest of its column, and that one
                    uint32_t own[WMT], most[WMT];
                    u32x4 wc[WMT];
                    f32x4 block[WMT][WNT];
#pragma unroll
                    for (int mt = 0; mt < WMT; ++mt) {
                        const uint32_t word = reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(st + TL::off_ws)[h * TL::cols + 16 * WMT * wm + WMT * r16 + mt];
                        most[mt] = largest_byte(word);
                        own[mt] = byte_over(word >> (8 * g4) & 0xffu, most[mt]);
                        wc[mt] = *reinterpret_cast<const lds_u32x4*>(stw + 16 * mt * kRowB + 16 * ((4 * h + g4) ^ swz(r16)));
                    }
                    clear<TL>(block);
                    // values 32 g4 .. + 31 of the row: 16-byte pieces 2 g4 and 2 g4 + 1
                    static_for<0, 2>([&](auto P) {
                        constexpr int piece = decltype(P)::value;
                        u32x4 xc[WNT];
#pragma unroll
                        for (int nt = 0; nt < WNT; ++nt) xc[nt] = *reinterpret_cast<const lds_u32x4*>(stx + 16 * nt * kRowB + 16 * ((2 * g4 + piece) ^ swz(r16)));
                        static_for<0, 2>([&](auto Q) {
                            constexpr int q = decltype(Q)::value;
                            bf16x8 x[WNT];
                            static_for<0, WNT>([&](auto NT) { x[decltype(NT)::value] = codes_to_bf16<FA>(xc[decltype(NT)::value][2 * q], xc[decltype(NT)::value][2 * q + 1], 127u); });
                            static_for<0, WMT>([&](auto MT) {
                                constexpr int mt = decltype(MT)::value;
                                const bf16x8 w = fp4_to_bf16(wc[mt][2 * piece + q], own[mt]);
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
    store<TL, OUT32>(p, acc, f0 + 16 * WNT * wn + WNT * 4 * g4, c0 + 16 * WMT * wm + WMT * r16);
}

}  // namespace
