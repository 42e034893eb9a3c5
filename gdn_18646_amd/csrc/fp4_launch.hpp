// Launches of the tiled kernels of the product with 4-bit weights: a tile's kernel and
// grid, instantiated for each format of the activations in fp4_mm_*.hip.
#pragma once

#include <algorithm>

#include "fp4_phased.hpp"
#include "fp4_tiles.hpp"

namespace gdn_fp4 {

template <class TL, bool STREAM, int FA, bool OUT32>
int launch_tiled(const MatmulParams& p, hipStream_t stream) {
    const int n_tok = (p.M + TL::toks - 1) / TL::toks, n_col = (p.N + TL::cols - 1) / TL::cols;
    const unsigned tiles = static_cast<unsigned>(n_tok) * n_col;
    const dim3 grid(STREAM ? std::min<unsigned>(tiles, 256 * TL::PER_CU) : tiles);
    if (!gdn_host::grid_fits(grid.x, TL::waves * 64))
        return gdn_host::fail(GDN_ERR_UNSUPPORTED, "fp4_matmul: M=%d N=%d are too large for a launch", p.M, p.N);
    if constexpr (STREAM)
        hipLaunchKernelGGL((gdn_fp4_stream_kernel<TL, FA, OUT32>), grid, dim3(TL::waves * 64), 0, stream, p, n_tok, n_col);
    else
        hipLaunchKernelGGL((gdn_fp4_ring_kernel<TL, FA, OUT32>), grid, dim3(TL::waves * 64), 0, stream, p, n_tok, n_col);
    return gdn_host::check_launch("gdn_fp4_matmul_kernel");
}

template <int FA>
int launch_phased(const MatmulParams& p, hipStream_t stream) {
    using TL = Phased;
    const int n_tok = (p.M + TL::toks - 1) / TL::toks, n_col = (p.N + TL::cols - 1) / TL::cols;
    const unsigned grid = std::min<unsigned>(static_cast<unsigned>(n_tok) * n_col, 256);
    hipLaunchKernelGGL(gdn_fp4_phased_kernel<FA>, dim3(grid), dim3(512), 0, stream, p, n_tok, n_col);
    return gdn_host::check_launch("gdn_fp4_phased_kernel");
}

// columns x tokens
template <int FA, bool OUT32>
int launch_out(int tile, const MatmulParams& p, hipStream_t stream) {
    constexpr bool X8 = FA != GDN_E2M1;
    constexpr bool kStream = !(X8 && OUT32);
    if constexpr (!X8) {
        switch (tile) {
            case k256x256: return launch_tiled<Fp4Tile<X8, 2, 4, 8, 4, 2, 1>, true, FA, OUT32>(p, stream);
            case k128x128: return launch_tiled<Fp4Tile<X8, 2, 2, 4, 4, 2, 2>, true, FA, OUT32>(p, stream);
            case k128x64: return launch_tiled<Fp4Tile<X8, 2, 2, 4, 2, 3, 2>, false, FA, OUT32>(p, stream);
            case k64x128: return launch_tiled<Fp4Tile<X8, 1, 4, 4, 2, 3, 1, 2>, false, FA, OUT32>(p, stream);
        }
    } else {
        if constexpr (kStream) {
            if (tile == k256x256) return launch_phased<FA>(p, stream);
            if (tile == k256x128) return launch_tiled<Fp4Tile<X8, 4, 2, 4, 4, 2, 1>, true, FA, OUT32>(p, stream);
        }
        switch (tile) {
            case k128x64: return launch_tiled<Fp4Tile<X8, 2, 2, 4, 2, 2, 2>, kStream, FA, OUT32>(p, stream);
            case k16x16Alone: return launch_tiled<Fp4Tile<X8, 1, 1, 1, 1, 3, 1, 8>, false, FA, OUT32>(p, stream);
        }
    }
    switch (tile) {
        case k64x64: return launch_tiled<Fp4Tile<X8, 2, 2, 2, 2, 3, 1, 2>, false, FA, OUT32>(p, stream);
        case k64x32: return launch_tiled<Fp4Tile<X8, 1, 2, 4, 1, X8 ? 2 : 3, 1, 4>, false, FA, OUT32>(p, stream);
        case k32x32: return launch_tiled<Fp4Tile<X8, 1, 2, 2, 1, X8 ? 2 : 3, 1, 4>, false, FA, OUT32>(p, stream);
        default: return launch_tiled<Fp4Tile<X8, 1, 1, 1, 1, X8 ? 2 : 3, 3, 4>, false, FA, OUT32>(p, stream);
    }
}

template <int FA>
int launch_tile(int tile, bool f32, const MatmulParams& p, hipStream_t stream) {
    return f32 ? launch_out<FA, true>(tile, p, stream) : launch_out<FA, false>(tile, p, stream);
}

}  // namespace gdn_fp4
