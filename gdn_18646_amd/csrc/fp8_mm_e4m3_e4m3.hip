// The tiled fp8 product of e4m3 codes by e4m3 codes (in a file of its own so that
// the pairs of formats build in parallel).
#include "fp8_tiles.hpp"

template int gdn_fp8::launch_tile<GDN_E4M3, GDN_E4M3>(int, int, bool, const gdn_fp8::MatmulParams&, hipStream_t);
