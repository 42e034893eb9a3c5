// The tiled product of e4m3 codes by 4-bit weights (in a file of its own so that the
// formats build in parallel).
#include "fp4_launch.hpp"

template int gdn_fp4::launch_tile<GDN_E4M3>(int, bool, const gdn_fp4::MatmulParams&, hipStream_t);
