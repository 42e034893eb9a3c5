// The tiled product of e2m1 codes by 4-bit weights (in a file of its own so that the
// formats build in parallel).
#include "fp4_launch.hpp"

template int gdn_fp4::launch_tile<GDN_E2M1>(int, bool, const gdn_fp4::MatmulParams&, hipStream_t);
