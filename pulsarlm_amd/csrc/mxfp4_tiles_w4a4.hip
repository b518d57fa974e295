// mx_tile_kernel with quantized x.
#include "mxfp4_tiles.hpp"

namespace plm {

void launch_mx_tiles_w4a4(const mx_product& p, hipStream_t s) {
    if (p.epilogue == kMxGatedCodes) launch_shape<true, true, kMxGatedCodes>(p, s);
    else if (p.bf16) launch_shape<true, true, kMxPlain>(p, s);
    else launch_shape<true, false, kMxPlain>(p, s);
}

}  // namespace plm
