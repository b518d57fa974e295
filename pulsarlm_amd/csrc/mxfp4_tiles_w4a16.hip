// mx_tile_kernel with 16-bit x.
#include "mxfp4_tiles.hpp"

namespace plm {

void launch_mx_tiles_w4a16(const mx_product& p, hipStream_t s) {
    if (p.epilogue == kMxGated) {
        if (p.bf16) launch_shape<false, true, kMxGated>(p, s);
        else launch_shape<false, false, kMxGated>(p, s);
    } else {
        if (p.bf16) launch_shape<false, true, kMxPlain>(p, s);
        else launch_shape<false, false, kMxPlain>(p, s);
    }
}

}  // namespace plm
