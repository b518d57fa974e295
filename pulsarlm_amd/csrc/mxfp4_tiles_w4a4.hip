// mx_tile_kernel with quantized x.
#include "mxfp4_tiles.hpp"

namespace plm {

void launch_mx_tiles_w4a4(const mx_product& p, hipStream_t s) {
    if (p.epilogue == kMxGatedCodes) launch_shape<true, true, kMxGatedCodes>(p, s);
    else if (p.bf16) launch_shape<true, true, kMxPlain>(p, s);
    else launch_shape<true, false, kMxPlain>(p, s);
}

// Workspace of the K splits' sums.
int64_t mx_tiles_w4a4_bytes(int64_t m, int64_t n, int64_t k) {
    const tile_choice c = choose_w4a4(m, n, k, true);
    return c.splits > 1 ? c.splits * m * n * 4 : 0;
}

}  // namespace plm
