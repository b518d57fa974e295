// Tiles of the 16-bit products by expert: y = x W_e^T.
#include "dense_tiles.hpp"

namespace plm {

void launch_tiles_16(const dense_product& p, hipStream_t s) {
    if (p.type == kBf16) launch_shape<kBf16, kByRows, false, false>(p, s);
    else launch_shape<kFp16, kByRows, false, false>(p, s);
}

}  // namespace plm
