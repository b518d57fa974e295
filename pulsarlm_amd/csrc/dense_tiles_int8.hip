// Tiles of the 8-bit products, dense and by expert.
#include "dense_tiles.hpp"

namespace plm {

void launch_tiles_int8(const dense_product& p, dense_mode mode, hipStream_t s) {
    if (mode == kDense) launch_shape<kInt8, kDense, false, false>(p, s);
    else launch_shape<kInt8, kByRows, false, false>(p, s);
}

}  // namespace plm
