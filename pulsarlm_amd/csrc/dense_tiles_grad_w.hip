// Tiles of the weights' gradient by expert: dW_e = dy_e^T x_e.
#include "dense_tiles.hpp"

namespace plm {

void launch_tiles_grad_w(const dense_product& p, hipStream_t s) {
    if (p.type == kBf16) launch_shape<kBf16, kByRanges, true, true>(p, s);
    else launch_shape<kFp16, kByRanges, true, true>(p, s);
}

}  // namespace plm
