// Tiles of the inputs' gradient by expert: dx = dy W_e.
#include "dense_tiles.hpp"

namespace plm {

void launch_tiles_grad_x(const dense_product& p, hipStream_t s) {
    if (p.type == kBf16) launch_shape<kBf16, kByRows, false, true>(p, s);
    else launch_shape<kFp16, kByRows, false, true>(p, s);
}

}  // namespace plm
