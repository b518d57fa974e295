// The products on unpacked weights for few rows, and which calls they take.
#include "dense_rows.hpp"

namespace plm {

namespace {

template <dense_type T, dense_mode MODE> void launch_blocks(const dense_product& p, int64_t rows, hipStream_t s) {
    if (rows <= 16) launch_rows<T, MODE, 1, 1, 4, 8>(p, s);
    else if (rows <= 32) launch_rows<T, MODE, 2, 1, 4, 8>(p, s);
    else launch_rows<T, MODE, 4, 2, 2, 8>(p, s);
}

}  // namespace

bool launch_dense_rows(const dense_product& p, dense_mode mode, hipStream_t s) {
    // Rows of a block: all of them, or twice the experts' average, as a router's choice is uneven.
    int64_t rows = mode == kByRows ? 2 * ceil_div(p.rows, p.experts) : p.rows;
    const int forced = knobs().dense_rows;
    if (forced == 0 || (forced < 0 && rows > 64) || !dense_grid_fits(dense_row_blocks(p, mode, 16) * ceil_div(p.cols, 16), 512)) return false;
    if (forced > 0) rows = forced;
    if (mode == kDense) launch_blocks<kInt8, kDense>(p, rows, s);
    else if (p.type == kInt8) launch_blocks<kInt8, kByRows>(p, rows, s);
    else if (p.type == kBf16) launch_blocks<kBf16, kByRows>(p, rows, s);
    else launch_blocks<kFp16, kByRows>(p, rows, s);
    return true;
}

}  // namespace plm
