// The products on unpacked weights for few rows: workgroup shapes.
#include "dense_rows.hpp"

namespace plm {

namespace {

template <dense_type T, dense_mode MODE> void launch_blocks(const dense_product& p, hipStream_t s) {
    const int rows = p.plan.rows_block;
    const bool wide = dense_rows_strips(dense_row_blocks(p, MODE, rows), p.cols) == 2;
    if (rows <= 16 && wide) launch_rows<T, MODE, 1, 2, 4, 4>(p, s);
    else if (rows <= 16) launch_rows<T, MODE, 1, 1, 2, 8>(p, s);
    else if (rows <= 32 && wide) launch_rows<T, MODE, 2, 2, 2, 4>(p, s);
    else if (rows <= 32) launch_rows<T, MODE, 2, 1, 2, 8>(p, s);
    else if (wide) launch_rows<T, MODE, 4, 2, 2, 8>(p, s);
    else launch_rows<T, MODE, 4, 1, 2, 8>(p, s);
}

}  // namespace

void launch_dense_rows(const dense_product& p, dense_mode mode, hipStream_t s) {
    if (mode == kDense) launch_blocks<kInt8, kDense>(p, s);
    else if (p.type == kInt8) launch_blocks<kInt8, kByRows>(p, s);
    else if (p.type == kBf16) launch_blocks<kBf16, kByRows>(p, s);
    else launch_blocks<kFp16, kByRows>(p, s);
}

}  // namespace plm
