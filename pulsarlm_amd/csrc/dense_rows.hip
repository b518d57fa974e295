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

// 16-bit x of a dense 8-bit product quantized in the kernel, by every workgroup for itself. Against a launch more, us: one
// row of N 6144, K 4096 10.2 and 12.4, two 12.2 and 12.4; N 4096, K 12288 one 13.2 and 15.3, four 19.2 and 15.3; N 1000,
// K 2048 four 4.9 and 6.5.
bool dense_rows_quantizes(const dense_product& p, int rows_block) {
    const int64_t bytes = p.rows * p.depth;
    return p.to_quantize && rows_block == 16 && p.rows <= kQuantRows && bytes <= (p.rows <= 2 ? kQuantBytes : 8192);
}
void launch_dense_rows_quantize(const dense_product& p, hipStream_t s) {
    if (dense_rows_strips(1, p.cols) == 2) launch_rows<kInt8, kDense, 1, 2, 4, 4, true>(p, s);
    else launch_rows<kInt8, kDense, 1, 1, 2, 8, true>(p, s);
}

void launch_dense_rows(const dense_product& p, dense_mode mode, hipStream_t s) {
    if (mode == kDense) launch_blocks<kInt8, kDense>(p, s);
    else if (p.type == kInt8) launch_blocks<kInt8, kByRows>(p, s);
    else if (p.type == kBf16) launch_blocks<kBf16, kByRows>(p, s);
    else launch_blocks<kFp16, kByRows>(p, s);
}

}  // namespace plm
