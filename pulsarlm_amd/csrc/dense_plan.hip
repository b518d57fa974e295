// Which kernel takes a product on unpacked weights, and the kernel that adds the parts of a split sum.
#include <algorithm>
#include <cmath>

#include "dense_gemm.hpp"

namespace plm {

namespace {

// Times in us, fitted to calls of 1 to 4096 rows, N 1000 to 24576, K 2048 to 17408 from captured graphs, weights cold.
//
// A tile shape's time is that of a stage, for each of its stages, one and a half a tile and two and a half a launch: `one`
// with one workgroup a CU, from few of them to one on every CU; `two` for a pair on a CU, where two fit.
struct tile_cost {
    int rows, cols;
    double one_few, one_all, two;
};
constexpr tile_cost kTileCosts[] = {{256, 256, 1.28, 1.58, 0.}, {128, 256, .88, .94, 0.}, {128, 128, .62, .63, 0.},
                                    {128, 128, .87, .87, 1.06}, {64, 128, .47, .50, .68}, {64, 64, .31, .33, .52}};
constexpr double kTileEnds = 1.5, kLaunchEnds = 2.5;
// Experts' weights through tiles with few rows: E 128, N 1536, K 2048 in 16 bits, 64 rows 74 to 67 us of the kernel for few
// rows, 256 rows 136 to 123, 512 rows 141 to 144.
constexpr double kRaggedTiles = 1.1;
// By ranges: both operands lie across the sum, sums of unequal length, of which the longest is taken as three times the
// average, or all there is.
constexpr double kRangesStage = 1.13, kRangesEnds = 3.;
double ranges_time(const tile_cost& c, double tiles, int64_t stages, int64_t experts) {
    const double each = std::max(1., tiles / cu_count() / (c.two > 0. ? 2. : 1.)), all = c.two > 0. ? c.two : c.one_all;
    return kRangesStage * std::max((each * (stages + kRangesEnds) + kLaunchEnds) * all, (std::min<int64_t>(3, experts) * stages + kRangesEnds + kLaunchEnds) * c.one_all);
}
// Workgroups of the busiest CU; where their number is a guess, the average and a half.
double rounds_of(double tiles, bool guess) {
    const double each = tiles / cu_count();
    return std::max(1., guess && each > 1. ? each + .5 : static_cast<double>(static_cast<int64_t>(each + .999)));
}
double rounds_time(const tile_cost& c, double tiles, bool guess, int64_t stages) {
    const double each = rounds_of(tiles, guess), one = c.one_few + (c.one_all - c.one_few) * std::min(1., tiles / cu_count());
    const double pairs = c.two > 0. ? static_cast<double>(static_cast<int64_t>(each) / 2) : 0.;
    return (pairs * c.two + (each - 2 * pairs) * one) * (stages + kTileEnds) + kLaunchEnds * one;
}
// The kernel for few rows: a CU takes in 33 GB/s of its workgroups' x and weights (64 bytes of a row a request), all of
// them 5.2 TB/s of weights.
constexpr double kStart = 3.3, kRowsRate = 33e3, kMemoryRate = 5.2e6;
// The launch that quantizes 16-bit rows, where the product does not; and where it does, a value a thread past the 32 that wait
// in registers, which is read again. M 1: N 1024, K 1024 4.3 us in the kernel for few rows and 7.5 through tiles, N 12288, K 16384 57
// and 52; M 2: N 4096, K 512 4.5 and 7.0, N 24576, K 12288 74 and 82, K 16384 99 and 89.
constexpr double kQuantizer = 2.2, kReadAgain = .06;
// A split sum's parts: a kernel more, and their way through memory and back.
constexpr double kCombine = 4.0, kPartRate = 4.5e6;

// By rows, how the rows fall on the experts is known on the device only. Taken: 1 - e^-a of them have any, with a rows
// an expert on average, and those have half a block more than whole ones, one at least.
dense_plan make_plan(const dense_product& p, dense_mode mode, bool rows_kernel, bool may_split) {
    const int64_t size = p.type == kInt8 ? 1 : 2, cus = cu_count();
    const int64_t depth = mode == kByRanges ? ceil_div(p.depth, p.experts) : p.depth;
    const int64_t stages = std::max<int64_t>(1, ceil_div(depth * size, 128));
    const tuning& t = knobs();
    dense_plan best;
    if (rows_kernel && t.dense_rows > 0) {
        best.rows_block = t.dense_rows;
        return best;
    }
    if (t.dense_tile >= 0) {
        best.shape = t.dense_tile;
        if (may_split) best.splits = static_cast<int>(ceil_div(stages, ceil_div(stages, std::min<int64_t>(stages, t.dense_splits))));
        return best;
    }
    const double used = mode == kByRows ? p.experts * (1. - std::exp(-static_cast<double>(p.rows) / p.experts)) : 1.;
    const double memory = kStart + (mode == kByRanges ? 1. * p.experts * p.rows * p.cols : used * p.cols * depth) * size / kMemoryRate;
    const bool guess = mode == kByRows && p.experts > 1;
    auto blocks_of = [&](int64_t rows) {
        if (!guess) return static_cast<double>(ceil_div(p.rows, rows));
        return used + std::max(0., static_cast<double>(p.rows) / rows - .5 * used);
    };
    // What takes longer hides most of the other.
    auto together = [](double a, double b) { return std::max(a, b) + .3 * std::min(a, b); };
    double least = 1e300;
    for (int i = 0; i < 6; ++i) {
        const tile_cost& c = kTileCosts[i];
        const int64_t cols = ceil_div(p.cols, c.cols), experts = mode == kByRanges ? p.experts : 1;
        const double tiles = blocks_of(c.rows) * cols * experts;
        const int64_t most = may_split ? std::max<int64_t>(1, std::min<int64_t>({16, stages / 4, static_cast<int64_t>(2 * cus / tiles)})) : 1;
        for (int64_t splits = 1; splits <= most; ++splits) {
            const int64_t each = ceil_div(stages, splits);
            if (ceil_div(stages, each) != splits) continue;  // no part without a stage
            double time = mode == kByRanges ? together(memory, ranges_time(c, tiles, stages, p.experts))
                                            : together(memory * (mode == kByRows ? kRaggedTiles : 1.), rounds_time(c, tiles * splits, guess, each));
            if (splits > 1) time += kCombine + splits * p.rows * p.cols * 8 / kPartRate;
            if (p.to_quantize) time += kQuantizer;
            if (time < least) least = time, best = {i, static_cast<int>(splits), 0};
        }
    }
    if (!rows_kernel || t.dense_rows == 0) return best;
    for (int block : {16, 32, 64}) {
        const int64_t blocks = dense_row_blocks(p, mode, block);
        if (!dense_grid_fits(blocks * ceil_div(p.cols, 16), 512)) continue;
        const int64_t strips = dense_rows_strips(blocks, p.cols);
        const double groups = blocks_of(block) * ceil_div(p.cols, 16 * strips);
        const double rows = std::min<double>(block, p.rows / used);
        double time = together(memory, kStart + rounds_of(groups, guess) * (16 * strips + rows) * depth * size / kRowsRate);
        if (p.to_quantize) {
            const double values = static_cast<double>(p.rows) * p.depth / (strips == 2 ? 256 : 512);  // a thread's
            time += dense_rows_quantizes(p, block) ? kReadAgain * std::max(0., values - 32) : kQuantizer;
        }
        if (time < least) least = time, best = {0, 1, block};
    }
    return best;
}

}  // namespace

dense_plan plan_dense(const dense_product& p, dense_mode mode, bool rows_kernel, bool may_split) {
    static thread_local plan_cache<dense_plan> cache;
    const int kind = mode * 16 + (p.to_quantize ? 8 : 0) + (p.type == kInt8 ? 4 : 0) + (rows_kernel ? 2 : 0) + (may_split ? 1 : 0);
    return cache.get(kind, p.rows, p.cols, p.depth, p.experts, [&] { return make_plan(p, mode, rows_kernel, may_split); });
}

namespace {

// y = the parts' sum, scaled; four columns a thread.
template <bool BF16>
__global__ void __launch_bounds__(256) combine_int8_kernel(const i32x4_t* __restrict__ partial, int splits, int64_t rows, int quads, int cols,
                                                           const float* __restrict__ p_scale, const float* __restrict__ q_scale, uint16_t* __restrict__ y, bool wide) {
    const int64_t total = rows * quads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / quads;
        const int col = static_cast<int>(i - row * quads) * 4;
        i32x4_t v = partial[i];
        for (int s = 1; s < splits; ++s) v = v + partial[s * total + i];
        dense_store4<BF16>(y + row * cols, col, cols, wide, dense_scaled(v, dense_channels(q_scale, col, cols), p_scale[row]));
    }
}

}  // namespace

void launch_combine_int8(const dense_product& p, hipStream_t s) {
    const int64_t quads = ceil_div(p.cols, 4), total = p.rows * quads;
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(total, 256), int64_t{32} * cu_count()));
    const bool wide = p.cols % 4 == 0 && aligned(p.y, 8);
    auto* y = static_cast<uint16_t*>(p.y);
    if (p.bf16) combine_int8_kernel<true><<<grid, 256, 0, s>>>(p.partial, p.plan.splits, p.rows, int(quads), int(p.cols), p.p_scale, p.q_scale, y, wide);
    else combine_int8_kernel<false><<<grid, 256, 0, s>>>(p.partial, p.plan.splits, p.rows, int(quads), int(p.cols), p.p_scale, p.q_scale, y, wide);
}

}  // namespace plm
