// Products on unpacked weights: 8-bit integers with a scale for each token and channel, and 16-bit experts with both
// gradients, dense or grouped by expert with ragged sizes. Shared by the tile kernel (dense_tiles.hpp), the kernel for
// few rows (dense_rows.hip) and the entry points (dense_api.hip).
//
// Every product is D[r, c] = sum_k P[r, k] Q[c, k]: P's rows are the output's rows, Q's its columns.
//   forward         P = x [rows, K],  Q = W_e [N, K], sum over K
//   input gradient  P = dy [rows, N], Q = W_e [N, K] read along N, sum over N
//   weight gradient P = dy [rows, N], Q = x [rows, K], both read along the rows, sum over the expert's rows
#pragma once

#include <algorithm>
#include <type_traits>

#include "plm_common.hpp"

namespace plm {

enum dense_type { kBf16 = 0, kFp16 = 1, kInt8 = 2 };
// What a workgroup's tile is found from.
enum dense_mode {
    kDense,    // one product
    kByRows,   // expert e's rows offsets[e - 1] .. offsets[e] of P times its own Q
    kByRanges  // expert e's product sums over rows offsets[e - 1] .. offsets[e] of both
};

constexpr int64_t kDenseMaxSize = int64_t{1} << 19;  // N and K
constexpr int64_t kDenseMaxRows = (int64_t{1} << 24) - 1;
constexpr int64_t kInt8MaxK = 131056;  // 128 * 128 * K fits 31 bits
constexpr int64_t kMaxExperts = 4096;

typedef __attribute__((ext_vector_type(4))) int i32x4_t;

struct dense_args {
    const uint8_t *p, *q;  // rows pitch_p and pitch_q bytes apart
    uint16_t* y;           // [rows][cols], an expert's product `rows * cols` after the one before (kByRanges)
    const float *p_scale, *q_scale;  // int8: per row of P, per column [experts][cols]
    const int32_t* offsets;
    int64_t q_expert;           // bytes of an expert's Q (kByRows)
    int pitch_p, pitch_q;       // bytes
    int rows, cols, depth;      // the output's, and the length of the sum in elements (kByRanges: all rows)
    int experts;
    int m_blocks, n_blocks, band;  // kByRows: m_blocks as many as there can be
    bool zero_rest;             // kByRows: rows past the last expert's are set to zero, else not written
    bool lines, wide;           // stores of 16 bytes (cols % 8 == 0, y 16-byte aligned), of 8
    bool bf16;                  // the output's type
    i32x4_t* partial;           // dense 8-bit: sums of split_stages stages each, [splits][rows][quads of columns], or null
    int split_stages, quads;
};

// The rows of the experts: offsets are their inclusive ends, each taken within [0, rows] and no less than the ones before
// it, so that the experts' rows never overlap whatever the offsets are.
template <int CTRL, int ROW_MASK> __device__ __forceinline__ int dpp_max(int x) {
    return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xf, true));
}
// Inclusive running maximum of non-negative values over the wavefront.
__device__ __forceinline__ int wave_inclusive_max(int x) {
    x = dpp_max<0x111, 0xf>(x);
    x = dpp_max<0x112, 0xf>(x);
    x = dpp_max<0x114, 0xf>(x);
    x = dpp_max<0x118, 0xf>(x);
    x = dpp_max<0x142, 0xa>(x);
    return dpp_max<0x143, 0xc>(x);
}

struct expert_range {
    int expert, lo, hi;
};

// A lane's value from lane `at`.
__device__ __forceinline__ int from_lane(int v, int at) { return __builtin_amdgcn_ds_bpermute(at * 4, v); }

// The rows of the expert at each lane's place `slot`. Up to 64 experts are placed by their rows, most first (their
// products' times go by them, and the longest should not begin last), more of them as they come. By a whole wavefront.
__device__ __forceinline__ expert_range find_experts(const int32_t* __restrict__ offsets, int n, int rows, int slot) {
    const int lane = __lane_id();
    if (n <= 64) {
        const int hi = wave_inclusive_max(lane < n ? min(max(offsets[lane], 0), rows) : 0);
        int lo = __shfl_up(hi, 1);
        if (lane == 0) lo = 0;
        const int count = lane < n ? hi - lo : -1;
        int place = 0;
        for (int i = 0; i < n; ++i) {
            const int other = __builtin_amdgcn_readlane(count, i);
            place += other > count || (other == count && i < lane) ? 1 : 0;
        }
        place = lane < n ? place : lane;
        const int e = from_lane(__builtin_amdgcn_ds_permute(place * 4, lane), slot);  // the lane that goes to the place
        return {e, from_lane(lo, e), from_lane(hi, e)};
    }
    expert_range r{slot, 0, 0};
    for (int base = 0, end = 0; base < n; base += 64) {
        const int i = base + lane;
        const int hi = max(wave_inclusive_max(i < n ? min(max(offsets[i], 0), rows) : 0), end);
        int lo = __shfl_up(hi, 1);
        if (lane == 0) lo = end;
        const int at_lo = from_lane(lo, slot & 63), at_hi = from_lane(hi, slot & 63);
        if ((slot & ~63) == base) r.lo = at_lo, r.hi = at_hi;
        end = __builtin_amdgcn_readlane(hi, 63);
    }
    return r;
}

// Row blocks of `1 << shift` rows, expert by expert; where rest is set, the rows past the last expert's count as
// expert n's. count_blocks: how many there are. find_block: block b's expert and rows. Both by one wavefront, 64
// experts at a time.
struct block_scan {
    int end, blocks;  // carried over the experts before
};
template <typename F>
__device__ __forceinline__ block_scan scan_blocks(const int32_t* __restrict__ offsets, int n, int rows, bool rest, int shift, F visit) {
    const int lane = __lane_id(), count = n + (rest ? 1 : 0);
    block_scan s{0, 0};
    for (int base = 0; base < count; base += 64) {
        const int i = base + lane;
        int v = 0;
        if (i < n) v = min(max(offsets[i], 0), rows);
        else if (i < count) v = rows;
        const int hi = max(wave_inclusive_max(v), s.end);
        int lo = __shfl_up(hi, 1);
        if (lane == 0) lo = s.end;
        const int blocks = (hi - lo + (1 << shift) - 1) >> shift;
        const int past = s.blocks + wave_inclusive_scan(blocks);
        if (visit(base, lo, hi, past - blocks, past)) break;
        s.end = __builtin_amdgcn_readlane(hi, 63);
        s.blocks = __builtin_amdgcn_readlane(past, 63);
    }
    return s;
}
__device__ __forceinline__ int count_blocks(const int32_t* offsets, int n, int rows, bool rest, int shift) {
    return scan_blocks(offsets, n, rows, rest, shift, [](int, int, int, int, int) { return false; }).blocks;
}
// b < count_blocks(...).
__device__ __forceinline__ expert_range find_block(const int32_t* offsets, int n, int rows, bool rest, int shift, int b) {
    expert_range r{0, 0, 0};
    scan_blocks(offsets, n, rows, rest, shift, [&](int base, int lo, int hi, int first, int past) {
        const uint64_t later = __ballot(past > b);
        if (later == 0) return false;
        const int at = __ffsll(static_cast<unsigned long long>(later)) - 1;
        const int row = __builtin_amdgcn_readlane(lo, at) + ((b - __builtin_amdgcn_readlane(first, at)) << shift);
        r = {base + at, row, min(row + (1 << shift), __builtin_amdgcn_readlane(hi, at))};
        return true;
    });
    return r;
}

// The same for each lane's own b (a result is only used where b < count_blocks(...)).
__device__ __forceinline__ expert_range find_blocks(const int32_t* offsets, int n, int rows, bool rest, int shift, int b) {
    expert_range r{0, 0, 0};
    int before = 0;  // blocks of the experts seen before
    scan_blocks(offsets, n, rows, rest, shift, [&](int base, int lo, int hi, int first, int past) {
        int at = 0;  // the first expert whose blocks end past b
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) at += from_lane(past, at + step - 1) <= b ? step : 0;
        const int row = from_lane(lo, at) + ((b - from_lane(first, at)) << shift), end = min(row + (1 << shift), from_lane(hi, at));
        const int blocks = __builtin_amdgcn_readlane(past, 63);
        if (b >= before && b < blocks) r = {base + at, row, end};
        before = blocks;
        return false;
    });
    return r;
}

// Sums, int32 or fp32, of the matrix instruction on 16 x 16 rows and columns and 64 bytes of K: a lane's operand is 16
// bytes, row lane % 16, K bytes 16 (lane / 16) on; its sums are P's row lane % 16 and Q's rows 4 (lane / 16) + 0..3.
template <dense_type T> using dense_acc = std::conditional_t<T == kInt8, i32x4_t, f32x4_t>;

template <dense_type T> __device__ __forceinline__ dense_acc<T> dense_mfma(u32x4_t q, u32x4_t p, dense_acc<T> c) {
    if constexpr (T == kInt8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, q), __builtin_bit_cast(i32x4_t, p), c, 0, 0, 0);
    else return mfma16x16x32<T == kBf16>(q, p, c);
}

// Four columns of a row, the 8-bit products' sums scaled: sum * channel scale * token scale. The scales' exponents come last, in
// one step, so that only a result that is out of range itself passes fp32's, whichever scale is the large one: the sum times
// both mantissas lies within 2^-2 and 2^31. Three roundings to fp32, the sum's and the two products', and one more of
// results below its normal range. Beside two plain products, whose bits it gives wherever they stay in range: 4096 rows, N 24576,
// K 4096 338 us for 333, 2000 rows, N = K = 4096 34.5 for 34.7.
__device__ __forceinline__ f32x4_t dense_scaled(const i32x4_t& v, const f32x4_t& channel, float token) {
    f32x4_t f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = __builtin_amdgcn_ldexpf(static_cast<float>(v[i]) * __builtin_amdgcn_frexp_mantf(channel[i]) * __builtin_amdgcn_frexp_mantf(token),
                                       __builtin_amdgcn_frexp_expf(channel[i]) + __builtin_amdgcn_frexp_expf(token));
    return f;
}
template <bool BF16> __device__ __forceinline__ uint2 dense_pack(const f32x4_t& f) {
    return make_uint2(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]));
}
// The channel scales of columns col .. col + 3, zeros past cols.
__device__ __forceinline__ f32x4_t dense_channels(const float* scale, int col, int cols) {
    f32x4_t f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = col + i < cols ? scale[col + i] : 0.f;
    return f;
}
// Columns col .. col + 3 of a row that starts at `row`, which lie below cols.
template <bool BF16> __device__ __forceinline__ void dense_store4(uint16_t* row, int col, int cols, bool wide, const f32x4_t& f) {
    if (wide) {  // cols % 4 == 0
        if (col < cols) *reinterpret_cast<uint2*>(row + col) = dense_pack<BF16>(f);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < cols) row[col + i] = static_cast<uint16_t>(to_bits16<BF16>(f[i]));
}

// Which kernel takes a call: for few rows, in blocks of rows_block, or where that is 0 a tile shape, with the sum split
// into parts.
struct dense_plan {
    int shape = 0, splits = 1, rows_block = 0;
};
// One call's product. type: the operands'.
struct dense_product {
    const void *p, *q;
    void* y;
    const float *p_scale, *q_scale;
    const int32_t* offsets;
    int64_t rows, cols, depth;  // kByRanges: rows N, cols K, depth the number of all rows
    int64_t experts;
    dense_type type;
    bool bf16, zero_rest;
    bool to_quantize;  // dense 8-bit: p is 16 bits and 16-byte aligned, quantized by the kernel for few rows or before
    dense_plan plan;
    i32x4_t* partial;
};

// Row blocks of `rows` that a call can have: by rows, each expert's last one can be a part.
inline int64_t dense_row_blocks(const dense_product& p, dense_mode mode, int64_t rows) {
    const int64_t whole = ceil_div(p.rows, rows);
    return mode == kByRows ? std::min(p.rows, whole + p.experts) : whole;
}
// A grid's work-items are counted in 32 bits.
inline bool dense_grid_fits(int64_t workgroups, int64_t threads) { return workgroups * threads < int64_t{1} << 32; }
// The kernels' arguments but for the blocks. across: the operand lies across the sum.
inline dense_args make_dense_args(const dense_product& p, bool p_across, bool q_across) {
    const int64_t size = p.type == kInt8 ? 1 : 2;
    dense_args a{};
    a.p = static_cast<const uint8_t*>(p.p);
    a.q = static_cast<const uint8_t*>(p.q);
    a.y = static_cast<uint16_t*>(p.y);
    a.p_scale = p.p_scale;
    a.q_scale = p.q_scale;
    a.offsets = p.offsets;
    a.rows = static_cast<int>(p.rows);
    a.cols = static_cast<int>(p.cols);
    a.depth = static_cast<int>(p.depth);
    a.pitch_p = static_cast<int>((p_across ? p.rows : p.depth) * size);
    a.pitch_q = static_cast<int>((q_across ? p.cols : p.depth) * size);
    a.q_expert = p.cols * p.depth * size;
    a.experts = static_cast<int>(p.experts);
    a.zero_rest = p.zero_rest;
    a.bf16 = p.bf16;
    a.lines = p.cols % 8 == 0 && aligned(p.y, 16);
    a.wide = p.cols % 4 == 0 && aligned(p.y, 8);
    a.quads = static_cast<int>(ceil_div(p.cols, 4));
    return a;
}

dense_plan plan_dense(const dense_product& p, dense_mode mode, bool rows_kernel, bool may_split);
// Strips of 16 columns of a workgroup of the kernel for few rows: two where that leaves work for every CU.
inline int64_t dense_rows_strips(int64_t blocks, int64_t cols) { return ceil_div(cols, 16) * blocks > cu_count() ? 2 : 1; }
// Workspace of a plan's parts.
inline int64_t dense_partial_bytes(const dense_plan& plan, int64_t rows, int64_t cols) {
    return plan.splits > 1 ? plan.splits * rows * ceil_div(cols, 4) * 16 : 0;
}
void launch_tiles_int8(const dense_product& p, dense_mode mode, hipStream_t s);
void launch_tiles_16(const dense_product& p, hipStream_t s);         // forward, by rows
void launch_tiles_grad_x(const dense_product& p, hipStream_t s);
void launch_tiles_grad_w(const dense_product& p, hipStream_t s);
void launch_combine_int8(const dense_product& p, hipStream_t s);
// The kernel for few rows, forward.
void launch_dense_rows(const dense_product& p, dense_mode mode, hipStream_t s);
// The same on 16-bit x [rows][depth] (p.p, 16-byte aligned), quantized in the kernel, for dense 8-bit products that it takes.
bool dense_rows_quantizes(const dense_product& p, int rows_block);
void launch_dense_rows_quantize(const dense_product& p, hipStream_t s);

// Rows of codes and their scales.
void launch_quantize_int8(const void* x, plm_dtype dtype, int64_t m, int64_t k, int8_t* codes, float* scale, hipStream_t s);

}  // namespace plm
