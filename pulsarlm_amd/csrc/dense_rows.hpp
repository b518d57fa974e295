// The kernel of the products on unpacked weights (dense_gemm.hpp) for few rows, where the weights' bytes are what
// counts: they go from memory to registers once, as the matrix instruction's A operand, and x's few rows, which the
// caches hold, as its B operand.
//
// * A workgroup owns 16 MT rows by 16 NS columns. Its NW wavefronts take chunks of 64 U bytes of K in turn, each with the
//   next chunk's loads in flight, and their sums meet in LDS in wavefront order: results do not depend on timing.
// * QUANT: a few rows of 16-bit x, quantized by every workgroup for itself while its first weights are on their way: each
//   reads the rows for their largest magnitudes, and keeps their codes in LDS. A launch less: N 6144, K 4096, one row 10.2 us for
//   12.4.
// What bounds it: memory, 16 rows of 8 bits, N 4096, K 12288 13.1 us (50 MB); 64 rows over 128 experts in 16 bits, N 1536,
// K 2048 53.6 us (284 MB). With more rows x: every workgroup reads them again, from the caches, at 33 GB/s a CU.
#pragma once

#include <algorithm>

#include "dense_gemm.hpp"
#include "int8_rows.hpp"

namespace plm {

namespace {

constexpr int kQuantRows = 4, kQuantBytes = 64 * 1024;  // QUANT: rows and bytes of their codes at most

template <dense_type T, dense_mode MODE, int MT, int NS, int U, int NW, bool QUANT>
__global__ void __launch_bounds__(NW * 64) dense_rows_kernel(dense_args a) {
    using acc_t = dense_acc<T>;
    constexpr int SIZE = T == kInt8 ? 1 : 2, CHUNK = 64 * U, BM = 16 * MT;
    constexpr int SHIFT = MT == 1 ? 4 : MT == 2 ? 5 : 6;
    static_assert(1 << SHIFT == BM, "row blocks are powers of two");
    static_assert(!QUANT || (T == kInt8 && MODE == kDense && MT == 1), "a few rows of the dense product");
    __shared__ acc_t sums[NW][MT * NS][64];
    extern __shared__ __attribute__((aligned(16))) uint8_t codes[];  // QUANT: [rows][K]
    __shared__ uint32_t tops[QUANT ? NW : 1];
    __shared__ float tokens[QUANT ? kQuantRows : 1];

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col16 = lane & 15, kq = lane >> 4;
    const int nb = blockIdx.x % a.n_blocks, mb = blockIdx.x / a.n_blocks;
    int row0 = mb * BM, rows = min(BM, a.rows - row0), expert = 0, depth = a.depth;
    bool rest = false;  // rows of no expert: zeros, whatever scales they have
    if constexpr (MODE == kByRows) {
        if (mb >= count_blocks(a.offsets, a.experts, a.rows, a.zero_rest, SHIFT)) return;
        const expert_range r = find_block(a.offsets, a.experts, a.rows, a.zero_rest, SHIFT, mb);
        expert = r.expert, row0 = r.lo, rows = r.hi - r.lo;
        if (expert == a.experts) rest = true, expert = 0, depth = 0;
    }
    const int col0 = nb * (16 * NS);
    const int bytes = depth * SIZE, chunks = (bytes + CHUNK - 1) / CHUNK;

    const uint8_t* q_base = a.q + (MODE == kByRows ? expert * a.q_expert : 0) + static_cast<int64_t>(col0) * a.pitch_q;
    const __amdgpu_buffer_rsrc_t qr = make_rsrc(q_base, static_cast<uint32_t>(min(16 * NS, a.cols - col0)) * a.pitch_q);
    const __amdgpu_buffer_rsrc_t pr = make_rsrc(a.p + static_cast<int64_t>(row0) * a.pitch_p, static_cast<uint32_t>(rows) * a.pitch_p);
    const int q_at = col16 * a.pitch_q + kq * 16, p_at = col16 * a.pitch_p + kq * 16;

    struct chunk {
        u32x4_t q[NS][U], p[MT][U];
    };
    auto load = [&](chunk& c, int at) {  // chunk `at`; past the end zeros
        const int from = at < chunks ? at * CHUNK : 0, left = bytes - at * CHUNK;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int past = u * 64 + kq * 16 < left ? u * 64 : kOOB;
#pragma unroll
            for (int j = 0; j < NS; ++j) c.q[j][u] = buffer_load16(qr, q_at + past, from + j * 16 * a.pitch_q);
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if constexpr (!QUANT) c.p[i][u] = buffer_load16(pr, p_at + past, from + i * 16 * a.pitch_p);
        }
    };
    acc_t acc[MT][NS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
    // The rows' codes of chunk `at`.
    auto take_codes = [&](chunk& c, int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = at * CHUNK + u * 64 + kq * 16;
            c.p[0][u] = col16 < rows && k < bytes ? *reinterpret_cast<const u32x4_t*>(codes + col16 * bytes + k) : u32x4_t{0, 0, 0, 0};
        }
    };
    auto multiply = [&](const chunk& c) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][j] = dense_mfma<T>(c.q[j][u], c.p[i][u], acc[i][j]);
    };
    chunk even, odd;
    load(even, wave);
    if constexpr (QUANT) {
        // A row's wavefronts (all of them; half; a quarter) take its pieces of eight values in turn; the first HELD of a
        // lane wait in registers for the row's largest, what is past them is read again, from the caches.
        constexpr int HELD = 4;
        const int row_waves = rows == 1 ? NW : rows == 2 ? NW / 2 : NW / 4;
        const int r = wave / row_waves, step = row_waves * 64, first = (wave % row_waves) * 64 + lane, pieces = depth / 8;
        auto piece = [&](int i) { return buffer_load16(pr, i < pieces ? r * a.pitch_p + i * 16 : kOOB); };  // past the rows zeros
        u32x4_t held[HELD];
#pragma unroll
        for (int h = 0; h < HELD; ++h) held[h] = piece(first + h * step);
        uint32_t top = 0;
        auto count = [&](const u32x4_t& v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) top = top_16(top, v[i]);
        };
#pragma unroll
        for (int h = 0; h < HELD; ++h) count(held[h]);
        for (int i = first + HELD * step; i < pieces; i += step) count(piece(i));
        top = a.bf16 ? top_bits<true>(top) : top_bits<false>(top);
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), s)));
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        for (int w = r * row_waves; w < (r + 1) * row_waves; ++w) top = max(top, tops[w]);
        const int8_scale k = make_int8_scale(top);
        if (lane == 0 && r < kQuantRows) tokens[r] = k.s;
        auto put = [&](int i, const u32x4_t& v) {
            if (r >= rows || i >= pieces) return;
            uint32_t q[2] = {0, 0};
            float x[8];
            if (a.bf16) eight_values<true>(v, x);
            else eight_values<false>(v, x);
            if (k.finite) int8_codes<8>(x, k, q);
            *reinterpret_cast<uint2*>(codes + r * depth + i * 8) = make_uint2(q[0], q[1]);
        };
#pragma unroll
        for (int h = 0; h < HELD; ++h) put(first + h * step, held[h]);
        for (int i = first + HELD * step; i < pieces; i += step) put(i, piece(i));
        __syncthreads();
    }
    for (int c = wave; c < chunks; c += 2 * NW) {
        load(odd, c + NW);
        if constexpr (QUANT) take_codes(even, c);
        multiply(even);
        load(even, c + 2 * NW);
        if constexpr (QUANT) take_codes(odd, c + NW);
        multiply(odd);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) sums[wave][i * NS + j][lane] = acc[i][j];
    __syncthreads();

    auto finish = [&](auto bf16) {
        constexpr bool BF16 = decltype(bf16)::value;
        for (int s = wave; s < MT * NS; s += NW) {
            const int i = s / NS, j = s % NS, r = i * 16 + col16, col = col0 + j * 16 + 4 * kq;
            acc_t v = sums[0][s][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) v = v + sums[w][s][lane];
            if (r >= rows) continue;
            f32x4_t f;
            float token = 0.f;
            if constexpr (QUANT) {
                token = tokens[r];
            } else if constexpr (T == kInt8) {
                token = a.p_scale[row0 + r];
            }
            if constexpr (T == kInt8) f = dense_scaled(v, dense_channels(a.q_scale + static_cast<int64_t>(expert) * a.cols, col, a.cols), token);
            else f = v;
            if (T == kInt8 && rest) f = f32x4_t{0.f, 0.f, 0.f, 0.f};
            dense_store4<BF16>(a.y + (static_cast<int64_t>(row0) + r) * a.cols, col, a.cols, a.wide, f);
        }
    };
    if constexpr (T == kBf16) finish(std::true_type{});
    else if constexpr (T == kFp16) finish(std::false_type{});
    else if (a.bf16) finish(std::true_type{});
    else finish(std::false_type{});
}

template <dense_type T, dense_mode MODE, int MT, int NS, int U, int NW, bool QUANT = false> void launch_rows(const dense_product& p, hipStream_t s) {
    dense_args a = make_dense_args(p, false, false);
    a.n_blocks = static_cast<int>(ceil_div(p.cols, 16 * NS));
    a.m_blocks = static_cast<int>(dense_row_blocks(p, MODE, 16 * MT));
    if (QUANT) a.pitch_p = 2 * a.depth;
    dense_rows_kernel<T, MODE, MT, NS, U, NW, QUANT>
        <<<static_cast<unsigned>(a.n_blocks) * a.m_blocks, NW * 64, QUANT ? static_cast<unsigned>(p.rows * p.depth) : 0u, s>>>(a);
}

}  // namespace

}  // namespace plm
