// Input gradients through MXFP4 weights: dx[M, K] = dy[M, N] @ W, and the gated block's, whose dy is
// [d gate | d up] against the two weights one after the other (the sum runs on from one into the other).
// The weights themselves are codes and have no gradient.
//
// The sum runs over N here, along which the tile layout is not contiguous and every row has its own block
// scales, so the scaled matrix instruction cannot take the codes. A workgroup decodes its 64 x 256 slice of
// W into LDS in 16 bits instead (exact in bf16), 32 codes to a lane under one scale, and the fragments are
// read back with the transposing LDS read: 16 lanes fetch four rows of 16 columns and receive one column each.
// * Tile (2 MT 16) x 256 columns, steps of 64 along N. dy and the codes of the step after next are requested
//   to registers and go, the codes decoded, into the other of two LDS slots a step ahead. (dy by loads to
//   LDS would be waited for in full before every transposing read: the compiler cannot tell them apart.)
// * One barrier a step, before the matrix instructions of its second half, as in the forward kernel
//   (mxfp4_tiles.hpp): their operands are in registers, and the next step's first half is read meanwhile.
// * Few tiles: the steps are split over workgroups, whose fp32 sums a second kernel adds in split order.
// * What bounds it: the way of W through LDS. At M = 2000, N = K = 4096 the matrix units are busy 42% of the cycles and LDS
//   48% (60% and 45% with tiles of 256 rows); without W's decoding and writes, its loads kept, a call takes 61 us of 73,
//   without dy's writes 66. M = 4096,
//   N 24576, K 4096: 627 us, 1314 TFLOP/s; M = 2000 70 us, 960; the gated block's M = 4096, intermediate 12288: 740 us,
//   150 of them the factors' kernel, which moves 704 MB at 4.6 TB/s.
#include "mxfp4.hpp"

namespace plm {

namespace {

constexpr int kGradStep = 64;    // N of a step
constexpr int kGradCols = 256;   // columns of a workgroup

struct grad_args {
    const uint16_t* dy;  // [M][pitch], zero past N up to a whole step
    mx_matrix w0, w1;
    uint16_t* dx;
    float* partial;  // [splits][M][K]
    int64_t pitch;
    int m, k, ktiles, strips;
    int side_steps, steps, split_steps, splits;
    int m_blocks, n_blocks;
    const float* row_scale;  // fp16 factors: what row m's sums are to be multiplied by; or null
};

typedef __attribute__((ext_vector_type(4))) short tr_t;

template <bool BF16, int MT>
__global__ void __launch_bounds__(512) mx_grad_kernel(grad_args a) {
    constexpr int WN = 4, NS = 4, NW = 8, BM = 2 * MT * 16;
    constexpr int XC = BM / 8, XPW = XC / NW;  // 1 KiB chunks of dy: 8 rows of 128 bytes
    constexpr int XS = BM * 128, WS = kGradStep * kGradCols * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * XS + 2 * WS];
    constexpr int S0 = 2 * XS;  // W's slots

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int col16 = lane & 15, kq = lane >> 4;

    // Workgroups go round the 8 XCDs by id; each takes a run of the tiles, row block fastest (they share W).
    const int tiles = a.m_blocks * a.n_blocks, xcd = blockIdx.x & 7;
    const int lin = xcd * (tiles >> 3) + min(xcd, tiles & 7) + (blockIdx.x >> 3);
    const int row0 = lin % a.m_blocks * BM, nb = lin / a.m_blocks;
    const int rows = min(BM, a.m - row0);
    const int split = blockIdx.y;
    const int lo = split * a.split_steps, hi = min(lo + a.split_steps, a.steps);

    const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.dy + row0 * a.pitch, static_cast<uint32_t>(rows * a.pitch * 2));
    struct step_data {
        u32x4_t x[XPW], c;
        uint32_t s;
    };
    // A load's range check covers both its offsets (checked on the GPU): past the end the wave-uniform one is kOOB,
    // and the lanes' own never change.
    const int x_from = static_cast<int>((lane >> 3) * a.pitch * 2) + (lane & 7) * 16;
    auto load_x = [&](step_data& b, int i, int s) {
        const int at = s * 128 + 8 * (wave * XPW + i) * static_cast<int>(a.pitch * 2);  // rows past the last are past the buffer's end
        b.x[i] = buffer_load16(xr, x_from, s < hi ? at : kOOB);
    };
    const int x_to = wave * XPW * 1024 + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);  // 16-byte columns swizzled by row
    auto write_x = [&](const step_data& b, int i, int slot) {
        *reinterpret_cast<u32x4_t*>(lds + slot * XS + x_to + i * 1024) = b.x[i];
    };

    // Wavefront w decodes one tile of a step: strip w / 2, K tile w % 2 (the second may lie past K).
    const int kt = 2 * nb + (wave & 1);
    auto load_w = [&](step_data& b, int s) {
        const int side = s >= a.side_steps ? 1 : 0, strip = 4 * (s - side * a.side_steps) + (wave >> 1);
        const uint8_t* base = side ? a.w1.codes : a.w0.codes;
        const uint32_t* sbase = side ? a.w1.scale : a.w0.scale;
        const bool in = s < hi && strip < a.strips && kt < a.ktiles;
        const int64_t at = in ? strip : 0, t = in ? kt : 0;
        b.c = buffer_load16(make_rsrc(base + (at * a.ktiles + t) * kSubTileBytes, kSubTileBytes), lane * 16, in ? 0 : kOOB);
        b.s = buffer_load_u32(make_rsrc(sbase + ((at >> 2) * a.ktiles + t) * 64, 256u), lane * 4, in ? 0 : kOOB);
    };
    // LDS row n (512 bytes): its 32-byte pieces are XOR-swizzled by f(n) = n % 4 + 4 ((n / 4 + n / 8) % 2),
    // which sets apart both the eight rows that one write covers and the rows of one transposing read.
    const int w_to = S0 + ((wave >> 1) * 16 + col16) * 512 +
                     ((((wave & 1) * 8 + 2 * kq) ^ ((col16 & 3) | ((((col16 >> 2) ^ (col16 >> 3)) & 1) << 2))) << 5);
    auto write_w = [&](const step_data& b, int q, int slot) {
        const float s = mx_scale(b.s >> (8 * (wave >> 1)) & 0xffu);
        *reinterpret_cast<u32x4_t*>(lds + slot * WS + (w_to ^ ((q >> 1) << 5)) + (q & 1) * 16) = mx_decode<BF16>(b.c[q], s);
    };

    u32x4_t x[MT], w[2][NS];  // fragments; x's are read again for the next half right after their use
    const int x_at = wm * MT * 2048 + col16 * 128 + ((kq ^ (col16 & 7)) << 4);
    const int w_at = S0 + (8 * kq + (col16 >> 2)) * 512 + (((wn * NS) ^ ((col16 >> 2) | ((kq & 1) << 2))) << 5) + (col16 & 3) * 8;
    auto read_x = [&](int i, int slot, int t) { x[i] = *reinterpret_cast<const u32x4_t*>(lds + slot * XS + (x_at ^ (t << 6)) + i * 2048); };
    auto read_w = [&](u32x4_t (&w)[NS], int j, int slot, int t) {
        const int at = slot * WS + w_at;
        const tr_t lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr_t*)(lds + (at ^ (j << 5)) + t * 16384));
        const tr_t hi4 =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr_t*)(lds + (at ^ ((j ^ 4) << 5)) + t * 16384 + 2048));
        const u32x2_t l = __builtin_bit_cast(u32x2_t, lo4), h = __builtin_bit_cast(u32x2_t, hi4);
        w[j] = u32x4_t{l[0], l[1], h[0], h[1]};
    };

    f32x4_t acc[MT][NS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    step_data b;
#pragma unroll
    for (int i = 0; i < XPW; ++i) load_x(b, i, lo);
    load_w(b, lo);
#pragma unroll
    for (int i = 0; i < XPW; ++i) write_x(b, i, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) write_w(b, q, 0);
#pragma unroll
    for (int i = 0; i < XPW; ++i) load_x(b, i, lo + 1);
    load_w(b, lo + 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) read_x(i, 0, 0);
#pragma unroll
    for (int j = 0; j < NS; ++j) read_w(w[0], j, 0, 0);
    int slot = 0;
    for (int s = lo; s < hi; ++s) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            // The other slot is filled over the first rows of matrix instructions, and the data of the step
            // after requested over the last ones into the same registers.
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q * MT / 8 == i) write_w(b, q, slot ^ 1);
#pragma unroll
            for (int q = 0; q < XPW; ++q) {
                if (q * MT / 8 == i) write_x(b, q, slot ^ 1);
                if (MT / 2 + q * MT / 8 == i) load_x(b, q, s + 2);
            }
            if (i == MT - 1) load_w(b, s + 2);
#pragma unroll
            for (int j = i * NS / MT; j < (i + 1) * NS / MT; ++j) read_w(w[1], j, slot, 1);
#pragma unroll
            for (int j = 0; j < NS; ++j) acc[i][j] = mfma16x16x32<BF16>(w[0][j], x[i], acc[i][j]);
            read_x(i, slot, 1);
            __builtin_amdgcn_sched_barrier(0);  // the reads stay among the matrix instructions, half a step ahead
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        slot ^= 1;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int j = i * NS / MT; j < (i + 1) * NS / MT; ++j) read_w(w[0], j, slot, 0);
#pragma unroll
            for (int j = 0; j < NS; ++j) acc[i][j] = mfma16x16x32<BF16>(w[1][j], x[i], acc[i][j]);
            read_x(i, slot, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int r = (wm * MT + i) * 16 + col16;
        if (r >= rows) continue;
        const int64_t row = row0 + r;
        float scale = 1.f;
        if constexpr (!BF16)
            if (a.row_scale != nullptr) scale = a.row_scale[row];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int col = nb * kGradCols + (wn * NS + j) * 16 + 4 * kq;  // K is a multiple of 32
            if (col >= a.k) continue;
            f32x4_t v = acc[i][j];
            if constexpr (!BF16) v = f32x4_t{v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale};
            if (a.splits > 1) *reinterpret_cast<f32x4_t*>(a.partial + (static_cast<int64_t>(split) * a.m + row) * a.k + col) = v;
            else *reinterpret_cast<uint2*>(a.dx + row * a.k + col) = make_uint2(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]));
        }
    }
}

// Sums over the splits, four values a thread.
template <bool BF16>
__global__ void __launch_bounds__(256) mx_combine_kernel(const f32x4_t* __restrict__ partial, int64_t quads, int splits,
                                                              uint2* __restrict__ dx) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= quads) return;
    f32x4_t v = partial[i];
    for (int s = 1; s < splits; ++s) v = v + partial[s * quads + i];
    dx[i] = make_uint2(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]));
}

// Eight values of a row from column col on, zeros past n. WIDE: rows of whole 16-byte pieces.
template <bool WIDE> __device__ __forceinline__ void row_load8(const uint16_t* p, int col, int n, uint32_t (&v)[8]) {
    if (WIDE && col < n) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = w[i] & 0xffffu, v[2 * i + 1] = w[i] >> 16;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < n ? p[col + i] : 0u;
    }
}
template <bool WIDE> __device__ __forceinline__ void row_load8(const float* p, int col, int n, float (&v)[8]) {
    if (WIDE && col < n) {
        const f32x4_t a = reinterpret_cast<const f32x4_t*>(p + col)[0], b = reinterpret_cast<const f32x4_t*>(p + col)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < n ? p[col + i] : 0.f;
    }
}
__device__ __forceinline__ void row_store8(uint16_t* p, const uint32_t (&v)[8]) {
    *reinterpret_cast<u32x4_t*>(p) = u32x4_t{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
}
// Eight columns of one row's factors in fp32: with s = sigmoid(g), d gate = dh u s (1 + g (1 - s)), d up = dh g s.
template <bool BF16, bool WIDE>
__device__ __forceinline__ void row_factors8(const uint16_t* dh, const float* gate_up, int col, int n, float (&dg)[8], float (&du)[8]) {
    uint32_t d[8];
    float g[8], u[8];
    row_load8<WIDE>(dh, col, n, d);
    row_load8<WIDE>(gate_up, col, n, g);
    row_load8<WIDE>(gate_up + n, col, n, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = from_bits16<BF16>(d[i]), s = mx_sigmoid(g[i]);
        dg[i] = f * u[i] * s * (1.f + g[i] * (1.f - s));
        du[i] = f * g[i] * s;
    }
}

// The gated block's [d gate | d up], each padded with zeros to a whole step, rounded to the matrix
// instruction's 16 bits. !GATED: a copy of dy padded so. Eight values a thread.
// bf16 holds every factor that fp32 does, to 8 bits: dx is off by 2.3e-3 of its size against float64 with them and by 1.7e-3
// with factors in fp32 (its own rounding). Two bf16 terms a factor would give that, but are the products of twice the
// rows: N 9728, K 2080 57 us at M = 1001 and 96 at 2002; N 24576, K 4096 620 at M = 4096 and 1320 at 8192.
template <bool BF16, bool GATED, bool WIDE>
__global__ void __launch_bounds__(256) mx_grad_rows_kernel(const uint16_t* __restrict__ dy, const float* __restrict__ gate_up,
                                                           int64_t m, int n, int padded, uint16_t* __restrict__ out) {
    const int per_row = padded / 8;
    const int64_t total = m * per_row, step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; c < total; c += step) {
        const int64_t row = c / per_row;
        const int col = static_cast<int>(c % per_row) * 8;
        uint32_t d[8];
        if constexpr (!GATED) {
            row_load8<WIDE>(dy + row * n, col, n, d);
            row_store8(out + row * padded + col, d);
        } else {
            float dg[8], du[8];
            row_factors8<BF16, WIDE>(dy + row * n, gate_up + row * 2 * n, col, n, dg, du);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = to_bits16<BF16>(dg[i]);
            row_store8(out + row * 2 * padded + col, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = to_bits16<BF16>(du[i]);
            row_store8(out + row * 2 * padded + padded + col, d);
        }
    }
}

// The factors in fp16. They pass its range at both ends where dx does not (dh of 100 by u of 1000; dh of 1e-5 by u of
// 1e-3), so each row is brought by a power of two to a largest factor in [2^14, 2^15), and its sums are multiplied by
// the inverse, row_scale, when they leave. Infinity and NaN do not count for that: they come through as such.
// A workgroup a row. The first kHeld pieces of eight columns a thread wait in registers for the row's largest; what is
// past them (N over 12288) is computed again, its reads mostly from the L2. M = 4096, N 12288, over and over on the
// same inputs: 127 us, the bf16 kernel 118.
constexpr int kRowThreads = 512, kHeld = 3;
template <bool WIDE>
__global__ void __launch_bounds__(kRowThreads) mx_grad_rows_fp16_kernel(const uint16_t* __restrict__ dh, const float* __restrict__ gate_up,
                                                                        int64_t m, int n, int padded, uint16_t* __restrict__ out,
                                                                        float* __restrict__ row_scale) {
    constexpr int kStep = kRowThreads * 8;
    __shared__ uint32_t tops[kRowThreads / 64];
    for (int64_t row = blockIdx.x; row < m; row += gridDim.x) {
        const uint16_t* d = dh + row * n;
        const float* gu = gate_up + row * 2 * n;
        uint16_t* to = out + row * 2 * padded;
        uint32_t top = 0;
        auto count = [&](const float (&dg)[8], const float (&du)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t a = mx_magnitude(dg[i]), b = mx_magnitude(du[i]);
                top = max(top, max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u));
            }
        };
        const int first = threadIdx.x * 8;
        float hg[kHeld][8], hu[kHeld][8];
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (first + h * kStep < padded) row_factors8<false, WIDE>(d, gu, first + h * kStep, n, hg[h], hu[h]);
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (first + h * kStep < padded) count(hg[h], hu[h]);
        float dg[8], du[8];
        for (int col = first + kHeld * kStep; col < n; col += kStep) {
            row_factors8<false, WIDE>(d, gu, col, n, dg, du);
            count(dg, du);
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), s)));
        __syncthreads();  // the last row's are read
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kRowThreads / 64; ++w) top = max(top, tops[w]);
        // 2^(141 - e) brings 2^(e - 127) to 2^14. Rows below 2^-86 (zeros among them) take that one's: |W| <= 65504 and N <=
        // 2^19, so their dx is zero in fp16 whatever the factors are.
        const uint32_t e = max(top >> 23, 41u);
        const float up = __uint_as_float((127u + 141u - e) << 23);
        if (threadIdx.x == 0) row_scale[row] = __uint_as_float((e - 14u) << 23);
        auto store = [&](int col, const float (&dg)[8], const float (&du)[8]) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_bits16<false>(dg[i] * up);
            row_store8(to + col, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_bits16<false>(du[i] * up);
            row_store8(to + padded + col, v);
        };
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (first + h * kStep < padded) store(first + h * kStep, hg[h], hu[h]);
        for (int col = first + kHeld * kStep; col < padded; col += kStep) {
            row_factors8<false, WIDE>(d, gu, col, n, dg, du);
            store(col, dg, du);
        }
    }
}

struct grad_plan {
    int mt;
    int64_t m_blocks, n_blocks, steps, splits, split_steps;
};
// The tile height and the split with the least estimated time (us): steps of the busiest CU, each 0.76 / 1.0 /
// 1.55 us at 64 / 128 / 256 rows, and the fp32 sums, written and read by a kernel more at 5.5 TB/s (they mostly stay in
// the caches). Measured against the best of 24 forced choices (N 4096, K 4096): M = 48 16.6 of 16.6 us, M = 333
// 29.7 of 29.7, M = 1000 47.4 of 47.4, M = 2000 72 of 72; 64, 256 and 256 rows unsplit take 20, 61 and 100 us there.
grad_plan make_grad_plan(int64_t m, int64_t k, int64_t steps) {
    grad_plan best{};
    double least = 1e300;
    const int64_t cus = cu_count();
    for (int mt = 2; mt <= 8; mt *= 2) {
        grad_plan p{};
        p.mt = mt;
        p.m_blocks = ceil_div(m, 32 * mt);
        p.n_blocks = ceil_div(k, kGradCols);
        p.steps = steps;
        const double step = mt == 2 ? 0.76 : (mt == 4 ? 1.0 : 1.55);
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(steps / 8, 2 * cus / (p.m_blocks * p.n_blocks)));
        for (int64_t splits = 1; splits <= most; ++splits) {
            p.split_steps = ceil_div(steps, splits);
            p.splits = ceil_div(steps, p.split_steps);
            const int64_t rounds = ceil_div(p.m_blocks * p.n_blocks * p.splits, cus);
            const double t = rounds * (p.split_steps * step + 4.) + (p.splits > 1 ? 2. + p.splits * m * k * 8 / 5.5e6 : 0.);
            if (t < least) least = t, best = p;
        }
    }
    return best;
}

int64_t padded_n(int64_t n) { return round_up(n, kGradStep); }
bool copies_dy(int64_t n, bool dy_aligned) { return n % kGradStep != 0 || !dy_aligned; }

// Workspace: [rows in 16 bits, where dy is not read in place][gated: a scale a row][fp32 partial sums].
int64_t rows_bytes(int64_t m, int64_t n, int sides) { return round_up(m * sides * padded_n(n) * 2, 256); }
int64_t row_scale_bytes(int64_t m, int sides) { return sides == 2 ? round_up(m * 4, 256) : 0; }
int64_t grad_bytes(int64_t m, int64_t n, int64_t k, int sides, bool rows) {
    const grad_plan p = make_grad_plan(m, k, sides * padded_n(n) / kGradStep);
    return (rows ? rows_bytes(m, n, sides) + row_scale_bytes(m, sides) : 0) + (p.splits > 1 ? p.splits * m * k * 4 : 0);
}

template <bool BF16, bool GATED>
void launch_rows(const void* dy, const void* gate_up, int64_t m, int64_t n, uint16_t* out, float* row_scale, hipStream_t s) {
    const int64_t padded = padded_n(n), most = int64_t{64} * cu_count();
    const int nn = static_cast<int>(n), pn = static_cast<int>(padded);
    const auto* d = static_cast<const uint16_t*>(dy);
    const auto* g = static_cast<const float*>(gate_up);
    const bool wide = n % 8 == 0 && aligned(dy, 16) && aligned(gate_up, 16);
    if constexpr (GATED && !BF16) {
        const unsigned grid = static_cast<unsigned>(std::min(m, most));
        if (wide) mx_grad_rows_fp16_kernel<true><<<grid, kRowThreads, 0, s>>>(d, g, m, nn, pn, out, row_scale);
        else mx_grad_rows_fp16_kernel<false><<<grid, kRowThreads, 0, s>>>(d, g, m, nn, pn, out, row_scale);
    } else {
        const unsigned grid = static_cast<unsigned>(std::min(ceil_div(m * padded / 8, 256), most));
        if (wide) mx_grad_rows_kernel<BF16, GATED, true><<<grid, 256, 0, s>>>(d, g, m, nn, pn, out);
        else mx_grad_rows_kernel<BF16, GATED, false><<<grid, 256, 0, s>>>(d, g, m, nn, pn, out);
    }
}

template <bool BF16>
int run(const char* op, bool gated, const void* dy, const void* gate_up, const mx_matrix& w0, const mx_matrix& w1, int64_t m, int64_t n,
        int64_t k, void* dx, void* workspace, hipStream_t s) {
    const int sides = gated ? 2 : 1;
    const mx_dims d = make_mx_dims(n, k);
    grad_args a{};
    auto* rows = static_cast<uint16_t*>(workspace);
    a.dy = static_cast<const uint16_t*>(dy);
    a.pitch = n;
    auto* sums = static_cast<uint8_t*>(workspace);
    if (gated || copies_dy(n, aligned(dy, 16))) {
        auto* row_scale = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + rows_bytes(m, n, sides));
        if (gated) launch_rows<BF16, true>(dy, gate_up, m, n, rows, row_scale, s);
        else launch_rows<BF16, false>(dy, nullptr, m, n, rows, nullptr, s);
        if (gated && !BF16) a.row_scale = row_scale;
        PLM_HIP_LAUNCH_CHECK(op);
        a.dy = rows;
        a.pitch = sides * padded_n(n);
        sums += rows_bytes(m, n, sides) + row_scale_bytes(m, sides);
    }
    a.side_steps = static_cast<int>(padded_n(n) / kGradStep);
    const grad_plan p = make_grad_plan(m, k, int64_t{sides} * a.side_steps);
    a.w0 = w0;
    a.w1 = w1;
    a.dx = static_cast<uint16_t*>(dx);
    a.partial = reinterpret_cast<float*>(sums);
    a.m = static_cast<int>(m);
    a.k = static_cast<int>(k);
    a.ktiles = static_cast<int>(d.ktiles);
    a.strips = static_cast<int>(d.strips);
    a.steps = static_cast<int>(p.steps);
    a.splits = static_cast<int>(p.splits);
    a.split_steps = static_cast<int>(p.split_steps);
    a.m_blocks = static_cast<int>(p.m_blocks);
    a.n_blocks = static_cast<int>(p.n_blocks);
    const dim3 grid(static_cast<unsigned>(p.m_blocks * p.n_blocks), static_cast<unsigned>(p.splits));
    if (p.mt == 2) mx_grad_kernel<BF16, 2><<<grid, 512, 0, s>>>(a);
    else if (p.mt == 4) mx_grad_kernel<BF16, 4><<<grid, 512, 0, s>>>(a);
    else mx_grad_kernel<BF16, 8><<<grid, 512, 0, s>>>(a);
    PLM_HIP_LAUNCH_CHECK(op);
    if (p.splits > 1) {
        launch_mx_combine(BF16, a.partial, m * k, a.splits, a.dx, s);
        PLM_HIP_LAUNCH_CHECK(op);
    }
    return PLM_OK;
}

}  // namespace

void launch_mx_combine(bool bf16, const float* partial, int64_t count, int splits, uint16_t* out, hipStream_t s) {
    const int64_t quads = count / 4;
    const unsigned grid = static_cast<unsigned>(ceil_div(quads, 256));
    const auto* p = reinterpret_cast<const f32x4_t*>(partial);
    auto* o = reinterpret_cast<uint2*>(out);
    if (bf16) mx_combine_kernel<true><<<grid, 256, 0, s>>>(p, quads, splits, o);
    else mx_combine_kernel<false><<<grid, 256, 0, s>>>(p, quads, splits, o);
}

int64_t mx_grad_bytes(int64_t m, int64_t n, int64_t k, bool gated, bool dy_aligned) {
    return grad_bytes(m, n, k, gated ? 2 : 1, gated || copies_dy(n, dy_aligned));
}

int launch_mx_grad(const char* op, bool gated, bool bf16, const void* dy, const void* gate_up, const mx_matrix& w0, const mx_matrix& w1,
                   int64_t m, int64_t n, int64_t k, void* dx, void* workspace, hipStream_t s) {
    return bf16 ? run<true>(op, gated, dy, gate_up, w0, w1, m, n, k, dx, workspace, s)
                : run<false>(op, gated, dy, gate_up, w0, w1, m, n, k, dx, workspace, s);
}

}  // namespace plm
