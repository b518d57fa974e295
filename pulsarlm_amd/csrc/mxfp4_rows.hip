// MXFP4 products for few rows (one token to short prompts): y[M, N] = x[M, K] @ W^T, the gated block's
// two products with its activation, and the same with 4-bit x.
//
// A workgroup owns the rows (RB blocks of 16, one or two) by SG strips of 16 weight rows over all of K; its wavefronts take
// the K tiles round-robin, each holding all RB x SG accumulators of its own tiles, and their sums are added
// through LDS in wavefront order. The weight bytes bound it (they are read once, by one wavefront each,
// DW K tiles ahead in registers, nontemporal), so nothing is shared before the end and no barrier stands in
// the K loop. K is not split over workgroups: 16-row strips alone give N / 16 of them, and with DW tiles in
// flight per wavefront fewer than one workgroup to a CU already draw the memory's rate. x comes as:
// * staged: all of x in LDS (`staged` says where). Rows past M are not stored, so their lanes read row M - 1 again. With 4-bit x the lane that holds a block's 32
//   values quantizes them there: one launch, no scratch.
// * a ring of two K tiles per wavefront, filled with loads to LDS.
// * codes in the tile layout, straight to registers.
// The weights are the matrix instruction's A operand and x its B operand, so that a lane ends with four
// neighbouring columns of one row: 8-byte stores, and gate and up of a column in one lane.
// One token, us (TB/s of weights), 16-bit x: N 6144, K 4096 5.6 (2.4; 4.9 of the kernel itself); N 4096, K 12288 8.0
// (3.3); gate and up of 12288, K 4096 13.4 (4.0). A copy of 2 GiB makes 4.9-5.06 TB/s; the rest is the launch and the
// first loads' latency, some 2.5 us.
#include "mxfp4.hpp"

namespace plm {

namespace {

enum mx_x { kXStaged, kXStagedQuantize, kXRing, kXCodes };

struct rows_args {
    const uint16_t* x;
    mx_matrix xq, w0, w1;
    mx_output out;
    int m, k, ktiles, strips;
};

constexpr int kWaves = 8;
constexpr int rows_ahead(int sg) { return sg <= 2 ? 4 : 2; }

template <int XM, bool BF16, int RB, int SG, mx_epilogue EPI>
__global__ void __launch_bounds__(kWaves * 64) mx_rows_kernel(rows_args a) {
    constexpr int NW = kWaves;
    constexpr int DW = rows_ahead(SG);
    constexpr bool STAGED = XM == kXStaged || XM == kXStagedQuantize;
    constexpr int P = EPI == kMxPlain ? SG : SG / 2;                 // strips of one matrix
    constexpr int SLOT = RB * 4096;                                  // ring: a K tile of x
    constexpr int XL = RB * 4;                                       // its loads of 1 KiB
    constexpr int WL = 2 * SG;                                       // loads of a K tile's weights and scales
    static_assert(RB == 1 || (!STAGED && RB == 2), "staged x is one row block");
    extern __shared__ __attribute__((aligned(1024))) uint8_t mx_lds[];

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int col16 = lane & 15, kq = lane >> 4;
    const int strip0 = blockIdx.x * P;
    const int mine = min(P, a.strips - strip0);  // strips past N read zeros

    const int64_t w_at = static_cast<int64_t>(strip0) * a.ktiles * kSubTileBytes, s_at = static_cast<int64_t>(strip0 >> 2) * a.ktiles * 64;
    const uint32_t w_bytes = static_cast<uint32_t>(mine) * a.ktiles * kSubTileBytes, s_bytes = static_cast<uint32_t>(a.ktiles) * 256;
    __amdgpu_buffer_rsrc_t wr[2] = {make_rsrc(a.w0.codes + w_at, w_bytes), make_rsrc(a.w0.codes + w_at, w_bytes)};
    __amdgpu_buffer_rsrc_t sr[2] = {make_rsrc(a.w0.scale + s_at, s_bytes), make_rsrc(a.w0.scale + s_at, s_bytes)};
    if constexpr (EPI != kMxPlain) {
        wr[1] = make_rsrc(a.w1.codes + w_at, w_bytes);
        sr[1] = make_rsrc(a.w1.scale + s_at, s_bytes);
    }
    const int x_pitch = STAGED ? (a.ktiles + 3) / 4 * 1024 : 0;
    const __amdgpu_buffer_rsrc_t xr =
        XM == kXCodes ? make_rsrc(a.xq.codes, static_cast<uint32_t>((a.m + 15) / 16) * a.ktiles * kSubTileBytes)
                      : make_rsrc(a.x, static_cast<uint32_t>(a.m) * a.k * 2);
    const __amdgpu_buffer_rsrc_t xsr = XM == kXCodes ? make_rsrc(a.xq.scale, static_cast<uint32_t>(a.ktiles) * 256) : xr;

    struct batch {
        u32x4_t w[SG], x[XM == kXCodes ? RB : 1];
        uint32_t s[SG], xs[XM == kXCodes ? RB : 1];
    };
    auto load = [&](batch& b, int kt) {
        const bool in = kt < a.ktiles;  // a load's range check covers both its offsets
#pragma unroll
        for (int j = 0; j < SG; ++j) {
            const int side = j / P, jj = j % P;
            b.w[j] = buffer_load16_stream(wr[side], lane * 16, in ? (jj * a.ktiles + kt) * kSubTileBytes : kOOB);
            b.s[j] = __builtin_amdgcn_raw_buffer_load_b8(sr[side], lane * 4, in ? kt * 256 + ((strip0 + jj) & 3) : kOOB, 0);
        }
        if constexpr (XM == kXCodes) {
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                b.x[i] = buffer_load16(xr, lane * 16, in ? (i * a.ktiles + kt) * kSubTileBytes : kOOB);
                b.xs[i] = __builtin_amdgcn_raw_buffer_load_b8(xsr, lane * 4, in ? kt * 256 + i : kOOB, 0);
            }
        }
    };
    // Ring: a load's 64 lanes fill four rows of 256 bytes; the 16-byte columns are XOR-swizzled by row, so
    // that the 16 rows of a fragment read fall in different banks.
    uint8_t* ring = mx_lds + wave * 2 * SLOT;
    auto load_x = [&](int kt, int slot) {
        if constexpr (XM == kXRing) {
            const bool in = kt < a.ktiles;
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int r = 4 * i + (lane >> 4), c = (lane & 15) ^ (r & 15);
                const bool ok = in && kt * kTileK + 8 * c < a.k;  // rows past M are past the buffer's end
                buffer_load_lds16(xr, ring + slot * SLOT + i * 1024, ok ? r * a.k * 2 + c * 16 : kOOB, in ? kt * 256 : 0);
            }
        }
    };

    f32x4_t acc[RB][SG];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < SG; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    int slot = 0;
    auto multiply = [&](const batch& b, int kt) {
        const uint8_t* xt[RB];
        int swz = 0;
        if constexpr (STAGED) {
            const int r = min(col16, a.m - 1);
            xt[0] = mx_lds + r * x_pitch + kt * 256;
            swz = r & 15;
        } else if constexpr (XM == kXRing) {
#pragma unroll
            for (int i = 0; i < RB; ++i) xt[i] = ring + slot * SLOT + (16 * i + col16) * 256;
            swz = col16;
        }
        if constexpr (XM == kXCodes) {
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int j = 0; j < SG; ++j) acc[i][j] = mx_mfma<0, 0>(b.w[j], b.s[j], b.x[i], b.xs[i], acc[i][j]);
        } else if constexpr (XM == kXStagedQuantize) {
            float v[4][8];
            uint32_t top = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const u32x4_t f = *reinterpret_cast<const u32x4_t*>(xt[0] + (((4 * kq + q) ^ swz) << 4));
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    v[q][2 * h] = from_bits16<BF16>(f[h] & 0xffffu);
                    v[q][2 * h + 1] = from_bits16<BF16>(f[h] >> 16);
                    top = max(top, max(mx_magnitude(v[q][2 * h]), mx_magnitude(v[q][2 * h + 1])));
                }
            }
            const uint32_t s = mx_scale_byte(top);
            u32x4_t x;
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = mx_encode8(v[q], s);
#pragma unroll
            for (int j = 0; j < SG; ++j) acc[0][j] = mx_mfma<0, 0>(b.w[j], b.s[j], x, s, acc[0][j]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                u32x4_t x[RB];
#pragma unroll
                for (int i = 0; i < RB; ++i) x[i] = *reinterpret_cast<const u32x4_t*>(xt[i] + (((4 * kq + q) ^ swz) << 4));
#pragma unroll
                for (int j = 0; j < SG; ++j) {
                    const u32x4_t w = mx_decode<BF16>(b.w[j][q], mx_scale(b.s[j]));
#pragma unroll
                    for (int i = 0; i < RB; ++i) acc[i][j] = mfma16x16x32<BF16>(w, x[i], acc[i][j]);
                }
            }
        }
    };

    batch b[DW];
    if constexpr (STAGED) {
        // Row r's K group q (512 values, 1 KiB), swizzled within each K tile.
        const int groups = x_pitch / 1024;
        for (int i = wave; i < a.m * groups; i += NW) {
            const int r = i / groups, q = i % groups;
            const int c = (lane & 48) | ((lane & 15) ^ (r & 15)), at = q * 512 + c * 8;
            buffer_load_lds16(xr, mx_lds + i * 1024, at < a.k ? (r * a.k + at) * 2 : kOOB, 0);
        }
    }
#pragma unroll
    for (int d = 0; d < DW - 1; ++d) load(b[d], wave + d * NW);
    if constexpr (STAGED) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((DW - 1) * WL) : "memory");  // x, not the weights
    load_x(wave, 0);
    for (int kt = wave; kt < a.ktiles; kt += DW * NW) {
#pragma unroll
        for (int d = 0; d < DW; ++d) {
            const int cur = kt + d * NW;
            if (cur >= a.ktiles) break;
            load(b[(d + DW - 1) % DW], cur + (DW - 1) * NW);
            if constexpr (XM == kXRing) {
                // The other slot's reads are over; this slot's loads are older than this step's.
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                load_x(cur + NW, slot ^ 1);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(WL + XL) : "memory");
            }
            multiply(b[d], cur);
            slot ^= 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // requests past the last tile
    __syncthreads();

    // Sums over the wavefronts, in wavefront order.
    f32x4_t* red = reinterpret_cast<f32x4_t*>(mx_lds);
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < SG; ++j) red[((i * SG + j) * NW + wave) * 64 + lane] = acc[i][j];
    __syncthreads();
    auto total = [&](int i, int j, int ln) {
        const f32x4_t* p = red + (i * SG + j) * NW * 64 + ln;
        f32x4_t v = p[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) v = v + p[w * 64];
        return v;
    };
    constexpr int PER = EPI == kMxGatedCodes ? 1 : P;  // items of 64 lanes per row block
    for (int u = threadIdx.x; u < RB * PER * 64; u += NW * 64) {
        const int ln = u & 63, i = (u >> 6) / PER, p = (u >> 6) % PER;
        const int r = 16 * i + (ln & 15);
        if constexpr (EPI == kMxGatedCodes) {
            static_assert(P == 2 || EPI != kMxGatedCodes, "a block is two strips");
            const f32x4_t g[2] = {total(i, 0, ln), total(i, 1, ln)}, h[2] = {total(i, P, ln), total(i, P + 1, ln)};
            if (16 * i < a.m) mx_store_codes(a.out, i, strip0 >> 1, g, h);  // wave-uniform
        } else {
            const int col = (strip0 + p) * kTileN + 4 * (ln >> 4);
            const f32x4_t v = total(i, p, ln);
            if constexpr (EPI == kMxPlain) {
                if (r < a.m) mx_store_plain<BF16>(a.out, r, col, v);
            } else {
                const f32x4_t up = total(i, P + p, ln);
                if (r < a.m) {
                    mx_store_plain<BF16>(a.out, r, col, mx_gated4(v, up));
                    mx_store_gate_up(a.out, r, col, v, up);
                }
            }
        }
    }
}

// M <= 16 RB.
template <int XM, bool BF16, int RB, int SG, mx_epilogue EPI> void launch(const mx_product& p, hipStream_t s) {
    const mx_dims d = make_mx_dims(p.n, p.k);
    rows_args a{};
    a.x = p.x16;
    a.xq = p.xq;
    a.w0 = p.w0;
    a.w1 = p.w1;
    a.out = p.out;
    a.m = static_cast<int>(p.m);
    a.k = static_cast<int>(p.k);
    a.ktiles = static_cast<int>(d.ktiles);
    a.strips = static_cast<int>(d.strips);
    constexpr int NW = kWaves;
    int64_t loop = 0;  // bytes of LDS in the K loop
    if (XM == kXStaged || XM == kXStagedQuantize) loop = p.m * ceil_div(d.ktiles, 4) * 1024;
    if (XM == kXRing) loop = int64_t{NW} * 2 * RB * 4096;
    const int64_t lds = std::max<int64_t>(loop, int64_t{RB} * SG * NW * 1024);
    constexpr int P = EPI == kMxPlain ? SG : SG / 2;
    const int64_t grid = ceil_div(d.strips, P);
    mx_rows_kernel<XM, BF16, RB, SG, EPI><<<static_cast<unsigned>(grid), NW * 64, static_cast<size_t>(lds), s>>>(a);
}

// Strips of a matrix in a workgroup: as few as fill the GPU in one round, since more leave fewer workgroups to
// draw on the memory, and fewer bring x once more each. One / two / four, us at M = 1 and 16: N 2048, K 2048
// 3.3 / 4.0 / 4.6 and 4.2 / 4.8 / 5.7; N 4096, K 12288 8.2 / 8.8 / 14.1 and 11.7 / 13.6 / 17.2; N 6144, K 4096
// 5.9 / 5.6 / 6.8 and 8.7 / 6.8 / 7.8; N 24576, K 4096 13.9 / 13.1 / 12.8 and 20.9 / 16.2 / 15.0.
template <int XM, bool BF16, int RB> void launch_sg(const mx_product& p, hipStream_t s) {
    const int64_t strips = ceil_div(p.n, kTileN), cus = cu_count();
    if (p.epilogue == kMxPlain) {
        if (strips <= cus) launch<XM, BF16, RB, 1, kMxPlain>(p, s);
        else if (strips <= 2 * cus) launch<XM, BF16, RB, 2, kMxPlain>(p, s);
        else launch<XM, BF16, RB, 4, kMxPlain>(p, s);
    }
    if constexpr (XM == kXCodes || XM == kXStagedQuantize) {
        if (p.epilogue == kMxGatedCodes) launch<XM, BF16, RB, 4, kMxGatedCodes>(p, s);  // a block is two strips of either
    } else if (p.epilogue == kMxGated) {
        if (strips <= cus) launch<XM, BF16, RB, 2, kMxGated>(p, s);
        else launch<XM, BF16, RB, 4, kMxGated>(p, s);
    }
}

int64_t all_strips(const mx_product& p) { return ceil_div(p.n, kTileN) * (p.epilogue == kMxPlain ? 1 : 2); }

// x in LDS: up to 64 KiB, so that two workgroups fit a CU; up to 128 KiB where one does, if x is quantized there (a
// launch less) or has at most 8 rows (the ring takes all 16). 128 / 64 KiB, us, quantized: M = 12, N 6144, K 4096
// 7.6 / 8.5, N 2048 6.5 / 7.2, but M = 16, N 24576 17.7 / 16.7; 16-bit: M = 5, N 4096, K 12288 9.2 / 10.8, but M = 12,
// N 2048, K 4096 5.3 / 4.9 and N 24576 16.4 / 14.5.
bool staged(const mx_product& p, bool quantize_x) {
    const bool more = all_strips(p) <= 2 * cu_count() && (quantize_x || p.m <= 8);
    return p.m <= 16 && p.m * ceil_div(p.k, 512) * 1024 <= (more ? 128 : 64) * 1024;
}

template <bool BF16> void launch_typed(const mx_product& p, bool quantize_x, hipStream_t s) {
    if (quantize_x) return launch_sg<kXStagedQuantize, BF16, 1>(p, s);
    if (p.xq.codes != nullptr) {
        if (p.m <= 16) launch_sg<kXCodes, BF16, 1>(p, s);
        else launch_sg<kXCodes, BF16, 2>(p, s);
    } else if (staged(p, false)) launch_sg<kXStaged, BF16, 1>(p, s);
    else if (p.m <= 16) launch_sg<kXRing, BF16, 1>(p, s);
    else launch_sg<kXRing, BF16, 2>(p, s);
}

}  // namespace

// Rows kernel or tiles, us. 16-bit x, M = 32: N 2048, K 2048 4.8 against 6.1; N 6144, K 4096 8.7, 10.3; N 4096, K 12288
// 16.3, 21.9; but N 24576, K 4096 20.1, 18.0. M = 48 (four row blocks): 6.5 against 6.1; 12, 10.0; 26.7, 21.2. With
// x as codes, M = 32: 7.1, 7.6; 9.8, 10.7; 14.7, 19.0; 18.1, 16.2 (M = 16 16.5, 15.1); M = 64: 8.9, 8.3; 12.3, 11.7;
// K 12288 18.6, 17.1 (the tiles' K split).
bool launch_mx_rows(const mx_product& p, bool quantize_x, hipStream_t s) {
    const int64_t strips = all_strips(p), cus = cu_count();
    const bool codes = p.xq.codes != nullptr;
    if (quantize_x) {
        if (!staged(p, true)) return false;
    } else if (strips > 4 * cus) {
        if (p.m > (codes ? 8 : 16)) return false;
    } else if (p.m > 32) {
        return false;
    }
    if (p.bf16) launch_typed<true>(p, quantize_x, s);
    else launch_typed<false>(p, quantize_x, s);
    return true;
}

}  // namespace plm
