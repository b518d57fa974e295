// MXFP4 products for many rows: y[M, N] = x[M, K] @ W^T on the matrix cores, with 16-bit x (the weights
// converted in registers, W4A16) or x quantized to the same format (raw codes and scales to the scaled
// matrix instruction, W4A4), plain or with the gated block's activation as the epilogue.
//
// * A workgroup owns BM = WM MT 16 rows by BS = WN NS strips; its WM x WN wavefronts own MT x NS products of
//   16 x 16 each. The large W4A4 tile is 256 x 256 with four wavefronts of 128 x 128: each operand byte
//   read from LDS then feeds eight matrix instructions, which is what LDS bandwidth needs (the operands of
//   one K tile take 64 KiB of reads in 1024 cycles of matrix instructions). W4A16 has four times the cycles
//   for 2.5 times the bytes: eight wavefronts of 128 x 64, whose sums fit the vector registers.
// * The operands of a K tile (128) go from memory straight into one of S LDS stages. One barrier a K tile
//   stands before its last slice's matrix instructions, whose operands are in registers by then: past it
//   every wavefront has read the stage, which the loads of K tile kt + S may overwrite, and K tile kt + 1 has
//   landed, so that its first slice is read while those instructions run. W4A4 has one slice a K tile,
//   W4A16 four of 32 K values.
// * The weights are the A operand and x the B operand: a lane ends with four neighbouring columns of a row.
// * Gated: local strips 2 p and 2 p + 1 are gate and up of one 16-column slice, so that both halves of an
//   output are in one lane.
#pragma once

#include <type_traits>

#include "mxfp4.hpp"

namespace plm {

namespace {

struct tile_args {
    const uint16_t* x;
    mx_matrix xq, w0, w1;
    mx_output out;
    int m, k, ktiles, kgroups, strips;
    int m_blocks, n_blocks, band;  // band: row blocks of an XCD's patch of work tiles
};

template <bool A4, bool BF16, mx_epilogue EPI, int WM, int WN, int MT, int NS, int S>
__global__ void __launch_bounds__(WM * WN * 64) mx_tile_kernel(tile_args a) {
    constexpr int NW = WM * WN;
    constexpr int BM = WM * MT * 16, BS = WN * NS;
    constexpr int XC = A4 ? WM * MT : WM * MT * 4;  // 1 KiB chunks of x in a stage
    constexpr int STAGE = (XC + BS) * 1024;
    constexpr int LOADS = (XC + BS) / NW;
    constexpr int SLICES = A4 ? 1 : 4;
    static_assert(XC % NW == 0 && BS % NW == 0, "every wavefront loads as many chunks");
    static_assert(EPI == kMxPlain || NS % 2 == 0, "gate and up in one wavefront");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S * STAGE];

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int col16 = lane & 15, kq = lane >> 4;

    // Workgroups go round the 8 XCDs by id: each takes one run of the work tiles, which are ordered in
    // bands of `band` row blocks, row block fastest, so that an XCD's L2 holds what its tiles share.
    const int tiles = a.m_blocks * a.n_blocks, xcd = blockIdx.x & 7;
    const int lin = xcd * (tiles >> 3) + min(xcd, tiles & 7) + (blockIdx.x >> 3);
    const int first = lin / (a.band * a.n_blocks) * a.band;
    const int band_rows = min(a.band, a.m_blocks - first), in_band = lin - first * a.n_blocks;
    const int nb = in_band / band_rows, row0 = (first + in_band % band_rows) * BM;
    const int rows = min(BM, a.m - row0);

    // Local strip s: strip nb BS + s, or slice nb BS / 2 + s / 2 of the gate (s even) or up weight.
    constexpr int SIDES = EPI == kMxPlain ? 1 : 2;
    const int strip0 = nb * (BS / SIDES);
    const int mine = min(BS / SIDES, a.strips - strip0);
    const int64_t w_at = static_cast<int64_t>(strip0) * a.ktiles * kSubTileBytes, s_at = static_cast<int64_t>(strip0) * a.kgroups * 64;
    const uint32_t w_bytes = static_cast<uint32_t>(mine) * a.ktiles * kSubTileBytes, s_bytes = static_cast<uint32_t>(mine) * a.kgroups * 256;
    __amdgpu_buffer_rsrc_t wr[2], sr[2];
    wr[0] = make_rsrc(a.w0.codes + w_at, w_bytes);
    sr[0] = make_rsrc(a.w0.scale + s_at, s_bytes);
    wr[1] = SIDES == 2 ? make_rsrc(a.w1.codes + w_at, w_bytes) : wr[0];
    sr[1] = SIDES == 2 ? make_rsrc(a.w1.scale + s_at, s_bytes) : sr[0];
    const int x_strips = (rows + 15) / 16;
    const __amdgpu_buffer_rsrc_t xr =
        A4 ? make_rsrc(a.xq.codes + static_cast<int64_t>(row0 / 16) * a.ktiles * kSubTileBytes, static_cast<uint32_t>(x_strips) * a.ktiles * kSubTileBytes)
           : make_rsrc(a.x + static_cast<int64_t>(row0) * a.k, static_cast<uint32_t>(rows) * a.k * 2);
    const __amdgpu_buffer_rsrc_t xsr =
        make_rsrc(a.xq.scale + static_cast<int64_t>(row0 / 16) * a.kgroups * 64, A4 ? static_cast<uint32_t>(x_strips) * a.kgroups * 256 : 0u);

    // Chunk c of a stage: x's first (codes: strip c; 16-bit: rows 4 c .. 4 c + 3, their 16-byte columns
    // XOR-swizzled by row), then the weight strips'. Past the end of either, zeros.
    auto issue = [&](int kt, int slot) {
        const bool in = kt < a.ktiles;
        const int past = in ? 0 : kOOB, off = in ? kt : 0;
        uint8_t* base = lds + slot * STAGE;
        // W4A16: an opaque copy of the lane id, so that the offsets are worked out here and not kept in registers.
        int lane = threadIdx.x & 63;
        if constexpr (!A4) asm volatile("" : "+v"(lane));
#pragma unroll
        for (int i = 0; i < XC / NW; ++i) {
            const int c = wave * (XC / NW) + i;
            if constexpr (A4) {
                buffer_load_lds16(xr, base + c * 1024, (c * a.ktiles * kSubTileBytes + lane * 16) | past, off * kSubTileBytes);
            } else {
                const int r = 4 * c + (lane >> 4), col = (lane & 15) ^ (r & 15);
                const int at = kt * kTileK + col * 8 < a.k ? r * a.k * 2 + col * 16 : kOOB;
                buffer_load_lds16(xr, base + c * 1024, at, off * 256);
            }
        }
#pragma unroll
        for (int i = 0; i < BS / NW; ++i) {
            const int c = wave * (BS / NW) + i, side = SIDES == 2 ? c & 1 : 0, strip = SIDES == 2 ? c >> 1 : c;
            buffer_load_lds16(wr[side], base + (XC + c) * 1024, (strip * a.ktiles * kSubTileBytes + lane * 16) | past,
                              off * kSubTileBytes);
        }
    };

    // Scale dwords of a group of 4 K tiles.
    struct scales {
        uint32_t w[NS], x[A4 ? MT : 1];
    };
    auto load_scales = [&](scales& s, int q) {
        const int past = q < a.kgroups ? 0 : kOOB, off = q < a.kgroups ? q * 256 : 0;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int sl = wn * NS + j, side = SIDES == 2 ? sl & 1 : 0, strip = SIDES == 2 ? sl >> 1 : sl;
            s.w[j] = buffer_load_u32(sr[side], (strip * a.kgroups * 256 + lane * 4) | past, off);
        }
        if constexpr (A4) {
#pragma unroll
            for (int i = 0; i < MT; ++i) s.x[i] = buffer_load_u32(xsr, ((wm * MT + i) * a.kgroups * 256 + lane * 4) | past, off);
        }
    };

    auto shift_scales = [&](scales& to, const scales& from, int by) {
#pragma unroll
        for (int j = 0; j < NS; ++j) to.w[j] = from.w[j] >> by;
        if constexpr (A4) {
#pragma unroll
            for (int i = 0; i < MT; ++i) to.x[i] = from.x[i] >> by;
        }
    };

    // Fragments. x's are read again for the next slice right after their use, the weights' a slice ahead.
    u32x4_t x[MT], w[2][NS];
    auto read_x = [&](int i, int slot, int t) {
        const uint8_t* base = lds + slot * STAGE;
        if constexpr (A4) x[i] = *reinterpret_cast<const u32x4_t*>(base + (wm * MT + i) * 1024 + lane * 16);
        else x[i] = *reinterpret_cast<const u32x4_t*>(base + (wm * MT * 16 + i * 16 + col16) * 256 + (((4 * kq + t) ^ col16) << 4));
    };
    auto read_w = [&](u32x4_t (&to)[NS], int j, int slot) {
        to[j] = *reinterpret_cast<const u32x4_t*>(lds + slot * STAGE + (XC + wn * NS + j) * 1024 + lane * 16);
    };

    f32x4_t acc[MT][NS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    scales sc, scn;
#pragma unroll
    for (int p = 0; p < S; ++p) {
        if (p == S - 2) load_scales(sc, 0);  // where a turn before the first would have asked for them (see the counts below)
        issue(p, p);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * LOADS) : "memory");

#pragma unroll
    for (int i = 0; i < MT; ++i) read_x(i, 0, 0);
#pragma unroll
    for (int j = 0; j < NS; ++j) read_w(w[0], j, 0);
    int slot = 0;
    if constexpr (A4) {
        // Loads after those of K tile kt + 1, which has to have landed: S - 2 K tiles' and the scales of the
        // turns begun since.
        constexpr int SC = NS + MT;
        auto step = [&](int kt, const u32x4_t (&cur)[NS], u32x4_t (&next)[NS], auto older) {
            const int ns = slot + 1 == S ? 0 : slot + 1;
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(older)::value) : "memory");
            issue(kt + S, slot);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = i * NS / MT; j < (i + 1) * NS / MT; ++j) read_w(next, j, ns);
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][j] = mx_mfma<0, 0>(cur[j], sc.w[j], x[i], sc.x[i], acc[i][j]);
                read_x(i, ns, 0);
                __builtin_amdgcn_sched_barrier(0);  // the reads stay among the matrix instructions, a K tile ahead
            }
            slot = ns;
        };
        // Two K tiles a turn; past an odd number of them one of zeros, whose scale bytes are zeros, too. No
        // branch in a turn: the compiler would sink the matrix instructions past it, and past the reads.
        for (int kt = 0; kt < a.ktiles; kt += 2) {
            load_scales(scn, (kt + 2) >> 2);
            step(kt, w[0], w[1], std::integral_constant<int, (S - 2) * LOADS + S / 2 * SC>{});
            shift_scales(sc, sc, 8);
            step(kt + 1, w[1], w[0], std::integral_constant<int, (S - 2) * LOADS + (S - 1) / 2 * SC>{});
            shift_scales(sc, scn, (kt & 2) ? 0 : 16);
        }
    } else {
        for (int kt = 0; kt < a.ktiles; ++kt) {
            load_scales(scn, (kt + 1) >> 2);
            const int ns = slot + 1 == S ? 0 : slot + 1;
            float s[NS];
#pragma unroll
            for (int j = 0; j < NS; ++j) s[j] = mx_scale(sc.w[j] & 0xffu);
#pragma unroll
            for (int t = 0; t < SLICES; ++t) {
                if (t == SLICES - 1) {
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LOADS) : "memory");
                    issue(kt + S, slot);
                }
                u32x4_t wf[NS];
#pragma unroll
                for (int j = 0; j < NS; ++j) wf[j] = mx_decode<BF16>(w[0][j][t], s[j]);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (t == SLICES - 1)
#pragma unroll
                        for (int j = i * NS / MT; j < (i + 1) * NS / MT; ++j) read_w(w[1], j, ns);
#pragma unroll
                    for (int j = 0; j < NS; ++j) acc[i][j] = mfma16x16x32<BF16>(wf[j], x[i], acc[i][j]);
                    read_x(i, t == SLICES - 1 ? ns : slot, (t + 1) & 3);
                    __builtin_amdgcn_sched_barrier(0);  // the reads stay among the matrix instructions, a slice ahead
                }
            }
#pragma unroll
            for (int j = 0; j < NS; ++j) w[0][j] = w[1][j];
            shift_scales(sc, scn, 8 * ((kt + 1) & 3));
            slot = ns;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // requests past the last K tile

#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int r = (wm * MT + i) * 16 + col16;
        const int64_t row = row0 + r;
        if constexpr (EPI == kMxPlain) {
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (r < rows) mx_store_plain<BF16>(a.out, row, (strip0 + wn * NS + j) * kTileN + 4 * kq, acc[i][j]);
        } else if constexpr (EPI == kMxGated) {
#pragma unroll
            for (int j = 0; j < NS; j += 2)
                if (r < rows) mx_store_gated<BF16>(a.out, row, (strip0 + (wn * NS + j) / 2) * kTileN + 4 * kq, acc[i][j], acc[i][j + 1]);
        } else {
            static_assert(EPI != kMxGatedCodes || NS % 4 == 0, "whole blocks");
#pragma unroll
            for (int j = 0; j + 3 < NS; j += 4) {
                const f32x4_t g[2] = {acc[i][j], acc[i][j + 2]}, u[2] = {acc[i][j + 1], acc[i][j + 3]};
                const int block = (strip0 + (wn * NS + j) / 2) / 2;
                if ((wm * MT + i) * 16 < rows && block * kMxBlock < a.out.n)  // wave-uniform
                    mx_store_codes(a.out, row0 / 16 + wm * MT + i, block, g, u);
            }
        }
    }
}

template <bool A4, bool BF16, mx_epilogue EPI, int WM, int WN, int MT, int NS, int S> void launch(const mx_product& p, hipStream_t s) {
    const mx_dims d = make_mx_dims(p.n, p.k);
    tile_args a{};
    a.x = p.x16;
    a.xq = p.xq;
    a.w0 = p.w0;
    a.w1 = p.w1;
    a.out = p.out;
    a.m = static_cast<int>(p.m);
    a.k = static_cast<int>(p.k);
    a.ktiles = static_cast<int>(d.ktiles);
    a.kgroups = static_cast<int>(d.kgroups);
    a.strips = static_cast<int>(d.strips);
    constexpr int BS = WN * NS / (EPI == kMxPlain ? 1 : 2);
    a.m_blocks = static_cast<int>(ceil_div(p.m, WM * MT * 16));
    a.n_blocks = static_cast<int>(ceil_div(d.strips, BS));
    a.band = 4;
    mx_tile_kernel<A4, BF16, EPI, WM, WN, MT, NS, S><<<static_cast<unsigned>(a.m_blocks) * a.n_blocks, WM * WN * 64, 0, s>>>(a);
}

template <bool A4, bool BF16, mx_epilogue EPI> void launch_shape(const mx_product& p, hipStream_t s) {
    const int64_t wide = ceil_div(p.m, 256) * ceil_div(p.n * (EPI == kMxPlain ? 1 : 2), 256);
    if constexpr (A4) {
        if (wide >= cu_count()) launch<A4, BF16, EPI, 2, 2, 8, 8, 4>(p, s);
        else launch<A4, BF16, EPI, 2, 2, 4, 4, 4>(p, s);
    } else {
        if (wide >= cu_count()) launch<A4, BF16, EPI, 2, 4, 8, 4, 2>(p, s);
        else launch<A4, BF16, EPI, 2, 2, 4, 4, 2>(p, s);
    }
}

}  // namespace

}  // namespace plm
