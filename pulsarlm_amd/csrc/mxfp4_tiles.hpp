// MXFP4 products for many rows: y[M, N] = x[M, K] @ W^T on the matrix cores, with 16-bit x (the weights
// converted in registers, W4A16) or x quantized to the same format (raw codes and scales to the scaled
// matrix instruction, W4A4), plain or with the gated block's activation as the epilogue.
//
// * A workgroup owns BM = WM MT 16 rows by BS = WN NS strips; its WM x WN wavefronts own MT x NS products of
//   16 x 16 each. The large tile is 256 x 256 with eight wavefronts of 128 x 64, whose 128 sums a lane leave the
//   registers for the operands of two K tiles. (Four of 128 x 128 read a third less from LDS, but LDS is busy a
//   quarter of the time, and one wavefront a SIMD leaves its matrix unit idle at every wait.)
// * The operands of a K tile (128) go from memory straight into one of S LDS stages. One barrier a K tile
//   stands before its last slice's matrix instructions, whose operands are in registers by then: past it
//   every wavefront has read the stage, which the loads of K tile kt + S may overwrite, and K tile kt + 1 has
//   landed, so that its first slice is read while those instructions run. W4A4 has one slice a K tile,
//   W4A16 four of 32 K values.
// * The weights are the A operand and x the B operand: a lane ends with four neighbouring columns of a row.
// * What bounds it (M = 4096, N 24576, K 4096): W4A16 546 us, 1511 TFLOP/s, what the library's 16-bit product makes
//   (1410-1455); W4A4 214 us with the quantizer's 10, of which the product takes 195, 4200 TFLOP/s, with the matrix units
//   busy 55% of the cycles at 1.83-1.95 GHz, and wavefronts waiting 27%. The same FLOPs at N 4096, K 24576, with a
//   sixth of the stores and as long a run a tile, take 167 us, 70% and 1.89-1.91 GHz.
// * Gated: local strips 2 p and 2 p + 1 are gate and up of one 16-column slice, so that both halves of an
//   output are in one lane.
#pragma once

#include <type_traits>
#include <utility>

#include "mxfp4.hpp"

namespace plm {

namespace {

struct tile_args {
    const uint16_t* x;
    mx_matrix xq, w0, w1;
    mx_output out;
    int m, k, ktiles, strips;
    float* partial;                // W4A4: [splits][M][N] sums of split_tiles K tiles each, or null
    int split_tiles;
    int m_blocks, n_blocks, band;  // band: row blocks of an XCD's patch of work tiles
};

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>): the byte of a scale register that a matrix
// instruction uses is part of the instruction.
template <typename F, int... I> __device__ __forceinline__ void unrolled_(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void unrolled(F f) {
    unrolled_(f, std::make_integer_sequence<int, N>{});
}

// SL: the scales go through the stages, too; else (W4A16 only) to registers, a K tile ahead.
// KG: groups of WM x WN wavefronts that take the K tiles in turn, each with stages of its own; their sums meet in LDS.
template <bool A4, bool BF16, mx_epilogue EPI, int WM, int WN, int MT, int NS, int S, int KG, bool SL>
__global__ void __launch_bounds__(WM * WN * KG * 64) mx_tile_kernel(tile_args a) {
    constexpr int NW = WM * WN;
    constexpr int BM = WM * MT * 16, BS = WN * NS;
    constexpr int XC = A4 ? WM * MT : WM * MT * 4;  // 1 KiB chunks of x in a stage
    // Scale chunks of 256 bytes (4 strips each): x's, then the weights' (gate's, then up's).
    constexpr int SIDES = EPI == kMxPlain ? 1 : 2;
    constexpr int XG = A4 ? (WM * MT + 3) / 4 : 0, WG = (BS / SIDES + 3) / 4, SCC = XG + SIDES * WG;
    constexpr int SCL = SL ? (SCC + NW - 1) / NW : 0;
    constexpr int STAGE = (XC + BS) * 1024 + (SL ? SCC * 256 : 0);
    constexpr int LOADS = (XC + BS) / NW + SCL;
    constexpr int SLICES = A4 ? 1 : 4;
    static_assert((NS & (NS - 1)) == 0 && (!A4 || ((MT & (MT - 1)) == 0 && WM % 2 == 0)), "a wavefront's strips lie in whole groups, or in one");
    static_assert(XC % NW == 0 && BS % NW == 0, "every wavefront loads as many chunks");
    static_assert(EPI == kMxPlain || NS % 2 == 0, "gate and up in one wavefront");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S * KG * STAGE];

    const int lane = threadIdx.x & 63;
    const int group = KG == 1 ? 0 : uniform(threadIdx.x >> 6) / NW, wave = uniform(threadIdx.x >> 6) % NW;
    const int wm = wave / WN, wn = wave % WN;
    uint8_t* stages = lds + group * STAGE;  // slot s at s KG STAGE
    const int col16 = lane & 15, kq = lane >> 4;

    // Workgroups go round the 8 XCDs by id: each takes one run of the work tiles, which are ordered in
    // bands of `band` row blocks, row block fastest, so that an XCD's L2 holds what its tiles share.
    const int tiles = a.m_blocks * a.n_blocks, xcd = blockIdx.x & 7;
    const int lin = xcd * (tiles >> 3) + min(xcd, tiles & 7) + (blockIdx.x >> 3);
    const int first = lin / (a.band * a.n_blocks) * a.band;
    const int band_rows = min(a.band, a.m_blocks - first), in_band = lin - first * a.n_blocks;
    const int nb = in_band / band_rows, row0 = (first + in_band % band_rows) * BM;
    const int rows = min(BM, a.m - row0);
    // The workgroup's K tiles.
    const int kt_first = A4 ? static_cast<int>(blockIdx.y) * a.split_tiles : 0;
    const int kt_end = A4 ? min(kt_first + a.split_tiles, a.ktiles) : a.ktiles;

    // Local strip s: strip nb BS + s, or slice nb BS / 2 + s / 2 of the gate (s even) or up weight.
    const int strip0 = nb * (BS / SIDES);
    const int mine = min(BS / SIDES, a.strips - strip0);
    const int64_t w_at = static_cast<int64_t>(strip0) * a.ktiles * kSubTileBytes, s_at = static_cast<int64_t>(strip0 >> 2) * a.ktiles * 64;
    const uint32_t w_bytes = static_cast<uint32_t>(mine) * a.ktiles * kSubTileBytes;
    const uint32_t s_bytes = static_cast<uint32_t>(((strip0 & 3) + mine + 3) / 4) * a.ktiles * 256;
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
        make_rsrc(a.xq.scale + static_cast<int64_t>(row0 / 64) * a.ktiles * 64, A4 ? static_cast<uint32_t>((row0 % 64 / 16 + x_strips + 3) / 4) * a.ktiles * 256 : 0u);

    // The scale chunks that this wavefront loads (the last one again where there are fewer): chunk, its group
    // of strips and buffer.
    int scc[SCL + 1], scg[SCL + 1];
    __amdgpu_buffer_rsrc_t scr[SCL + 1];
#pragma unroll
    for (int i = 0; i < SCL; ++i) {
        const int c = min(wave * SCL + i, SCC - 1), w = c - XG;
        scc[i] = c;
        scg[i] = c < XG ? c : w % WG;
        scr[i] = c < XG ? xsr : (w < WG ? sr[0] : sr[1]);
    }

    // Load l of the wavefront's LOADS for K tile kt. Chunk c of a stage: x's first (codes: strip c; 16-bit: rows
    // 4 c .. 4 c + 3, their 16-byte columns XOR-swizzled by row), then the weight strips', then the scales'. Past
    // the end of any, zeros.
    // A load's range check covers both its offsets (checked on the GPU): the lanes' own hardly change, and past the
    // end the wave-uniform one is kOOB.
    constexpr int XL = XC / NW, WL = BS / NW;
    const int x_row = (lane >> 4) * a.k * 2, x_col = ((lane & 15) ^ (lane >> 4)) << 4;
    auto issue_one = [&](int l, int turn, int slot) {
        const int kt = kt_first + turn * KG + group;
        const bool in = kt < kt_end;
        uint8_t* base = stages + slot * (KG * STAGE);
        if (l < XL) {
            const int c = wave * XL + l;
            if constexpr (A4) {
                buffer_load_lds16(xr, base + c * 1024, lane * 16, in ? (c * a.ktiles + kt) * kSubTileBytes : kOOB);
            } else {
                const int col = x_col ^ ((c & 3) << 6);  // the lane's row 4 c + lane / 16, its column swizzled by row % 16
                buffer_load_lds16(xr, base + c * 1024, col < (a.k - kt * kTileK) * 2 ? x_row + col : kOOB, in ? kt * 256 + c * a.k * 8 : kOOB);
            }
        } else if (l < XL + WL) {
            const int c = wave * WL + l - XL, side = SIDES == 2 ? c & 1 : 0, strip = SIDES == 2 ? c >> 1 : c;
            buffer_load_lds16(wr[side], base + (XC + c) * 1024, lane * 16, in ? (strip * a.ktiles + kt) * kSubTileBytes : kOOB);
        } else {
            const int i = l - XL - WL;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(scr[i], (__attribute__((address_space(3))) void*)(base + (XC + BS) * 1024 + scc[i] * 256), 4,
                                                     lane * 4, in ? (scg[i] * a.ktiles + kt) * 256 : kOOB, 0, 0);
        }
    };
    // The loads of a K tile stand among the matrix instructions, at places 0 .. SPREAD - 1 (one row of them
    // each): requested all at once, a wavefront waits for the memory pipeline to take them (16 cycles each,
    // one pipeline a CU) with its matrix unit idle.
    auto issue_at = [&](int place, auto spread, int kt, int slot) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
            if (l * decltype(spread)::value / LOADS == place) issue_one(l, kt, slot);
    };
    auto issue = [&](int kt, int slot) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l) issue_one(l, kt, slot);
    };

    const int x_at = row0 / 16 & 3, g_at = strip0 & 3;  // where the workgroup's first strips lie in their groups
    // A lane's scale dwords of a K tile: the bytes of four strips each, shifted to start at the wavefront's own.
    constexpr int XN = A4 ? (MT + 3) / 4 : 0, PN = NS / SIDES, WN4 = (PN + 3) / 4;
    struct scales {
        uint32_t x[A4 ? XN : 1], w[SIDES][WN4];
    };
    auto read_scales = [&](scales& s, int slot) {
        const uint8_t* base = stages + slot * (KG * STAGE) + (XC + BS) * 1024 + lane * 4;
        if constexpr (A4) {
#pragma unroll
            for (int g = 0; g < XN; ++g)
                s.x[g] = *reinterpret_cast<const uint32_t*>(base + ((x_at + wm * MT) / 4 + g) * 256) >> (8 * ((x_at + wm * MT) & 3));
        }
#pragma unroll
        for (int d = 0; d < SIDES; ++d)
#pragma unroll
            for (int g = 0; g < WN4; ++g)
                s.w[d][g] = *reinterpret_cast<const uint32_t*>(base + (XG + d * WG + (g_at + wn * PN) / 4 + g) * 256) >> (8 * ((g_at + wn * PN) & 3));
    };

    auto load_scales = [&](scales& s, int turn) {
        const int kt = turn * KG + group;
        const int past = kt < a.ktiles ? 0 : kOOB, off = kt < a.ktiles ? kt * 256 : 0;
#pragma unroll
        for (int d = 0; d < SIDES; ++d)
#pragma unroll
            for (int g = 0; g < WN4; ++g)
                s.w[d][g] = buffer_load_u32(sr[d], (((g_at + wn * PN) / 4 + g) * a.ktiles * 256 + lane * 4) | past, off);
    };
    auto shift_scales = [&](scales& s) {
#pragma unroll
        for (int d = 0; d < SIDES; ++d)
#pragma unroll
            for (int g = 0; g < WN4; ++g) s.w[d][g] >>= 8 * ((g_at + wn * PN) & 3);
    };

    // Fragments. x's are read again right after their use, XB slices ahead (XB: as many as make that some hundred
    // cycles, the time of an LDS read); the weights' a K tile ahead.
    constexpr int XB = A4 ? 1 : (MT * NS >= 16 ? 1 : (MT * NS >= 8 ? 2 : 4));
    u32x4_t x[XB][MT], w[2][NS];
    auto read_x = [&](int i, int slot, int t) {
        const uint8_t* base = stages + slot * (KG * STAGE);
        if constexpr (A4) x[0][i] = *reinterpret_cast<const u32x4_t*>(base + (wm * MT + i) * 1024 + lane * 16);
        else x[t % XB][i] = *reinterpret_cast<const u32x4_t*>(base + (wm * MT * 16 + i * 16 + col16) * 256 + (((4 * kq + t) ^ col16) << 4));
    };
    auto read_w = [&](u32x4_t (&to)[NS], int j, int slot) {
        to[j] = *reinterpret_cast<const u32x4_t*>(stages + slot * (KG * STAGE) + (XC + wn * NS + j) * 1024 + lane * 16);
    };

    f32x4_t acc[MT][NS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // W4A16: K tile kt's barrier stands before slice BAR, past which no wavefront reads its stage; the loads of
    // K tile kt + S into it are spread over the slices from there on into the next K tile.
    constexpr int BAR = SLICES - XB;
    constexpr int SPREAD = A4 ? MT : std::min(SLICES * MT, (XB + 1) * MT);
    using spread_t = std::integral_constant<int, SPREAD>;
#pragma unroll
    for (int p = 0; p < S - 1; ++p) issue(p, p);
    // Of K tile S - 1 the loads that the first K tile's slices before BAR do not make.
#pragma unroll
    for (int place = 0; place < (A4 ? SPREAD : XB * MT); ++place) issue_at(place, spread_t{}, S - 1, S - 1);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 2) * LOADS) : "memory");
#pragma unroll
    for (int t = 0; t < XB; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) read_x(i, 0, t);
#pragma unroll
    for (int j = 0; j < NS; ++j) read_w(w[0], j, 0);
    scales sc[2];
    if constexpr (SL) {
        read_scales(sc[0], 0);
    } else {
        load_scales(sc[0], 0);
        shift_scales(sc[0]);
    }
    int slot = 0;
    const int turns = (kt_end - kt_first + KG - 1) / KG;  // past the last K tile one of zeros
    // K tile kt + 1 has landed when only the loads of S - 2 K tiles after it are left.
    constexpr int LEFT = (S - 2) * LOADS;
    static_assert(LEFT <= 63 && (SL || S == 2), "the counter's range; loads to registers are not counted");
    if constexpr (A4) {
        auto step = [&](int kt, const u32x4_t (&cur)[NS], u32x4_t (&next)[NS], const scales& s, scales& s_next) {
            const int ns = slot + 1 == S ? 0 : slot + 1;
            unrolled<MT>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                if constexpr (i == 0) {
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
                    read_scales(s_next, ns);
                }
                issue_at(i, spread_t{}, kt + S, slot);
#pragma unroll
                for (int j = i * NS / MT; j < (i + 1) * NS / MT; ++j) read_w(next, j, ns);
                unrolled<NS>([&](auto jc) {
                    constexpr int j = decltype(jc)::value, p = j / SIDES;
                    acc[i][j] = mx_mfma<p & 3, i & 3>(cur[j], s.w[j % SIDES][p / 4], x[0][i], s.x[i / 4], acc[i][j]);
                });
                read_x(i, ns, 0);
                __builtin_amdgcn_sched_barrier(0);  // reads and loads stay where they are
            });
            slot = ns;
        };
        // Two K tiles a turn; past an odd number of them one of zeros. No branch in a turn: the compiler would
        // sink the matrix instructions past it, and past the reads.
        for (int kt = 0; kt < turns; kt += 2) {
            step(kt, w[0], w[1], sc[0], sc[1]);
            step(kt + 1, w[1], w[0], sc[1], sc[0]);
        }
    } else {
        int load_kt = S - 1, load_slot = S - 1;
        for (int kt = 0; kt < turns; ++kt) {
            const int ns = slot + 1 == S ? 0 : slot + 1;
            if constexpr (!SL) load_scales(sc[1], kt + 1);
            float s[NS];
#pragma unroll
            for (int j = 0; j < NS; ++j) s[j] = mx_scale(sc[0].w[j % SIDES][j / SIDES / 4] >> (8 * (j / SIDES & 3)) & 0xffu);
#pragma unroll
            for (int t = 0; t < SLICES; ++t) {
                u32x4_t wf[NS];
#pragma unroll
                for (int j = 0; j < NS; ++j) wf[j] = mx_decode<BF16>(w[0][j][t], s[j]);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (t == BAR && i == 0) {
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
                        load_kt = kt + S;
                        load_slot = slot;
                        if constexpr (SL) read_scales(sc[1], ns);
                    }
                    issue_at(((t - BAR + SLICES) * MT + i) % (SLICES * MT), spread_t{}, load_kt, load_slot);
                    if (t == SLICES - 1)
#pragma unroll
                        for (int j = i * NS / MT; j < (i + 1) * NS / MT; ++j) read_w(w[1], j, ns);
#pragma unroll
                    for (int j = 0; j < NS; ++j) acc[i][j] = mfma16x16x32<BF16>(wf[j], x[t % XB][i], acc[i][j]);
                    read_x(i, t >= BAR ? ns : slot, (t + XB) % SLICES);
                    __builtin_amdgcn_sched_barrier(0);  // reads and loads stay where they are
                }
            }
#pragma unroll
            for (int j = 0; j < NS; ++j) w[0][j] = w[1][j];
            if constexpr (!SL) shift_scales(sc[1]);
            sc[0] = sc[1];
            slot = ns;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // requests past the last K tile; LDS is free

    if constexpr (KG > 1) {
        // In group order, so that the result does not depend on which is done first.
        static_assert((KG - 1) * NW * MT * NS * 1024 <= S * KG * STAGE, "the sums fit");
        f32x4_t* sums = reinterpret_cast<f32x4_t*>(lds);
        if (group > 0)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) sums[(((group - 1) * NW + wave) * MT * NS + i * NS + j) * 64 + lane] = acc[i][j];
        __syncthreads();
        if (group == 0)
#pragma unroll
            for (int g = 0; g < KG - 1; ++g)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NS; ++j) acc[i][j] = acc[i][j] + sums[((g * NW + wave) * MT * NS + i * NS + j) * 64 + lane];
        __syncthreads();
        if (group > 0) return;
    }

    if constexpr (EPI == kMxGatedCodes) {
        static_assert(EPI != kMxGatedCodes || NS % 4 == 0, "whole blocks");
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j + 3 < NS; j += 4) {
                const f32x4_t g[2] = {acc[i][j], acc[i][j + 2]}, u[2] = {acc[i][j + 1], acc[i][j + 3]};
                const int block = (strip0 + (wn * NS + j) / 2) / 2;
                if ((wm * MT + i) * 16 < rows && block * kMxBlock < a.out.n)  // wave-uniform
                    mx_store_codes(a.out, row0 / 16 + wm * MT + i, block, g, u);
            }
    } else {
        // A lane has four columns of one row, a quarter of a 32-byte piece. RB row blocks at a time go through the
        // wavefront's own part of LDS (pitch padded by 16 bytes) and leave as 16 bytes a lane, whole rows of the
        // wavefront's tile.
        constexpr int COLS = PN * 16, PITCH = COLS * 2 + 16, CH = COLS / 8;
        constexpr int FIT = S * KG * STAGE / (NW * 16 * PITCH), RB = FIT >= MT ? MT : (FIT >= 4 ? 4 : 2);
        static_assert(FIT >= 2 || MT == 1, "the rows fit");
        uint8_t* mine_lds = lds + wave * RB * 16 * PITCH;
        const int col0 = (strip0 + wn * PN) * kTileN;
        auto value = [&](int i, int p) {
            return EPI == kMxPlain ? acc[i][p] : mx_gated4(acc[i][SIDES * p], acc[i][SIDES * p + SIDES - 1]);
        };
        if (EPI == kMxGated && a.out.gate_up != nullptr) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int r = (wm * MT + i) * 16 + col16;
                if (r < rows)
#pragma unroll
                    for (int p = 0; p < PN; ++p)
                        mx_store_gate_up(a.out, row0 + r, col0 + p * 16 + 4 * kq, acc[i][SIDES * p], acc[i][SIDES * p + SIDES - 1]);
            }
        }
        if constexpr (A4 && EPI == kMxPlain) {
            if (a.partial != nullptr) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int r = (wm * MT + i) * 16 + col16;
                    float* to = a.partial + (static_cast<int64_t>(blockIdx.y) * a.m + row0 + r) * a.out.n;
                    if (r < rows)
#pragma unroll
                        for (int p = 0; p < PN; ++p) {
                            const int col = col0 + p * 16 + 4 * kq;  // N is a multiple of 4
                            if (col < a.out.n) *reinterpret_cast<f32x4_t*>(to + col) = acc[i][p];
                        }
                }
                return;
            }
        }
        if (!a.out.lines) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int r = (wm * MT + i) * 16 + col16;
                if (r < rows)
#pragma unroll
                    for (int p = 0; p < PN; ++p) mx_store_plain<BF16>(a.out, row0 + r, col0 + p * 16 + 4 * kq, value(i, p));
            }
            return;
        }
#pragma unroll
        for (int i0 = 0; i0 < MT; i0 += RB) {
            const int r0 = (wm * MT + i0) * 16;
            if (r0 >= rows) break;
#pragma unroll
            for (int i = i0; i < i0 + RB; ++i)
#pragma unroll
                for (int p = 0; p < PN; ++p) {
                    const f32x4_t v = value(i, p);
                    *reinterpret_cast<uint2*>(mine_lds + ((i - i0) * 16 + col16) * PITCH + (p * 16 + 4 * kq) * 2) =
                        make_uint2(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]));
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int c0 = 0; c0 < RB * 16 * CH; c0 += 64) {
                const int c = c0 + lane, r = c / CH, col = col0 + c % CH * 8;
                if (c < RB * 16 * CH && r0 + r < rows && col < a.out.n)
                    *reinterpret_cast<u32x4_t*>(a.out.y + (row0 + r0 + r) * static_cast<int64_t>(a.out.n) + col) =
                        *reinterpret_cast<const u32x4_t*>(mine_lds + r * PITCH + c % CH * 16);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <bool A4, bool BF16, mx_epilogue EPI, int WM, int WN, int MT, int NS, int S, int KG = 1, bool SL = true> void launch(const mx_product& p, int splits, hipStream_t s) {
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
    a.strips = static_cast<int>(d.strips);
    constexpr int BS = WN * NS / (EPI == kMxPlain ? 1 : 2);
    a.m_blocks = static_cast<int>(ceil_div(p.m, WM * MT * 16));
    a.n_blocks = static_cast<int>(ceil_div(d.strips, BS));
    a.band = 4;
    a.split_tiles = static_cast<int>(ceil_div(d.ktiles, splits));
    a.partial = splits > 1 ? p.partial : nullptr;
    const dim3 grid(static_cast<unsigned>(a.m_blocks) * a.n_blocks, static_cast<unsigned>(splits));
    mx_tile_kernel<A4, BF16, EPI, WM, WN, MT, NS, S, KG, SL><<<grid, WM * WN * KG * 64, 0, s>>>(a);
}

// The tile shapes, and which of them takes a call: the least of rounds x K tiles x time of a K tile. The times (us)
// were measured with one workgroup on the GPU and with every slot taken; between the two they grow with the
// share of slots taken, as the workgroups share the L2s and the clock. 192 rows are there for what 128 and 256 waste:
// M = 333, N 24576, K 4096 70 us with them and 87 without; gate and up of 4864, K 2080, M = 1001 45 and 54.
// {rows, columns, workgroups a CU, lone, full}
struct tile_cost {
    int rows, cols, per_cu;
    double lone, full;
};
constexpr tile_cost kTiles16[] = {{256, 256, 1, 2.35, 2.70}, {192, 256, 1, 1.61, 2.03}, {128, 256, 1, 1.10, 1.50}, {128, 128, 2, 1.20, 1.70}, {128, 128, 1, 0.69, 0.95},
                                  {64, 128, 1, 0.36, 0.52},  {64, 64, 1, 0.29, 0.36},   {32, 64, 1, 0.18, 0.27},   {32, 64, 2, 0.20, 0.38}};
constexpr tile_cost kTiles4[] = {{256, 256, 1, 0.60, 0.95}, {128, 256, 1, 0.40, 0.62}, {128, 128, 2, 0.33, 0.62},
                                 {64, 128, 2, 0.23, 0.38},  {64, 64, 2, 0.18, 0.24}};

struct tile_choice {
    int shape, splits;
};
// The first `count` shapes, and up to most_splits parts of the K tiles, whose fp32 sums a kernel more adds: that and
// their way through memory take 8 us and more, which only a long K with few tiles gives back. Split / not, us: M = 64,
// N 5120, K 17408 23.6 / 28.9; M = 48, N 4096, K 12288 15.6 / 19.9; but M = 200, N 4096, K 12288 26.7 / 21.2, and
// M = 24, N 6144, K 4096 13.2 / 10.7.
template <int N> tile_choice choose_tile(const tile_cost (&shapes)[N], int count, int64_t m, int64_t n, int64_t ktiles, int64_t most_splits) {
    tile_choice best{0, 1};
    double least = 1e300;
    for (int i = 0; i < count; ++i) {
        const tile_cost& c = shapes[i];
        const int64_t tiles = ceil_div(m, c.rows) * ceil_div(n, c.cols), slots = int64_t{c.per_cu} * cu_count();
        const int64_t most = std::max<int64_t>(1, std::min({most_splits, ktiles / 4, slots / tiles}));
        for (int64_t splits = 1; splits <= most; ++splits) {
            const int64_t each = ceil_div(ktiles, splits);
            if (ceil_div(ktiles, each) != splits) continue;  // no part without a K tile
            const double fill = std::min(1.0, static_cast<double>(tiles * splits) / slots);
            const double t = ceil_div(tiles * splits, slots) * each * (c.lone + (c.full - c.lone) * fill) +
                             (splits > 1 ? 8. + splits * m * n * 8 / 5.5e6 : 0.);
            if (t < least) least = t, best = {i, static_cast<int>(splits)};
        }
    }
    return best;
}
// W4A4, plain: where N is not a multiple of 4, the sums are not whole quads.
tile_choice choose_w4a4(int64_t m, int64_t n, int64_t k, bool may_split) {
    return choose_tile(kTiles4, 5, m, n, ceil_div(k, kTileK), may_split && n % 4 == 0 ? 16 : 1);
}

template <bool A4, bool BF16, mx_epilogue EPI> void launch_shape(const mx_product& p, hipStream_t s) {
    tile_choice c;
    if constexpr (A4 && EPI == kMxPlain) c = choose_w4a4(p.m, p.n, p.k, p.partial != nullptr && p.out.wide);
    else if constexpr (A4) c = choose_tile(kTiles4, 4, p.m, 2 * p.n, ceil_div(p.k, kTileK), 1);  // a block is in one wavefront: NS = 4
    else c = choose_tile(kTiles16, 9, p.m, p.n * (EPI == kMxPlain ? 1 : 2), ceil_div(p.k, kTileK), 1);
    const int shape = c.shape, splits = c.splits;
    if constexpr (A4) {
        switch (shape) {
            case 0: launch<A4, BF16, EPI, 2, 4, 8, 4, 4>(p, splits, s); break;
            case 1: launch<A4, BF16, EPI, 2, 4, 4, 4, 6>(p, splits, s); break;
            case 2: launch<A4, BF16, EPI, 2, 2, 4, 4, 4>(p, splits, s); break;
            case 3: launch<A4, BF16, EPI, 2, 2, 2, 4, 6>(p, splits, s); break;
            default:
                if constexpr (EPI != kMxGatedCodes) launch<A4, BF16, EPI, 2, 2, 2, 2, 4, 2>(p, splits, s);
        }
        if (splits > 1) launch_mx_combine(p.bf16, p.partial, p.m * p.n, splits, p.out.y, s);
    } else {
        constexpr bool G = EPI == kMxGated;  // gate and up in one wavefront: an even number of strips
        switch (shape) {
            case 0: return launch<A4, BF16, EPI, 2, 4, 8, 4, 2, 1, false>(p, splits, s);
            case 1: return launch<A4, BF16, EPI, 2, 4, 6, 4, 2>(p, splits, s);
            case 2: return launch<A4, BF16, EPI, 1, 8, 8, 2, 3>(p, splits, s);
            case 3: return launch<A4, BF16, EPI, 1, 4, 8, 2, 2, 1, false>(p, splits, s);
            case 4: return launch<A4, BF16, EPI, 2, 4, 4, 2, 3>(p, splits, s);
            case 5: return launch<A4, BF16, EPI, 1, 4, 4, 2, 3, 2>(p, splits, s);
            case 6: return launch<A4, BF16, EPI, 2, 2, 2, 2, 3, 2>(p, splits, s);
            case 7: return launch<A4, BF16, EPI, 2, 2, 1, 2, 3, 4>(p, splits, s);
            default: return launch<A4, BF16, EPI, G ? 2 : 1, G ? 2 : 4, G ? 1 : 2, G ? 2 : 1, 3, 2>(p, splits, s);
        }
    }
}

}  // namespace

}  // namespace plm
