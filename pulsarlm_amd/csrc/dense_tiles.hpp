// The tile kernel of the products on unpacked weights (dense_gemm.hpp): a workgroup owns a tile of (WM MT 16) rows by
// (WN NT 16) columns, its WM x WN wavefronts MT x NT products of 16 x 16 each.
//
// * A stage is 128 bytes of K, two slices of the matrix instruction's (32 values in 16 bits, 64 in 8). P's and Q's
//   parts of it go from memory straight into LDS, into rings of S + PX and S. Where an operand lies along the sum, its
//   rows are there with their 16-byte pieces XOR-swizzled by row; where it lies across (gradients), 64 rows of the sum's
//   index, 32-byte pieces swizzled, and the fragments are read with the transposing LDS read.
// * One barrier a stage, before its last slice's matrix instructions, whose operands are in registers by then: past it
//   the stage's room is free for loads, and stage kt + 1 has landed and is read while they run.
// * Q is the A operand and P the B operand: a lane ends with four neighbouring columns of a row.
// * A workgroup takes every gridDim.x-th tile of the launch, as many workgroups as are resident at once: the loads of the
//   next tile's first stages go on while a tile's sums are stored. (A workgroup a tile instead: 8 bits, 4096 rows, N 24576,
//   K 4096 353 us for 338; 32768 rows over 128 experts, N 2048, K 768 176 for 164.)
// What bounds it: 8192^3 takes 848 us in bf16 (1.30 PFLOP/s), 418 in 8 bits; without its loads and LDS reads 662 to 722, at the
// clock that the power leaves. Short sums: the stores' time (128 KB a tile at the memory's rate), and loads that wait behind
// them, as requests end in order. Few tiles: one round, a stage as long as a CU takes to bring it in, 50 to 60 GB/s.
#pragma once

#include <algorithm>
#include <type_traits>
#include <utility>

#include "dense_gemm.hpp"
#include "dense_turns.hpp"

namespace plm {

namespace {

// 16 bytes a lane from memory straight to LDS, as buffer_load_lds16, but written out: the compiler would wait for every
// such load in flight before a transposing LDS read, as it cannot tell their addresses apart. No register is written;
// the kernel counts these loads itself. `lds` and `soffset` are wave-uniform. m0 is these loads' own: the compiler takes no
// clobber of a reserved register, so nothing else in the kernel may use it (a builtin that loads to LDS, indexed registers).
__device__ __forceinline__ void dma16(i32x4_t buffer, uint32_t lds, int lds_more, int voffset, int soffset) {
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds" ::"s"(lds), "i"(lds_more), "v"(voffset), "s"(buffer), "s"(soffset) : "memory", "scc");
}
// make_rsrc's four words: a raw buffer of `bytes` from a wave-uniform address.
__device__ __forceinline__ i32x4_t buffer_words(const uint8_t* base, uint32_t bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return i32x4_t{static_cast<int>(at), static_cast<int>(at >> 32) & 0xffff, static_cast<int>(bytes), 0x00020000};
}

typedef __attribute__((ext_vector_type(4))) short tr16_t;

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>).
template <typename F, int... I> __device__ __forceinline__ void unrolled_(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void unrolled(F f) {
    unrolled_(f, std::make_integer_sequence<int, N>{});
}

// One operand: BLOCK rows or columns of the tile.
template <bool CROSS, int BLOCK, int NW> struct dense_operand {
    static constexpr int kBytes = BLOCK * 128;          // of a stage
    static constexpr int kLoads = kBytes / 1024 / NW;   // of a wavefront
    static_assert(kBytes % (1024 * NW) == 0, "every wavefront loads as much");
    // Along: rows of 128 bytes. Across: rows of the sum's index, BLOCK values each.
    static constexpr int kPitch = CROSS ? BLOCK * 2 : 128;
    static constexpr int kRowsLoad = 1024 / kPitch;
    static_assert(!CROSS || (NW * kRowsLoad) % 8 == 0, "the swizzle repeats");
};

// Across: piece (32 bytes) c of the sum's row k lies at piece c ^ f(k), so that the rows and pieces that 32 lanes of a
// transposing read touch fall on different banks.
__device__ __forceinline__ constexpr int cross_swizzle(int k, int pieces) {
    return pieces >= 8 ? (k & 3) << 1 | (((k >> 2) ^ (k >> 3)) & 1) : pieces == 4 ? (k & 2) | ((k >> 3) & 1) : (k >> 3) & 1;
}

template <dense_type T, dense_mode MODE, bool PC, bool QC, int WM, int WN, int MT, int NT, int S, int PX>
__global__ void __launch_bounds__(WM * WN * 64) dense_tile_kernel(dense_args a) {
    constexpr int NW = WM * WN, BM = WM * MT * 16, BN = WN * NT * 16;
    using P = dense_operand<PC, BM, NW>;
    using Q = dense_operand<QC, BN, NW>;
    using acc_t = dense_acc<T>;
    constexpr int P_RING = (S + PX) * P::kBytes, LDS = P_RING + S * Q::kBytes;
    constexpr int SIZE = T == kInt8 ? 1 : 2;
    constexpr int STAGE = 128, DEPTH = STAGE / SIZE;  // of the sum, bytes and elements
    constexpr bool SPLITS = T == kInt8 && MODE == kDense;
    static_assert(T != kInt8 || (!PC && !QC), "8-bit operands lie along the sum");
    static_assert(LDS <= 160 * 1024, "LDS");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, col16 = lane & 15, kq = lane >> 4;

    // The workgroup's tiles, one a lane: every gridDim.x-th of the launch's (dense_turns.hpp).
    constexpr int SHIFT = BM == 256 ? 8 : BM == 128 ? 7 : BM == 64 ? 6 : 5;
    static_assert(1 << SHIFT == BM, "row blocks are powers of two");
    int m_blocks = a.m_blocks;
    if constexpr (MODE == kByRows) m_blocks = count_blocks(a.offsets, a.experts, a.rows, a.zero_rest, SHIFT);
    // (By ranges, of an expert's tiles: experts can differ in depth by far.)
    const int block_tiles = m_blocks * a.n_blocks, all_tiles = block_tiles * (MODE == kByRanges ? a.experts : 1);
    const int each = static_cast<int>(gridDim.x), self = static_cast<int>(blockIdx.x);
    // By ranges, whose longest sums come first, the turns go back and forth.
    const int tiles = dense_turns(all_tiles, each, self, MODE == kByRanges);  // <= 64
    if (tiles == 0) return;
    int lane_expert = 0, lane_row0, lane_col0, lane_lo, lane_hi;  // rows of the output (by ranges, of the sum): lo .. hi
    {
        int id = min(lane * each + dense_place(lane, each, self, MODE == kByRanges), all_tiles - 1);
        if constexpr (MODE == kByRanges) lane_expert = id / block_tiles, id -= lane_expert * block_tiles;
        const auto [mb, nb] = dense_block_of(id, m_blocks, a.n_blocks, a.band);
        lane_col0 = nb * BN, lane_row0 = lane_lo = mb * BM, lane_hi = min(lane_lo + BM, a.rows);
        if constexpr (MODE == kByRows) {
            const expert_range r = find_blocks(a.offsets, a.experts, a.rows, a.zero_rest, SHIFT, mb);
            lane_expert = r.expert, lane_row0 = lane_lo = r.lo, lane_hi = r.hi;
        } else if constexpr (MODE == kByRanges) {
            const expert_range r = find_experts(a.offsets, a.experts, a.depth, lane_expert);
            lane_expert = r.expert, lane_lo = r.lo, lane_hi = r.hi;
        }
    }
    // The workgroup's part of the sum: from stage `skipped` on, split_stages of them.
    const int skipped = SPLITS ? static_cast<int>(blockIdx.y) * a.split_stages : 0;
    struct tile {
        int expert, row0, rows, col0;
        int first, depth;  // of the sum
        int stages;        // at least one, of zeros where there is nothing to add
        bool rest;         // rows of no expert: zeros, their scales are taken as zeros too
    };
    auto take = [&](int i) {
        tile t{__builtin_amdgcn_readlane(lane_expert, i), __builtin_amdgcn_readlane(lane_row0, i), 0, __builtin_amdgcn_readlane(lane_col0, i), 0, a.depth, 1, false};
        const int lo = __builtin_amdgcn_readlane(lane_lo, i), hi = __builtin_amdgcn_readlane(lane_hi, i);
        if constexpr (MODE == kByRanges) t.rows = min(BM, a.rows - t.row0), t.first = lo, t.depth = hi - lo;
        else t.rows = hi - lo;
        if constexpr (MODE == kByRows)
            if (t.expert == a.experts) t.rest = true, t.expert = 0, t.depth = 0;
        if constexpr (SPLITS) t.depth = min(t.depth, (skipped + a.split_stages) * DEPTH);
        t.stages = max(1, (t.depth + DEPTH - 1) / DEPTH - skipped);
        return t;
    };

    // Along: the lane's row and 16-byte piece of a load, swizzled.
    const int along_row = lane / 8, along_piece = lane % 8 ^ along_row;
    // Across: its row of the sum and where its 16 bytes lie in it; the swizzle of loads an odd number apart differs by 4
    // where a turn of the wavefronts is 8 rows.
    auto across = [&](auto operand, int parity, int limit) {
        using O = decltype(operand);
        const int r = lane * 16 / O::kPitch, at = lane * 16 % O::kPitch;
        const int k = (parity * NW + wave) * O::kRowsLoad + r;
        const int bytes = (((at >> 5) ^ cross_swizzle(k, O::kPitch / 32)) << 5) + (at & 16);
        return bytes < limit * 2 ? bytes : kOOB;
    };
    // Where the loads are: a tile ahead of the products when its last stage is in flight. Along: the tile's rows from the
    // first on, the range check ends past the last. Across: the sum's rows from the first on; a stage's base moves with it,
    // as all of them can pass 2 GiB.
    int load_tile = 0, load_kt, load_end, load_depth, load_rows, load_cols, load_row0, load_col0;
    const uint8_t *p_base, *q_base;
    int p_cross[2], q_cross[2];
    auto load_from = [&](const tile& t) {
        load_kt = skipped, load_end = skipped + t.stages, load_depth = t.depth;
        load_rows = t.rows, load_cols = min(BN, a.cols - t.col0), load_row0 = t.row0, load_col0 = t.col0;
        p_base = a.p + (PC ? static_cast<int64_t>(t.first) * a.pitch_p + t.row0 * 2 : static_cast<int64_t>(t.row0) * a.pitch_p);
        q_base = a.q + (MODE == kByRows ? t.expert * a.q_expert : 0) +
                 (QC ? static_cast<int64_t>(t.first) * a.pitch_q + t.col0 * 2 : static_cast<int64_t>(t.col0) * a.pitch_q);
        if constexpr (PC) {
#pragma unroll
            for (int i = 0; i < 2; ++i) p_cross[i] = across(P{}, i, load_rows) + lane * 16 / P::kPitch * a.pitch_p;
        }
        if constexpr (QC) {
#pragma unroll
            for (int i = 0; i < 2; ++i) q_cross[i] = across(Q{}, i, load_cols) + lane * 16 / Q::kPitch * a.pitch_q;
        }
    };
    // To the next stage. Past the last tile there is nothing left of the sum, and zeros are written.
    auto load_next = [&] {
        if (++load_kt < load_end) return;
        if (++load_tile < tiles) load_from(take(load_tile));
        else load_kt = 0, load_end = 1 << 30, load_depth = 0;
    };

    // What a stage's loads of an operand have in common: its buffer, from the stage's part of the sum on, and the lanes'
    // offsets. A load's range check covers both its offsets: past the end of the sum, or of the operand, zeros are written.
    struct source {
        i32x4_t buffer;
        int v[2];  // of even and odd loads
    };
    auto along = [&](int kt, const uint8_t* base, int block_rows, int pitch) {
        const int left = load_depth * SIZE - kt * STAGE;  // bytes of the sum
        const int v = along_piece * 16 < left ? along_row * pitch + along_piece * 16 : kOOB;
        return source{buffer_words(base + kt * STAGE, left > 0 ? static_cast<uint32_t>(block_rows) * pitch - kt * STAGE : 0u), {v, v}};
    };
    auto cross = [&](int kt, const uint8_t* base, int pitch, int column, const int (&v)[2]) {
        const int left = min(load_depth - kt * DEPTH, DEPTH);
        return source{buffer_words(base + static_cast<int64_t>(kt) * DEPTH * pitch, left > 0 ? static_cast<uint32_t>(left) * pitch - column * 2 : 0u), {v[0], v[1]}};
    };
    auto source_p = [&] {
        if constexpr (PC) return cross(load_kt, p_base, a.pitch_p, load_row0, p_cross);
        else return along(load_kt, p_base, load_rows, a.pitch_p);
    };
    auto source_q = [&] {
        if constexpr (QC) return cross(load_kt, q_base, a.pitch_q, load_col0, q_cross);
        else return along(load_kt, q_base, load_cols, a.pitch_q);
    };
    // Load l of the wavefront's.
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds)) + wave * 1024;
    auto issue_p = [&](const source& s, auto l, int slot) {
        constexpr int n = decltype(l)::value;
        dma16(s.buffer, lds0 + slot * P::kBytes, n * NW * 1024, s.v[n & 1], (n * NW + wave) * P::kRowsLoad * a.pitch_p);
    };
    auto issue_q = [&](const source& s, auto l, int slot) {
        constexpr int n = decltype(l)::value;
        dma16(s.buffer, lds0 + slot * Q::kBytes, P_RING + n * NW * 1024, s.v[n & 1], (n * NW + wave) * Q::kRowsLoad * a.pitch_q);
    };

    // Fragment f of slice t.
    auto read_along = [&](const uint8_t* base, int f, int t) {
        return *reinterpret_cast<const u32x4_t*>(base + (f * 16 + col16) * STAGE + (((4 * t + kq) ^ (col16 & 7)) << 4));
    };
    auto read_across = [&](const uint8_t* base, int f, int t, auto operand) {
        using O = decltype(operand);
        const int k = 32 * t + 8 * kq + (col16 >> 2);
        const uint8_t* at = base + k * O::kPitch + (col16 & 3) * 8;
        const int s = cross_swizzle(k, O::kPitch / 32), s4 = cross_swizzle(k + 4, O::kPitch / 32);
        const tr16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr16_t*)(at + ((f ^ s) << 5)));
        const tr16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr16_t*)(at + 4 * O::kPitch + ((f ^ s4) << 5)));
        const u32x2_t l = __builtin_bit_cast(u32x2_t, lo), h = __builtin_bit_cast(u32x2_t, hi);
        return u32x4_t{l[0], l[1], h[0], h[1]};
    };
    auto read_p = [&](int f, int slot, int t) {
        const uint8_t* base = lds + slot * P::kBytes;
        if constexpr (PC) return read_across(base, wm * MT + f, t, P{});
        else return read_along(base, wm * MT + f, t);
    };
    auto read_q = [&](int f, int slot, int t) {
        const uint8_t* base = lds + P_RING + slot * Q::kBytes;
        if constexpr (QC) return read_across(base, wn * NT + f, t, Q{});
        else return read_along(base, wn * NT + f, t);
    };

    acc_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = acc_t{0, 0, 0, 0};

    load_from(take(0));
    // Q's loads of stage kt + S follow the barrier of stage kt, among the matrix instructions of its second slice: the
    // memory pipeline takes a load in 16 cycles, one pipeline a CU, and a wavefront that waits for it leaves its matrix
    // unit idle. With PX, P's loads of stage kt + S + 1 stand in the next stage's first slice: both slices' time is the
    // pipeline's then, and they have a slice more to land.
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const source from_p = source_p(), from_q = source_q();
        unrolled<P::kLoads>([&](auto l) { issue_p(from_p, l, s); });
        unrolled<Q::kLoads>([&](auto l) { issue_q(from_q, l, s); });
        load_next();
    }
    // Stage 0 has landed; later, at stage kt's barrier, stage kt + 1, when only these are left:
    constexpr int LEFT = (S - 2) * (P::kLoads + Q::kLoads) + PX * P::kLoads, LEFT0 = (S - 1) * (P::kLoads + Q::kLoads);
    static_assert(S >= 2 && LEFT0 <= 63 && LEFT <= 63, "the counter's range");
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LEFT0) : "memory");
    u32x4_t p[2][MT], q[2][NT];
#pragma unroll
    for (int f = 0; f < MT; ++f) p[0][f] = read_p(f, 0, 0);
#pragma unroll
    for (int f = 0; f < NT; ++f) q[0][f] = read_q(f, 0, 0);
    int ps = 0, qs = 0, p_to = S;  // the stage's slots, and with PX where P's next loads go
    // Stores of the tile before count as loads do, and are later than the loads of this tile's first S stages.
    constexpr int STORES = MT * NT / 2;
    static_assert(LEFT + STORES <= 63, "the counter's range");
    int behind = 0;  // stages whose loads they are behind
    // One slice of a turn's stage. Among its matrix instructions, one behind each, stand the reads of the next slice's
    // fragments, over the first three quarters, so that they are there when it begins, and the loads: a wavefront issues
    // in order, and two such in a row would take longer than a matrix instruction and leave its unit idle.
    constexpr int STEPS = MT * NT, READS = MT + NT, EARLY = STEPS * 3 / 4;
    // which: the stage's first or its last, and which set of fragments is multiplied.
    auto slice = [&](auto which) {
        constexpr int w = decltype(which)::value, last = w;
        constexpr int next_t = last ? 0 : 1;
        constexpr int PL = PX != last ? P::kLoads : 0, QL = last ? Q::kLoads : 0, LOADS = PL + QL;
        const int pn = last ? (ps + 1 == S + PX ? 0 : ps + 1) : ps, qn = last ? (qs + 1 == S ? 0 : qs + 1) : qs;
        source from_p, from_q;
        if constexpr (PL > 0) from_p = source_p();
        if constexpr (QL > 0) from_q = source_q();
        if constexpr (last) {
            if (behind > 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT + STORES) : "memory");
            else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            --behind;
        }
        unrolled<STEPS>([&](auto step) {
            constexpr int s = decltype(step)::value, i = s / NT, j = s % NT;
            acc[i][j] = dense_mfma<T>(q[w][j], p[w][i], acc[i][j]);
            unrolled<READS>([&](auto read) {
                constexpr int f = decltype(read)::value;
                if constexpr (f * EARLY / READS == s) {
                    if constexpr (f < NT) q[w ^ 1][f] = read_q(f, qn, next_t);
                    else p[w ^ 1][f - NT] = read_p(f - NT, pn, next_t);
                }
            });
            unrolled<LOADS>([&](auto load) {
                constexpr int l = decltype(load)::value;
                if constexpr (std::min(l * STEPS / LOADS + 1, STEPS - 1) == s) {
                    if constexpr (l < PL) issue_p(from_p, load, PX ? p_to : ps);
                    else issue_q(from_q, std::integral_constant<int, l - PL>{}, qs);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (last) {
            p_to = ps;
            ps = pn, qs = qn;
            load_next();
        }
    };
    constexpr std::integral_constant<int, 0> zero{};
    constexpr std::integral_constant<int, 1> one{};
    // Tile i's sums to memory. Returns whether exactly STORES stores were issued.
    auto finish_tile = [&](int i_tile) {
        const tile t = take(i_tile);
        // Kept from the compiler, which would hold every lane's offsets in registers throughout the main loop.
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int col16 = lane & 15, kq = lane >> 4;
        if constexpr (SPLITS) {
            if (a.partial != nullptr) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int r = (wm * MT + i) * 16 + col16;
                    i32x4_t* to = a.partial + ((static_cast<int64_t>(blockIdx.y) * a.rows + t.row0 + r) * a.quads + (t.col0 >> 2));
                    if (r < t.rows)
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const int quad = (wn * NT + j) * 4 + kq;
                            if ((t.col0 >> 2) + quad < a.quads) to[quad] = acc[i][j];
                        }
                }
                return false;
            }
        }
        const int c0 = t.col0 + wn * NT * 16;
        uint16_t* y = a.y + (MODE == kByRanges ? t.expert * static_cast<int64_t>(a.rows) * a.cols : 0) + static_cast<int64_t>(t.row0) * a.cols;
        const float* scales = T == kInt8 ? a.q_scale + static_cast<int64_t>(t.expert) * a.cols : nullptr;
        auto value = [&](int i, int j, const f32x4_t& channel, float token) {
            if constexpr (T == kInt8) return dense_scaled(acc[i][j], channel, token);
            else return acc[i][j];
        };
        auto store = [&](auto bf16) {
            constexpr bool BF16 = decltype(bf16)::value;
            if (!a.lines) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int r = (wm * MT + i) * 16 + col16;
                    if (r >= t.rows) continue;
                    const float token = T == kInt8 && !t.rest ? a.p_scale[t.row0 + r] : 0.f;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int col = c0 + j * 16 + 4 * kq;
                        const f32x4_t channel = T == kInt8 ? dense_channels(scales, col, t.rest ? 0 : a.cols) : f32x4_t{};
                        dense_store4<BF16>(y + static_cast<int64_t>(r) * a.cols, col, a.cols, a.wide, value(i, j, channel, token));
                    }
                }
                return;
            }
            // A lane has four columns of one row. Lanes 16 apart exchange theirs between two products, so that each has eight
            // neighbouring ones and four lanes 64 bytes of a row. Past the tile's rows and the columns nothing is stored.
            const __amdgpu_buffer_rsrc_t yr = make_rsrc(y, static_cast<uint32_t>(t.rows) * a.cols * 2);
            f32x4_t channel[NT];
            float token[MT];
            if constexpr (T == kInt8) {
                const __amdgpu_buffer_rsrc_t cr = make_rsrc(scales, t.rest ? 0u : static_cast<uint32_t>(a.cols) * 4);
                const __amdgpu_buffer_rsrc_t tr = make_rsrc(a.p_scale + t.row0, t.rest ? 0u : static_cast<uint32_t>(t.rows) * 4);
#pragma unroll
                for (int j = 0; j < NT; ++j) channel[j] = __builtin_bit_cast(f32x4_t, buffer_load16(cr, (c0 + j * 16 + 4 * kq) * 4));
#pragma unroll
                for (int i = 0; i < MT; ++i) token[i] = __uint_as_float(buffer_load_u32(tr, ((wm * MT + i) * 16 + col16) * 4, 0));
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int r = (wm * MT + i) * 16 + col16;
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    const uint2 even = dense_pack<BF16>(value(i, j, channel[j], token[i])), odd = dense_pack<BF16>(value(i, j + 1, channel[j + 1], token[i]));
                    const auto lo = __builtin_amdgcn_permlane16_swap(even.x, odd.x, false, false);
                    const auto hi = __builtin_amdgcn_permlane16_swap(even.y, odd.y, false, false);
                    const int col = c0 + (j + (kq & 1)) * 16 + (kq >> 1) * 8;
                    __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{lo[0], hi[0], lo[1], hi[1]}, yr, col < a.cols ? (r * a.cols + col) * 2 : kOOB, 0, 0);
                }
            }
        };
        if constexpr (T == kBf16) store(std::true_type{});
        else if constexpr (T == kFp16) store(std::false_type{});
        else if (a.bf16) store(std::true_type{});
        else store(std::false_type{});
        return a.lines;
    };
    for (int t = 0;;) {
        for (int turn = take(t).stages; turn > 0; --turn) {
            slice(zero);
            slice(one);
        }
        if (t + 1 == tiles) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // requests past the end
        behind = finish_tile(t) ? S - 1 : 0;
        if (++t == tiles) return;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
    }
}

template <dense_type T, dense_mode MODE, bool PC, bool QC, int WM, int WN, int MT, int NT, int S, int PX>
void launch_tile(const dense_product& p, hipStream_t s) {
    constexpr int BM = WM * MT * 16, BN = WN * NT * 16;
    dense_args a = make_dense_args(p, PC, QC);
    a.band = 8;
    a.n_blocks = static_cast<int>(ceil_div(p.cols, BN));
    a.m_blocks = static_cast<int>(dense_row_blocks(p, MODE, BM));
    const int64_t tiles = int64_t{1} * a.m_blocks * a.n_blocks * (MODE == kByRanges ? p.experts : 1);
    // As many workgroups as are resident at once, which is in whole rounds of the XCDs, or as there are tiles.
    constexpr int LDS = 128 * ((S + PX) * BM + S * BN);
    const int64_t resident = ceil_div(int64_t{cu_count()} * (2 * LDS <= 160 * 1024 ? 2 : 1), 8) * 8;
    dim3 grid(static_cast<unsigned>(dense_grid(tiles, resident, MODE == kByRanges)));
    if (T == kInt8 && MODE == kDense && p.plan.splits > 1) {
        grid.y = static_cast<unsigned>(p.plan.splits);
        a.split_stages = static_cast<int>(ceil_div(ceil_div(p.depth, 128), p.plan.splits));
        a.partial = p.partial;
    } else {
        a.split_stages = 1 << 20;
    }
    dense_tile_kernel<T, MODE, PC, QC, WM, WN, MT, NT, S, PX><<<grid, WM * WN * 64, 0, s>>>(a);
}

template <dense_type T, dense_mode MODE, bool PC, bool QC> void launch_shape(const dense_product& p, hipStream_t s) {
    switch (p.plan.shape) {
        case 0: return launch_tile<T, MODE, PC, QC, 2, 4, 8, 4, 2, 1>(p, s);
        case 1: return launch_tile<T, MODE, PC, QC, 2, 4, 4, 4, 3, 0>(p, s);
        case 2: return launch_tile<T, MODE, PC, QC, 2, 2, 4, 4, 5, 0>(p, s);
        case 3: return launch_tile<T, MODE, PC, QC, 2, 2, 4, 4, 2, 0>(p, s);
        case 4: return launch_tile<T, MODE, PC, QC, 2, 2, 2, 4, 3, 0>(p, s);
        default: return launch_tile<T, MODE, PC, QC, 2, 2, 2, 2, 4, 0>(p, s);
    }
}

}  // namespace

}  // namespace plm
