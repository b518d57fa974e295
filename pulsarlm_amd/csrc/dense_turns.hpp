// Which tiles a workgroup of dense_tiles.hpp takes: whole numbers only, the same on the device, in the launch, and in a program
// that goes through them on the host.
#pragma once

#include <cstdint>

namespace plm {

// Workgroups of a launch of `tiles`, of which `resident` (a multiple of 8) are on the GPU at once: each keeps count of up
// to 64 tiles. XCDs are gone round by id, 8 at a time. Back and forth in whole rounds of them, which dense_place counts on:
// of a launch of few tiles the workgroups past the last one have no turn.
constexpr int64_t dense_grid(int64_t tiles, int64_t resident, bool back_and_forth) {
    const int64_t most = (tiles + 511) / 512 * 8, each = resident > most ? resident : most;
    return tiles >= each ? each : back_and_forth ? (tiles + 7) / 8 * 8 : tiles;
}
// Workgroup `self`'s place in turn `turn` of the grid's `each`. Back and forth, so that those who had the longest tiles of
// one turn have the shortest of the next, each on its XCD; `each` is a multiple of 8 then.
constexpr int dense_place(int turn, int each, int self, bool back_and_forth) {
    return back_and_forth && (turn & 1) ? each - 8 - (self & ~7) + (self & 7) : self;
}
// How many tiles it takes. Its tile in a turn is dense_place(...) past the turn's first, turn * each.
constexpr int dense_turns(int tiles, int each, int self, bool back_and_forth) {
    const int whole = tiles / each;
    return whole + (tiles - whole * each > dense_place(whole, each, self, back_and_forth) ? 1 : 0);
}

// Tile `id` of block_tiles = m_blocks * n_blocks: ids go round the XCDs, each of which takes one run of the tiles, ordered in
// bands of `band` row blocks, row block fastest, so that an XCD's L2 holds what its tiles share.
struct dense_block {
    int mb, nb;
};
constexpr dense_block dense_block_of(int id, int m_blocks, int n_blocks, int band) {
    const int block_tiles = m_blocks * n_blocks, xcd = id & 7, extra = block_tiles & 7;
    const int lin = xcd * (block_tiles >> 3) + (xcd < extra ? xcd : extra) + (id >> 3);
    const int band0 = lin / (band * n_blocks) * band;
    const int band_rows = band < m_blocks - band0 ? band : m_blocks - band0, in_band = lin - band0 * n_blocks;
    const int nb = in_band / band_rows;
    return {band0 + in_band - nb * band_rows, nb};
}

}  // namespace plm
