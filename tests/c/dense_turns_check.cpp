// Every tile of a launch of the tile kernel exactly once (pulsarlm_amd/csrc/dense_turns.hpp): goes through the workgroups and
// turns of launches of m_blocks x n_blocks tiles for each of `experts` (back and forth) or of one product, and prints how many
// launches it went through, tiles outside, tiles that no workgroup takes and tiles taken again.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../pulsarlm_amd/csrc/dense_turns.hpp"

int main() {
    long launches = 0, outside = 0, left = 0, again = 0;
    std::vector<int> taken;
    auto launch = [&](int m_blocks, int n_blocks, int experts, long resident, bool back_and_forth) {
        ++launches;
        const int block_tiles = m_blocks * n_blocks, tiles = block_tiles * experts;
        const int each = static_cast<int>(plm::dense_grid(tiles, resident, back_and_forth));
        taken.assign(tiles, 0);
        for (int self = 0; self < each; ++self) {
            const int turns = plm::dense_turns(tiles, each, self, back_and_forth);
            if (turns > 64) ++outside;
            for (int turn = 0; turn < turns; ++turn) {
                const int id = turn * each + plm::dense_place(turn, each, self, back_and_forth);
                if (id < 0 || id >= tiles) {
                    ++outside;
                    continue;
                }
                const plm::dense_block at = plm::dense_block_of(id % block_tiles, m_blocks, n_blocks, 8);
                if (at.mb < 0 || at.mb >= m_blocks || at.nb < 0 || at.nb >= n_blocks) ++outside;
                else ++taken[(id / block_tiles * m_blocks + at.mb) * n_blocks + at.nb];
            }
        }
        for (int t : taken) left += t == 0, again += t > 1;
    };
    for (bool back_and_forth : {false, true})
        for (long resident : {8, 256, 304, 512}) {
            for (int tiles = 1; tiles <= 1100; ++tiles) {
                launch(tiles, 1, 1, resident, back_and_forth);
                launch(1, tiles, 1, resident, back_and_forth);
            }
            for (int experts = 1; experts <= 130; ++experts)
                for (int m_blocks = 1; m_blocks <= 11; ++m_blocks)
                    for (int n_blocks : {1, 2, 5, 9}) launch(m_blocks, n_blocks, experts, resident, back_and_forth);
            launch(183, 183, 1, resident, back_and_forth);
            launch(3, 7, 4096, resident, back_and_forth);
        }
    std::printf("%ld %ld %ld %ld\n", launches, outside, left, again);
    return 0;
}
