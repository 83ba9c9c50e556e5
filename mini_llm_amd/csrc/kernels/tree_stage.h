// How tree attention's keys come in stages and tiles, and which words of a node's ancestors a tile needs. Plain arithmetic, which the host can walk too.
#pragma once

#include <algorithm>

// The kernels that there are, as (KERNEL, ONE, TWO) calls KERNEL(NT, RT, 16-key groups of a tile, wavefronts, key groups): of 16 RT rows a wavefront, for heads of
// more than 16 NT, up to 32 NT columns (NT = 1: from the first). 16-key groups of a tile: as many as the registers hold beside the outputs where few wavefronts
// share the keys, so that there is independent work for the latencies from keys to outputs; where many do, as few as one product takes (ONE), so that a stage is not too large.
#define TREE_NARROW_KERNELS(KERNEL, N, ONE, TWO) \
    KERNEL(N, 1, ONE, 4, 4) KERNEL(N, 1, ONE, 8, 4) KERNEL(N, 1, TWO, 8, 2) KERNEL(N, 2, ONE, 8, 2) KERNEL(N, 2, ONE, 8, 1)
#define TREE_COMMON_KERNELS(KERNEL, ONE, TWO) \
    TREE_NARROW_KERNELS(KERNEL, 1, ONE, TWO) TREE_NARROW_KERNELS(KERNEL, 2, ONE, TWO) \
    KERNEL(4, 1, ONE, 2, 2) KERNEL(4, 1, ONE, 4, 2) KERNEL(4, 1, ONE, 8, 2) KERNEL(8, 1, ONE, 1, 1) KERNEL(8, 1, ONE, 2, 1) KERNEL(8, 1, ONE, 4, 1)
#define TREE_BF16_KERNELS(KERNEL) TREE_COMMON_KERNELS(KERNEL, 2, 4) KERNEL(4, 2, 2, 8, 2) KERNEL(4, 2, 2, 8, 1)
#define TREE_F32_KERNELS(KERNEL) TREE_COMMON_KERNELS(KERNEL, 1, 2) KERNEL(4, 1, 1, 8, 1)

// Sizes of a tile. A row has a power of two of columns in LDS, so that whole rows fill a load instruction; narrower heads leave some of them unused (96
// columns as 128: 1.5 times as fast as rows packed without a gap).
template <typename T, int NT, int KEY_GROUPS_OF_16>
struct Shape {
    static constexpr int KT = KEY_GROUPS_OF_16;            // 16-key groups of a tile (bfloat16: a product step of values takes two)
    static constexpr int KEYS = 16 * KT;
    static constexpr int CH = NT * sizeof(T) / 2;          // 64-byte pieces of a row
    static constexpr int PER = 4 / sizeof(T);              // elements of a word
    static constexpr int TILES = 2 * NT;                   // 16-column tiles of the output
    static constexpr int LEAST = NT / 2;                   // heads are wider than 32 LEAST
    static_assert((NT & (NT - 1)) == 0, "a power of two");
    static constexpr int BLOCK = std::min(CH, 4);          // 32 bits: words of a value row that lie together in a lane
    static constexpr int WORDS = 4 * KT / PER;             // words of a lane's keys in a column
    static_assert(64 % KEYS == 0, "a tile of nodes lies in one word of their ancestors");
};

template <typename T, int NT, int K16, int NW, int KG>
struct Stage {
    using S = Shape<T, NT, K16>;
    static constexpr int ROW = S::CH * 64, PIECES = 4 * S::CH, LEAST = S::KEYS * KG;      // a key group has one tile of a stage at least
    static constexpr int keys() {          // 24 KB of keys and values at least, in whole instructions of all wavefronts
        int n = LEAST;
        while (n * 2 * ROW < 24576 || n * PIECES % (64 * NW) != 0) n *= 2;
        return n;
    }
    static constexpr int KEYS = keys();
    static constexpr int TURNS = KEYS / LEAST;                            // tiles of a key group in a stage
    static constexpr int MATRIX = KEYS * ROW, BYTES = 2 * MATRIX;
    static constexpr int NUMBER = 4;          // of stages in LDS: one is read, the next has come, the others are on their way
    static_assert(NUMBER * BYTES <= 131072, "beside the table and the states");
    static constexpr int LOADS = KEYS * PIECES / 64 / NW;                 // of a wavefront, a stage and matrix
    static_assert(LOADS * 64 * NW == KEYS * PIECES, "whole instructions");
    static constexpr int MINE = KEYS / NW, PER_LOAD = 64 / PIECES;        // rows of a wavefront (it loads these), rows of a load instruction
    static_assert(MINE <= 64 && KEYS % NW == 0, "a bit a row");
};

// The word of a node's ancestors that a tile of the nodes from `at0` on needs; -1: no node is in it. (A stage has up to 256 keys whatever the
// nodes: a tile behind the last of them has no word either, where the word at its place lies behind the row's, and the last row's behind the array.)
constexpr int word_of_nodes(int at0, int nodes) { return at0 < nodes ? at0 / 64 : -1; }
