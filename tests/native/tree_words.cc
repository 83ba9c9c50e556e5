// Walks the nodes' stages of every tree attention kernel on the host, for every number of nodes, as the kernel does: the word of a
// node's ancestors that a tile reads lies among the row's own `words`, so that the last row's lies inside the array, and a tile that has a node
// has the word of it. Exit code 0 and "ok <tiles>" on success.
#include <cstdint>
#include <cstdio>

#include "tree_stage.h"

struct half_t { uint16_t bits; };

static long g_tiles = 0, g_bad = 0;

template <typename T, int NT, int RT, int K16, int NW, int KG>
static void walk(const char* name) {
    using St = Stage<T, NT, K16, NW, KG>;
    constexpr int KEYS = Shape<T, NT, K16>::KEYS;
    for (int nodes = 1; nodes <= 256; ++nodes) {
        const int words = (nodes + 63) / 64;
        for (int tile = 0; tile < (nodes + St::KEYS - 1) / St::KEYS; ++tile)
            for (int turn = 0; turn < St::TURNS; ++turn)
                for (int kg = 0; kg < KG; ++kg) {
                    const int at0 = tile * St::KEYS + (turn * KG + kg) * KEYS, word = word_of_nodes(at0, nodes);
                    ++g_tiles;
                    if (word >= words || (at0 < nodes && word != at0 / 64)) {
                        if (g_bad++ < 20) std::fprintf(stderr, "%s<%d,%d,%d,%d,%d>: %d nodes, %d words: the tile at %d reads word %d\n", name, NT, RT, K16, NW, KG, nodes, words, at0, word);
                    }
                }
    }
}

int main() {
#define WALK_BF16(N, R, K, W, G) walk<half_t, N, R, K, W, G>("bf16");
#define WALK_F32(N, R, K, W, G) walk<float, N, R, K, W, G>("f32");
    TREE_BF16_KERNELS(WALK_BF16)
    TREE_F32_KERNELS(WALK_F32)
    if (g_bad != 0) {
        std::fprintf(stderr, "%ld of %ld tiles\n", g_bad, g_tiles);
        return 1;
    }
    std::printf("ok %ld\n", g_tiles);
    return 0;
}
