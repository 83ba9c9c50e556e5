// Attention of drafted trees over the paged cache, for gfx950. Node t of sequence b (rows cu_q[b] to cu_q[b + 1] of the step) sees the
// sequence's cached positions j < cached[b], whose keys and values lie in the pages, and of the sequence's own nodes those whose bit is set
// in ancestors[t]; their keys and values lie in the step's rows. With a window, what stands at positions[t] - window or in front of it is not
// seen. With z_j = scale q_t . k_j over what is seen:
//   o_t = sum_j exp(z_j - max z) v_j / sum_j exp(z_j - max z),   a node that sees nothing gets zeros.
// What is not seen counts for nothing whatever stands there (infinities and NaN among it), and a block table's entry that names no page of
// the pool holds nothing that is seen.
//
// All nodes of a sequence and all query heads of a key/value head read the same keys, so these are the rows of one product: a workgroup
// has 16 RT of them (row r is node r / group, head r % group of the key head's), and its wavefronts take the key tiles in turn, each
// with all rows. Keys and values then go from memory straight into the registers that the matrix instructions read, each once a
// workgroup, and nothing but the few page rows of a tile passes through LDS until the wavefronts' states meet at the end.
//
// As in prompt attention everything is transposed, so that a lane owns one query row of each 16:
//   S^T = K Q^T   the lane with row c, group G (lane = 16 G + c) loads key c of each 16, 16 bytes at 64 i + 16 G of its row: the product's k
//                 index runs over the columns in an order of its own, the same for queries and keys;
//   O^T = V^T P^T the lane has the weights of keys 4 G .. 4 G + 3 of each 16 from the first product, in the place where the second wants
//                 them. As the other operand it loads, of just these keys, 16 (8, 4) bytes at the same place c of a block of 256 (128, 64) bytes:
//                 column m of the product's tile x is column E m + x of the block, E elements to 16 bytes. In 32 bits the loaded words are
//                 the operand; in bfloat16 a byte permutation joins two keys' halves, one instruction a register, shared by all rows.
// Softmax statistics, sums and outputs are fp32; the weights are rounded to the values' type for the second product (in bfloat16: by half a step,
// which averages over the keys; the sum is over the weights before they are rounded).
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct TreeAttentionParams {
    const char *q, *k, *v, *k_pages, *v_pages;
    long long ldq, ldk, ldv, ldo;                 // bytes between rows
    unsigned page_pitch;                          // bytes between rows of the pages
    const int *block_tables, *cached, *cu_q, *positions;
    const unsigned long long* ancestors;
    int n_seqs, max_blocks, tokens, words, n_heads, n_kv_heads, head_dim, page_size, n_pages, window, max_new;
    unsigned page_magic;                          // at / page_size = (at * page_magic) >> page_shift for 0 <= at < 2^31
    int page_shift;
    int row_tiles, nsplit, units;
    float scale_log2e;
    char* out;
    float* ws;
};

// Sizes of a kernel for heads of more than 32 (NT - 1), up to 32 NT columns (less for the NT that stand for two).
template <typename T, int NT>
struct Shape {
    static constexpr int KT = sizeof(T) == 2 ? 2 : 1;      // 16-key groups of a tile: one product step of values takes 32 keys in bfloat16
    static constexpr int KEYS = 16 * KT;
    static constexpr int CH = NT * sizeof(T) / 2;          // 64-byte pieces of a row; words of a value row in a lane
    static constexpr int PER = 4 / sizeof(T);              // elements of a word
    static constexpr int TILES = 2 * NT;                   // 16-column tiles of the output
    static constexpr int LEAST = NT == 6 ? 4 : NT == 8 ? 6 : NT - 1;       // heads are wider than 32 LEAST
    // of word w: the first word of its block (of 4, 2 or 1 words a lane) and the block's words
    static constexpr int block_words(int w) { return w < CH / 4 * 4 ? 4 : w < CH / 2 * 2 ? 2 : 1; }
    static constexpr int block_first(int w) { return w / block_words(w) * block_words(w); }
};

// Ones (1 in the lowest bit of each element) where a word's elements are not finite. In whole-number arithmetic on all elements of the word at
// once: as comparisons, the lanes' answers to all words of a tile fill the scalar registers several times over.
__device__ __forceinline__ uint32_t not_finite(uint32_t w, float) { return ((w & 0x7f800000u) + 0x00800000u) >> 31; }
__device__ __forceinline__ uint32_t not_finite(uint32_t w, bf16_t) { return ((w & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u; }
// kind 0: the elements that are finite, zeros for the others; 1, 2, 3: one where the element is NaN, +inf, -inf, else 0.
__device__ __forceinline__ uint32_t sifted(uint32_t w, int kind, float) {
    const uint32_t special = not_finite(w, 0.f), mantissa = (w & 0x7fffffu) + 0x7fffffu >> 23, sign = w >> 31;
    if (kind == 0) return w & (special - 1);
    return (special & (kind == 1 ? mantissa : ~mantissa & (kind == 2 ? ~sign : sign))) * 0x3f800000u;
}
__device__ __forceinline__ uint32_t sifted(uint32_t w, int kind, bf16_t) {
    const uint32_t special = not_finite(w, bf16_t{}), mantissa = (w & 0x007f007fu) + 0x007f007fu >> 7, sign = w >> 15;
    if (kind == 0) return w & ~(special * 0xffffu);
    return (special & (kind == 1 ? mantissa : ~mantissa & (kind == 2 ? ~sign : sign))) * 0x3f80u;
}

template <typename T, int NT, int RT, int MAXW>
__global__ void __launch_bounds__(MAXW * 64) tree_attention_kernel(TreeAttentionParams a) {
    using S = Shape<T, NT>;
    constexpr int KT = S::KT, KEYS = S::KEYS, CH = S::CH, TILES = S::TILES, DIMS = 32 * NT, PITCH = DIMS + 4;
    extern __shared__ __attribute__((aligned(16))) float state_s[];       // [wavefront][16 RT][PITCH], then maxima and sums
    __shared__ int row_s[MAXW][KEYS];

    // Workgroups that share keys have numbers 8 apart, so that they run on one XCD and the second finds the keys in its L2.
    const int residue = blockIdx.x % 8, rest = blockIdx.x / 8;
    const int unit = rest / a.row_tiles * 8 + residue, row_tile = rest % a.row_tiles;
    if (unit >= a.units) return;
    const int split = unit % a.nsplit, hk = unit / a.nsplit % a.n_kv_heads, b = unit / a.nsplit / a.n_kv_heads;
    const int group = a.n_heads / a.n_kv_heads;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, n_waves = blockDim.x / 64;
    const int G = lane / 16, c16 = lane % 16;

    const int first = min(max(a.cu_q[b], 0), a.tokens);
    const int nodes = min(min(max(a.cu_q[b + 1] - first, 0), a.tokens - first), a.max_new);
    const int rows = nodes * group, row0 = row_tile * 16 * RT;
    if (row0 >= rows) return;
    const int cached = static_cast<int>(min(min(static_cast<long long>(max(a.cached[b], 0)), static_cast<long long>(a.max_blocks) * a.page_size), INT32_MAX - 64ll));
    const int row_bytes = a.head_dim * static_cast<int>(sizeof(T));
    const int* table = a.block_tables + static_cast<size_t>(b) * a.max_blocks;

    // The lane's query row of each 16 (beyond the last: zeros, never written).
    uint4 q[RT][CH];
    int low[RT], token[RT];
    int low_least = INT32_MAX, low_most = INT32_MIN;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(row0 + 16 * rt + c16, rows - 1), node = r / group;
        token[rt] = first + node;
        const char* at = a.q + token[rt] * a.ldq + (hk * group + r - node * group) * row_bytes;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int off = 64 * c + 16 * G;
            const bool in = off < row_bytes;
            q[rt][c] = *reinterpret_cast<const uint4*>(at + (in ? off : 0));
            if (!in) q[rt][c] = make_uint4(0, 0, 0, 0);
        }
        low[rt] = a.window > 0 ? a.positions[token[rt]] - a.window + 1 : INT32_MIN;
        low_least = min(low_least, low[rt]);
        low_most = max(low_most, low[rt]);
    }
    int first_tile = 0;
    if (a.window > 0) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            low_least = min(low_least, __shfl_xor(low_least, off, 64));
            low_most = max(low_most, __shfl_xor(low_most, off, 64));
        }
        low_least = __builtin_amdgcn_readfirstlane(low_least);
        low_most = __builtin_amdgcn_readfirstlane(low_most);
        first_tile = min(max(low_least, 0), cached) / KEYS;
    }

    // Tiles: those of the cache from first_tile on, then the nodes'. A split has `per` neighbouring ones.
    const int cache_tiles = (cached + KEYS - 1) / KEYS - first_tile, all_tiles = cache_tiles + (nodes + KEYS - 1) / KEYS;
    const int per = (all_tiles + a.nsplit - 1) / a.nsplit, begin = split * per, end = min(all_tiles, begin + per);
    const bool whole_pages = a.page_size % 16 == 0;        // 16 neighbouring keys lie in one page

    f32x4 o[TILES][RT];
    float m[RT], ref[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY; ref[rt] = 0.f; l[rt] = 0.f;
#pragma unroll
        for (int x = 0; x < TILES; ++x) o[x][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // Asks for the page of this lane's key of a tile (of a tile of nodes, or beyond the last: some entry, not used).
    const int key = lane % KEYS;
    auto block_of = [&](int at) { return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(at)) * a.page_magic) >> a.page_shift); };
    auto ask_entry = [&](int tile) { return table[min(block_of((max(min(tile, cache_tiles - 1), 0) + first_tile) * KEYS + key), a.max_blocks - 1)]; };
    struct Tile {
        uint4 k[KT][CH];
        uint32_t v[4 * KT][CH];
        unsigned valid;          // a bit a key
    };
    const char* k_head = a.k_pages + static_cast<size_t>(hk) * row_bytes;
    const char* v_head = a.v_pages + static_cast<size_t>(hk) * row_bytes;
    // Asks for a tile's keys and values. All loads are unconditional (keys that are not seen read some row that exists).
    auto ask = [&](int tile, int entry, Tile& t) {
        const bool of_nodes = tile >= cache_tiles;
        int row;
        bool there;
        if (of_nodes) {
            const int j = (tile - cache_tiles) * KEYS + key;
            there = j < nodes;
            row = first + min(j, nodes - 1);
        } else {
            const int at = (tile + first_tile) * KEYS + key;
            there = at < cached && static_cast<unsigned>(entry) < static_cast<unsigned>(a.n_pages);
            row = there ? entry * a.page_size + at - block_of(at) * a.page_size : 0;
        }
        t.valid = static_cast<unsigned>(__ballot(there && lane < KEYS));
        const char *kb = of_nodes ? a.k + static_cast<size_t>(hk) * row_bytes : k_head, *vb = of_nodes ? a.v + static_cast<size_t>(hk) * row_bytes : v_head;
        const char *kp[KT], *vp[4 * KT];
        if (whole_pages && !of_nodes && t.valid == (KEYS == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const size_t base = static_cast<size_t>(__builtin_amdgcn_readlane(row, 16 * kt)) * a.page_pitch;
                kp[kt] = kb + base + c16 * a.page_pitch;
#pragma unroll
                for (int i = 0; i < 4; ++i) vp[4 * kt + i] = vb + base + (4 * G + i) * a.page_pitch;
            }
        } else {
            const size_t k_pitch = of_nodes ? a.ldk : a.page_pitch, v_pitch = of_nodes ? a.ldv : a.page_pitch;
            if (lane < KEYS) row_s[wave][lane] = row;
            wave_lds_sync();
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                kp[kt] = kb + row_s[wave][16 * kt + c16] * k_pitch;
#pragma unroll
                for (int i = 0; i < 4; ++i) vp[4 * kt + i] = vb + row_s[wave][16 * kt + 4 * G + i] * v_pitch;
            }
            wave_lds_sync();
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int off = 64 * c + 16 * G;
                const bool check = 64 * (c + 1) > 32 * S::LEAST * static_cast<int>(sizeof(T));
                t.k[kt][c] = *reinterpret_cast<const uint4*>(kp[kt] + (!check || off < row_bytes ? off : 0));
            }
#pragma unroll
        for (int j = 0; j < 4 * KT; ++j)
#pragma unroll
            for (int w = 0; w < CH; w += S::block_words(w)) {
                const int off = 64 * w + 4 * S::block_words(w) * c16;
                const char* p = vp[j] + (off < row_bytes ? off : 0);
                if (S::block_words(w) == 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p);
                    t.v[j][w] = x.x; t.v[j][w + 1] = x.y; t.v[j][w + 2] = x.z; t.v[j][w + 3] = x.w;
                } else if (S::block_words(w) == 2) {
                    const uint2 x = *reinterpret_cast<const uint2*>(p);
                    t.v[j][w] = x.x; t.v[j][w + 1] = x.y;
                } else {
                    t.v[j][w] = *reinterpret_cast<const uint32_t*>(p);
                }
            }
    };

    // The second product: into(x, rt, product) for every tile x of columns and 16 rows. With `sift` of the values' elements of a kind (sifted), and
    // for kinds 1 to 3 with ones in place of the weights.
    auto weigh = [&](const uint32_t (&v)[4 * KT][CH], const float (&p)[RT][4 * KT], auto sift, int kind, auto&& into) {
        constexpr bool SIFT = decltype(sift)::value;
        auto value = [&](int j, int w) { return SIFT ? sifted(v[j][w], kind, T{}) : v[j][w]; };
        auto weight = [&](int rt, int j) { return SIFT && kind > 0 ? (p[rt][j] == 0.f ? 0.f : 1.f) : p[rt][j]; };
        if constexpr (sizeof(T) == 2) {
            uint4 pb[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                pb[rt] = make_uint4(pack_bf16x2(weight(rt, 0), weight(rt, 1)), pack_bf16x2(weight(rt, 2), weight(rt, 3)), pack_bf16x2(weight(rt, 4), weight(rt, 5)),
                                    pack_bf16x2(weight(rt, 6), weight(rt, 7)));
#pragma unroll
            for (int w = 0; w < CH; ++w) {
                uint32_t vw[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) vw[j] = value(j, w);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t sel = e == 0 ? 0x05040100u : 0x07060302u;
                    const uint4 va = make_uint4(__builtin_amdgcn_perm(vw[1], vw[0], sel), __builtin_amdgcn_perm(vw[3], vw[2], sel),
                                                __builtin_amdgcn_perm(vw[5], vw[4], sel), __builtin_amdgcn_perm(vw[7], vw[6], sel));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        into(2 * w + e, rt, [&](f32x4 c) {
                            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, pb[rt]), c, 0, 0, 0);
                        });
                }
                if (SIFT) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int w = 0; w < CH; ++w) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    into(w, rt, [&](f32x4 c) {
#pragma unroll
                        for (int j = 0; j < 4 * KT; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, value(j, w)), weight(rt, j), c, 0, 0, 0);
                        return c;
                    });
                if (SIFT) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    auto take = [&](int tile, Tile& t) {
        const bool of_nodes = tile >= cache_tiles;
        const int at0 = of_nodes ? (tile - cache_tiles) * KEYS : (tile + first_tile) * KEYS;
        const bool all_seen = !of_nodes && t.valid == (KEYS == 32 ? 0xffffffffu : 0xffffu) && (a.window <= 0 || at0 >= low_most);
        // (columns behind the head's last: zero on both sides)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const bool check = 64 * (c + 1) > 32 * S::LEAST * static_cast<int>(sizeof(T));
                if (check && 64 * c + 16 * G >= row_bytes) t.k[kt][c] = make_uint4(0, 0, 0, 0);
            }
        float p[RT][4 * KT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    if constexpr (sizeof(T) == 2) {
                        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t.k[kt][c]), __builtin_bit_cast(bf16x8, q[rt][c]), s, 0, 0, 0);
                    } else {
                        const f32x4 kf = __builtin_bit_cast(f32x4, t.k[kt][c]), qf = __builtin_bit_cast(f32x4, q[rt][c]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[i], qf[i], s, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) p[rt][4 * kt + i] = s[i] * a.scale_log2e;
            }
        bool special = false;
        if (!all_seen) {
            unsigned mine = 0, odd = 0;       // which of the lane's keys exist; whether one of them holds what is not finite
#pragma unroll
            for (int j = 0; j < 4 * KT; ++j) {
                const unsigned there = t.valid >> (16 * (j / 4) + 4 * G + j % 4) & 1;
                mine |= there << j;
#pragma unroll
                for (int w = 0; w < CH; ++w) {
                    t.v[j][w] &= 0u - there;
                    odd |= not_finite(t.v[j][w], T{});
                }
            }
            special = __any(odd != 0);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                unsigned seen = mine;
                if (of_nodes) {
                    const unsigned bits = static_cast<unsigned>(a.ancestors[static_cast<size_t>(token[rt]) * a.words + at0 / 64] >> (at0 % 64)) >> (4 * G);
                    seen &= (bits & 15u) | (KT == 2 ? (bits >> 16 & 15u) << 4 : 0u);
                }
                if (a.window > 0)
#pragma unroll
                    for (int j = 0; j < 4 * KT; ++j) {
                        const int k = at0 + 16 * (j / 4) + 4 * G + j % 4;
                        const int at = of_nodes ? a.positions[first + min(k, nodes - 1)] : k;
                        seen &= ~((at < low[rt] ? 1u : 0u) << j);
                    }
#pragma unroll
                for (int j = 0; j < 4 * KT; ++j) p[rt][j] = seen >> j & 1 ? p[rt][j] : -INFINITY;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mx = p[rt][0];
#pragma unroll
            for (int j = 1; j < 4 * KT; ++j) mx = fmaxf(mx, p[rt][j]);
            mx = rows_max(mx);
            // The maximum that weights are taken against follows only when one lies 8 above it: weights then reach 2^8, which costs no
            // accuracy, and most tiles leave sum and outputs as they are.
            const bool more = mx > m[rt] + 8.f;
            if (__any(more)) {
                const float fix = more ? exp2_for<T>(m[rt] - mx) : 1.f;
                m[rt] = more ? mx : m[rt];
                ref[rt] = more ? mx : ref[rt];
                l[rt] *= fix;
#pragma unroll
                for (int x = 0; x < TILES; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[x][rt][i] *= fix;
            }
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4 * KT; ++j) {
                p[rt][j] = exp2_for<T>(p[rt][j] - ref[rt]);
                sum += p[rt][j];
            }
            l[rt] += sum;
        }
        auto add = [&](int x, int rt, auto&& product) { o[x][rt] = product(o[x][rt]); };
        if (!special) {
            weigh(t.v, p, std::false_type{}, 0, add);
            return;
        }
        // A tile of which some rows see less than others holds a value that is not finite: zero times it would reach those that do not see
        // it. The finite values are weighed as ever; whether a row gives weight to a NaN, +inf or -inf of a column is a product of ones and zeros.
        weigh(t.v, p, std::true_type{}, 0, add);
#pragma unroll 1
        for (int kind = 1; kind <= 3; ++kind) {
            const float value = kind == 1 ? __builtin_nanf("") : kind == 2 ? INFINITY : -INFINITY;
            weigh(t.v, p, std::true_type{}, kind, [&](int x, int rt, auto&& product) {
                const f32x4 count = product(f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int i = 0; i < 4; ++i) o[x][rt][i] += count[i] > 0.f ? value : 0.f;
            });
        }
    };

    // One tile is multiplied while the wavefront's next is on its way and the page of the one after it is asked for.
    {
        Tile t0, t1;
        int tile = begin + wave, entry = 0, entry1 = 0;
        if (tile < end) {
            entry = ask_entry(tile);
            entry1 = ask_entry(tile + n_waves);
            ask(tile, entry, t0);
        }
        while (tile < end) {
            const int next = tile + n_waves;
            entry = ask_entry(next + n_waves);
            if (next < end) ask(next, entry1, t1);
            take(tile, t0);
            if (next >= end) break;
            const int after = next + n_waves;
            entry1 = ask_entry(after + n_waves);
            if (after < end) ask(after, entry, t0);
            take(next, t1);
            tile = after;
        }
    }

    // The wavefronts' states meet in LDS; every thread merges some rows' columns in the wavefronts' order.
    float2* ml_s = reinterpret_cast<float2*>(state_s + n_waves * 16 * RT * PITCH);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = rows_sum(l[rt]);
        if (G == 0) ml_s[wave * 16 * RT + 16 * rt + c16] = make_float2(m[rt], sum);
        float* to = state_s + (wave * 16 * RT + 16 * rt + c16) * PITCH;
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
            const int w = x / S::PER, E = S::block_words(w) * S::PER, base = S::block_first(w) * 16 * S::PER, e = (w - S::block_first(w)) * S::PER + x % S::PER;
#pragma unroll
            for (int i = 0; i < 4; ++i) to[base + E * (4 * G + i) + e] = o[x][rt][i];
        }
    }
    __syncthreads();
    const int quads = a.head_dim / 4, count = min(16 * RT, rows - row0);
    for (int item = threadIdx.x; item < count * quads; item += blockDim.x) {
        const int r = item / quads, d = (item - r * quads) * 4;
        float top = -INFINITY, sum = 0.f;
        for (int w = 0; w < n_waves; ++w) top = fmaxf(top, ml_s[w * 16 * RT + r].x);
        const float against = top == -INFINITY ? 0.f : top;
        f32x4 v{0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < n_waves; ++w) {
            const float2 ml = ml_s[w * 16 * RT + r];
            const f32x4 part = *reinterpret_cast<const f32x4*>(state_s + (w * 16 * RT + r) * PITCH + d);
            const float weight = exp2_for<T>(ml.x - against);
            if (ml.y == 0.f) continue;          // (a wavefront whose keys nobody saw)
            sum += weight * ml.y;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += weight * part[i];
        }
        const int node = (row0 + r) / group, t = first + node, h = hk * group + row0 + r - node * group;
        if (a.nsplit == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            T* to = reinterpret_cast<T*>(a.out + t * a.ldo) + h * a.head_dim + d;
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = from_float<T>(v[i] * inv);
        } else {
            const size_t pair = (static_cast<size_t>(t) * a.n_heads + h) * a.nsplit + split;
            *reinterpret_cast<f32x4*>(a.ws + pair * a.head_dim + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(a.ws + static_cast<size_t>(a.tokens) * a.n_heads * a.nsplit * a.head_dim + 2 * pair) = make_float2(top, sum);
        }
    }
}

// Joins the splits' states. A workgroup has a node; a thread four columns of a head.
template <typename T>
__global__ void __launch_bounds__(256) tree_attention_join_kernel(TreeAttentionParams a) {
    const int b = blockIdx.y, node = blockIdx.x;
    const int first = min(max(a.cu_q[b], 0), a.tokens);
    if (node >= min(min(max(a.cu_q[b + 1] - first, 0), a.tokens - first), a.max_new)) return;
    const int t = first + node, quads = a.head_dim / 4;
    const float* state = a.ws + static_cast<size_t>(a.tokens) * a.n_heads * a.nsplit * a.head_dim;
    for (int item = blockIdx.z * 256 + threadIdx.x; item < a.n_heads * quads; item += gridDim.z * 256) {
        const int h = item / quads, d = (item - h * quads) * 4;
        const size_t pair = (static_cast<size_t>(t) * a.n_heads + h) * a.nsplit;
        float top = -INFINITY, sum = 0.f;
        for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, state[2 * (pair + s)]);
        const float against = top == -INFINITY ? 0.f : top;
        f32x4 v{0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.nsplit; ++s) {
            const float2 ml = *reinterpret_cast<const float2*>(state + 2 * (pair + s));
            const f32x4 part = *reinterpret_cast<const f32x4*>(a.ws + (pair + s) * a.head_dim + d);
            const float weight = exp2_for<T>(ml.x - against);
            if (ml.y == 0.f) continue;
            sum += weight * ml.y;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += weight * part[i];
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* to = reinterpret_cast<T*>(a.out + t * a.ldo) + h * a.head_dim + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = from_float<T>(v[i] * inv);
    }
}

// How a call is shared out: rows of a workgroup, wavefronts, workgroups that share a row's keys.
struct Plan {
    int nt, rt, waves, row_tiles, nsplit;
};

Plan plan_of(int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_new, int max_cached, int window, int dtype) {
    Plan p;
    p.nt = (head_dim + 31) / 32;
    if (p.nt == 5) p.nt = 6;
    if (p.nt == 7) p.nt = 8;
    const long long rows = static_cast<long long>(max_new) * (n_heads / n_kv_heads);
    p.rt = rows <= 16 ? 1 : rows <= 32 || p.nt > 4 || (dtype == MLLM_F32 && p.nt > 2) ? 2 : 4;
    if (dtype == MLLM_F32 && p.nt > 4) p.rt = 1;
    p.waves = p.rt == 4 || p.nt >= 4 || p.nt * p.rt >= 6 || (dtype == MLLM_F32 && p.nt > 2) ? 4 : 8;
    p.row_tiles = static_cast<int>((rows + 16 * p.rt - 1) / (16 * p.rt));
    const int keys = dtype == MLLM_F32 ? 16 : 32;
    const long long seen = window > 0 ? std::min<long long>(max_cached, static_cast<long long>(window) + max_new) : max_cached;
    const long long tiles = (seen + keys - 1) / keys + (max_new + keys - 1) / keys;
    const long long groups = static_cast<long long>(n_seqs) * n_kv_heads * p.row_tiles;
    p.nsplit = static_cast<int>(std::max<long long>(1, std::min<long long>({512 / groups, tiles / (4 * p.waves), 64})));
    return p;
}

template <typename T, int NT, int RT, int MAXW>
int launch(const TreeAttentionParams& p, int waves, hipStream_t stream) {
    const size_t lds = static_cast<size_t>(waves) * 16 * RT * ((32 * NT + 4) * 4 + 8);
    auto kernel = tree_attention_kernel<T, NT, RT, MAXW>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return static_cast<int>(e);
    const long long blocks = (static_cast<long long>(p.units) + 7) / 8 * 8 * p.row_tiles;
    if (blocks > INT32_MAX) return -1;
    kernel<<<static_cast<unsigned>(blocks), waves * 64, lds, stream>>>(p);
    return 0;
}

template <typename T>
int dispatch(const TreeAttentionParams& p, const Plan& plan, hipStream_t stream) {
#define TREE_CASE(N, R, W) if (plan.nt == N && plan.rt == R) return launch<T, N, R, W>(p, plan.waves, stream);
    if constexpr (sizeof(T) == 2) {
        TREE_CASE(1, 1, 8) TREE_CASE(1, 2, 8) TREE_CASE(1, 4, 4) TREE_CASE(2, 1, 8) TREE_CASE(2, 2, 8) TREE_CASE(2, 4, 4)
        TREE_CASE(3, 1, 8) TREE_CASE(3, 2, 4) TREE_CASE(3, 4, 4) TREE_CASE(4, 1, 4) TREE_CASE(4, 2, 4) TREE_CASE(4, 4, 4)
        TREE_CASE(6, 1, 4) TREE_CASE(6, 2, 4) TREE_CASE(8, 1, 4) TREE_CASE(8, 2, 4)
    } else {
        TREE_CASE(1, 1, 8) TREE_CASE(1, 2, 8) TREE_CASE(1, 4, 4) TREE_CASE(2, 1, 8) TREE_CASE(2, 2, 8) TREE_CASE(2, 4, 4)
        TREE_CASE(3, 1, 4) TREE_CASE(3, 2, 4) TREE_CASE(4, 1, 4) TREE_CASE(4, 2, 4) TREE_CASE(6, 1, 4) TREE_CASE(8, 1, 4)
    }
#undef TREE_CASE
    return -1;
}

}  // namespace

extern "C" {

// Floats of workspace for a call of these sizes.
long long mllm_tree_attention_ws_floats(int tokens, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_new, int max_cached, int window, int dtype) {
    const Plan plan = plan_of(n_seqs, n_heads, n_kv_heads, head_dim, max_new, max_cached, window, dtype);
    return plan.nsplit == 1 ? 0 : static_cast<long long>(tokens) * n_heads * plan.nsplit * (head_dim + 2);
}

// Returns 0, a HIP error code, or -1 for sizes the kernel refuses. Strides in elements.
int mllm_tree_attention(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* k_pages, const void* v_pages,
                        int n_pages, int page_size, const int* block_tables, int n_seqs, int max_blocks, const int* cached, const int* cu_q,
                        const unsigned long long* ancestors, int words, const int* positions, int tokens, int n_heads, int n_kv_heads, int head_dim,
                        float scale, int window, int max_new, int max_cached, void* out, long long ldo, float* ws, int dtype, hipStream_t stream) {
    if (tokens < 1 || n_seqs < 1) return 0;
    if (n_kv_heads < 1 || n_heads % n_kv_heads != 0 || head_dim < 8 || head_dim > 256 || head_dim % 8 != 0 || words < 1 || words > 4 || page_size < 1) return -1;
    if (static_cast<long long>(n_pages) * page_size > INT32_MAX || max_new < 1 || max_new > 64 * words) return -1;
    const Plan plan = plan_of(n_seqs, n_heads, n_kv_heads, head_dim, max_new, max_cached, window, dtype);
    const long long units = static_cast<long long>(n_seqs) * n_kv_heads * plan.nsplit;
    if (units > INT32_MAX / 8 || (plan.nsplit > 1 && (ws == nullptr || n_seqs > 65535))) return -1;
    const int esz = dtype == MLLM_F32 ? 4 : 2;
    int bits = 0;
    while ((1ll << bits) < page_size) ++bits;
    TreeAttentionParams p{};
    p.q = static_cast<const char*>(q); p.k = static_cast<const char*>(k); p.v = static_cast<const char*>(v);
    p.k_pages = static_cast<const char*>(k_pages); p.v_pages = static_cast<const char*>(v_pages);
    p.ldq = ldq * esz; p.ldk = ldk * esz; p.ldv = ldv * esz; p.ldo = ldo * esz;
    p.page_pitch = static_cast<unsigned>(n_kv_heads) * head_dim * esz;
    p.block_tables = block_tables; p.cached = cached; p.cu_q = cu_q; p.positions = positions; p.ancestors = ancestors;
    p.n_seqs = n_seqs; p.max_blocks = max_blocks; p.tokens = tokens; p.words = words; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
    p.head_dim = head_dim; p.page_size = page_size; p.n_pages = n_pages; p.window = window; p.max_new = max_new;
    p.page_shift = 31 + bits;
    p.page_magic = static_cast<unsigned>(((1ull << p.page_shift) + page_size - 1) / page_size);
    p.row_tiles = plan.row_tiles; p.nsplit = plan.nsplit; p.units = static_cast<int>(units);
    p.scale_log2e = scale * MLLM_LOG2E;
    p.out = static_cast<char*>(out); p.ws = ws;
    const int rc = dtype == MLLM_F32 ? dispatch<float>(p, plan, stream) : dispatch<bf16_t>(p, plan, stream);
    if (rc != 0) return rc;
    if (plan.nsplit > 1) {
        const dim3 grid(max_new, n_seqs, std::min(64, (n_heads * (head_dim / 4) + 255) / 256));
        if (dtype == MLLM_F32) tree_attention_join_kernel<float><<<grid, 256, 0, stream>>>(p);
        else tree_attention_join_kernel<bf16_t><<<grid, 256, 0, stream>>>(p);
    }
    MLLM_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
