// Attention of drafted trees over the paged cache, for gfx950. Node t of sequence b (rows cu_q[b] to cu_q[b + 1] of the step) sees the
// sequence's cached positions j < cached[b], whose keys and values lie in the pages, and of the sequence's own nodes those whose bit is set
// in ancestors[t]; their keys and values lie in the step's rows. With a window, what stands at positions[t] - window or in front of it is not
// seen. With z_j = scale q_t . k_j over what is seen:
//   o_t = sum_j exp(z_j - max z) v_j / sum_j exp(z_j - max z),   a node that sees nothing gets zeros.
// What is not seen counts for nothing whatever stands there (infinities and NaN among it), and a block table's entry that names no page of
// the pool holds nothing that is seen. What is seen counts as in the formula: a value that is not finite makes its column so in the rows that see it (NaN, where
// its weight is zero in 32 bits), and a row all of whose seen keys score -inf is NaN.
//
// All nodes of a sequence and all query heads of a key/value head read the same keys, so these are the rows of one product (row r is node r /
// group, head r % group of the key head's), of which a workgroup has up to 256. Keys and values come through LDS in four stages of 32 KB, loaded straight
// into it three stages ahead, so that what is on its way holds no register: 96 KB behind a request, of which 64 are still on their way when the next
// stage is read. A workgroup's wavefronts are row groups x key groups: each has 16 RT rows, and of every stage the keys of its key
// group; the key groups' states meet in LDS at the end. Few rows: one row group, many key groups, and memory is what bounds it; many rows: a
// stage is read by all row groups, and the matrix instructions are.
//
// As in prompt attention everything is transposed, so that a lane owns one query row of each 16:
//   S^T = K Q^T   the lane with row c, group G (lane = 16 G + c) takes key c of each 16, 16 bytes at 64 i + 16 G of its row: the product's k
//                 index runs over the columns in an order of its own, the same for queries and keys;
//   O^T = V^T P^T the lane has the weights of keys 4 G .. 4 G + 3 of each 16 from the first product, in the place where the second wants
//                 them, and takes the values of just these keys in 16 columns as the other operand. In bfloat16 these come out of LDS turned by
//                 the read itself; in 32 bits a lane reads 16 (8) bytes at the same place c of a block of 256 (128) bytes: column m of the
//                 product's tile x is column E m + x of the block, E words to a read.
// Softmax statistics, sums and outputs are fp32; the weights are rounded to the values' type for the second product. In bfloat16 that is half a step of each
// (2^-8), which averages over the keys; the sum is over the rounded weights, as a product of ones with them, so that a row whose values are all alike gets that value. In 32 bits
// nothing is rounded. (Weights kept in 32 bits would need the second product in 32 bits, at a sixteenth of the rate.)
//
// What bounds it, as measured in bfloat16 (a copy of 1 GiB reaches 5.2 TB/s, a product of 8,192 cubed 1.35 PFLOP/s):
//   64 nodes over 31,000 positions, 25 heads of 64: 45 us, 4.5 TB/s: memory, and the join of 8 splits behind it (4 us).
//   32 trees of up to 64 nodes over 4,096 to 8,192 positions, 32 query heads that share 8 of 128: 262 to 276 us by the machine, 0.59 PFLOP/s, 3.1 TB/s: what a unit has
//   to do for a tile, and units that are done: they are busy in 73% of the kernel's cycles (at 2.4 GHz), of which matrix instructions take 44%, softmax and addresses 34%; without
//   loads from memory it takes 4% less; with the longest sequences' ends shared out to units that are done it took as long.
//   8 sequences of one node over 1,000 positions, 12 heads of 64: 11.9 us, of which 8 are a launch, three loads that wait for each other (lengths, table,
//   keys) and the merge.
// What the steps to this gave (us; these three calls, and one of 3 trees of 37 nodes with a window of 1,000, 10 heads of 80 that share 5): a workgroup a
// row and head, keys straight from memory: 17,689, 101,655, 501, 732; on the matrix cores with LDS stages: 51, 313, 15, 27; the way of sharing
// a call out by measured times: 46, 302, 12, 16; values turned by the read: 45, 266, 12, 15.
#include "common.h"
#include "lds_loads.h"
#include "tree_stage.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename V> __device__ __forceinline__ V from_lds(unsigned at) { return *(const __attribute__((address_space(3))) V*)(at); }

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
    float scale;              // of the products, in base 2, above zero: a negative one is its size, and the queries' sign is turned
    bool negative;
    char* out;
    float* ws;
};

// Ones (1 in the lowest bit of each element) where a word's elements are not finite. In whole-number arithmetic on all elements of the word at
// once: as comparisons, the lanes' answers to all words of a tile fill the scalar registers several times over.
__device__ __forceinline__ uint32_t not_finite(uint32_t w, float) { return ((w & 0x7f800000u) + 0x00800000u) >> 31; }
__device__ __forceinline__ uint32_t not_finite(uint32_t w, bf16_t) { return ((w & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u; }
// The elements that are finite, zeros for the others.
__device__ __forceinline__ uint32_t finite(uint32_t w, float) { return w & (not_finite(w, 0.f) - 1); }
__device__ __forceinline__ uint32_t finite(uint32_t w, bf16_t) { return w & ~(not_finite(w, bf16_t{}) * 0xffffu); }
// 1 where the element is NaN, 2^7 for +inf, 2^14 for -inf, else 0: sums of up to 127 of them tell how many of each there were.
__device__ __forceinline__ uint32_t counted(uint32_t w, float) {
    const uint32_t special = not_finite(w, 0.f), nan = ((w & 0x7fffffu) + 0x7fffffu) >> 23;
    return special * (0x3f800000u + (1 - nan) * (0x03800000u << (w >> 31)));
}
__device__ __forceinline__ uint32_t counted(uint32_t w, bf16_t) {
    const uint32_t special = not_finite(w, bf16_t{}), inf = special & ~(((w & 0x007f007fu) + 0x007f007fu) >> 7);
    return special * 0x3f80u + (inf + (inf & w >> 15)) * 0x0380u;
}

// What a row's weights are taken against before it has seen a key: finite, so that no difference of two of them is NaN, and no finite score is below it.
constexpr float LEAST_SCORE = -FLT_MAX;

// a / b for 0 <= a < 2^20, 1 <= b < 2^20, by the reciprocal: half a unit more than `a` lies further from the next quotient than it errs.
__device__ __forceinline__ int lane_quotient(int a, int b) { return static_cast<int>((static_cast<float>(a) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(b))); }

// The first position that a row at `position` sees through a window, or the least number if that lies below it.
__device__ __forceinline__ int low_of(int position, int window) { return max(position, INT32_MIN + window) - window + 1; }

// One wavefront's rows, 16 RT of them, and what it has summed up for them.
template <typename T, int NT, int RT, int KEY_GROUPS_OF_16>
struct Rows {
    using S = Shape<T, NT, KEY_GROUPS_OF_16>;
    static constexpr int KT = S::KT, KEYS = S::KEYS, CH = S::CH, TILES = S::TILES;
    static constexpr unsigned long long ALL = ~0ull >> (64 - KEYS);

    uint4 q[RT][CH];
    f32x4 o[TILES][RT];
    f32x4 sum[RT];                     // of the weights: bfloat16: in every element, of all lanes' keys; 32 bits: in the first, of the lane's
    float m[RT];                       // what weights are taken against, the same in the four lanes of a row
    int low[RT], token[RT];            // (what stands in front of `low` is not seen)
    unsigned long long above[RT];      // the first word of the nodes seen (few rows: asked for ahead)
    int low_least, low_most;

    // Asks for the rows' queries (beyond the last: the last again, never written).
    __device__ __forceinline__ void begin(const TreeAttentionParams& a, int first, int rows, int group, int hk, int row0, int row_bytes) {
        const int G = threadIdx.x % 64 / 16, c16 = threadIdx.x % 16;
        low_least = INT32_MAX;
        low_most = INT32_MIN;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = min(row0 + 16 * rt + c16, rows - 1), node = rows < 1 << 20 ? lane_quotient(r, group) : r / group;
            token[rt] = first + node;
            const char* at = a.q + token[rt] * a.ldq + (hk * group + r - node * group) * row_bytes;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int off = 64 * c + 16 * G;
                q[rt][c] = *reinterpret_cast<const uint4*>(at + (off < row_bytes ? off : 0));
            }
            if (RT == 1) above[rt] = a.ancestors[static_cast<size_t>(token[rt]) * a.words];
            low[rt] = a.window > 0 ? low_of(a.positions[token[rt]], a.window) : INT32_MIN;
            low_least = min(low_least, low[rt]);
            low_most = max(low_most, low[rt]);
        }
        if (a.window > 0) {
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) {
                low_least = min(low_least, __shfl_xor(low_least, off, 64));
                low_most = max(low_most, __shfl_xor(low_most, off, 64));
            }
        }
        low_least = __builtin_amdgcn_readfirstlane(low_least);
        low_most = __builtin_amdgcn_readfirstlane(low_most);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = LEAST_SCORE; sum[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < TILES; ++x) o[x][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Columns behind the head's last are zero in queries and keys.
    static constexpr bool maybe_behind(int c) { return 64 * (c + 1) > 32 * S::LEAST * static_cast<int>(sizeof(T)); }
    __device__ __forceinline__ void wait_for_queries(int row_bytes, bool negative) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            if (RT == 1) asm volatile("" : "+v"(above[rt]));
        const uint32_t sign = !negative ? 0u : sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (maybe_behind(c) && 64 * c + 16 * static_cast<int>(threadIdx.x % 64 / 16) >= row_bytes) q[rt][c] = make_uint4(0, 0, 0, 0);
                q[rt][c].x ^= sign; q[rt][c].y ^= sign; q[rt][c].z ^= sign; q[rt][c].w ^= sign;
                asm volatile("" : "+v"(q[rt][c].x), "+v"(q[rt][c].y), "+v"(q[rt][c].z), "+v"(q[rt][c].w));
            }
    }

    // The second product: into(x, rt, product) for every tile x of columns and 16 rows, of the words word(j, x) of the lane's keys (PER in a word) and the weights
    // weight(rt, j).
    // In bfloat16 added(rt, product) is handed the product of ones with the weights, whose rows are the weights' sum.
    template <bool ONE_BY_ONE, typename V, typename W, typename F, typename A>
    __device__ __forceinline__ static void weigh(V&& word, W&& weight, F&& into, A&& added) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < 4 * KT; h += 8) {
                uint4 pb[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    pb[rt] = make_uint4(pack_bf16x2(weight(rt, h), weight(rt, h + 1)), pack_bf16x2(weight(rt, h + 2), weight(rt, h + 3)),
                                        pack_bf16x2(weight(rt, h + 4), weight(rt, h + 5)), pack_bf16x2(weight(rt, h + 6), weight(rt, h + 7)));
                const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    added(rt, [&](f32x4 c) {
                        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ones), __builtin_bit_cast(bf16x8, pb[rt]), c, 0, 0, 0);
                    });
#pragma unroll
                for (int x = 0; x < TILES; ++x) {
                    const uint4 va = make_uint4(word(h / 2, x), word(h / 2 + 1, x), word(h / 2 + 2, x), word(h / 2 + 3, x));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        into(x, rt, [&](f32x4 c) {
                            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, pb[rt]), c, 0, 0, 0);
                        });
                    if (ONE_BY_ONE) __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
#pragma unroll
            for (int w = 0; w < TILES; ++w) {
                float vw[4 * KT];
#pragma unroll
                for (int j = 0; j < 4 * KT; ++j) vw[j] = __builtin_bit_cast(float, word(j, w));
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    into(w, rt, [&](f32x4 c) {
#pragma unroll
                        for (int j = 0; j < 4 * KT; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(vw[j], weight(rt, j), c, 0, 0, 0);
                        return c;
                    });
                if (ONE_BY_ONE) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // The products of a tile's keys (the lane's operands k) with the queries.
    __device__ __forceinline__ void scores(float (&p)[RT][4 * KT], int row_bytes, uint4 (&k)[KT][CH]) const {
        const int G = threadIdx.x % 64 / 16;
        if (row_bytes != 64 * CH)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (maybe_behind(c) && 64 * c + 16 * G >= row_bytes) k[kt][c] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    if constexpr (sizeof(T) == 2) {
                        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[kt][c]), __builtin_bit_cast(bf16x8, q[rt][c]), s, 0, 0, 0);
                    } else {
                        const f32x4 kf = __builtin_bit_cast(f32x4, k[kt][c]), qf = __builtin_bit_cast(f32x4, q[rt][c]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[i], qf[i], s, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) p[rt][4 * kt + i] = s[i];
            }
        }
    }
    // Products to weights 2^(scale p - m), scale > 0 (what is not seen is -inf). What weights are taken against is put 8 above the maximum, and follows
    // only when a product lies above it: the largest weight then lies between 2^-8 and 1, which costs no accuracy, and most tiles leave sums and outputs as
    // they are and need not know the maximum over a row's four lanes. (No weight is above 1, so that values add up as far as they would by the maximum itself.)
    __device__ __forceinline__ void weights(float (&p)[RT][4 * KT], float scale) {
        float mx[RT];
        bool any = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            mx[rt] = p[rt][0];
#pragma unroll
            for (int j = 1; j < 4 * KT; ++j) mx[rt] = fmaxf(mx[rt], p[rt][j]);
            mx[rt] *= scale;
            any |= mx[rt] > m[rt];
        }
        if (__any(any))
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float top = rows_max(mx[rt]);
                const bool more = top > m[rt];
                const float fix = more ? exp2_for<T>(m[rt] - (top + 8.f)) : 1.f;
                m[rt] = more ? top + 8.f : m[rt];
                sum[rt] *= fix;
#pragma unroll
                for (int x = 0; x < TILES; ++x) o[x][rt] *= fix;
            }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < 4 * KT; ++j) {
                p[rt][j] = exp2_for<T>(fmaf(p[rt][j], scale, -m[rt]));
                if (sizeof(T) == 4) sum[rt][0] += p[rt][j];
            }
    }
    __device__ __forceinline__ float sum_of(int rt) const { return sizeof(T) == 4 ? rows_sum(sum[rt][0]) : sum[rt][0]; }

    // A tile whose keys all rows see, from its products on, with the lane's words of its values.
    __device__ __forceinline__ void take(float (&p)[RT][4 * KT], float scale, const uint32_t (&v)[TILES][S::WORDS]) {
        // (The weights' chain of dependent instructions goes first on the unit, so that the other wavefront's products run beside it: 256 rows of 128
        // columns over 8,192 positions, 32 sequences: in short runs 310 > 288 us, in long ones 312 > 301; the products first: 290; products and scores first: 300.)
        __builtin_amdgcn_s_setprio(1);
        weights(p, scale);
        __builtin_amdgcn_s_setprio(0);
        weigh<false>([&](int j, int w) { return v[w][j]; }, [&](int rt, int j) { return p[rt][j]; },
                     [&](int x, int rt, auto&& product) { o[x][rt] = product(o[x][rt]); }, [&](int rt, auto&& product) { sum[rt] = product(sum[rt]); });
    }
    // Any tile: keys [at0, at0 + KEYS) of the cache, or of the nodes; `valid` has a bit for each that exists. stored(j, w) gives a word of the values again;
    // seen_by, the lane's own word of LDS, keeps which of the lane's keys its rows see (a register more all the way does not fit beside 32 rows of 128 columns).
    template <typename W>
    __device__ __forceinline__ void take_some(float (&p)[RT][4 * KT], const uint32_t (&v)[TILES][S::WORDS], const TreeAttentionParams& a, bool of_nodes, int at0,
                                              unsigned long long valid, int first, int nodes, unsigned* seen_by, W&& stored) {
        const int G = threadIdx.x % 64 / 16;
        unsigned mine = 0;                   // which of the lane's keys exist
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) mine |= static_cast<unsigned>(valid >> (16 * kt + 4 * G) & 15) << (4 * kt);
        static_assert(RT * 4 * KT <= 32, "a bit a row and key");
        unsigned all_seen = 0;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            unsigned seen = mine;
            if (of_nodes) {
                const int word = word_of_nodes(at0, nodes);
                unsigned long long bits = RT == 1 ? above[rt] : 0;
                if (word > 0 || (RT > 1 && word == 0)) bits = a.ancestors[static_cast<size_t>(token[rt]) * a.words + word];
                bits >>= at0 % 64 + 4 * G;
                unsigned nodes_seen = 0;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) nodes_seen |= static_cast<unsigned>(bits >> (16 * kt) & 15) << (4 * kt);
                seen &= nodes_seen;
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
            all_seen |= seen << (4 * KT * rt);
        }
        *seen_by = all_seen;
        weights(p, a.scale);
        // A key that does not exist has some other row's values. A value that is not finite, in a tile of which some rows see less than others,
        // would reach those that do not see it as zero times it: the finite values are weighed as ever, and how many NaN, +inf and -inf a row gives weight
        // to in a column, and whether it sees any of these and gives it none (zero times it: NaN, as where all rows see all keys), comes out of a product of their
        // marks with ones, and 2^21 for the keys of the last kind. (For these products the words are read anew, which keeps them out of the registers.)
        auto exists = [&](int j) {           // (of the keys of word j)
            return sizeof(T) == 2 ? (mine >> 2 * j & 1 ? 0xffffu : 0u) | (mine >> 2 * j & 2 ? 0xffff0000u : 0u) : 0u - (mine >> j & 1);
        };
        auto weight = [&](int rt, int j) { return p[rt][j]; };
        auto add = [&](int x, int rt, auto&& product) { o[x][rt] = product(o[x][rt]); };
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < S::WORDS; ++j) {
            uint32_t each = 0;
#pragma unroll
            for (int w = 0; w < TILES; ++w) each |= not_finite(v[w][j], T{});
            odd |= each & exists(j);
        }
        auto added = [&](int rt, auto&& product) { sum[rt] = product(sum[rt]); };
        int plain = !__any(odd != 0);
        asm volatile("" : "+v"(plain));          // (a lane's register, as where this function is called)
        if (plain) {
            weigh<true>([&](int j, int w) { return v[w][j] & exists(j); }, weight, add, added);
            return;
        }
        auto word = [&](int j, int w) { return stored(j, w) & exists(j); };
        weigh<true>([&](int j, int w) { return finite(word(j, w), T{}); }, weight, add, added);
        asm volatile("" ::: "memory");
        static_assert(KEYS <= 127, "as many marks");
        const unsigned seen = *seen_by;
        weigh<true>([&](int j, int w) { return counted(word(j, w), T{}); }, [&](int rt, int j) { return p[rt][j] != 0.f ? 1.f : seen >> (4 * KT * rt + j) & 1 ? 2097152.f : 0.f; },
                    [&](int x, int rt, auto&& product) {
                        const f32x4 marks = product(f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int n = static_cast<int>(fminf(marks[i], 4194304.f));
                            const float up = n & 0x3f80 ? INFINITY : 0.f, down = n & 0x1fc000 ? -INFINITY : 0.f;
                            o[x][rt][i] += n & 127 || n >= 1 << 21 ? __builtin_nanf("") : up + down;
                        }
                    }, [](int, auto&&) {});
    }

    // o[x][rt][i] stands in column column(x) + EACH (4 G + i) of its row.
    static constexpr int EACH = sizeof(T) == 2 ? 1 : S::BLOCK;
    __device__ __forceinline__ static constexpr int column(int x) { return x / EACH * 16 * EACH + x % EACH; }
};

__device__ __forceinline__ int cached_of(const TreeAttentionParams& a, int b) {
    return static_cast<int>(min(min(static_cast<long long>(max(a.cached[b], 0)), static_cast<long long>(a.max_blocks) * a.page_size), INT32_MAX - 65536ll));
}

// What a workgroup works on, the same in all its threads.
struct Work {
    int b, hk, split, row_tile, group, first, nodes, rows, cached;
    // Workgroups that share keys have numbers 8 apart, so that they run on one XCD and the second finds the keys in its L2.
    __device__ __forceinline__ bool find(const TreeAttentionParams& a, int rows_each) {
        const int residue = blockIdx.x % 8, rest = blockIdx.x / 8;
        const int eight = uniform_quotient(rest, a.row_tiles), unit = eight * 8 + residue;
        row_tile = rest - eight * a.row_tiles;
        if (unit >= a.units) return false;
        const int pair = uniform_quotient(unit, a.nsplit);
        split = unit - pair * a.nsplit;
        b = uniform_quotient(pair, a.n_kv_heads);
        hk = pair - b * a.n_kv_heads;
        group = small_quotient(a.n_heads, a.n_kv_heads);
        first = min(max(a.cu_q[b], 0), a.tokens);
        nodes = min(min(max(a.cu_q[b + 1] - first, 0), a.tokens - first), a.max_new);
        rows = nodes * group;
        cached = cached_of(a, b);
        return row_tile * rows_each < rows;
    }
};

__device__ __forceinline__ int block_of(const TreeAttentionParams& a, int at) {
    return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(at)) * a.page_magic) >> a.page_shift);
}
// The factor of a row whose weights add up to zero: zero if it sees nothing; else all that it sees scores -inf, no weights can be found, and it is NaN. (What it takes
// is read anew from the arguments, which are all that either kernel has: kept in scalar registers from the start it costs every call 0.2 us.)
__device__ __forceinline__ float factor_of_none(int b, int t) {
    auto at = reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(at));
    const auto& a = *reinterpret_cast<const TreeAttentionParams*>(at);
    const int first = min(max(a.cu_q[b], 0), a.tokens), nodes = min(min(max(a.cu_q[b + 1] - first, 0), a.tokens - first), a.max_new), cached = cached_of(a, b);
    const int low = a.window > 0 ? low_of(a.positions[t], a.window) : 0;
#pragma unroll 1
    for (int i = 0; i < nodes; ++i)
        if (a.ancestors[static_cast<size_t>(t) * a.words + i / 64] >> i % 64 & 1 && (a.window <= 0 || a.positions[first + i] >= low)) return __builtin_nanf("");
    if (low < cached)
#pragma unroll 1
        for (int block = max(low, 0) / a.page_size; static_cast<long long>(block) * a.page_size < cached; ++block)
            if (static_cast<unsigned>(a.block_tables[static_cast<size_t>(b) * a.max_blocks + block]) < static_cast<unsigned>(a.n_pages)) return __builtin_nanf("");
    return 0.f;
}
__device__ __forceinline__ float2* split_state(const TreeAttentionParams& a, size_t pair) {
    return reinterpret_cast<float2*>(a.ws + static_cast<size_t>(a.tokens) * a.n_heads * a.nsplit * a.head_dim) + pair;
}

// 16-byte piece p of row k of a stage lies at piece p ^ turned(k). A 16-byte read serves lanes 0-3, 12-15 and 20-27 at once, then the others of 32 alike:
// of keys that is one piece of rows 0-3 and 12-15 and its neighbour of rows 4-11; the values' turning read serves 32 lanes, 32 bytes of each of eight
// rows; a 16-byte read of values has eight pieces of a row and the other eight of the row four further on. None meets a bank twice. (By k % 16 alone the
// reads of values took twice as long, a third of all LDS cycles.)
constexpr int TABLE_ENTRIES = 2048;
template <typename T, int NT, int RT, int K16, int NW, int KG>
__global__ void __launch_bounds__(NW * 64) tree_attention_kernel(TreeAttentionParams a) {
    using R = Rows<T, NT, RT, K16>;
    using S = Shape<T, NT, K16>;
    using St = Stage<T, NT, K16, NW, KG>;
    constexpr int KT = S::KT, KEYS = S::KEYS, CH = S::CH, TILES = S::TILES, PIECES = St::PIECES, SK = St::KEYS, RG = NW / KG, PITCH = 32 * NT + 4;
    auto turned = [](int k) {
        if (PIECES < 16) return k & (PIECES - 1);
        return sizeof(T) == 2 ? (k & 7) << 1 ^ (k & 8 ? 9 : 0) : (k ^ (k & 4) << 1) & 15;
    };
    // the stages [keys, values][SK][PIECES * 16]; at the end the states [wavefront][16 RT][PITCH], then their maxima and sums
    extern __shared__ __attribute__((aligned(512))) unsigned char stage_s[];
    __shared__ int table_s[TABLE_ENTRIES];
    __shared__ unsigned seen_s[NW * 64];                                  // of each lane
    __shared__ unsigned long long valid_s[St::NUMBER][NW];                // of each wavefront's rows of a stage: a bit a key that exists
    Work w;
    if (!w.find(a, 16 * RT * RG)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int kg = wave % KG, rg = wave / KG, group0 = w.row_tile * RG * 16 * RT, row0 = group0 + rg * 16 * RT;
    const int G = lane / 16, c16 = lane % 16, row_bytes = a.head_dim * static_cast<int>(sizeof(T));
    const int first = w.first, nodes = w.nodes, hk = w.hk, cached = w.cached;
    const int* table = a.block_tables + static_cast<size_t>(w.b) * a.max_blocks;

    // A part of the block table lies in LDS, from entry `base` on; all of the workgroup meet here. Returns whether all of its entries that the
    // cache reaches name pages.
    int base = 0, filled = 0;
    auto fill_table = [&](int from) {
        lds_barrier();
        base = from;
        filled = min(TABLE_ENTRIES, a.max_blocks - from);
        const int reached = min(filled, block_of(a, cached - 1) + 1 - from);
        int good = 1;
        for (int i = threadIdx.x; i < filled; i += NW * 64) {
            const int entry = table[from + i];
            table_s[i] = entry;
            good &= i >= reached || static_cast<unsigned>(entry) < static_cast<unsigned>(a.n_pages);
        }
        return __syncthreads_and(good) != 0;
    };
    // Tiles of SK keys: those of the cache from the window's first on, then the nodes'. A split has `per` neighbouring ones.
    int first_tile = 0;
    if (a.window > 0) {        // the least position of the workgroup's rows
        int least = INT32_MAX;
        const int last = min(group0 + 16 * RT * RG, w.rows) - 1;
        for (int node = group0 / w.group + static_cast<int>(threadIdx.x); node <= last / w.group; node += NW * 64) least = min(least, a.positions[first + node]);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) least = min(least, __shfl_xor(least, off, 64));
        if (lane == 0) table_s[wave] = least;
        __syncthreads();
        for (int i = 0; i < NW; ++i) least = min(least, table_s[i]);
        first_tile = __builtin_amdgcn_readfirstlane(min(max(low_of(least, a.window), 0), cached) / SK);
    }
    const int cache_tiles = (cached + SK - 1) / SK - first_tile, all_tiles = cache_tiles + (nodes + SK - 1) / SK;
    const int per = (all_tiles + a.nsplit - 1) / a.nsplit, begin = w.split * per, end = min(all_tiles, begin + per);
    // The queries come with the table, and are waited for here: a load that the compiler knows of and has not waited for in front of the loop
    // would have it wait in the loop, every time, for all that is on its way.
    R r;
    r.begin(a, first, w.rows, w.group, hk, row0, row_bytes);
    // Tiles below whole_end have SK keys that exist, and load instructions that take whole rows of one page each.
    int whole_end = a.page_size % St::PER_LOAD == 0 ? cached / SK - first_tile : 0;
    if (begin < cache_tiles && !fill_table(min(block_of(a, (begin + first_tile) * SK), a.max_blocks - 1))) whole_end = min(whole_end, begin);
    r.wait_for_queries(row_bytes, a.negative);

    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)stage_s));
    const size_t head = static_cast<size_t>(hk) * row_bytes;
    // Asks for stage after stage. (All of the workgroup come here, behind a barrier after which nobody reads what it fills.) A wavefront has MINE
    // neighbouring rows of it. Of tiles below whole_end an instruction's address is its first row's and an offset that the lane keeps, and the
    // rows are found AHEAD tiles at a time, from tile ready_from on: lane s * LOADS + i has instruction i of tile ready_from + s. A few scalar
    // instructions a load are left: between two barriers there is nothing else to do for a unit. Otherwise a lane finds a row, and hands it to those
    // that load it.
    constexpr unsigned long long ALL_MINE = St::MINE == 64 ? ~0ull : (1ull << (St::MINE % 64)) - 1;
    constexpr int AHEAD = 64 / St::LOADS;
    unsigned offset[St::LOADS];
#pragma unroll
    for (int i = 0; i < St::LOADS; ++i) {
        const int k = wave * St::MINE + i * St::PER_LOAD + lane / PIECES, piece = (lane % PIECES) ^ turned(k);
        offset[i] = (lane / PIECES) * a.page_pitch + (16 * piece < row_bytes ? 16 * piece : 0);
    }
    const unsigned char *k_head = reinterpret_cast<const unsigned char*>(a.k_pages) + head, *v_head = reinterpret_cast<const unsigned char*>(a.v_pages) + head;
    unsigned long long row_at = 0;
    int ready_from = 0, ready_end = 0, ask_place = 0;      // (tiles from ready_from to ready_end; the stage that is filled next)
    auto ask = [&](int tile) {
        const int place = ask_place;
        ask_place = place + 1 == St::NUMBER ? 0 : place + 1;
        const unsigned to = lds0 + place * St::BYTES + wave * St::LOADS * 1024;
        const bool of_nodes = tile >= cache_tiles;
        const int at0 = (of_nodes ? tile - cache_tiles : tile + first_tile) * SK;
        if (tile >= ready_end) {
            if (!of_nodes && block_of(a, min(at0 + SK, cached) - 1) >= base + filled && !fill_table(block_of(a, at0))) whole_end = min(whole_end, tile);
            if (tile < whole_end) {
                // (of a tile behind the table's part some entry: it is found again when that part is there)
                const int at = at0 + lane / St::LOADS * SK + wave * St::MINE + lane % St::LOADS * St::PER_LOAD, block = min(block_of(a, at), base + filled - 1);
                row_at = static_cast<unsigned long long>(static_cast<unsigned>(table_s[block - base] * a.page_size + at - block * a.page_size)) * a.page_pitch;
                const long long covered = (static_cast<long long>(base + filled) * a.page_size - at0) / SK;
                ready_from = tile;
                ready_end = min(tile + static_cast<int>(min(covered, static_cast<long long>(AHEAD))), whole_end);
            }
        }
        if (tile < ready_end) {
            const int from = (tile - ready_from) * St::LOADS, low = static_cast<int>(row_at), high = static_cast<int>(row_at >> 32);
#pragma unroll
            for (int i = 0; i < St::LOADS; ++i) {
                const size_t row = static_cast<size_t>(static_cast<unsigned>(__builtin_amdgcn_readlane(high, from + i))) << 32 |
                                   static_cast<unsigned>(__builtin_amdgcn_readlane(low, from + i));
                load_to_lds(k_head + row, offset[i], to + 1024 * i);
                load_to_lds(v_head + row, offset[i], to + St::MATRIX + 1024 * i);
            }
            return;
        }
        const int mine = at0 + wave * St::MINE + lane % St::MINE;
        bool there;
        int row;
        if (of_nodes) {
            there = mine < nodes;
            row = first + min(mine, nodes - 1);
        } else {
            const int at = min(mine, cached - 1), block = block_of(a, at), entry = table_s[block - base];
            there = mine < cached && static_cast<unsigned>(entry) < static_cast<unsigned>(a.n_pages);
            row = there ? entry * a.page_size + at - block * a.page_size : 0;
        }
        const unsigned long long bits = __ballot(there) & ALL_MINE;
        if (lane == 0) valid_s[place][wave] = bits;
        const unsigned char* kb = reinterpret_cast<const unsigned char*>(of_nodes ? a.k : a.k_pages) + head;
        const unsigned char* vb = reinterpret_cast<const unsigned char*>(of_nodes ? a.v : a.v_pages) + head;
        const size_t k_pitch = of_nodes ? a.ldk : a.page_pitch, v_pitch = of_nodes ? a.ldv : a.page_pitch;
#pragma unroll 1
        for (int i = 0; i < St::LOADS; ++i) {
            const int k = i * St::PER_LOAD + lane / PIECES, piece = (lane % PIECES) ^ turned(wave * St::MINE + k);
            const int off = 16 * piece < row_bytes ? 16 * piece : 0;
            const size_t from = __shfl(row, k, 64);
            load_to_lds(kb, from * k_pitch + off, to + 1024 * i);
            load_to_lds(vb, from * v_pitch + off, to + St::MATRIX + 1024 * i);
        }
    };
    auto place_of = [&](int k, int piece) { return 16 * (piece ^ turned(k)); };

    // One loop over the wavefront's tiles of all stages: in two loops, one in the other, the outputs would be copied from the one's registers
    // to the other's for every tile. (A wavefront whose rows lie behind the last works on the last again, and writes nothing.)
    constexpr int TURNS = St::TURNS;
    // Everything comes from LDS a phase before it is multiplied: a tile's keys while the tile in front of it is weighed (its stage has come by then),
    // its values while its own products are made.
    constexpr bool SHORT = sizeof(T) == 2;
    // Where the lane's pieces of 16 rows lie; those of the next 16 lie 16 rows behind. A row starts at a multiple of its (two) powers of two of bytes, so a
    // piece further on in it is the first one's address with some bits turned.
    static_assert(St::BYTES % 512 == 0 && KEYS * St::ROW % 512 == 0 && St::ROW <= (SHORT ? 512 : 1024), "rows start at multiples of their size");
    const int key_at = c16 * St::ROW + place_of(c16, G);
    int value_at[SHORT ? 1 : 4 * CH];
    if constexpr (SHORT) {
        value_at[0] = St::MATRIX + (4 * G + c16 / 4) * St::ROW + place_of(4 * G + c16 / 4, c16 % 4 / 2) + c16 % 2 * 8;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < CH; ++x) {
                const int row = 4 * G + i, byte = 64 * (x / S::BLOCK * S::BLOCK) + 4 * S::BLOCK * c16;
                value_at[i * CH + x] = St::MATRIX + row * St::ROW + place_of(row, byte / 16) + byte % 16;
            }
    }
    // (16 bits) Of two words of column 16 x + c16 the keys 4 G .. 4 G + 3 of a 16: the sixteen lanes of a G give the addresses of four keys' 32 bytes in pieces of
    // eight, and each gets a column of them.
    auto two_words = [&](unsigned keys, int kt, int x) {
        const unsigned at = ((keys + value_at[0]) ^ (32 * x)) + kt * 16 * St::ROW;
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at)));
    };
    uint4 k[KT][CH];
    auto read_keys = [&](unsigned keys) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int c = 0; c < CH; ++c)
                k[kt][c] = __builtin_bit_cast(uint4, from_lds<u32x4>((St::ROW <= 512 ? (keys + key_at) ^ (64 * c) : keys + c16 * St::ROW + place_of(c16, 4 * c + G)) + kt * 16 * St::ROW));
    };
    const int steps = (end - begin) * TURNS;
    // (not unrolled: code that runs once waits for its instructions to come)
#pragma unroll 1
    for (int i = 0; i < St::NUMBER - 1; ++i)
        if (begin + i < end) ask(begin + i);
    if (steps > 0) {
        wait_tiles_and_meet<St::NUMBER - 3, 2 * St::LOADS>(min(St::NUMBER - 3, end - 1 - begin));
        read_keys(lds0 + kg * (KEYS * St::ROW));
    }
    // (tiles from seen_begin to whole_end: every row sees all keys)
    const int seen_begin = a.window > 0 ? (max(r.low_most, 0) + SK - 1) / SK - first_tile : 0;
    int turn = 0, tile = begin, place = 0;
    for (int step = 0; step < steps; ++step) {
        const unsigned keys = lds0 + place * St::BYTES + (turn * KG + kg) * (KEYS * St::ROW);
        if (turn == 0) {
            // the next stage has come (those behind it may be on their way), and all have read the one in front of this
            wait_tiles_and_meet<St::NUMBER - 3, 2 * St::LOADS>(max(0, min(St::NUMBER - 3, end - 2 - tile)));
            if (tile + St::NUMBER - 1 < end) ask(tile + St::NUMBER - 1);
        }
        uint32_t v[TILES][S::WORDS];
        if constexpr (SHORT) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int x = 0; x < TILES; ++x) {
                    const u32x2 u = two_words(keys, kt, x);
                    v[x][2 * kt] = u.x; v[x][2 * kt + 1] = u.y;
                }
        } else {
#pragma unroll
            for (int j = 0; j < 4 * KT; ++j)
#pragma unroll
                for (int x = 0; x < CH; x += S::BLOCK) {
                    const unsigned at = keys + value_at[j % 4 * CH + x] + j / 4 * 16 * St::ROW;
                    if (S::BLOCK == 4) {
                        const u32x4 u = from_lds<u32x4>(at);
                        v[x][j] = u.x; v[x + 1][j] = u.y; v[x + 2][j] = u.z; v[x + 3][j] = u.w;
                    } else {
                        const u32x2 u = from_lds<u32x2>(at);
                        v[x][j] = u.x; v[x + 1][j] = u.y;
                    }
                }
        }
        __builtin_amdgcn_sched_barrier(0);
        float p[RT][4 * KT];
        r.scores(p, row_bytes, k);
        __builtin_amdgcn_sched_barrier(0);
        const int here = place, tile_here = tile, k0 = (turn * KG + kg) * KEYS;
        if (++turn == TURNS) {
            turn = 0;
            ++tile;
            place = place + 1 == St::NUMBER ? 0 : place + 1;
        }
        if (step + 1 < steps) read_keys(lds0 + place * St::BYTES + (turn * KG + kg) * (KEYS * St::ROW));
        __builtin_amdgcn_sched_barrier(0);
        // (The condition is kept in a lane's register: as a scalar branch, which the same one in all lanes could be, the compiler gives the outputs other
        // registers on either side of a product, and moves or spills them every time.)
        int all_seen = tile_here >= seen_begin && tile_here < whole_end;
        asm volatile("" : "+v"(all_seen));
        if (all_seen) {
            r.take(p, a.scale, v);
        } else {
            unsigned long long some = 0;
            const bool of_nodes = tile_here >= cache_tiles;
            const int at0 = (of_nodes ? tile_here - cache_tiles : tile_here + first_tile) * SK;
            if (tile_here < whole_end) {
                some = R::ALL;
            } else if (St::MINE >= KEYS) {
                some = valid_s[here][k0 / St::MINE] >> (k0 % St::MINE) & R::ALL;
            } else {
#pragma unroll
                for (int i = 0; i < KEYS / St::MINE; ++i) some |= valid_s[here][k0 / St::MINE + i] << (i * St::MINE);
            }
            some = static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(some >> 32)))) << 32 |
                   static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(some)));
            r.take_some(p, v, a, of_nodes, at0 + k0, some, first, nodes, seen_s + threadIdx.x, [&](int j, int x) {
                if constexpr (SHORT) {
                    const u32x2 u = two_words(keys, j / 2, x);
                    return j % 2 == 0 ? u.x : u.y;
                } else {
                    return from_lds<uint32_t>(keys + value_at[j % 4 * CH + x] + j / 4 * 16 * St::ROW + 4 * (x % S::BLOCK));
                }
            });
        }
    }

    if constexpr (KG == 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int row = row0 + 16 * rt + c16;
            const float sum = r.sum_of(rt);
            if (row >= w.rows) continue;
            const int node = row / w.group, t = first + node, h = hk * w.group + row - node * w.group;
            const float inv = a.nsplit > 1 ? 1.f : sum == 0.f ? factor_of_none(w.b, t) : 1.f / sum;
            T* to = reinterpret_cast<T*>(a.out + t * a.ldo) + h * a.head_dim;
            const size_t pair = (static_cast<size_t>(t) * a.n_heads + h) * a.nsplit + w.split;
            float* part = a.ws + pair * a.head_dim;
            if constexpr (SHORT) {
#pragma unroll
                for (int x = 0; x < TILES; ++x) {
                    const int d = R::column(x) + 4 * G;
                    if (d >= a.head_dim) continue;
                    const f32x4 o = r.o[x][rt];
                    if (a.nsplit == 1) *reinterpret_cast<uint2*>(to + d) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
                    else *reinterpret_cast<f32x4*>(part + d) = o;
                }
            } else {
#pragma unroll
                for (int x = 0; x < TILES; x += R::EACH)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = R::column(x) + R::EACH * (4 * G + i);
                        if (d >= a.head_dim) continue;
#pragma unroll
                        for (int e = 0; e < R::EACH; ++e) {
                            if (a.nsplit == 1) to[d + e] = from_float<T>(r.o[x + e][rt][i] * inv);
                            else part[d + e] = r.o[x + e][rt][i];
                        }
                    }
            }
            if (a.nsplit > 1 && G == 0) *split_state(a, pair) = make_float2(r.m[rt], sum);
        }
        return;
    }
    // The key groups' states meet in LDS; every thread merges some rows' columns in the groups' order.
    lds_barrier();              // (the last stage has been read; no load is on its way)
    float* state_s = reinterpret_cast<float*>(stage_s);
    float2* ml_s = reinterpret_cast<float2*>(state_s + NW * 16 * RT * PITCH);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = r.sum_of(rt);
        if (G == 0) ml_s[wave * 16 * RT + 16 * rt + c16] = make_float2(r.m[rt], sum);
        float* to = state_s + (wave * 16 * RT + 16 * rt + c16) * PITCH;
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
            if constexpr (SHORT) *reinterpret_cast<f32x4*>(to + R::column(x) + 4 * G) = r.o[x][rt];
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) to[R::column(x) + R::EACH * (4 * G + i)] = r.o[x][rt][i];
        }
    }
    lds_barrier();
    const int quads = a.head_dim / 4, count = min(16 * RT * RG, w.rows - group0);
    for (int item = threadIdx.x; item < count * quads; item += NW * 64) {
        const int row = item / quads, d = (item - row * quads) * 4;
        const int at = row / (16 * RT) * KG * 16 * RT + row % (16 * RT);        // in the first key group's state; the others' lie 16 RT rows apart
        float top = LEAST_SCORE, sum = 0.f;
#pragma unroll
        for (int i = 0; i < KG; ++i) top = fmaxf(top, ml_s[at + i * 16 * RT].x);
        f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            const float2 ml = ml_s[at + i * 16 * RT];
            const f32x4 part = *reinterpret_cast<const f32x4*>(state_s + (at + i * 16 * RT) * PITCH + d);
            const float weight = exp2_for<T>(ml.x - top);
            sum += weight * ml.y;               // (a key group whose keys nobody saw has zeros)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += weight * part[e];
        }
        const int node = (group0 + row) / w.group, t = first + node, h = hk * w.group + group0 + row - node * w.group;
        if (a.nsplit == 1) {
            const float inv = sum == 0.f ? factor_of_none(w.b, t) : 1.f / sum;
            T* to = reinterpret_cast<T*>(a.out + t * a.ldo) + h * a.head_dim + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = from_float<T>(v[e] * inv);
        } else {
            const size_t pair = (static_cast<size_t>(t) * a.n_heads + h) * a.nsplit + w.split;
            *reinterpret_cast<f32x4*>(a.ws + pair * a.head_dim + d) = v;
            if (d == 0) *split_state(a, pair) = make_float2(top, sum);
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
        float top = LEAST_SCORE, sum = 0.f;
        f32x4 v{0.f, 0.f, 0.f, 0.f};
        // (eight splits' loads at once: one behind the other, 64 nodes of 25 heads in 8 to 10 splits took 8.7 us where this takes 4.3)
        for (int s0 = 0; s0 < a.nsplit; s0 += 8) {
            float2 ml[8];
            f32x4 part[8];
            const int last = a.nsplit - 1;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ml[i] = *reinterpret_cast<const float2*>(state + 2 * (pair + min(s0 + i, last)));
                part[i] = *reinterpret_cast<const f32x4*>(a.ws + (pair + min(s0 + i, last)) * a.head_dim + d);
            }
            const float before = top;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, ml[i].x);
            const float kept = exp2_for<T>(before - top);
            sum *= kept;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= kept;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool counts = s0 + i <= last;
                const float weight = exp2_for<T>(ml[i].x - top);
                sum += counts ? weight * ml[i].y : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += counts ? weight * part[i][j] : 0.f;
            }
        }
        const float inv = sum == 0.f ? factor_of_none(b, t) : 1.f / sum;
        T* to = reinterpret_cast<T*>(a.out + t * a.ldo) + h * a.head_dim + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = from_float<T>(v[i] * inv);
    }
}

// How a call is shared out: 16-row tiles of a wavefront, wavefronts of a workgroup, key groups among them, workgroups that share a row's keys.
struct Plan {
    int nt, rt, waves, key_groups, row_tiles, nsplit;
};
struct Way {
    int rt, waves, key_groups;
};
// The ways that there are kernels for.
constexpr Way NARROW[] = {{1, 4, 4}, {1, 8, 4}, {1, 8, 2}, {2, 8, 2}, {2, 8, 1}}, MIDDLE[] = {{1, 2, 2}, {1, 4, 2}, {1, 8, 2}, {2, 8, 2}, {2, 8, 1}},
              MIDDLE_F32[] = {{1, 2, 2}, {1, 4, 2}, {1, 8, 2}, {1, 8, 1}}, WIDE[] = {{1, 1, 1}, {1, 2, 1}, {1, 4, 1}};

// Of every way and number of splits the one whose time is the least by a sum of what was measured, in us: a step (a wavefront's keys of a
// stage) takes 0.8 and its products, workgroups beyond the compute units take turns, all stages together come at 4.2 TB/s, and a
// join takes 6 and 0.2 a split (2.5 of it on the unit's side, the rest the host's: a second launch and a workspace, 14 us a call instead of 11). Over 180 calls
// in all ways of sharing them out the times taken, the host's among them, lie 4.5% above the best on average (58% at most), and 5% by the GPU's alone.
Plan plan_of(int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_new, int max_cached, int window, int dtype) {
    const bool f32 = dtype == MLLM_F32;
    const int nt = head_dim <= 32 ? 1 : head_dim <= 64 ? 2 : head_dim <= 128 ? 4 : 8, keys = f32 ? 16 : 32;
    const long long rows = static_cast<long long>(max_new) * (n_heads / n_kv_heads);
    const long long seen = window > 0 ? std::min<long long>(max_cached, static_cast<long long>(window) + max_new) : max_cached;
    const long long tiles = (seen + keys - 1) / keys + (max_new + keys - 1) / keys;
    const Way* ways = nt <= 2 ? NARROW : nt == 8 ? WIDE : f32 ? MIDDLE_F32 : MIDDLE;
    const int n_ways = nt <= 2 || (nt == 4 && !f32) ? 5 : nt == 8 ? 3 : 4;
    const float tile_kb = keys * nt * 64 * (f32 ? 4 : 2) / 1024.f;
    Plan best{};
    float least = INFINITY;
    for (const Way* w = ways; w < ways + n_ways; ++w) {
        const int each = 16 * w->rt * w->waves / w->key_groups;
        if (w != ways && each >= 2 * rows) break;
        const long long row_tiles = (rows + each - 1) / each, groups = row_tiles * n_seqs * n_kv_heads, all = (tiles + w->key_groups - 1) / w->key_groups;
        const float step = 0.8f + 0.105f * (f32 ? 4 : 1) * nt * w->rt * w->waves / 4;
        for (int n = 1; n <= 64 && (n == 1 || (n < 2 * all && groups * n <= 1024)); n += n < 4 ? 1 : n < 8 ? 2 : n < 16 ? 4 : n < 32 ? 8 : 16) {
            const float turns = static_cast<float>((groups * n + 255) / 256), steps = static_cast<float>((all + n - 1) / n);
            const float came = static_cast<float>(groups * n) * steps * w->key_groups * tile_kb * 0.00024f;
            const float us = 6.5f * (turns - 1) + std::max(turns * steps * step, came) + (n > 1 ? 6.f + 0.2f * n : 0.f);
            if (us < least) {
                least = us;
                best = {nt, w->rt, w->waves, w->key_groups, static_cast<int>(row_tiles), n};
            }
        }
    }
    return best;
}

template <typename T, int NT, int RT, int K16, int NW, int KG>
int launch(const TreeAttentionParams& p, hipStream_t stream) {
    using St = Stage<T, NT, K16, NW, KG>;
    const long long blocks = (static_cast<long long>(p.units) + 7) / 8 * 8 * p.row_tiles;
    if (blocks * NW * 64 > UINT32_MAX) return -1;          // (what one launch can have)
    constexpr int STATES = KG == 1 ? 0 : NW * 16 * RT * ((32 * NT + 4) * 4 + 8), LDS = std::max(St::NUMBER * St::BYTES, STATES);
    static_assert(LDS + TABLE_ENTRIES * 4 + NW * 256 + 1024 <= 163840, "LDS of a compute unit");
    auto kernel = tree_attention_kernel<T, NT, RT, K16, NW, KG>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return static_cast<int>(e);
    kernel<<<static_cast<unsigned>(blocks), NW * 64, LDS, stream>>>(p);
    return 0;
}

template <typename T>
int dispatch(const TreeAttentionParams& p, const Plan& plan, hipStream_t stream) {
#define TREE_CASE(N, R, K, W, G) if (plan.nt == N && plan.rt == R && plan.waves == W && plan.key_groups == G) return launch<T, N, R, K, W, G>(p, stream);
    if constexpr (sizeof(T) == 2) {
        TREE_BF16_KERNELS(TREE_CASE)
    } else {
        TREE_F32_KERNELS(TREE_CASE)
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
    if (units > INT32_MAX / 8 || (plan.nsplit > 1 && ws == nullptr)) return -1;
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
    // (a scale of zero, or one next to it: so small that products up to 2^98 move no weight by more than half a step, and -inf stays)
    p.scale = std::max(std::fabs(scale) * MLLM_LOG2E, 1e-37f);
    p.negative = scale < 0.f;
    p.out = static_cast<char*>(out); p.ws = ws;
    const int rc = dtype == MLLM_F32 ? dispatch<float>(p, plan, stream) : dispatch<bf16_t>(p, plan, stream);
    if (rc != 0) return rc;
    if (plan.nsplit > 1) {
        const dim3 grid(max_new, n_seqs, std::min(64, (n_heads * (head_dim / 4) + 255) / 256));          // (split: 1,024 workgroups at most, so as many sequences)
        if (dtype == MLLM_F32) tree_attention_join_kernel<float><<<grid, 256, 0, stream>>>(p);
        else tree_attention_join_kernel<bf16_t><<<grid, 256, 0, stream>>>(p);
    }
    MLLM_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
