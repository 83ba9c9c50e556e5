// What a step over drafted trees needs beside its attention, for gfx950: the step's arrays from request lengths, and the path of
// drafted tokens that the model's choices confirm. Both are small whole-number work that would otherwise send the host a result and
// wait for it between two steps: they are bound by the latency of a launch and of three or four dependent loads, not by bytes. Step maps of 8 trees of 16
// nodes take 5.7 us, of 256 trees of 128 nodes over up to 100,000 positions in pages of 16 (12 MB of tables) 9.0; paths of 1 tree of 26 nodes 3.0 us, of 512
// of up to 200 nodes 4.8. (Tables copied 16 bytes a thread took as long; lengths read before the counts are added up saved 0.4 us.)
//
// One workgroup has one sequence. Nothing passes between workgroups: each finds the place of its first token by adding up the
// counts in front of it itself (256 counts are one load a thread), so one launch does everything and the result has no order of
// arrival in it.
//
// What the host cannot see is checked here: a count, a length, a parent, a page number or a request row that names nothing is taken
// as none, so that no read or write leaves its array.
#include "common.h"

#include <algorithm>

#define TREE_MAX_NODES 256          // of one sequence: a thread has a node, and its nodes above fill four words of 64 bits
#define TREE_THREADS 256

namespace {

// Sum over the workgroup of a whole number; every thread gets it. `scratch`: one int a wavefront.
__device__ __forceinline__ int block_sum_int(int v, int* scratch) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, MLLM_WAVE);
    if (threadIdx.x % MLLM_WAVE == 0) scratch[threadIdx.x / MLLM_WAVE] = v;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x) / MLLM_WAVE; ++w) t += scratch[w];
    return t;
}

// Page row of position `at`, or -1 where the list names no page of the pool.
__device__ __forceinline__ int page_row(const int* __restrict__ list, int max_blocks, int page_size, int n_pages, int at) {
    const int block = at / page_size;
    if (at < 0 || block >= max_blocks) return -1;
    const int page = list[block];
    return static_cast<unsigned>(page) < static_cast<unsigned>(n_pages) ? page * page_size + (at - block * page_size) : -1;
}

struct StepMapsParams {
    const int *rows, *n_new, *lengths, *pages, *parents;
    long long ld_pages;
    int n_seqs, n_requests, tokens, page_size, n_pages, max_blocks, max_new, words;
    int *cu_q, *cached, *ctx_len, *token_seq, *positions, *slots, *block_tables;
    unsigned long long* ancestors;
};

// Workgroup (b, part) of (n_seqs + 1, parts): sequence b's share of its tokens and of its row of the table; the last b has the tokens
// behind the last sequence.
__global__ void __launch_bounds__(TREE_THREADS) step_maps_kernel(StepMapsParams a) {
    __shared__ int sums[TREE_THREADS / MLLM_WAVE];
    __shared__ int up_s[TREE_MAX_NODES], depth_s[TREE_MAX_NODES];
    __shared__ unsigned long long above_s[TREE_MAX_NODES / 64][TREE_MAX_NODES];
    const int b = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
    auto row_of = [&](int i) {
        const int r = a.rows != nullptr ? a.rows[i] : i;
        return static_cast<unsigned>(r) < static_cast<unsigned>(a.n_requests) ? r : -1;
    };
    auto count_of = [&](int i) { return row_of(i) < 0 ? 0 : min(max(a.n_new[i], 0), a.max_new); };
    // (what does not need the place of the first token is read while the counts come)
    const bool behind = b == a.n_seqs;
    const int row = behind ? -1 : row_of(b), count = behind ? 0 : count_of(b);
    const int cached = row < 0 ? 0 : min(max(a.lengths[row], 0), INT32_MAX - a.max_new);
    int before = 0;
    for (int i = tid; i < b; i += TREE_THREADS) before += count_of(i);
    const int first = min(block_sum_int(before, sums), a.tokens);
    if (behind) {
        for (int t = first + part * TREE_THREADS + tid; t < a.tokens; t += parts * TREE_THREADS) {
            a.token_seq[t] = 0;
            a.positions[t] = 0;
            a.slots[t] = -1;
            for (int w = 0; w < a.words; ++w) a.ancestors[static_cast<size_t>(t) * a.words + w] = 0;
        }
        if (part == 0 && tid == 0) a.cu_q[b] = first;
        return;
    }
    const int n = min(count, a.tokens - first);
    const int* list = a.pages + static_cast<size_t>(max(row, 0)) * a.ld_pages;
    if (part == 0 && tid == 0) {
        a.cu_q[b] = first;
        a.cached[b] = cached;
        a.ctx_len[b] = cached + n;
    }
    const int have = static_cast<int>(min((static_cast<long long>(cached) + n + a.page_size - 1) / a.page_size, static_cast<long long>(a.max_blocks)));
    int* table = a.block_tables + static_cast<size_t>(b) * a.max_blocks;
    for (int j = part * TREE_THREADS + tid; j < a.max_blocks; j += parts * TREE_THREADS) table[j] = j < have ? list[j] : 0;
    if (a.parents == nullptr) {
        for (int i = part * TREE_THREADS + tid; i < n; i += parts * TREE_THREADS) {
            a.token_seq[first + i] = b;
            a.positions[first + i] = cached + i;
            a.slots[first + i] = page_row(list, a.max_blocks, a.page_size, a.n_pages, cached + i);
            for (int w = 0; w < a.words; ++w) {          // (a chain: bits 0 to i)
                const int bits = i + 1 - 64 * w;
                a.ancestors[static_cast<size_t>(first + i) * a.words + w] = bits <= 0 ? 0 : bits >= 64 ? ~0ull : (1ull << bits) - 1;
            }
        }
        return;
    }
    if (part != 0) return;
    // A node's depth and the nodes above it, by doubling: in every round a node takes what the node its jump leads to has gathered, and
    // that node's jump, so that a chain of 2^k nodes takes k rounds.
    int up = -1, depth = 0;
    unsigned long long above[TREE_MAX_NODES / 64] = {};
    if (tid < n) {
        const int p = a.parents[first + tid];
        up = p >= 0 && p < tid ? p : -1;
        depth = up >= 0 ? 1 : 0;
        above[0] = tid < 64 ? 1ull << tid : 0;
        above[1] = tid >= 64 && tid < 128 ? 1ull << (tid - 64) : 0;
        above[2] = tid >= 128 && tid < 192 ? 1ull << (tid - 128) : 0;
        above[3] = tid >= 192 ? 1ull << (tid - 192) : 0;
    }
    while (__syncthreads_or(up >= 0)) {
        up_s[tid] = up;
        depth_s[tid] = depth;
#pragma unroll
        for (int w = 0; w < TREE_MAX_NODES / 64; ++w) above_s[w][tid] = above[w];
        __syncthreads();
        if (up >= 0) {
            const int to = up;
            depth += depth_s[to];
            up = up_s[to];
#pragma unroll
            for (int w = 0; w < TREE_MAX_NODES / 64; ++w) above[w] |= above_s[w][to];
        }
    }
    if (tid < n) {
        a.token_seq[first + tid] = b;
        a.positions[first + tid] = cached + depth;
        a.slots[first + tid] = -1;
#pragma unroll
        for (int w = 0; w < TREE_MAX_NODES / 64; ++w)
            if (w < a.words) a.ancestors[static_cast<size_t>(first + tid) * a.words + w] = above[w];
    }
}

struct TreeAcceptParams {
    const int *choices, *ids, *parents, *cu_q, *cached, *block_tables, *rows;
    int n_seqs, tokens, page_size, n_pages, max_blocks, max_new, n_requests;
    int *kept, *path, *next, *slots, *lengths;
};

// A node's confirmed child is the first of its children whose drafted token the model chose at the node. Following these from the
// root gives the path; by doubling, as above, so that a path of 2^k nodes takes k rounds and not 2^k dependent reads.
__global__ void __launch_bounds__(TREE_THREADS) tree_accept_kernel(TreeAcceptParams a) {
    __shared__ int choice_s[TREE_MAX_NODES], child_s[TREE_MAX_NODES], place_s[TREE_MAX_NODES];
    constexpr int NONE = INT32_MAX;
    const int b = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
    const int first = min(max(a.cu_q[b], 0), a.tokens);
    if (b == a.n_seqs) {
        for (int t = first + tid; t < a.tokens; t += threads) a.slots[t] = -1;
        const int ahead = min(max(a.cu_q[0], 0), a.tokens);          // (rows in front of the first sequence, where there are any)
        for (int t = tid; t < ahead; t += threads) a.slots[t] = -1;
        return;
    }
    const int all = min(max(a.cu_q[b + 1] - first, 0), a.tokens - first), n = min(all, a.max_new);
    const int cached = min(max(a.cached[b], 0), INT32_MAX - a.max_new);
    int id = 0, parent = -1, child = NONE, place = -1;
    if (tid < n) {
        id = a.ids[first + tid];
        parent = a.parents[first + tid];
        choice_s[tid] = a.choices[first + tid];
        place = tid == 0 ? 0 : -1;
    }
    child_s[tid] = NONE;
    place_s[tid] = place;
    __syncthreads();
    if (tid < n && parent >= 0 && parent < tid && choice_s[parent] == id) atomicMin(&child_s[parent], tid);
    __syncthreads();
    for (int step = 1; child_s[0] != NONE; step <<= 1) {
        child = child_s[tid];
        place = place_s[tid];
        const int further = child != NONE ? child_s[child] : NONE;
        __syncthreads();
        if (child != NONE && place >= 0) place_s[child] = place + step;
        child_s[tid] = further;
        __syncthreads();
    }
    place = place_s[tid];
    const int kept = __syncthreads_count(place >= 0);
    int* path = a.path + static_cast<size_t>(b) * a.max_new;
    // Of several sequences of one request the last one's length stands, and its nodes alone go to the pages: two sequences' keys in one row would be
    // those that arrive last.
    const int request = a.lengths == nullptr ? -1 : a.rows != nullptr ? a.rows[b] : b;
    const bool named = static_cast<unsigned>(request) < static_cast<unsigned>(a.n_requests);
    int later = 0;
    if (named && a.rows != nullptr)
        for (int i = b + 1 + tid; i < a.n_seqs; i += threads) later |= a.rows[i] == request;
    later = __syncthreads_or(later);
    if (tid < n) {
        a.slots[first + tid] = place >= 0 && !later ? page_row(a.block_tables + static_cast<size_t>(b) * a.max_blocks, a.max_blocks, a.page_size, a.n_pages, cached + place) : -1;
        if (place >= 0) path[place] = first + tid;
        if (place == kept - 1) a.next[b] = choice_s[tid];
    }
    for (int i = kept + tid; i < a.max_new; i += threads) path[i] = -1;
    for (int i = n + tid; i < all; i += threads) a.slots[first + i] = -1;
    if (tid == 0) {
        a.kept[b] = kept;
        if (kept == 0) a.next[b] = -1;
        if (named && !later) a.lengths[request] = cached + kept;
    }
}

}  // namespace

extern "C" {

int mllm_tree_max_nodes(void) { return TREE_MAX_NODES; }

// Returns 0, a HIP error code, or -1 for sizes the kernel refuses. parents null: portions of a text; otherwise trees. Where `ancestors` is not null it
// takes `words` words a token, of trees and of portions (a chain each), which have at most mllm_tree_max_nodes() nodes then.
int mllm_step_maps(const int* rows, const int* n_new, const int* lengths, const int* pages, long long ld_pages, const int* parents, int n_seqs,
                   int n_requests, int tokens, int page_size, int n_pages, int max_blocks, int max_new, int words, int* cu_q, int* cached,
                   int* ctx_len, int* token_seq, int* positions, int* slots, int* block_tables, unsigned long long* ancestors, hipStream_t stream) {
    if (n_seqs < 1 || n_requests < 1 || tokens < 1 || page_size < 1 || n_pages < 1 || max_blocks < 1 || max_new < 1) return -1;
    if (static_cast<long long>(n_seqs) * max_new > INT32_MAX || static_cast<long long>(n_pages) * page_size > INT32_MAX) return -1;
    if (parents != nullptr && ancestors == nullptr) return -1;
    if (ancestors != nullptr && (max_new > TREE_MAX_NODES || words < (max_new + 63) / 64 || words > TREE_MAX_NODES / 64)) return -1;
    const StepMapsParams p{rows, n_new, lengths, pages, parents, ld_pages, n_seqs, n_requests, tokens, page_size, n_pages, max_blocks, max_new,
                           ancestors != nullptr ? words : 0, cu_q, cached, ctx_len, token_seq, positions, slots, block_tables, ancestors};
    // (a workgroup for every 1,024 entries of a table or tokens of a portion)
    const int parts = std::min(64, (std::max(max_blocks, parents != nullptr ? 1 : max_new) + 1023) / 1024);
    step_maps_kernel<<<dim3(n_seqs + 1, parts), TREE_THREADS, 0, stream>>>(p);
    MLLM_LAUNCH_CHECK();
    return 0;
}

int mllm_tree_accept(const int* choices, const int* ids, const int* parents, const int* cu_q, const int* cached, const int* block_tables,
                     const int* rows, int n_seqs, int tokens, int page_size, int n_pages, int max_blocks, int max_new, int n_requests, int* kept,
                     int* path, int* next, int* slots, int* lengths, hipStream_t stream) {
    if (n_seqs < 1 || tokens < 1 || page_size < 1 || n_pages < 1 || max_blocks < 1 || max_new < 1 || max_new > TREE_MAX_NODES) return -1;
    if (static_cast<long long>(n_pages) * page_size > INT32_MAX) return -1;
    const TreeAcceptParams p{choices, ids, parents, cu_q, cached, block_tables, rows, n_seqs, tokens, page_size, n_pages, max_blocks, max_new, n_requests,
                             kept, path, next, slots, lengths};
    tree_accept_kernel<<<n_seqs + 1, (max_new + MLLM_WAVE - 1) / MLLM_WAVE * MLLM_WAVE, 0, stream>>>(p);
    MLLM_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
