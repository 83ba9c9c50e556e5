// Checked dispatch of what a step over trees of drafted tokens needs: its arrays, rotary positions, attention, acceptance.
#include "ops.h"

#include <climits>

#include "kernels.h"

namespace minillm {

static void check(int rc, const char* what) {
    if (rc == 0) return;
    if (rc < 0) fail("%s: the kernel refuses these sizes (code %d)", what, rc);
    fail("%s: HIP error %d (%s) at launch", what, rc, hipGetErrorString(static_cast<hipError_t>(rc)));
}

static bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

static void need_dtype(const Tensor2& t, const char* name) {
    if (t.dtype != F32 && t.dtype != BF16) fail("%s: unsupported dtype code %d (float32 or bfloat16)", name, t.dtype);
    if (t.data == nullptr && t.rows * t.cols > 0) fail("%s: null data pointer", name);
    if (t.rows < 0 || t.cols < 0 || t.stride < t.cols) fail("%s: rows of %lld columns lie %lld apart", name, (long long)t.cols, (long long)t.stride);
}

static void need_pool(int64_t n_pages, int64_t page_size, const char* what) {
    if (n_pages < 1 || page_size < 1 || n_pages > INT_MAX / page_size) fail("%s: %lld pages of %lld rows", what, (long long)n_pages, (long long)page_size);
}

// (every sequence looks at the others', so that the work grows with the square of their number)
static constexpr int MOST_SEQS = 65536;
static void need_seqs(int n_seqs, const char* what) {
    if (n_seqs > MOST_SEQS) fail("%s: %d sequences (at most %d)", what, n_seqs, MOST_SEQS);
}

// Arrays of one call. What one workgroup writes another may read, or write too: outputs lie apart from inputs and from each other.
struct Span {
    const char* name;
    const void* at;
    int64_t bytes;
};
template <size_t N, size_t M>
static void need_apart(const char* what, const Span (&outs)[N], const Span (&ins)[M]) {
    auto check_two = [&](const Span& a, const Span& b) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
        if (a.at != nullptr && b.at != nullptr && a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes) fail("%s: %s shares memory with %s", what, a.name, b.name);
    };
    for (size_t i = 0; i < N; ++i) {
        for (size_t j = i + 1; j < N; ++j) check_two(outs[i], outs[j]);
        for (const Span& in : ins) check_two(outs[i], in);
    }
}

int tree_max_nodes() { return mllm_tree_max_nodes(); }

void step_maps(const StepMapsArgs& a, hipStream_t stream) {
    if (a.n_seqs < 1 || a.n_requests < 1 || a.tokens < 1 || a.max_blocks < 1 || a.max_new < 1)
        fail("step_maps: %d sequences of %d requests, %d tokens, %d blocks, at most %d tokens a sequence", a.n_seqs, a.n_requests, a.tokens, a.max_blocks, a.max_new);
    need_pool(a.n_pages, a.page_size, "step_maps");
    if (static_cast<int64_t>(a.n_seqs) * a.max_new > INT_MAX) fail("step_maps: %d sequences of up to %d tokens", a.n_seqs, a.max_new);
    if (a.ld_pages < a.max_blocks) fail("step_maps: rows of %d pages lie %lld apart", a.max_blocks, (long long)a.ld_pages);
    if (a.n_new == nullptr || a.lengths == nullptr || a.pages == nullptr || a.cu_q == nullptr || a.cached == nullptr || a.ctx_len == nullptr ||
        a.token_seq == nullptr || a.positions == nullptr || a.slots == nullptr || a.block_tables == nullptr)
        fail("step_maps: an array is missing");
    if (a.rows == nullptr && a.n_seqs > a.n_requests) fail("step_maps: %d sequences without rows, %d requests", a.n_seqs, a.n_requests);
    if (a.parents != nullptr || a.ancestors != nullptr) {
        if (a.max_new > tree_max_nodes()) fail("step_maps: a tree has at most %d nodes, not %d", tree_max_nodes(), a.max_new);
        if (a.ancestors == nullptr || a.words < (a.max_new + 63) / 64 || a.words > tree_max_nodes() / 64)
            fail("step_maps: trees of up to %d nodes need %d words of ancestors a node, not %d", a.max_new, (a.max_new + 63) / 64, a.words);
    }
    need_seqs(a.n_seqs, "step_maps");
    const int64_t n = 4ll * a.n_seqs, t = 4ll * a.tokens;
    need_apart("step_maps", {{"cu_q", a.cu_q, n + 4}, {"cached", a.cached, n}, {"ctx_len", a.ctx_len, n}, {"token_seq", a.token_seq, t}, {"positions", a.positions, t},
                             {"slots", a.slots, t}, {"block_tables", a.block_tables, n * a.max_blocks}, {"ancestors", a.ancestors, a.ancestors == nullptr ? 0 : 2 * t * a.words}},
               {{"rows", a.rows, n}, {"n_new", a.n_new, n}, {"lengths", a.lengths, 4ll * a.n_requests},
                {"pages", a.pages, 4 * ((a.n_requests - 1) * a.ld_pages + a.max_blocks)}, {"parents", a.parents, t}});
    check(mllm_step_maps(a.rows, a.n_new, a.lengths, a.pages, a.ld_pages, a.parents, a.n_seqs, a.n_requests, a.tokens, a.page_size, a.n_pages, a.max_blocks,
                         a.max_new, a.words, a.cu_q, a.cached, a.ctx_len, a.token_seq, a.positions, a.slots, a.block_tables, a.ancestors, stream), "step_maps");
}

void rotary(const Tensor2& x, const int* positions, const unsigned long long* turns, int pairs, int n_heads, int head_dim, bool interleaved,
            float amplitude, const Tensor2& out, hipStream_t stream) {
    need_dtype(x, "rotary x");
    need_dtype(out, "rotary out");
    if (n_heads < 1 || n_heads > 65535 || head_dim < 2 || head_dim % 2 != 0 || head_dim > INT_MAX / 65535) fail("rotary: %d heads of %d columns (an even number)", n_heads, head_dim);
    if (pairs < 1 || pairs > head_dim / 2) fail("rotary: %d pairs in heads of %d columns", pairs, head_dim);
    if (x.cols != static_cast<int64_t>(n_heads) * head_dim || out.cols != x.cols || out.rows != x.rows || out.dtype != x.dtype)
        fail("rotary: x is [%lld, %lld], out [%lld, %lld], %d heads of %d in one dtype expected", (long long)x.rows, (long long)x.cols, (long long)out.rows,
             (long long)out.cols, n_heads, head_dim);
    if (x.rows > INT_MAX || x.rows * head_dim > 1ll << 38) fail("rotary: %lld rows", (long long)x.rows);
    if (positions == nullptr || turns == nullptr) fail("rotary: positions and frequencies are needed");
    if (!(x.data == out.data && x.stride == out.stride) && overlap(x, out)) fail("rotary: out shares memory with x and is not x");
    check(mllm_rotary(x.data, x.stride, positions, turns, static_cast<int>(x.rows), pairs, n_heads, head_dim, interleaved ? 1 : 0, amplitude, out.data,
                      out.stride, x.dtype, stream), "rotary");
}

static void check_tree_attention(const TreeAttentionArgs& a) {
    for (const Tensor2* t : {&a.q, &a.k, &a.v, &a.k_pages, &a.v_pages, &a.out}) {
        need_dtype(*t, "tree_attention");
        if (t->dtype != a.q.dtype) fail("tree_attention: queries, keys, values, pages and output are of one dtype");
    }
    const int64_t T = a.q.rows, esz = static_cast<int64_t>(a.q.esz());
    if (a.n_heads < 1 || a.n_kv_heads < 1 || a.n_heads % a.n_kv_heads != 0 || a.n_heads > 65535)
        fail("tree_attention: n_heads=%d is not a multiple of n_kv_heads=%d", a.n_heads, a.n_kv_heads);
    if (a.head_dim % 8 != 0 || a.head_dim < 8 || a.head_dim > 256) fail("tree_attention: head_dim=%d is not supported (multiples of 8 up to 256)", a.head_dim);
    const int64_t q_dim = static_cast<int64_t>(a.n_heads) * a.head_dim, kv_dim = static_cast<int64_t>(a.n_kv_heads) * a.head_dim;
    if (a.q.cols != q_dim || a.out.rows != T || a.out.cols != q_dim) fail("tree_attention: q and out must be [%lld, %lld]", (long long)T, (long long)q_dim);
    if (a.k.rows != T || a.v.rows != T || a.k.cols != kv_dim || a.v.cols != kv_dim) fail("tree_attention: k and v must be [%lld, %lld]", (long long)T, (long long)kv_dim);
    if (T > INT_MAX) fail("tree_attention: %lld rows", (long long)T);
    if (!a.k_pages.contiguous() || !a.v_pages.contiguous() || a.k_pages.cols != kv_dim || a.v_pages.cols != kv_dim || a.k_pages.rows != a.v_pages.rows)
        fail("tree_attention: key and value pages must be contiguous [rows, %lld] of one shape", (long long)kv_dim);
    if (a.page_size < 1 || a.k_pages.rows < 1 || a.k_pages.rows % a.page_size != 0) fail("tree_attention: the page pool is not a whole number of pages");
    need_pool(a.k_pages.rows / a.page_size, a.page_size, "tree_attention");
    for (const Tensor2* t : {&a.q, &a.k, &a.v, &a.k_pages, &a.v_pages, &a.out})
        if (!aligned(t->data, 16) || t->stride * esz % 16 != 0) fail("tree_attention: rows and heads must be 16-byte aligned");
    if (a.n_seqs < 1 || a.max_blocks < 1 || a.block_tables == nullptr || a.cached == nullptr || a.cu_q == nullptr || a.ancestors == nullptr)
        fail("tree_attention: block tables, cached lengths, sequence bounds and ancestors are needed");
    if (a.words < 1 || a.words > tree_max_nodes() / 64 || a.max_new < 1 || a.max_new > 64 * a.words)
        fail("tree_attention: %d words of ancestors for trees of up to %d nodes (at most %d)", a.words, a.max_new, tree_max_nodes());
    need_seqs(a.n_seqs, "tree_attention");
    if (a.max_cached < 0 || a.window < 0) fail("tree_attention: max_cached=%d, window=%d", a.max_cached, a.window);
    if (a.window > 0 && a.positions == nullptr) fail("tree_attention: positions are needed with a window");
    for (const Tensor2* t : {&a.q, &a.k, &a.v, &a.k_pages, &a.v_pages})
        if (overlap(a.out, *t)) fail("tree_attention: out shares memory with an input");
}

size_t tree_attention_workspace_floats(int tokens, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_new, int max_cached, int window, int dtype) {
    if (tokens < 1 || n_seqs < 1 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 || head_dim < 8 || head_dim > 256 || max_new < 1 ||
        max_new > tree_max_nodes() || max_cached < 0 || window < 0) return 0;
    return static_cast<size_t>(mllm_tree_attention_ws_floats(tokens, n_seqs, n_heads, n_kv_heads, head_dim, max_new, max_cached, window, dtype));
}

void tree_attention(const TreeAttentionArgs& a, hipStream_t stream) {
    check_tree_attention(a);
    const size_t floats = tree_attention_workspace_floats(static_cast<int>(a.q.rows), a.n_seqs, a.n_heads, a.n_kv_heads, a.head_dim, a.max_new, a.max_cached, a.window,
                                                          a.q.dtype);
    if (floats > 0 && (a.workspace == nullptr || a.workspace_floats < floats || !aligned(a.workspace, 16)))
        fail("tree_attention: a workspace of %zu floats is needed (16-byte aligned), %zu are there", floats, a.workspace_floats);
    check(mllm_tree_attention(a.q.data, a.q.stride, a.k.data, a.k.stride, a.v.data, a.v.stride, a.k_pages.data, a.v_pages.data,
                              static_cast<int>(a.k_pages.rows / a.page_size), a.page_size, a.block_tables, a.n_seqs, a.max_blocks, a.cached, a.cu_q,
                              a.ancestors, a.words, a.positions, static_cast<int>(a.q.rows), a.n_heads, a.n_kv_heads, a.head_dim, a.scale, a.window,
                              a.max_new, a.max_cached, a.out.data, a.out.stride, a.workspace, a.q.dtype, stream), "tree_attention");
}

void tree_accept(const TreeAcceptArgs& a, hipStream_t stream) {
    if (a.n_seqs < 1 || a.tokens < 1 || a.max_blocks < 1) fail("tree_accept: %d sequences, %d tokens, %d blocks", a.n_seqs, a.tokens, a.max_blocks);
    need_pool(a.n_pages, a.page_size, "tree_accept");
    if (a.max_new < 1 || a.max_new > tree_max_nodes()) fail("tree_accept: a tree has at most %d nodes, not %d", tree_max_nodes(), a.max_new);
    if (a.choices == nullptr || a.ids == nullptr || a.parents == nullptr || a.cu_q == nullptr || a.cached == nullptr || a.block_tables == nullptr ||
        a.kept == nullptr || a.path == nullptr || a.next == nullptr || a.slots == nullptr)
        fail("tree_accept: an array is missing");
    if (a.lengths != nullptr && a.rows == nullptr && a.n_seqs > a.n_requests) fail("tree_accept: %d sequences without rows, %d lengths", a.n_seqs, a.n_requests);
    need_seqs(a.n_seqs, "tree_accept");
    const int64_t n = 4ll * a.n_seqs, t = 4ll * a.tokens;
    need_apart("tree_accept", {{"kept", a.kept, n}, {"path", a.path, n * a.max_new}, {"next_token", a.next, n}, {"slots", a.slots, t}, {"lengths", a.lengths, 4ll * a.n_requests}},
               {{"choices", a.choices, t}, {"ids", a.ids, t}, {"parents", a.parents, t}, {"cu_q", a.cu_q, n + 4}, {"cached", a.cached, n},
                {"block_tables", a.block_tables, n * a.max_blocks}, {"rows", a.rows, n}});
    check(mllm_tree_accept(a.choices, a.ids, a.parents, a.cu_q, a.cached, a.block_tables, a.rows, a.n_seqs, a.tokens, a.page_size, a.n_pages, a.max_blocks,
                           a.max_new, a.n_requests, a.kept, a.path, a.next, a.slots, a.lengths, stream), "tree_accept");
}

}  // namespace minillm
