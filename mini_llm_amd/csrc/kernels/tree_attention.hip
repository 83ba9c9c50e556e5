// Attention of drafted trees over the paged cache, for gfx950. Node t of sequence b (rows cu_q[b] to cu_q[b + 1] of the step) sees the
// sequence's cached positions j < cached[b], whose keys and values lie in the pages, and of the sequence's own nodes those whose bit is set
// in ancestors[t]; their keys and values lie in the step's rows. With a window, what stands at positions[t] - window or in front of it is not
// seen. With z_j = scale q_t . k_j over what is seen:
//   o_t = sum_j exp(z_j - max z) v_j / sum_j exp(z_j - max z),   a node that sees nothing gets zeros.
// What is not seen counts for nothing whatever stands there (infinities and NaN among it), and a block table's entry that names no page of
// the pool holds nothing that is seen.
//
// One wavefront a node and head: a lane has a key of 64 for the scores, and columns of the head for the values.
#include "common.h"

#define TREE_WAVES 4

struct TreeAttentionParams {
    const void *q, *k, *v, *k_pages, *v_pages;
    long long ldq, ldk, ldv, ldo;
    const int *block_tables, *cached, *cu_q, *positions;
    const unsigned long long* ancestors;
    int n_seqs, max_blocks, tokens, words, n_heads, n_kv_heads, head_dim, page_size, n_pages, window;
    float scale;
    void* out;
};

template <typename T>
__global__ void __launch_bounds__(TREE_WAVES * 64) tree_attention_kernel(TreeAttentionParams a) {
    __shared__ float q_s[TREE_WAVES][256], p_s[TREE_WAVES][64];
    __shared__ int row_s[TREE_WAVES][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, t = blockIdx.y * TREE_WAVES + wave, h = blockIdx.x;
    if (t >= a.tokens) return;
    int lo = 0, hi = a.n_seqs;              // the sequence whose rows hold t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.cu_q[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
    }
    const int b = lo;
    if (b >= a.n_seqs) return;
    const int first = a.cu_q[b], nodes = min(min(a.cu_q[b + 1], a.tokens) - first, 64 * a.words);
    if (t < first || t - first >= nodes) return;
    const int dim = a.head_dim, hk = h / (a.n_heads / a.n_kv_heads);
    const size_t kv_dim = static_cast<size_t>(a.n_kv_heads) * dim;
    const T* q = static_cast<const T*>(a.q) + t * a.ldq + h * dim;
    for (int d = lane; d < dim; d += 64) q_s[wave][d] = to_float(q[d]);
    const int low = a.window > 0 ? a.positions[t] - a.window + 1 : INT32_MIN;
    const long long room = static_cast<long long>(a.max_blocks) * a.page_size;
    const int cached = static_cast<int>(min(static_cast<long long>(max(a.cached[b], 0)), room));
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    wave_lds_sync();
    for (int pass = 0; pass < 2; ++pass) {
        const T* keys = static_cast<const T*>(pass == 0 ? a.k_pages : a.k) + hk * dim;
        const T* values = static_cast<const T*>(pass == 0 ? a.v_pages : a.v) + hk * dim;
        const size_t ldk = pass == 0 ? kv_dim : a.ldk, ldv = pass == 0 ? kv_dim : a.ldv;
        const int n = pass == 0 ? cached : nodes;
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int j = j0 + lane;
            int row = -1;
            if (pass == 0) {
                if (j < n && j >= low) {
                    const int page = a.block_tables[static_cast<size_t>(b) * a.max_blocks + j / a.page_size];
                    if (static_cast<unsigned>(page) < static_cast<unsigned>(a.n_pages)) row = page * a.page_size + j % a.page_size;
                }
            } else if (j < n && (a.ancestors[static_cast<size_t>(t) * a.words + j0 / 64] >> lane & 1)) {
                if (a.window <= 0 || a.positions[first + j] >= low) row = first + j;
            }
            float z = -INFINITY;
            if (row >= 0) {
                float d = 0.f;
                for (int e = 0; e < dim; ++e) d = fmaf(q_s[wave][e], to_float(keys[row * ldk + e]), d);
                z = d * (a.scale * MLLM_LOG2E);
            }
            const float mn = fmaxf(m, wave_max(z)), ref = mn == -INFINITY ? 0.f : mn;
            const float p = row >= 0 ? exp2_for<T>(z - ref) : 0.f, fix = exp2_for<T>(m - ref);
            p_s[wave][lane] = p;
            row_s[wave][lane] = row;
            wave_lds_sync();
            l = l * fix + wave_sum(p);
            for (int i = 0; i < 4; ++i) o[i] *= fix;
            for (int kk = 0; kk < 64; ++kk) {
                if (row_s[wave][kk] < 0) continue;
                for (int i = 0; i < 4; ++i)
                    if (lane + 64 * i < dim) o[i] = fmaf(p_s[wave][kk], to_float(values[row_s[wave][kk] * ldv + lane + 64 * i]), o[i]);
            }
            m = mn;
            wave_lds_sync();
        }
    }
    T* out = static_cast<T*>(a.out) + t * a.ldo + h * dim;
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < dim) out[lane + 64 * i] = from_float<T>(l == 0.f ? 0.f : o[i] / l);
}

extern "C" {

// Floats of workspace for a call of these sizes.
long long mllm_tree_attention_ws_floats(int, int, int, int, int, int, int, int, int) { return 0; }

// Returns 0, a HIP error code, or -1 for sizes the kernel refuses.
int mllm_tree_attention(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* k_pages, const void* v_pages,
                        int n_pages, int page_size, const int* block_tables, int n_seqs, int max_blocks, const int* cached, const int* cu_q,
                        const unsigned long long* ancestors, int words, const int* positions, int tokens, int n_heads, int n_kv_heads, int head_dim,
                        float scale, int window, int max_new, int max_cached, void* out, long long ldo, float*, int dtype, hipStream_t stream) {
    if (tokens < 1 || n_seqs < 1) return 0;
    if (n_kv_heads < 1 || n_heads % n_kv_heads != 0 || head_dim < 8 || head_dim > 256 || head_dim % 8 != 0 || words < 1 || words > 4 || page_size < 1) return -1;
    if (static_cast<long long>(n_pages) * page_size > INT32_MAX) return -1;
    const TreeAttentionParams p{q, k, v, k_pages, v_pages, ldq, ldk, ldv, ldo, block_tables, cached, cu_q, positions, ancestors, n_seqs, max_blocks, tokens, words,
                                n_heads, n_kv_heads, head_dim, page_size, n_pages, window, scale, out};
    (void)max_new; (void)max_cached;
    const dim3 grid(n_heads, (tokens + TREE_WAVES - 1) / TREE_WAVES);
    if (dtype == MLLM_F32) tree_attention_kernel<float><<<grid, TREE_WAVES * 64, 0, stream>>>(p);
    else tree_attention_kernel<bf16_t><<<grid, TREE_WAVES * 64, 0, stream>>>(p);
    MLLM_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
