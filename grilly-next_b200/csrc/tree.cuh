// A step of several drafted tokens over the paged cache: what its append, its attention and the keeping of the accepted path share.
// Sequence b has n nodes, the rows behind its cached tokens; parents[t] < t is the node that node t follows, -1 for the cached tokens.
#pragma once
#include "common.cuh"

namespace grl {

// Device status word, kind 6: a sequence whose numbers do not fit ([1] = what, [2] = sequence, [3] = the number).
enum { TREE_BAD_PARENT = 1, TREE_BAD_COUNT = 2, TREE_BAD_LENGTH = 3, TREE_BAD_PAGE = 4, TREE_BAD_PATH = 5 };

int check_tree_layout(const grl_kv_layout& kv);
inline int pool_pages(const grl_kv_layout& kv) { return kv.num_pages > 0 ? kv.num_pages : kv.batch * kv.max_pages; }

// ---- tree attention
struct TreeArgs {
    const void* k_pages;
    const void* v_pages;
    const int32_t* block_table;
    const int32_t* seq_lens;
    const void* q;
    void* out;
    const int32_t* parents;
    const int32_t* n_nodes;
    // [split][ O (rows, D) | (m, l) (rows) ], rows = (sequence, kv head, node, head of the group); m in the exp2 domain.  l = 0: the split has no
    // weight in the row (nothing seen, or scores of -inf only); l < 0: no node's row, 0 in the result.
    float* part;
    size_t part_stride;     // floats of a split, rows * (D + 2) rounded up to 16 bytes
    int32_t* status;
    int B, Hq, Hkv, G, T, R, D, P, max_pages, num_pages, n_splits;      // R = T * G rows of a (sequence, kv head)
    float scale_log2;
    long long wait_limit;
};

// How the tensor-core kernel lays a call out (tree_sm100.cu).
struct TreeTensorPlan {
    int splits;         // CTAs of a (sequence, kv head, group of rows)
    int groups;         // of rows of a (sequence, kv head)
    size_t workspace;
};
TreeTensorPlan tree_sm100_plan(const grl_device* dev, int B, int Hkv, int R, int D, int longest, int asked);
int tree_sm100_launch(grl_device* dev, const TreeArgs& a, const TreeTensorPlan& plan);

// The parts of n_splits splits of every (sequence, kv head), `rows` rows each (tree_sm100.cu).
int tree_join_launch(grl_device* dev, const TreeArgs& a, int rows);
// How the kernel for few rows lays a call out (tree_mma.cu): up to kTreeFewRows rows of a (sequence, kv head).
// us, 16 rows of 8 kv heads, this kernel / the one of 128-row tiles: 1 x 300 tokens 8.8 / 9.9, 1 x 1001 9.8 / 12.9, 4 x 600 10.0 / 12.8, 4 x 4096
// 18.5 / 24.9, 16 x 4096 46.2 / 56.1, 32 x 600 17.9 / 31.3, 32 x 4096 82.6 / 109, 1 x 131072 106 / 102.  With 32 rows as two operands of a warp,
// one CTA an SM: 10.6 / 9.6, 11.6 / 11.8, 17.8 / 12.9, 32 / 25, 78 / 56, 33 / 31.5, 136 / 109; so it takes 16.
constexpr int kTreeFewRows = 16;
struct TreeMmaPlan {
    int splits, cluster;
    bool alone;         // CTAs that must not share an SM
    size_t workspace;
};
TreeMmaPlan tree_mma_plan(grl_device* dev, int B, int Hkv, int D, int longest, int asked);
int tree_mma_launch(grl_device* dev, const TreeArgs& a, const TreeMmaPlan& plan);

// A row that has met a score that is no number (l is NaN then) has no maximum, which such scores do not raise: 0 stands for it, so that the row is not
// taken for one that saw nothing, whose maximum is -inf.  Its sum makes the result NaN, as the definition has it.
#ifdef __CUDACC__
__device__ __forceinline__ float tree_row_max(float m, float l) { return l != l ? 0.f : m; }
#endif

inline size_t tree_part_stride(size_t rows, int D) { return (rows * (D + 2) + 3) / 4 * 4; }

#ifdef __CUDACC__
// A look at a barrier that does not suspend the thread; it costs a third of a wait where the phase is over.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void tree_fail(int32_t* status, int what, int b, int value) {
    if (status && atomicCAS(status, 0, GRL_ERR_INVALID) == 0) {
        status[1] = (6 << 28) | what;
        status[2] = b;
        status[3] = value;
    }
}
__device__ __forceinline__ int tree_count(const int32_t* n_nodes, int T, int b) { return n_nodes ? n_nodes[b] : T; }
// Nodes of a sequence and the cached tokens ahead of them, where seq_lens counts both; -1 (and the status word) where they do not fit.
__device__ __forceinline__ int tree_nodes(const TreeArgs& a, int b, int* prefix, bool tell) {
    const int n = tree_count(a.n_nodes, a.T, b), len = a.seq_lens[b];
    *prefix = len - n;
    if (n < 0 || n > a.T) {
        if (tell) tree_fail(a.status, TREE_BAD_COUNT, b, n);
        return -1;
    }
    if (len < n || len > a.max_pages * a.P) {
        if (tell) tree_fail(a.status, TREE_BAD_LENGTH, b, len);
        return -1;
    }
    return n;
}

// Ancestors of the first n <= GRL_MAX_TREE nodes, each one's own bit among them, by doubling: after round i a node knows 2^i generations.
struct TreeMasks {
    uint4 seen[GRL_MAX_TREE];
    int up[GRL_MAX_TREE];
};
__device__ __forceinline__ uint4 low_bits(int n) {      // bits 0 .. n-1 of 128
    const auto word = [n](int w) { const int k = n - 32 * w; return k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u; };
    return make_uint4(word(0), word(1), word(2), word(3));
}
// The whole CTA (at least GRL_MAX_TREE threads) calls it, thread t with the parent of node t; returns whether the parents are a tree.
__device__ __forceinline__ bool tree_masks(TreeMasks& m, int p, int n) {
    const int t = threadIdx.x;
    if (t >= n) p = -1;
    const bool bad = t < n && (p < -1 || p >= t);
    if (bad) p = -1;
    uint4 own = make_uint4(0u, 0u, 0u, 0u);
    if (t < n) {
        const uint32_t bit = 1u << (t & 31);
        own = make_uint4(t >> 5 == 0 ? bit : 0u, t >> 5 == 1 ? bit : 0u, t >> 5 == 2 ? bit : 0u, t >> 5 == 3 ? bit : 0u);
        m.seen[t] = own;
        m.up[t] = p;
    }
    if (__syncthreads_or(bad)) return false;
    while (__syncthreads_or(p >= 0)) {
        int next = -1;
        if (p >= 0) {
            const uint4 s = m.seen[p];
            own = make_uint4(own.x | s.x, own.y | s.y, own.z | s.z, own.w | s.w);
            next = m.up[p];
        }
        __syncthreads();
        if (t < n) { m.seen[t] = own; m.up[t] = next; }
        p = next;
    }
    return true;
}
__device__ __forceinline__ int mask_depth(const uint4 m) { return __popc(m.x) + __popc(m.y) + __popc(m.z) + __popc(m.w) - 1; }
#endif

}  // namespace grl
