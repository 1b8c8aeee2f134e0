// Attention of drafted trees over the paged cache: float32 kernel for every geometry, the merge of splits, and the entry points.
//   out[t] = softmax(scale q[t] K^T over the rows that node t sees) V:  all cached tokens, its ancestors and itself
#include "tree.cuh"

namespace grl {

constexpr int kTreeKeys = 32;       // keys of a tile of the float32 kernel
constexpr int kTreeRows = 8;        // rows of a CTA of it, a warp each

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// grid (splits, Hkv x chunks of rows, B).  A tile of 32 keys lies in shared memory as float32; a lane forms the score of one key, then
// the warp's lanes share out the columns of the output.
template <typename TIO, typename TC, int D>
__global__ void __launch_bounds__(32 * kTreeRows) tree_rows_kernel(const __grid_constant__ TreeArgs a) {
    extern __shared__ float smem[];
    __shared__ TreeMasks masks;
    float* ks = smem;                               // [32][D + 1]
    float* vs = ks + kTreeKeys * (D + 1);           // [32][D]
    float* qs = vs + kTreeKeys * D;                 // [8][D]
    const int chunks = (a.R + kTreeRows - 1) / kTreeRows;
    const int split = blockIdx.x, kvh = blockIdx.y / chunks, b = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.y % chunks * kTreeRows + warp, t = r / a.G, g = r % a.G;
    int prefix;
    int n = tree_nodes(a, b, &prefix, tid == 0);
    if (n > 0 && !tree_masks(masks, a.parents ? a.parents + (size_t)b * a.T : nullptr, n)) {
        if (tid == 0) tree_fail(a.status, TREE_BAD_PARENT, b, n);
        n = 0;
    }
    if (n < 0) n = 0;
    const int len = n ? prefix + n : 0;
    const int tiles = (len + kTreeKeys - 1) / kTreeKeys, per = (tiles + a.n_splits - 1) / a.n_splits;
    const int k_begin = min(len, split * per * kTreeKeys), k_end = min(len, (split + 1) * per * kTreeKeys);
    const bool live = r < a.R && t < n;
    const size_t io = (((size_t)b * a.T + t) * a.Hq + kvh * a.G + g) * D;
    for (int d = lane; d < D; d += 32) qs[warp * D + d] = live ? load_as_float<TIO>(reinterpret_cast<const TIO*>(a.q) + io + d) * a.scale_log2 : 0.f;
    const uint4 seen = live ? masks.seen[t] : make_uint4(0u, 0u, 0u, 0u);
    float m = -INFINITY, l = 0.f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
    const TC* kp = reinterpret_cast<const TC*>(a.k_pages);
    const TC* vp = reinterpret_cast<const TC*>(a.v_pages);
    const int32_t* table = a.block_table + (size_t)b * a.max_pages;
    for (int k0 = k_begin; k0 < k_end; k0 += kTreeKeys) {
        __syncthreads();
        for (int idx = tid; idx < kTreeKeys * (D / 4); idx += 32 * kTreeRows) {
            const int key = idx / (D / 4), d = idx % (D / 4) * 4, at = k0 + key;
            float4 kx = make_float4(0.f, 0.f, 0.f, 0.f), vx = kx;
            if (at < k_end) {
                const int page = table[at / a.P];
                if ((unsigned)page < (unsigned)a.num_pages) {
                    const size_t off = (((size_t)page * a.Hkv + kvh) * a.P + at % a.P) * D + d;
                    kx = load4<TC>(kp + off);
                    vx = load4<TC>(vp + off);
                } else if (d == 0) {
                    tree_fail(a.status, TREE_BAD_PAGE, b, page);
                }
            }
            float* kd = ks + key * (D + 1) + d;
            kd[0] = kx.x; kd[1] = kx.y; kd[2] = kx.z; kd[3] = kx.w;
            *reinterpret_cast<float4*>(vs + key * D + d) = vx;
        }
        __syncthreads();
        if (!live) continue;
        const int u = k0 + lane - prefix;       // node of this key, below 0 a cached token
        const uint32_t word = u < 64 ? (u < 32 ? seen.x : seen.y) : (u < 96 ? seen.z : seen.w);
        const bool vis = k0 + lane < k_end && (u < 0 || (word >> (u & 31) & 1u));
        float s = 0.f;
#pragma unroll 16
        for (int d = 0; d < D; ++d) s = fmaf(qs[warp * D + d], ks[lane * (D + 1) + d], s);
        float mx = vis ? s : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const uint32_t any = __ballot_sync(0xffffffffu, vis);
        if (!any) continue;
        const float m_new = fmaxf(m, mx), f = exp2f(m - m_new), p = vis ? exp2f(s - m_new) : 0.f;
        float sum = p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, f, sum);
        m = m_new;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= f;
        for (int key = 0; key < kTreeKeys; ++key) {
            const float w = __shfl_sync(0xffffffffu, p, key);
            if (any >> key & 1u) {      // a row that is not seen may hold anything
#pragma unroll
                for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(w, vs[key * D + lane + 32 * i], acc[i]);
            }
        }
    }
    if (r >= a.R) return;
    if (a.n_splits == 1) {
        TIO* out = reinterpret_cast<TIO*>(a.out) + io;
        const float inv = live ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) store_from_float<TIO>(out + lane + 32 * i, live ? acc[i] * inv : 0.f);
        return;
    }
    const size_t rows = (size_t)a.B * a.Hkv * a.R, row = ((size_t)b * a.Hkv + kvh) * a.R + r;
    float* part = a.part + split * a.part_stride;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) part[row * D + lane + 32 * i] = acc[i];
    if (lane == 0) *reinterpret_cast<float2*>(part + rows * D + 2 * row) = make_float2(m, l);
}

// A warp a row: the splits' sums at their common maximum.
template <typename TIO>
__global__ void __launch_bounds__(128) tree_merge_kernel(const __grid_constant__ TreeArgs a) {
    const size_t rows = (size_t)a.B * a.Hkv * a.R, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5), stride = a.part_stride;
    const int lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if (row >= rows) return;
    const float* ml = a.part + rows * a.D + 2 * row;
    float m = -INFINITY;
    for (int s = lane; s < a.n_splits; s += 32) {
        const float2 v = *reinterpret_cast<const float2*>(ml + s * stride);
        if (v.y != 0.f) m = fmaxf(m, v.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int s = 0; s < a.n_splits; ++s) {
        const float2 v = *reinterpret_cast<const float2*>(ml + s * stride);
        if (v.y == 0.f) continue;       // saw nothing: its O is not written
        const float w = exp2f(v.x - m);
        l = fmaf(w, v.y, l);
        const float* o = a.part + s * stride + row * a.D;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.D) acc[i] = fmaf(w, o[lane + 32 * i], acc[i]);
    }
    const int r = (int)(row % a.R), kvh = (int)(row / a.R % a.Hkv);
    const size_t b = row / a.R / a.Hkv;
    TIO* out = reinterpret_cast<TIO*>(a.out) + ((b * a.T + r / a.G) * a.Hq + kvh * a.G + r % a.G) * a.D;
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.D) store_from_float<TIO>(out + lane + 32 * i, acc[i] * inv);
}

template <typename TIO, typename TC, int D>
static int launch_rows(grl_device* dev, const TreeArgs& a) {
    const int smem = (kTreeKeys * (2 * D + 1) + kTreeRows * D) * (int)sizeof(float);
    static bool attr_set[64] = {};
    if (!attr_set[dev->ordinal & 63]) {
        GRL_CUDA(cudaFuncSetAttribute(tree_rows_kernel<TIO, TC, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        attr_set[dev->ordinal & 63] = true;
    }
    dim3 grid(a.n_splits, a.Hkv * ((a.R + kTreeRows - 1) / kTreeRows), a.B);
    tree_rows_kernel<TIO, TC, D><<<grid, 32 * kTreeRows, smem, dev->stream>>>(a);
    GRL_LAUNCHED("tree_rows_kernel");
    return GRL_OK;
}

template <typename TIO, typename TC>
static int launch_rows_d(grl_device* dev, const TreeArgs& a) {
    switch (a.D) {
        case 32: return launch_rows<TIO, TC, 32>(dev, a);
        case 64: return launch_rows<TIO, TC, 64>(dev, a);
        case 128: return launch_rows<TIO, TC, 128>(dev, a);
        default: return launch_rows<TIO, TC, 256>(dev, a);
    }
}

int check_tree_layout(const grl_kv_layout& kv) {
    GRL_REQUIRE(kv.k_pages && kv.v_pages && kv.block_table && kv.seq_lens, "NULL cache pointer");
    GRL_REQUIRE(kv.batch > 0 && kv.num_kv_heads > 0 && kv.page_tokens > 0 && kv.max_pages > 0 && kv.num_pages >= 0, "bad cache shape");
    GRL_REQUIRE((long long)kv.max_pages * kv.page_tokens < (1LL << 31), "a sequence of more than 2^31 tokens");
    GRL_REQUIRE(kv.batch <= 65535 && kv.num_kv_heads <= 4096, "at most 65535 sequences of 4096 kv heads");
    GRL_REQUIRE(kv.head_dim > 0 && kv.head_dim % 2 == 0 && kv.head_dim <= 256, "head_dim must be even and <= 256");
    if (kv.cache_dtype == GRL_FP8_INT4)
        return set_error(GRL_ERR_UNSUPPORTED, "steps of drafted tokens are not built for the quantised (FP8 / INT4) cache: its value bytes live "
                                              "in token pairs; use a bf16 or fp32 cache, or grl_qk_norm_rope, grl_kv_append and grl_gqa_decode");
    GRL_REQUIRE(kv.cache_dtype == GRL_BF16 || kv.cache_dtype == GRL_F32, "unknown cache dtype");
    return GRL_OK;
}

static bool tensor_cores_apply(const grl_tree_params* p) {
    const grl_kv_layout& kv = p->kv;
    return kv.cache_dtype == GRL_BF16 && p->io_dtype == GRL_BF16 && (kv.head_dim == 128 || kv.head_dim == 64) &&
           (kv.page_tokens == 64 || kv.page_tokens == 32 || kv.page_tokens == 16) &&
           (long long)pool_pages(kv) * kv.num_kv_heads * kv.page_tokens < (1LL << 31) &&
           (long long)p->n_tree * (p->num_q_heads / kv.num_kv_heads) < (1LL << 15);
}

static int check_tree(const grl_tree_params* p) {
    GRL_REQUIRE(p, "params is NULL");
    const grl_kv_layout& kv = p->kv;
    int rc = check_tree_layout(kv);
    if (rc) return rc;
    GRL_REQUIRE(p->q && p->out, "q or out is NULL");
    GRL_REQUIRE(p->io_dtype == GRL_F32 || p->io_dtype == GRL_BF16, "io_dtype must be GRL_F32 or GRL_BF16");
    GRL_REQUIRE(p->num_q_heads > 0 && p->num_q_heads % kv.num_kv_heads == 0, "num_q_heads (%d) must be a multiple of num_kv_heads (%d)",
                p->num_q_heads, kv.num_kv_heads);
    GRL_REQUIRE(p->n_tree > 0 && p->n_tree <= GRL_MAX_TREE, "n_tree must be 1 to %d, got %d", GRL_MAX_TREE, p->n_tree);
    GRL_REQUIRE(p->max_seq_len >= 0 && p->n_splits >= 0, "max_seq_len and n_splits must not be negative");
    GRL_REQUIRE(p->n_splits <= 4096, "at most 4096 splits");
    GRL_REQUIRE(p->scale >= 0.f, "scale must be positive, or 0 for 1/sqrt(head_dim)");
    GRL_REQUIRE(p->kernel == GRL_KERNEL_AUTO || p->kernel == GRL_KERNEL_SIMT_F32 || p->kernel == GRL_KERNEL_TCGEN05, "unknown kernel");
    if (kv.head_dim != 32 && kv.head_dim != 64 && kv.head_dim != 128 && kv.head_dim != 256)
        return set_error(GRL_ERR_UNSUPPORTED, "head_dim %d not supported (32, 64, 128 or 256)", kv.head_dim);
    if (p->kernel == GRL_KERNEL_TCGEN05 && !tensor_cores_apply(p))
        return set_error(GRL_ERR_UNSUPPORTED, "the tensor-core kernel takes bf16 queries over a bf16 cache, head_dim 128 or 64, pages of 64, 32 or 16 tokens");
    GRL_REQUIRE((uintptr_t)kv.k_pages % 16 == 0 && (uintptr_t)kv.v_pages % 16 == 0, "page pools must be 16-byte aligned");
    GRL_REQUIRE((uintptr_t)p->q % 16 == 0 && (uintptr_t)p->out % 16 == 0, "q and out must be 16-byte aligned");
    const long long chunks = ((long long)p->n_tree * (p->num_q_heads / kv.num_kv_heads) + kTreeRows - 1) / kTreeRows;
    GRL_REQUIRE(chunks * kv.num_kv_heads <= 65535, "too many query heads");
    return GRL_OK;
}

struct TreePlan {
    bool tensor;
    int splits;
    size_t workspace;
    bool few;
    TreeTensorPlan t;
    TreeMmaPlan m;
};
static TreePlan tree_plan(grl_device* dev, const grl_tree_params* p) {
    const grl_kv_layout& kv = p->kv;
    const int cap = kv.max_pages * kv.page_tokens, longest = p->max_seq_len > 0 && p->max_seq_len < cap ? p->max_seq_len : cap;
    const int R = p->n_tree * (p->num_q_heads / kv.num_kv_heads);
    TreePlan t{};
    t.tensor = p->kernel != GRL_KERNEL_SIMT_F32 && tensor_cores_apply(p);
    t.few = t.tensor && R <= kTreeFewRows;
    if (t.few) {
        t.m = tree_mma_plan(dev, kv.batch, kv.num_kv_heads, kv.head_dim, longest, p->n_splits);
        t.splits = t.m.splits;
        t.workspace = t.m.workspace;
        return t;
    }
    if (t.tensor) {
        t.t = tree_sm100_plan(dev, kv.batch, kv.num_kv_heads, R, kv.head_dim, longest, p->n_splits);
        t.splits = t.t.splits;
        t.workspace = t.t.workspace;
        return t;
    }
    // some four CTAs an SM, every split at least four tiles
    const long long ctas = (long long)kv.batch * kv.num_kv_heads * ((R + kTreeRows - 1) / kTreeRows);
    long long s = 4LL * dev->prop.multiProcessorCount / ctas, most = longest / (4 * kTreeKeys);
    if (s > most) s = most;
    t.splits = p->n_splits > 0 ? p->n_splits : (int)(s < 1 ? 1 : s > 256 ? 256 : s);
    t.workspace = t.splits == 1 ? 0 : sizeof(float) * t.splits * tree_part_stride((size_t)kv.batch * p->n_tree * p->num_q_heads, kv.head_dim);
    return t;
}

}  // namespace grl

using namespace grl;

extern "C" {

int grl_tree_workspace_bytes(grl_device* dev, const grl_tree_params* p, size_t* bytes) {
    int rc = check_tree(p);
    if (rc) return rc;
    GRL_REQUIRE(dev && bytes, "NULL argument");
    *bytes = tree_plan(dev, p).workspace;
    return GRL_OK;
}

int grl_tree_attention(grl_device* dev, const grl_tree_params* p) {
    int rc = check_tree(p);
    if (rc) return rc;
    GRL_REQUIRE(dev, "dev is NULL");
    const grl_kv_layout& kv = p->kv;
    TreeArgs a{};
    a.k_pages = kv.k_pages; a.v_pages = kv.v_pages; a.block_table = kv.block_table; a.seq_lens = kv.seq_lens;
    a.q = p->q; a.out = p->out; a.parents = p->parents; a.n_nodes = p->n_nodes; a.status = dev->d_status;
    a.B = kv.batch; a.Hq = p->num_q_heads; a.Hkv = kv.num_kv_heads; a.G = a.Hq / a.Hkv; a.T = p->n_tree; a.R = a.T * a.G;
    a.D = kv.head_dim; a.P = kv.page_tokens; a.max_pages = kv.max_pages; a.num_pages = pool_pages(kv);
    a.scale_log2 = (p->scale == 0.f ? 1.f / sqrtf((float)a.D) : p->scale) * 1.4426950408889634f;
    a.wait_limit = dev->wait_limit_cycles;
    const TreePlan plan = tree_plan(dev, p);
    a.n_splits = plan.splits;
    const size_t need = plan.workspace;
    GRL_REQUIRE(!need || (p->workspace && p->workspace_bytes >= need), "tree attention workspace too small: %zu < %zu",
                p->workspace ? p->workspace_bytes : 0, need);
    GRL_REQUIRE((uintptr_t)p->workspace % 16 == 0, "workspace must be 16-byte aligned");
    a.part = static_cast<float*>(p->workspace);
    a.part_stride = tree_part_stride((size_t)a.B * a.Hkv * a.R, a.D);
    DeviceGuard g(dev->ordinal);
    dev->status_dirty = true;
    const bool c32 = kv.cache_dtype == GRL_F32, io32 = p->io_dtype == GRL_F32;
    if (plan.few) return tree_mma_launch(dev, a, plan.m);
    if (plan.tensor) return tree_sm100_launch(dev, a, plan.t);
    rc = io32 ? (c32 ? launch_rows_d<float, float>(dev, a) : launch_rows_d<float, __nv_bfloat16>(dev, a))
       : (c32 ? launch_rows_d<__nv_bfloat16, float>(dev, a) : launch_rows_d<__nv_bfloat16, __nv_bfloat16>(dev, a));
    if (rc || a.n_splits == 1) return rc;
    const size_t rows = (size_t)a.B * a.Hkv * a.R;
    GRL_CUDA(launch_pdl(io32 ? tree_merge_kernel<float> : tree_merge_kernel<__nv_bfloat16>, dim3((unsigned)((rows + 3) / 4)), 128, 0, dev->stream, a));
    GRL_LAUNCHED("tree_merge_kernel");
    return GRL_OK;
}

}  // extern "C"
