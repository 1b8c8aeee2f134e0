// Attention of drafted trees over the paged cache: float32 kernel for every geometry, the merge of splits, and the entry points.
//   out[t] = softmax(scale q[t] K^T over the rows that node t sees) V:  all cached tokens, its ancestors and itself
#include "tree.cuh"

namespace grl {

constexpr int kTreeKeys = 32;       // keys of a tile of the float32 kernel
constexpr int kTreeRun = 4;         // rows of a warp of it
constexpr int kTreeWarps = 8;       // of a CTA
inline int tree_chunks(int R) { return (R + kTreeWarps * kTreeRun - 1) / (kTreeWarps * kTreeRun); }

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// grid (splits, Hkv x chunks of rows, B), the fours of rows shared out evenly.  A tile of 32 keys lies in shared memory as float32; a
// lane forms the scores of one key with the four rows of its warp, then the warp's lanes share out the columns of the output: a key, or a value,
// that has been read from shared memory meets four rows.  The next tile is on its way to registers meanwhile.
// Bound by shared-memory reads where there are many rows (8 x 8 heads x 4000 tokens, 64 rows of 128: 468 us, 18 TFLOP/s, 553 over a bf16 cache), by the chain of length, page
// and tile where there are few.  us, a row a warp / four: 5 x 2 heads x 777 tokens, 33 rows of 64 24.0 / 18.5; one row, 1 x 8 x 4000, 108 with a warp's
// loads to a CTA, 26 with eight.
template <typename TIO, typename TC, int D>
__global__ void __launch_bounds__(32 * kTreeWarps) tree_rows_kernel(const __grid_constant__ TreeArgs a) {
    extern __shared__ __align__(16) float smem[];
    __shared__ int up[GRL_MAX_TREE];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* ks = smem;                               // [32][D + 4]
    float* vs = ks + kTreeKeys * (D + 4);           // [32][D]
    float* qs = vs + kTreeKeys * D + warp * kTreeRun * D;                                        // this warp's [4][D]
    float* ps = vs + kTreeKeys * D + kTreeWarps * kTreeRun * D + warp * kTreeRun * kTreeKeys;   // and its weights [4][32]
    const int chunks = (a.R + kTreeWarps * kTreeRun - 1) / (kTreeWarps * kTreeRun), fours = ((a.R + kTreeRun - 1) / kTreeRun + chunks - 1) / chunks;
    const int split = blockIdx.x, kvh = blockIdx.y / chunks, b = blockIdx.z;
    const int r0 = warp < fours ? (blockIdx.y % chunks * fours + warp) * kTreeRun : a.R;
    pdl_wait();
    pdl_trigger();
    int prefix;
    int n = tree_nodes(a, b, &prefix, tid == 0);
    bool bad = false;
    if (a.parents)
        for (int t = tid; t < n; t += 32 * kTreeWarps) {
            up[t] = a.parents[(size_t)b * a.T + t];
            bad |= up[t] < -1 || up[t] >= t;
        }
    if (__syncthreads_or(bad)) {
        if (tid == 0) tree_fail(a.status, TREE_BAD_PARENT, b, n);
        n = 0;
    }
    if (n < 0) n = 0;
    const int len = n ? prefix + n : 0;
    const int tiles = (len + kTreeKeys - 1) / kTreeKeys, per = (tiles + a.n_splits - 1) / a.n_splits;
    const int k_begin = min(len, split * per * kTreeKeys), k_end = min(len, (split + 1) * per * kTreeKeys);
    // row x of the warp: element of the first of its head in q and out, whether it is a node's, and the nodes it sees
    size_t io[kTreeRun];
    bool live[kTreeRun], some = false;
#pragma unroll
    for (int x = 0; x < kTreeRun; ++x) {
        const int r = r0 + x, t = r / a.G;
        live[x] = r < a.R && t < n;
        some |= live[x];
        io[x] = (((size_t)b * a.T + t) * a.Hq + kvh * a.G + r - t * a.G) * D;
        for (int d = lane; d < D; d += 32) qs[x * D + d] = live[x] ? load_as_float<TIO>(reinterpret_cast<const TIO*>(a.q) + io[x] + d) * a.scale_log2 : 0.f;
    }
    uint4 seen = make_uint4(0u, 0u, 0u, 0u);        // lane x: of row x
    if (lane < kTreeRun && r0 + lane < a.R && (r0 + lane) / a.G < n) {
        const int node = (r0 + lane) / a.G;
        if (!a.parents) seen = low_bits(node + 1);
        else
            for (int u = node; u >= 0; u = up[u]) {
                const uint32_t bit = 1u << (u & 31);
                seen.x |= u < 32 ? bit : 0u;
                seen.y |= u >> 5 == 1 ? bit : 0u;
                seen.z |= u >> 5 == 2 ? bit : 0u;
                seen.w |= u >> 5 == 3 ? bit : 0u;
            }
    }
    __syncwarp();
    float m[kTreeRun], l[kTreeRun], acc[kTreeRun][D / 32];
#pragma unroll
    for (int x = 0; x < kTreeRun; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[x][i] = 0.f;
    }
    const TC* kp = reinterpret_cast<const TC*>(a.k_pages);
    const TC* vp = reinterpret_cast<const TC*>(a.v_pages);
    const int32_t* table = a.block_table + (size_t)b * a.max_pages;
    constexpr int PER = kTreeKeys * (D / 4) / (32 * kTreeWarps);       // 16-byte pieces of a tile of keys, of a thread
    float4 kx[PER], vx[PER];
    const auto fetch = [&](int k0) {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int idx = tid + e * 32 * kTreeWarps, d = idx % (D / 4) * 4, at = k0 + idx / (D / 4);
            kx[e] = vx[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at >= k_end) continue;
            const int page = table[at / a.P];
            if ((unsigned)page < (unsigned)a.num_pages) {
                const size_t off = (((size_t)page * a.Hkv + kvh) * a.P + at % a.P) * D + d;
                kx[e] = load4<TC>(kp + off);
                vx[e] = load4<TC>(vp + off);
            } else if (d == 0) {
                tree_fail(a.status, TREE_BAD_PAGE, b, page);
            }
        }
    };
    if (k_begin < k_end) fetch(k_begin);
    for (int k0 = k_begin; k0 < k_end; k0 += kTreeKeys) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int idx = tid + e * 32 * kTreeWarps, key = idx / (D / 4), d = idx % (D / 4) * 4;
            *reinterpret_cast<float4*>(ks + key * (D + 4) + d) = kx[e];
            *reinterpret_cast<float4*>(vs + key * D + d) = vx[e];
        }
        __syncthreads();
        if (k0 + kTreeKeys < k_end) fetch(k0 + kTreeKeys);
        if (!some) continue;
        float s[kTreeRun] = {};
#pragma unroll 8
        for (int d = 0; d < D; d += 4) {
            const float4 k = *reinterpret_cast<const float4*>(ks + lane * (D + 4) + d);
#pragma unroll
            for (int x = 0; x < kTreeRun; ++x) {
                const float4 q = *reinterpret_cast<const float4*>(qs + x * D + d);
                s[x] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[x]))));
            }
        }
        const bool nodes = k0 + kTreeKeys > prefix;
        uint32_t vis[kTreeRun];
#pragma unroll
        for (int x = 0; x < kTreeRun; ++x) {
            vis[x] = 0xffffffffu;
            if (nodes) {
                const int u = k0 + lane - prefix;       // node of this key, below 0 a cached token
                const uint32_t s0 = __shfl_sync(0xffffffffu, seen.x, x), s1 = __shfl_sync(0xffffffffu, seen.y, x), s2 = __shfl_sync(0xffffffffu, seen.z, x),
                               s3 = __shfl_sync(0xffffffffu, seen.w, x);
                const uint32_t word = u < 64 ? (u < 32 ? s0 : s1) : (u < 96 ? s2 : s3);
                vis[x] = __ballot_sync(0xffffffffu, k0 + lane < k_end && (u < 0 || (word >> (u & 31) & 1u)));
            }
            if (!(vis[x] >> lane & 1u)) s[x] = -INFINITY;
            float mx = s[x];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(m[x], mx), off = m_new == -INFINITY ? 0.f : m_new;       // a row that has seen nothing yet
            const float f = exp2f(m[x] - off), p = vis[x] >> lane & 1u ? exp2f(s[x] - off) : 0.f;
            l[x] = fmaf(l[x], f, p);
            m[x] = m_new;
            ps[x * kTreeKeys + lane] = p;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) acc[x][i] *= f;
        }
        __syncwarp();
#pragma unroll 2
        for (int k4 = 0; k4 < kTreeKeys; k4 += 4) {
            float4 w[kTreeRun];
#pragma unroll
            for (int x = 0; x < kTreeRun; ++x) w[x] = *reinterpret_cast<const float4*>(ps + x * kTreeKeys + k4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v[D / 32];
#pragma unroll
                for (int i = 0; i < D / 32; ++i) v[i] = vs[(k4 + e) * D + lane + 32 * i];
#pragma unroll
                for (int x = 0; x < kTreeRun; ++x) {
                    if (nodes && !(vis[x] >> (k4 + e) & 1u)) continue;       // a row that is not seen may hold anything
                    const float y = e == 0 ? w[x].x : e == 1 ? w[x].y : e == 2 ? w[x].z : w[x].w;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) acc[x][i] = fmaf(y, v[i], acc[x][i]);
                }
            }
        }
        __syncwarp();
    }
    const size_t rows = (size_t)a.B * a.Hkv * a.R;
    float* part = a.part + split * a.part_stride;
#pragma unroll
    for (int x = 0; x < kTreeRun; ++x) {
        float sum = l[x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (r0 + x >= a.R) continue;
        if (a.n_splits == 1) {
            TIO* out = reinterpret_cast<TIO*>(a.out) + io[x];
            const float inv = live[x] ? 1.f / sum : 0.f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) store_from_float<TIO>(out + lane + 32 * i, live[x] ? acc[x][i] * inv : 0.f);
            continue;
        }
        const size_t row = ((size_t)b * a.Hkv + kvh) * a.R + r0 + x;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) part[row * D + lane + 32 * i] = acc[x][i];
        if (lane == 0) *reinterpret_cast<float2*>(part + rows * D + 2 * row) = live[x] ? make_float2(tree_row_max(m[x], sum), sum) : make_float2(-INFINITY, -1.f);
    }
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
    const float* o_at = a.part + row * a.D + lane;
    float m = -INFINITY, l = 0.f, acc[8];
    bool nobody = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    constexpr int AT_ONCE = 8;
    for (int s0 = 0; s0 < a.n_splits; s0 += AT_ONCE) {
        float2 v[AT_ONCE];
        float o[AT_ONCE][8], top = m;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            v[j] = make_float2(-INFINITY, 0.f);
            if (s0 + j >= a.n_splits) continue;
            v[j] = *reinterpret_cast<const float2*>(ml + (s0 + j) * stride);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < a.D) o[j][i] = o_at[(s0 + j) * stride + 32 * i];
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
            if (!(v[j].y <= 0.f)) top = fmaxf(top, v[j].x);
        const float f = m == -INFINITY ? 0.f : exp2f(m - top);
        m = top;
        l *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= f;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            nobody |= v[j].y < 0.f;
            if (v[j].y <= 0.f) continue;       // saw nothing
            const float w = exp2f(v[j].x - m);
            l = fmaf(w, v[j].y, l);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < a.D) acc[i] = fmaf(w, o[j][i], acc[i]);
        }
    }
    const int r = (int)(row % a.R), kvh = (int)(row / a.R % a.Hkv);
    const size_t b = row / a.R / a.Hkv;
    TIO* out = reinterpret_cast<TIO*>(a.out) + ((b * a.T + r / a.G) * a.Hq + kvh * a.G + r % a.G) * a.D;
    const float inv = nobody ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.D) store_from_float<TIO>(out + lane + 32 * i, acc[i] * inv);
}

template <typename TIO, typename TC, int D>
static int launch_rows(grl_device* dev, const TreeArgs& a) {
    const int smem = (kTreeKeys * (2 * D + 4) + kTreeWarps * kTreeRun * (D + kTreeKeys)) * (int)sizeof(float);
    static bool attr_set[64] = {};
    if (!attr_set[dev->ordinal & 63]) {
        GRL_CUDA(cudaFuncSetAttribute(tree_rows_kernel<TIO, TC, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        attr_set[dev->ordinal & 63] = true;
    }
    GRL_CUDA(launch_pdl(tree_rows_kernel<TIO, TC, D>, dim3(a.n_splits, a.Hkv * tree_chunks(a.R), a.B), 32 * kTreeWarps, smem, dev->stream, a));
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
    const long long chunks = ((long long)p->n_tree * (p->num_q_heads / kv.num_kv_heads) + 7) / 8;
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
    // Some two CTAs an SM, every split at least two tiles.  us, splits: 5 x 2 x 777 tokens, 33 rows 1: 90, 3: 37, 6: 23.1, 12: 19.3; 1 x 8 x 4000, one row
    // 4: 114, 16: 34.7, 37: 26.3, 62: 38, 124: 43; 1 x 8 x 16000, 128 rows 4: 613, 8: 465, 9: 415, 16: 475.
    const long long ctas = (long long)kv.batch * kv.num_kv_heads * tree_chunks(R);
    long long s = 2LL * dev->prop.multiProcessorCount / ctas, most = longest / (2 * kTreeKeys);
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
