// Attention of drafted trees of few rows over the bf16 cache: up to 16 rows (nodes x heads of the group) of a (sequence, kv head), head_dim 128 or
// 64, pages of 64, 32 or 16 tokens.
//
// Bound by HBM where there is much to read, by latency where there is little, so 128-row tiles (tree_sm100.cu) are the wrong tool: their
// set-up and epilogue take longer than a short cache.  One CTA is a split of a (sequence, kv head): a producer warp brings stages of 64 tokens
// by TMA (boxes of 64 columns, 128-byte swizzle) into a ring; four compute warps take 16 tokens of each stage, with the rows as
// an operand of mma.sync m16n8k16, and a running maximum and sum of their own for every row.  Two CTAs an SM.  The warps' sums meet in
// shared memory, those of splits in the shared memory of a cluster where the splits of a head are one, else in tree_join_kernel.
// Measured, 16 rows: 32 x 8 heads x 4096 tokens 80 to 82 us (6.6 TB/s), 1 x 8 x 131072 86 (6.2 TB/s); 4 x 8 x 4096 18.5, 1 x 8 x 1001 9.8, 1 x 8 x 300 8.8,
// and 14.9, 8.6, 7.7 where call follows call and the rows are in L2.
// P is rounded to bf16 for its product with V, half a step of each probability; maxima, sums and O are float32.
// The predicate, and the cleaning of what lies past a sequence's end, concern the last stages only, as in tree_sm100.cu.
#include <cuda.h>

#include "decode_plan.h"
#include "sm100_ptx.cuh"
#include "tree.cuh"

namespace grl {
namespace treemma {

using sm100::cluster_map;
using sm100::fence_async_smem;
using sm100::lds128;
using sm100::ld_cluster_f32x4;
using sm100::mbar_arrive;
using sm100::mbar_expect_tx;
using sm100::mbar_init;
using sm100::mbar_try_wait;
using sm100::ex2;
using sm100::smem_u32;
using sm100::sts128;
using sm100::tma_load_2d;

constexpr int BN = 64;                  // tokens of a stage
constexpr int kThreads = 160;           // four compute warps and the producer
constexpr int kRows = kTreeFewRows;     // rows of a CTA: one operand
constexpr long long kDrainCycles = 200000000;
constexpr int kAloneSmem = 120 * 1024;  // more than half of an SM's: CTAs that must not share one
template <int HD> struct Form {
    static constexpr int SLAB = BN * HD * 2, STAGE = 2 * SLAB, NST = 96 * 1024 / STAGE;
    static constexpr int Q = NST * STAGE;               // query rows, 16-byte pieces XOR-swizzled by row
    static constexpr int BLOCK = Q + kRows * HD * 2;
    static constexpr int TOTAL = BLOCK + 1024 + 1024;   // + Block, + slack for 1024-byte alignment
    // after the stream, in the ring: the warps' rows, their (m, l), the CTA's rows, its (m, l)
    static constexpr int WARP_ML = 4 * kRows * HD * 4, CTA_O = WARP_ML + 4 * kRows * 8, CTA_ML = CTA_O + kRows * HD * 4;
    static_assert(CTA_ML + kRows * 8 <= Q, "the sums fit the ring");
};
struct Block {
    uint64_t full[6], empty[6];
    int abort, bad_tree;
    uint32_t bad[4];
    int8_t up[GRL_MAX_TREE];
    uint4 seen[kRows];
};
static_assert(sizeof(Block) <= 1024, "block");

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ bool wait_bar(uint32_t addr, uint32_t parity, Block& k, const TreeArgs& a, int what) {
    if (mbar_test(addr, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (clock64() - t0 > a.wait_limit) {
            *reinterpret_cast<volatile int*>(&k.abort) = 1;
            if (a.status && atomicCAS(a.status, 0, GRL_ERR_TIMEOUT) == 0) {
                a.status[1] = (7 << 28) | what;
                a.status[2] = blockIdx.x;
                a.status[3] = blockIdx.y | (blockIdx.z << 16);
            }
            return false;
        }
        if (mbar_try_wait(addr, parity)) return true;
        if (*reinterpret_cast<volatile int*>(&k.abort)) return false;
    }
}
// byte offset inside a slab of element (token row, column d): 64-column boxes, 128-byte swizzle
__device__ __forceinline__ uint32_t slab_off(int row, int d) {
    return (uint32_t)((d >> 6) * (BN * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4));
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Args {
    TreeArgs a;
    uint32_t per_group;         // row / G by its product's upper half; 0: G is 1
    int cluster;                // > 1: the splits of a head are one cluster
};

// grid (splits, Hkv, B)
template <int HD>
__global__ void __launch_bounds__(kThreads, 2)
tree_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Args args) {
    using F = Form<HD>;
    constexpr int NST = F::NST;
    const TreeArgs& a = args.a;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw), base = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_addr);
    Block& blk = *reinterpret_cast<Block*>(smem + F::BLOCK);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const auto node_of = [&](int r) { return args.per_group ? (int)__umulhi((uint32_t)r, args.per_group) : r; };
    const auto full = [&](int s) { return base + F::BLOCK + (uint32_t)s * 8u; };
    const auto empty = [&](int s) { return base + F::BLOCK + 48u + (uint32_t)s * 8u; };
    if (tid == 0) {
        for (int s = 0; s < NST; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 4); }
        blk.abort = blk.bad_tree = 0;
        blk.bad[0] = blk.bad[1] = blk.bad[2] = blk.bad[3] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmK)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmV)) : "memory");
    }
    __syncthreads();
    // everything above ran beside the kernel before this one; nothing below may
    pdl_wait();
    // what does not depend on the length is read beside it: parents, queries
    const int up = a.parents && tid < a.T ? a.parents[(size_t)b * a.T + tid] : -1;
    constexpr int CH = HD / 8, PER = (kRows * CH + 127) / 128;
    uint4 qv[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int idx = tid + 128 * e, r = idx / CH, c = idx % CH, node = node_of(r);
        qv[e] = make_uint4(0u, 0u, 0u, 0u);
        if (tid < 128 && r < a.R)
            qv[e] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) +
                                                         (((size_t)b * a.T + node) * a.Hq + kvh * a.G + r - node * a.G) * HD) + c);
    }
    int prefix, n = tree_nodes(a, b, &prefix, tid == 0);
    if (n < 0) { n = 0; prefix = 0; }
    const int len = n ? prefix + n : 0;
    const int stages = (len + BN - 1) / BN, per = (stages + a.n_splits - 1) / a.n_splits;
    const int p_begin = min(stages, split * per), p_end = min(stages, (split + 1) * per);
    const int32_t* table = a.block_table + (size_t)b * a.max_pages;

    // the producer: a lane a copy; its first stages leave ahead of the barrier below
    const int ppt = BN / a.P;
    int first = p_begin * ppt, entry = 0, next = 0, last = -1;
    auto issue = [&](int p) {
        const int i = p - p_begin, s = i % NST;
        if (p * ppt - first >= 32) {
            first += 32;
            entry = next;
            next = table[min(first + 32 + lane, a.max_pages - 1)];
        }
        const int np = min(ppt, (len - p * BN + a.P - 1) / a.P);
        if (lane == 0) mbar_expect_tx(full(s), (uint32_t)(np * a.P * HD * 4));
        __syncwarp();
        constexpr int BOXES = HD / 64;
        const int j = lane / (2 * BOXES), v = lane / BOXES & 1, x = lane % BOXES;
        int page = __shfl_sync(0xffffffffu, entry, (p * ppt - first + j) & 31);
        if (j < np) {
            if ((unsigned)page >= (unsigned)a.num_pages) { tree_fail(a.status, TREE_BAD_PAGE, b, page); page = 0; }
            tma_load_2d(base + s * F::STAGE + v * F::SLAB + x * (BN * 128) + j * a.P * 128, v ? &tmV : &tmK, x * 64, (page * a.Hkv + kvh) * a.P, full(s));
        }
        __syncwarp();
        last = i;
    };
    if (warp == 4) {
        entry = table[min(first + lane, a.max_pages - 1)];
        next = table[min(first + 32 + lane, a.max_pages - 1)];
        for (int p = p_begin; p < min(p_end, p_begin + NST); ++p) issue(p);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int idx = tid + 128 * e, r = idx / CH, c = idx % CH;
            if (r < kRows) sts128(base + F::Q + r * (HD * 2) + ((c ^ (r & 7)) << 4), qv[e]);
        }
        if (a.parents && tid < n) {
            if (up < -1 || up >= tid) blk.bad_tree = 1;
            blk.up[tid] = (int8_t)up;
        }
    }
    __syncthreads();
    const bool bad_tree = blk.bad_tree != 0;
    if (bad_tree && tid == 0) tree_fail(a.status, TREE_BAD_PARENT, b, n);
    const int live_nodes = bad_tree ? 0 : n;
    if (tid < kRows) {
        const int node = node_of(tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (tid < a.R && node < live_nodes) {
            if (!a.parents) seen = low_bits(node + 1);
            else
                for (int u = node; u >= 0; u = blk.up[u]) {
                    const uint32_t bit = 1u << (u & 31);
                    seen.x |= u < 32 ? bit : 0u;
                    seen.y |= u >> 5 == 1 ? bit : 0u;
                    seen.z |= u >> 5 == 2 ? bit : 0u;
                    seen.w |= u >> 5 == 3 ? bit : 0u;
                }
        }
        blk.seen[tid] = seen;
    }
    __syncthreads();

    const int g = lane >> 2, t4 = lane & 3;
    float o[HD / 8][4], m_ref[2], l[2];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    m_ref[0] = m_ref[1] = -INFINITY;
    l[0] = l[1] = 0.f;
    bool ok = true;
    if (warp == 4) {
        for (int p = p_begin + NST; p < p_end; ++p) {
            const int i = p - p_begin;
            if (!__all_sync(0xffffffffu, wait_bar(empty(i % NST), (i / NST - 1) & 1, blk, a, 6 + i % NST))) break;
            __syncwarp();
            issue(p);
        }
    } else {
        const int mat = lane >> 3;
        // operand rows of this lane's ldmatrix addresses: queries, keys (two 8-token tiles), values (transposed)
        const int q_row = (lane & 7) + ((mat & 1) << 3), q_col = mat >> 1;
        const int k_row = 16 * warp + (lane & 7) + ((mat >> 1) << 3), k_col = (mat & 1) << 3;
        const int v_row = 16 * warp + (lane & 7) + ((mat & 1) << 3), v_col = (mat >> 1) << 3;
        uint32_t qf[HD / 16][4];
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) ldmatrix_x4(base + F::Q + q_row * (HD * 2) + (((2 * ks + q_col) ^ (q_row & 7)) << 4), qf[ks]);
        for (int p = p_begin; p < p_end && ok; ++p) {
            const int i = p - p_begin, s = i % NST;
            ok = __all_sync(0xffffffffu, wait_bar(full(s), (i / NST) & 1, blk, a, s));
            __syncwarp();
            if (!ok) break;
            const uint32_t kb = base + (uint32_t)s * F::STAGE, vb = kb + F::SLAB;
            const int tok0 = p * BN + 16 * warp;            // this warp's first token
            if (tok0 < len) {
                const bool nodes = tok0 + 16 > prefix;
                if (nodes) {
                    // rows of V from the sequence's end on are cleared, and elements that are no finite number, whose nodes are remembered
                    for (int c = lane; c < 16 * CH; c += 32) {
                        const int row = 16 * warp + c / CH, key = p * BN + row;
                        if (key < prefix) continue;
                        const uint32_t addr = vb + slab_off(row, c % CH * 8);
                        if (key >= len) {
                            sts128(addr, make_uint4(0u, 0u, 0u, 0u));
                        } else {
                            const uint4 v = lds128(addr);
                            uint32_t w[4] = {v.x, v.y, v.z, v.w};
                            bool any = false;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const bool lo = (w[e] & 0x7f80u) == 0x7f80u, hi = (w[e] & 0x7f800000u) == 0x7f800000u;
                                any |= lo | hi;
                                w[e] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu);
                            }
                            if (any) {
                                atomicOr(&blk.bad[(key - prefix) >> 5], 1u << ((key - prefix) & 31));
                                sts128(addr, make_uint4(w[0], w[1], w[2], w[3]));
                            }
                        }
                    }
                    __syncwarp();
                }
                // ---- S = Q K^T, 16 tokens in two tiles of 8
                float sc[2][4];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    uint32_t kf[4];
                    ldmatrix_x4(kb + slab_off(k_row, 16 * ks + k_col), kf);
                    mma_bf16(sc[0], qf[ks], kf[0], kf[1]);
                    mma_bf16(sc[1], qf[ks], kf[2], kf[3]);
                }
                uint32_t pf[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {           // rows g and g + 8
                    float v[4] = {sc[0][2 * h], sc[0][2 * h + 1], sc[1][2 * h], sc[1][2 * h + 1]};
                    if (nodes) {
                        const uint4 seen = blk.seen[8 * h + g];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = tok0 + (e >> 1) * 8 + 2 * t4 + (e & 1), u = key - prefix;
                            const uint32_t w = u < 64 ? (u < 32 ? seen.x : seen.y) : (u < 96 ? seen.z : seen.w);
                            if (key >= len || (u >= 0 && !(w >> (u & 31) & 1u))) v[e] = -INFINITY;
                        }
                    }
                    const float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) * a.scale_log2;
                    // a new maximum, by more than 2^8: seldom, after the first few tiles
                    if (__any_sync(0xffffffffu, mx > m_ref[h] + 8.f)) {
                        float top = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        const float m_new = top > m_ref[h] + 8.f ? top : m_ref[h];
                        const float f = m_new == m_ref[h] ? 1.f : ex2(m_ref[h] - m_new);
                        m_ref[h] = m_new;
                        l[h] *= f;
#pragma unroll
                        for (int j = 0; j < HD / 8; ++j) { o[j][2 * h] *= f; o[j][2 * h + 1] *= f; }
                    }
                    const float off = m_ref[h] == -INFINITY ? 0.f : -m_ref[h];       // a row that has seen nothing yet
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = ex2(fmaf(v[e], a.scale_log2, off));
                    l[h] += (v[0] + v[1]) + (v[2] + v[3]);
                    pf[h] = pack_bf16(v[0], v[1]);
                    pf[2 + h] = pack_bf16(v[2], v[3]);
                }
                // ---- O += P V
#pragma unroll
                for (int dn = 0; dn < HD / 16; ++dn) {
                    uint32_t vf[4];
                    ldmatrix_x4_trans(vb + slab_off(v_row, 16 * dn + v_col), vf);
                    mma_bf16(o[2 * dn], pf, vf[0], vf[1]);
                    mma_bf16(o[2 * dn + 1], pf, vf[2], vf[3]);
                }
            }
            if (tok0 + 16 > prefix) fence_async_smem();         // cleaned rows, ahead of the copy that takes their place
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            m_ref[h] = tree_row_max(m_ref[h], l[h]);
        }
    }
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(&blk.abort)) {
        // A wait ran out, maybe behind the producer's last look at the flag: copies in flight land before the ring is used again.  No wait of
        // the stream is left, so that the whole CTA finds the flag as it is.
        if (warp == 4) {
            const long long t0 = clock64();
            for (int x = last; x >= 0 && x > last - NST; --x)
                while (!mbar_try_wait(full(x % NST), (x / NST) & 1) && clock64() - t0 < kDrainCycles) {}
        }
        __syncthreads();
    }
    // the ring is free: every copy has come in and been read
    pdl_trigger();
    float* warp_o = reinterpret_cast<float*>(smem);
    float2* warp_ml = reinterpret_cast<float2*>(smem + F::WARP_ML);
    float* cta_o = reinterpret_cast<float*>(smem + F::CTA_O);
    float2* cta_ml = reinterpret_cast<float2*>(smem + F::CTA_ML);
    ok = *reinterpret_cast<volatile int*>(&blk.abort) == 0;
    // blocks of eight columns XOR-swizzled by row, so that neither the stores nor the reads meet in a bank
    if (warp < 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = warp * kRows + 8 * h + g;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j)
                *reinterpret_cast<float2*>(warp_o + row * HD + ((j ^ g) << 3) + 2 * t4) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
            if (t4 == 0) warp_ml[row] = make_float2(m_ref[h], l[h]);
        }
    }
    __syncthreads();
    // who writes row r, its columns 4 c..: v un-normalised
    const auto write = [&](int r, int c, float4 v, float sum) {
        const int node = node_of(r);
        const float inv = node < live_nodes ? 1.f / sum : 0.f;
        uint2 w = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        if (node >= live_nodes) w = make_uint2(0u, 0u);
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + node) * a.Hq + kvh * a.G + r - node * a.G) * HD;
        reinterpret_cast<uint2*>(out)[c] = w;
    };
    const uint4 bad = make_uint4(blk.bad[0], blk.bad[1], blk.bad[2], blk.bad[3]);
    float* part = a.part + (((size_t)b * a.Hkv + kvh) * a.n_splits + split) * (size_t)(kRows * (HD + 2));
    for (int idx = tid; idx < a.R * (HD / 4); idx += kThreads) {
        const int r = idx / (HD / 4), c = idx % (HD / 4);
        float m = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, warp_ml[w * kRows + r].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 ml = warp_ml[w * kRows + r];
            if (ml.x == -INFINITY) continue;
            const float f = ex2(ml.x - m);
            const float4 u = *reinterpret_cast<const float4*>(warp_o + (w * kRows + r) * HD + (((c >> 1) ^ (r & 7)) << 3) + ((c & 1) << 2));
            v.x = fmaf(f, u.x, v.x); v.y = fmaf(f, u.y, v.y); v.z = fmaf(f, u.z, v.z); v.w = fmaf(f, u.w, v.w);
            sum = fmaf(f, ml.y, sum);
        }
        if ((bad.x | bad.y | bad.z | bad.w) != 0u) {        // rare: what is no finite number, for the rows that see it
            const uint4 seen = blk.seen[r];
            for (int u = 0; u < n; ++u) {
                const uint32_t w = u < 64 ? (u < 32 ? seen.x & bad.x : seen.y & bad.y) : (u < 96 ? seen.z & bad.z : seen.w & bad.w);
                if (!(w >> (u & 31) & 1u)) continue;
                const int at = prefix + u, page = table[at / a.P];
                if ((unsigned)page >= (unsigned)a.num_pages) continue;
                const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.v_pages) + (((size_t)page * a.Hkv + kvh) * a.P + at % a.P) * HD + 4 * c;
                const float y[4] = {__bfloat162float(x[0]), __bfloat162float(x[1]), __bfloat162float(x[2]), __bfloat162float(x[3])};
                if (!isfinite(y[0])) v.x += y[0];
                if (!isfinite(y[1])) v.y += y[1];
                if (!isfinite(y[2])) v.z += y[2];
                if (!isfinite(y[3])) v.w += y[3];
            }
        }
        if (!ok) continue;
        if (a.n_splits == 1) {
            write(r, c, v, sum);
        } else if (args.cluster > 1) {
            reinterpret_cast<float4*>(cta_o)[r * (HD / 4) + c] = v;
            if (c == 0) cta_ml[r] = make_float2(m, sum);
        } else {
            reinterpret_cast<float4*>(part)[r * (HD / 4) + c] = v;
            if (c == 0) reinterpret_cast<float2*>(part + kRows * HD)[r] = node_of(r) < live_nodes ? make_float2(m, sum) : make_float2(-INFINITY, -1.f);
        }
    }
    if (args.cluster > 1) {
        // every CTA of the head's cluster joins its share of the rows' pieces, from all of them
        cluster_sync();
        const int size = args.cluster;
        for (int idx = split + size * tid; idx < a.R * (HD / 4) && ok; idx += size * kThreads) {
            const int r = idx / (HD / 4), c = idx % (HD / 4);
            const uint32_t o_addr = smem_u32(cta_o) + (uint32_t)idx * 16u, ml_addr = smem_u32(cta_ml) + (uint32_t)r * 8u;
            float m = -INFINITY, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p0 = 0; p0 < size; p0 += 8) {
                float4 u[8];
                float2 ml[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    ml[j] = make_float2(-INFINITY, 0.f);
                    u[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (p0 + j < size) {
                        u[j] = ld_cluster_f32x4(cluster_map(o_addr, p0 + j));
                        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(ml[j].x), "=f"(ml[j].y) : "r"(cluster_map(ml_addr, p0 + j)) : "memory");
                    }
                }
                float m_new = m;
#pragma unroll
                for (int j = 0; j < 8; ++j) m_new = fmaxf(m_new, ml[j].x);
                const float f = m == -INFINITY ? 0.f : ex2(m - m_new);
                v.x *= f; v.y *= f; v.z *= f; v.w *= f;
                sum *= f;
                m = m_new;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (ml[j].x == -INFINITY) continue;
                    const float w = ex2(ml[j].x - m);
                    v.x = fmaf(w, u[j].x, v.x); v.y = fmaf(w, u[j].y, v.y); v.z = fmaf(w, u[j].z, v.z); v.w = fmaf(w, u[j].w, v.w);
                    sum = fmaf(w, ml[j].y, sum);
                }
            }
            write(r, c, v, sum);
        }
        cluster_sync();         // a CTA leaves only when nobody reads its rows any more
    }
}

static int make_pool_map(grl_device* dev, CUtensorMap* tm, const void* pool, const TreeArgs& a) {
    TmapKey k{};
    k.ptr = pool; k.rank = 2; k.swizzle_128b = 1;
    k.dims[0] = (uint64_t)a.D; k.dims[1] = (uint64_t)a.num_pages * a.Hkv * a.P;
    k.strides[0] = (uint64_t)a.D * 2;
    k.box[0] = 64; k.box[1] = (uint32_t)a.P;
    return get_tensor_map(dev, k, tm);
}

using Kernel = void (*)(CUtensorMap, CUtensorMap, Args);
static Kernel kernel_of(int D) { return D == 128 ? tree_mma_kernel<128> : tree_mma_kernel<64>; }
static int smem_of(int D) { return D == 128 ? Form<128>::TOTAL : Form<64>::TOTAL; }

static int set_attributes(grl_device* dev) {
    static bool attr_set[64] = {};
    if (!attr_set[dev->ordinal & 63]) {      // a function attribute belongs to the device that was current
        for (int D : {64, 128}) {
            GRL_CUDA(cudaFuncSetAttribute(kernel_of(D), cudaFuncAttributeMaxDynamicSharedMemorySize, kAloneSmem));
            GRL_CUDA(cudaFuncSetAttribute(kernel_of(D), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        }
        attr_set[dev->ordinal & 63] = true;
    }
    return GRL_OK;
}

}  // namespace treemma

// The split of a decode of as many heads and stages (decode_plan.h); the splits of a head are a cluster while they are short and clusters fit the GPU
// at once.
TreeMmaPlan tree_mma_plan(grl_device* dev, int B, int Hkv, int D, int longest, int asked) {
    using namespace treemma;
    DecodeShape d;
    d.heads = B * Hkv;
    d.stages = (longest + BN - 1) / BN;
    d.sms = dev->prop.multiProcessorCount;
    d.mma = true;
    const auto fits = [&](bool, int c) {
        DeviceGuard g(dev->ordinal);
        return set_attributes(dev) != GRL_OK ? 0 : max_active_clusters(dev, (const void*)kernel_of(D), kThreads, smem_of(D), c);
    };
    TreeMmaPlan p{};
    p.splits = asked > 0 ? asked : decode_splits(d, fits);
    p.cluster = 1;
    if (p.splits > 1 && p.splits <= kMaxCluster && (d.stages + p.splits - 1) / p.splits <= kClusterStages && d.heads <= fits(false, p.splits)) p.cluster = p.splits;
    p.workspace = p.splits > 1 && p.cluster == 1 ? sizeof(float) * (size_t)d.heads * p.splits * kRows * (D + 2) : 0;
    p.alone = p.splits > 1 && p.cluster == 1 && (long long)d.heads * p.splits <= d.sms;
    return p;
}

int tree_mma_launch(grl_device* dev, const TreeArgs& a, const TreeMmaPlan& plan) {
    using namespace treemma;
    CUtensorMap tk, tv;
    int rc = make_pool_map(dev, &tk, a.k_pages, a);
    if (!rc) rc = make_pool_map(dev, &tv, a.v_pages, a);
    if (!rc) rc = set_attributes(dev);
    if (rc) return rc;
    const Args args{a, a.G == 1 ? 0u : (uint32_t)(((1ull << 32) + a.G - 1) / a.G), plan.cluster};
    GRL_CUDA(launch_pdl_cluster(kernel_of(a.D), dim3(a.n_splits, a.Hkv, a.B), kThreads, plan.alone ? kAloneSmem : smem_of(a.D), dev->stream, plan.cluster, tk, tv, args));
    GRL_LAUNCHED("tree_mma_kernel");
    return a.n_splits > 1 && plan.cluster == 1 ? tree_join_launch(dev, a, kRows) : GRL_OK;
}

}  // namespace grl
