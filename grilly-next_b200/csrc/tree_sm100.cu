// Attention of drafted trees over the bf16 cache on the tensor cores: head_dim 128 or 64, pages of 64, 32 or 16 tokens.
//
// The T * G rows (node, head of the group) of a (sequence, kv head) are the rows of the products, 128 to a tile; a CTA streams its
// share of the cached keys and values once, 64 tokens a stage, through a shared-memory ring filled by TMA:
//   warps 1, 3   TMA, every second stage each: the stage's pages (boxes of 64 columns, 128-byte swizzle) of K and V
//   warps 0, 2   one elected lane each issues tcgen05.mma:  S = Q K^T (64 keys) into TMEM,  O += P V  with P from TMEM
//   warps 4-7 / 8-11   softmax: a thread a row; S from TMEM, running maximum and sum in the exp2 domain, P back as bf16; the accumulator is
//                scaled only where a maximum grew by more than 2^8
// The two chains of products and softmax (t = 0, 1) are
//   PAIR    two row tiles over the same stages, where there are more than 128 rows: a stage crosses shared memory once for 256 rows
//   SPLIT   the even and the odd stages of one row tile, joined in the epilogue
//   FOLD    up to 64 rows, twice in the tile: the first half of a chain's threads takes one stage of a pair, the second half the other.  P has zeros
//           where a half's rows meet the other's keys, so that one product sums both; four streams are joined in the epilogue
// The predicate is applied to the last stages only, those with nodes in them: a row has one bit for each of 128 nodes.  There, rows
// of V past the sequence's end, which may hold anything, are cleared in shared memory ahead of the product, and so are elements
// that are no finite number; rows that see such an element add it again in the epilogue, so that it reaches nobody else.
//
// Every mbarrier wait is bounded; on expiry the CTA records an error, drains its copies and returns.
#include <cuda.h>

#include "sm100_ptx.cuh"
#include "tmem_ops.cuh"
#include "tree.cuh"

namespace grl {
namespace tree {

using namespace sm100;

constexpr int BM = 128;             // rows of a tile (TMEM lanes)
constexpr int BN = 64;              // tokens of a stage
constexpr int kThreads = 384;
constexpr int WARP_MMA0 = 0, WARP_TMA0 = 1, WARP_MMA1 = 2, WARP_TMA1 = 3, WARP_SOFTMAX = 4;
// Registers: the softmax warpgroups take what the first one gives up.  setmaxnreg.inc is served from what the CTA was launched with only.
constexpr int REGS_LAUNCH = 168, REGS_SOFTMAX = 208, REGS_MISC = 80;
static_assert(2 * REGS_SOFTMAX + REGS_MISC <= 3 * REGS_LAUNCH && REGS_LAUNCH * kThreads <= 65536, "register budgets");
constexpr int Q_BOX = BM * 128, KV_BOX = BN * 128;      // bytes of a 64-column box
constexpr uint32_t TMEM_COLS = 512, TMEM_CHAIN = 256, TMEM_O = 128;     // a chain: two buffers of S (P overlays them), then O

enum Mode { SPLIT, PAIR, FOLD };
template <int HD, Mode MODE> struct Form {
    static constexpr int BOXES = HD / 64;
    static constexpr int SLAB = BOXES * KV_BOX;             // K (or V) of a stage
    static constexpr int STAGE = 2 * SLAB;
    static constexpr int Q_TILE = BOXES * Q_BOX;
    static constexpr int Q_BYTES = (MODE == PAIR ? 2 : 1) * Q_TILE;
    static constexpr int NST = (226 * 1024 - Q_BYTES - 1280) / STAGE < 8 ? (226 * 1024 - Q_BYTES - 1280) / STAGE : 8;
    static constexpr int SMEM_RING = Q_BYTES, SMEM_BAR = SMEM_RING + NST * STAGE;
    static constexpr int TOTAL = SMEM_BAR + 256 + 1024;     // + barriers and flags, + slack for 1024-byte alignment
    static_assert(TOTAL <= 227 * 1024, "shared memory");
    static_assert(sizeof(TreeMasks) <= Q_TILE, "the masks are formed where the query rows go");
    // barriers
    static constexpr int FULL = 0, EMPTY = NST, S_FULL = 2 * NST, P_READY = S_FULL + 4, O_PREV = P_READY + 4, O_DONE = O_PREV + 2, NUM = O_DONE + 2;
    static_assert(NUM * 8 <= 232 && NUM <= 28, "barrier block; the status word has 28 bits for them");
};

constexpr uint32_t IDESC_QK = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
template <int HD> struct IdescPV {      // N = head_dim columns, V is MN-major
    static constexpr uint32_t value = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BM >> 4) << 24) | (1u << 16);
};

struct Ctx {
    uint32_t bars;
    volatile int* abort;
    int32_t* status;
    long long limit;
};
__device__ __forceinline__ bool wait_bar(const Ctx& c, int bar, uint32_t parity) {
    const uint32_t addr = c.bars + bar * 8;
    if (mbar_try_wait(addr, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (mbar_try_wait(addr, parity)) return true;
        if (*c.abort) return false;
        if (clock64() - t0 > c.limit) {
            *c.abort = 1;
            if (c.status && atomicCAS(c.status, 0, GRL_ERR_TIMEOUT) == 0) {
                c.status[1] = (7 << 28) | bar;
                c.status[2] = blockIdx.x;
                c.status[3] = blockIdx.y | (blockIdx.z << 16);
            }
            return false;
        }
    }
}
__device__ __forceinline__ bool wait_bar_warp(const Ctx& c, int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_bar(c, bar, parity)); }

__device__ __forceinline__ void store32(float* dst, const uint32_t (&r)[32]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        reinterpret_cast<float4*>(dst)[i] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]),
                                                        __uint_as_float(r[4 * i + 3]));
}
__device__ __forceinline__ void store32(__nv_bfloat16* dst, const uint32_t (&r)[32]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(r[8 * i + 2 * e]), __uint_as_float(r[8 * i + 2 * e + 1]));
            w[e] = *reinterpret_cast<const uint32_t*>(&v);
        }
        reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Which of 32 tokens a row sees, the first of them node `at` (below 0: a cached token, seen by all).
__device__ __forceinline__ uint32_t window32(const uint4& seen, int at) {
    if (at <= -32) return 0xffffffffu;
    if (at < 0) return (seen.x << -at) | ((1u << -at) - 1u);
    const int w = at >> 5;
    const uint32_t lo = w == 0 ? seen.x : w == 1 ? seen.y : w == 2 ? seen.z : w == 3 ? seen.w : 0u;
    const uint32_t hi = w == 0 ? seen.y : w == 1 ? seen.z : w == 2 ? seen.w : 0u;
    return __funnelshift_r(lo, hi, at & 31);
}

// Rows of V of a stage that has nodes in it, token k0 first, by the 128 threads of a softmax warpgroup: cleared from the sequence's end
// on; elements that are no finite number cleared too, and their nodes remembered in bad.
template <int HD>
__device__ __forceinline__ void clean_values(uint32_t slab, int k0, int prefix, int len, uint32_t* bad, int wt) {
    const int row = wt >> 1, key = k0 + row;
    if (key < prefix) return;
    constexpr int CHUNKS = HD / 16;             // 16-byte pieces of half a row
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int chunk = (wt & 1) * CHUNKS + c;
        const uint32_t addr = slab + (chunk >> 3) * KV_BOX + row * 128 + ((chunk & 7) << 4);      // the swizzle permutes pieces inside a row
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
                atomicOr(bad + ((key - prefix) >> 5), 1u << ((key - prefix) & 31));
                __threadfence_block();
                sts128(addr, make_uint4(w[0], w[1], w[2], w[3]));
            }
        }
    }
}

// Columns 32 ch .. of the nodes in hit that are no finite number, for a row that sees them: rare.
template <int HD>
__device__ __noinline__ void add_bad(const TreeArgs& a, const int32_t* table, int kvh, int prefix, int n, const uint4 hit, int ch, uint32_t (&o)[32]) {
    for (int u = 0; u < n; ++u) {
        const uint32_t w = u < 64 ? (u < 32 ? hit.x : hit.y) : (u < 96 ? hit.z : hit.w);
        if (!(w >> (u & 31) & 1u)) continue;
        const int at = prefix + u, page = table[at / a.P];
        if ((unsigned)page >= (unsigned)a.num_pages) continue;
        const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(a.v_pages) + (((size_t)page * a.Hkv + kvh) * a.P + at % a.P) * HD + ch * 32;
        for (int e = 0; e < 32; ++e) {
            const float x = __bfloat162float(v[e]);
            if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
        }
    }
}

// grid (splits, Hkv * CTAs of row tiles, B)
template <int HD, Mode MODE>
__global__ void __launch_bounds__(kThreads, 1)
tree_sm100_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeArgs a) {
    using F = Form<HD, MODE>;
    constexpr bool PAIR = MODE == tree::PAIR, FOLD = MODE == tree::FOLD;
    constexpr int NST = F::NST;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_addr);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + F::SMEM_BAR + 232);
    int* abort_flag = reinterpret_cast<int*>(smem + F::SMEM_BAR + 236);
    uint32_t* bad = reinterpret_cast<uint32_t*>(smem + F::SMEM_BAR + 240);          // 128 bits
    const Ctx ctx{base + F::SMEM_BAR, abort_flag, a.status, a.wait_limit};
    auto bar = [&](int i) { return ctx.bars + (uint32_t)i * 8u; };
    if (warp == WARP_TMA0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmK)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmV)) : "memory");
        for (int s = 0; s < NST; ++s) {
            mbar_init(bar(F::FULL + s), 1);
            mbar_init(bar(F::EMPTY + s), PAIR ? 2 : 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(F::S_FULL + i), 1);
            mbar_init(bar(F::P_READY + i), 128);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar(F::O_PREV + t), 1);
            mbar_init(bar(F::O_DONE + t), 1);
        }
        *abort_flag = 0;
        bad[0] = bad[1] = bad[2] = bad[3] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == WARP_MMA0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // all of the above beside the tail of the kernel before this one, nothing below
    pdl_wait();

    const int groups = PAIR ? (a.R + 2 * BM - 1) / (2 * BM) : (a.R + BM - 1) / BM;
    const int split = blockIdx.x, kvh = blockIdx.y / groups, b = blockIdx.z;
    const int r0 = blockIdx.y % groups * (PAIR ? 2 * BM : BM);
    const int32_t* table = a.block_table + (size_t)b * a.max_pages;
    TreeMasks& masks = *reinterpret_cast<TreeMasks*>(smem);
    const bool tell = tid == 0;
    int prefix, n = tree_nodes(a, b, &prefix, tell);
    if (n > 0 && !tree_masks(masks, a.parents ? a.parents + (size_t)b * a.T : nullptr, n)) {
        if (tell) tree_fail(a.status, TREE_BAD_PARENT, b, n);
        n = 0;
    }
    if (n < 0) n = 0;
    const int len = n ? prefix + n : 0;
    const int stages = (len + BN - 1) / BN, per = (stages + a.n_splits - 1) / a.n_splits;
    const int st0 = min(stages, split * per), ns = min(stages, (split + 1) * per) - st0;       // this CTA's stages
    const int chain = warp >= WARP_SOFTMAX ? (warp - WARP_SOFTMAX) >> 2 : warp == WARP_MMA1 ? 1 : 0;
    const int row = tid & 127, sub = FOLD ? row >> 6 : 0, r = r0 + (PAIR ? chain * BM : 0) + (FOLD ? row & 63 : row);                         // softmax threads: their row
    const int node = r / a.G;
    const bool live = r < a.R && node < n;
    const uint4 seen = live ? masks.seen[node] : make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();                // the masks are read: query rows take their place
    {   // query rows as the K-major operand, rows past the last one zero
        constexpr int CH = HD / 8, ROWS = PAIR ? 2 * BM : BM;
        for (int idx = tid; idx < ROWS * CH; idx += kThreads) {
            const int qr = idx / CH, c = idx % CH, g = r0 + (FOLD ? qr & 63 : qr), t = g / a.G;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (g < a.R && t < n)
                v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) +
                                                         (((size_t)b * a.T + t) * a.Hq + kvh * a.G + g % a.G) * HD) + c);
            sts128(base + (qr >> 7) * F::Q_TILE + (c >> 3) * Q_BOX + (qr & 127) * 128 + (((c & 7) ^ (qr & 7)) << 4), v);
        }
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    // steps of a chain: all stages, or every second one; a tile without rows takes none
    auto steps_of = [&](int t) { return PAIR ? (r0 + t * BM < a.R ? ns : 0) : FOLD ? ((ns + 1) / 2 - t + 1) / 2 : (ns - t + 1) / 2; };
    const int nh = steps_of(chain);
    auto stage_of = [&](int i) { return PAIR ? i : FOLD ? 4 * i + 2 * chain : 2 * i + chain; };     // FOLD: the first of two

    if (warp < WARP_SOFTMAX) {
      reg_dec<REGS_MISC>();
      if (warp == WARP_TMA0 || warp == WARP_TMA1) {
        // ------------------------------------------------------------------ TMA: a warp the even stages, a warp the odd ones
        // A lane a copy: one lane's chain of waits and copies took some 1700 cycles a stage, longer than HBM takes to bring it.
        const int ppt = BN / a.P, odd = uniform(warp == WARP_TMA1);
        int first = st0 * ppt, issued = 0;
        int entry = table[min(first + lane, a.max_pages - 1)], next = table[min(first + 32 + lane, a.max_pages - 1)];
        for (int i = odd; i < ns; i += 2) {
            const int p = st0 + i, s = i % NST, it = i / NST;
            if (p * ppt - first >= 32) {
                first += 32;
                entry = next;
                next = table[min(first + 32 + lane, a.max_pages - 1)];
            }
            if (it > 0 && !wait_bar_warp(ctx, F::EMPTY + s, (it - 1) & 1)) break;
            const int np = min(ppt, (len - p * BN + a.P - 1) / a.P);       // pages of the stage that hold tokens
            if (lane == 0) mbar_expect_tx(bar(F::FULL + s), (uint32_t)(np * a.P * HD * 4));
            __syncwarp();
            // lane: page j, then K or V, then the box
            constexpr int COPIES = 2 * F::BOXES;
            const int j = lane / COPIES, v = lane / F::BOXES & 1, x = lane % F::BOXES;
            int page = __shfl_sync(0xffffffffu, entry, (p * ppt - first + j) & 31);
            if (j < np) {
                if ((unsigned)page >= (unsigned)a.num_pages) { tree_fail(a.status, TREE_BAD_PAGE, b, page); page = 0; }
                tma_load_2d(base + F::SMEM_RING + s * F::STAGE + v * F::SLAB + x * KV_BOX + j * a.P * 128, v ? &tmV : &tmK, x * 64,
                            (page * a.Hkv + kvh) * a.P, bar(F::FULL + s));
            }
            __syncwarp();
            issued = i + 1;
        }
        if (*ctx.abort && lane == 0) {      // copies in flight land before the shared memory is given back
            const long long t0 = clock64();
            for (int i = odd; i < issued; i += 2)
                if (i >= issued - NST) while (!mbar_try_wait(bar(F::FULL + i % NST), (i / NST) & 1) && clock64() - t0 < ctx.limit) {}
        }
      } else if (warp == WARP_MMA0 || warp == WARP_MMA1) {
        // ------------------------------------------------------------------ products of chain t
        const int steps = uniform(nh), t = uniform(chain);
        if (steps > 0) {
            const uint32_t qa = desc_lo(base + (PAIR ? t * F::Q_TILE : 0), 16);
            const uint32_t k_lo = desc_lo(base + F::SMEM_RING, 16), v_lo = desc_lo(base + F::SMEM_RING + F::SLAB, KV_BOX);
            const uint32_t s_tmem = (uint32_t)uniform((int)tmem_base) + (uint32_t)t * TMEM_CHAIN, o_tmem = s_tmem + TMEM_O;
            // S of a step: 64 columns of buffer i & 1; FOLD: both buffers, a stage each
            auto issue_qk = [&](int i) -> bool {
#pragma unroll
                for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                    const int st = stage_of(i) + half, s = st % NST;
                    if (FOLD && st >= ns) break;
                    if (!wait_bar_warp(ctx, F::FULL + s, (st / NST) & 1)) return false;
                    tc_fence_after();
                    const uint32_t kb = k_lo + (uint32_t)s * (F::STAGE >> 4), d = s_tmem + (uint32_t)(FOLD ? half : i & 1) * BN;
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        mma_ss2(d, qa + (uint32_t)(((ks >> 2) * Q_BOX + (ks & 3) * 32) >> 4), kb + (uint32_t)(((ks >> 2) * KV_BOX + (ks & 3) * 32) >> 4),
                                IDESC_QK, ks != 0);
                }
                mma_commit(bar(F::S_FULL + 2 * t + (FOLD ? 0 : i & 1)));
                return true;
            };
            bool ok = true;
            for (int i = 0; i < (FOLD ? 1 : 2) && i < steps && ok; ++i) ok = issue_qk(i);
            for (int i = 0; i < steps && ok; ++i) {
                ok = wait_bar_warp(ctx, F::P_READY + 2 * t + (FOLD ? 0 : i & 1), (FOLD ? i : i >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                if constexpr (FOLD) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int st = stage_of(i) + half, s = st % NST;
                        if (st >= ns) break;
                        const uint32_t p_tmem = s_tmem + (uint32_t)half * (BN / 2), vb = v_lo + (uint32_t)s * (F::STAGE >> 4);
#pragma unroll
                        for (int ks = 0; ks < BN / 16; ++ks)
                            mma_ts2(o_tmem, p_tmem + ks * 8, vb + (uint32_t)ks * (2048 >> 4), IdescPV<HD>::value, i > 0 || half > 0 || ks > 0);
                        mma_commit(bar(F::EMPTY + s));
                    }
                    if (i + 1 == steps) mma_commit(bar(F::O_DONE + t));
                    else ok = issue_qk(i + 1);      // S takes the place of P: in order behind its product
                    continue;
                }
                const int s = stage_of(i) % NST;
                const uint32_t p_tmem = s_tmem + (uint32_t)(i & 1) * BN, vb = v_lo + (uint32_t)s * (F::STAGE >> 4);
                mma_ts2(o_tmem, p_tmem, vb, IdescPV<HD>::value, i > 0);
#pragma unroll
                for (int ks = 1; ks < BN / 16; ++ks) mma_ts2(o_tmem, p_tmem + ks * 8, vb + (uint32_t)ks * (2048 >> 4), IdescPV<HD>::value, 1u);
                if (i + 2 >= steps) mma_commit(bar((i + 2 == steps ? F::O_PREV : F::O_DONE) + t));
                mma_commit(bar(F::EMPTY + s));
                // a stage that the other tile does not read is released for it too
                if (PAIR && steps_of(t ^ 1) == 0) mma_commit(bar(F::EMPTY + s));
                if (i + 2 < steps) ok = issue_qk(i + 2);       // overwrites the buffer of P(i): in order behind its product
            }
        }
      }
    } else {
        // ------------------------------------------------------------------ softmax and epilogue
        reg_inc<REGS_SOFTMAX>();
        const int t = chain;
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_addr + (uint32_t)t * TMEM_CHAIN, o_addr = s_addr + TMEM_O;
        float m_ref = -INFINITY, l = 0.f;
        bool ok = true;
        for (int i = 0; i < nh && ok; ++i) {
            const int bf = FOLD ? 0 : i & 1, st = stage_of(i) + sub, k0 = (st0 + st) * BN;
            const bool none = FOLD && st >= ns, nodes = none || k0 + BN > prefix;       // none: the pair's second stage is another CTA's, or past the end
            // stages with nodes in them: their values are there when their scores are
#pragma unroll
            for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                const int vs = stage_of(i) + half, v0 = (st0 + vs) * BN;
                if (vs < ns && v0 + BN > prefix) {
                    ok = ok && wait_bar_warp(ctx, F::FULL + vs % NST, (vs / NST) & 1);
                    if (!ok) break;
                    clean_values<HD>(base + F::SMEM_RING + (vs % NST) * F::STAGE + F::SLAB, v0, prefix, len, bad, row);
                    fence_async_smem();
                }
            }
            if (!ok) break;
            ok = wait_bar_warp(ctx, F::S_FULL + 2 * t + bf, (FOLD ? i : i >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            uint32_t sr[BN];
            tmem_ld_x64_sync(s_addr + (FOLD ? sub : bf) * BN, sr);
            if (nodes) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t vis = none ? 0u : window32(seen, k0 + 32 * w - prefix);
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(vis >> c & 1u)) sr[32 * w + c] = 0xff800000u;
                }
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < BN; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx4[e] = max3(mx4[e], __uint_as_float(sr[c + 2 * e]), __uint_as_float(sr[c + 2 * e + 1]));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            const float m_new = fmaxf(m_ref, mx * a.scale_log2);
            if (i == 0) {
                m_ref = m_new;
            } else {
                const bool need = m_new > m_ref + 8.f;
                if (__any_sync(0xffffffffu, need)) {
                    // P V of the step before must be in O: it is once S of the next step is there (FOLD: of this one), issued behind it
                    if constexpr (!FOLD) ok = i + 1 < nh ? wait_bar_warp(ctx, F::S_FULL + 2 * t + (bf ^ 1), ((i + 1) >> 1) & 1) : wait_bar_warp(ctx, F::O_PREV + t, 0);
                    if (!ok) break;
                    tc_fence_after();
                    const float f = need ? ex2(m_ref - m_new) : 1.f;
                    if (need) m_ref = m_new;
                    l *= f;
#pragma unroll
                    for (int ch = 0; ch < HD / 32; ++ch) {
                        uint32_t o[32];
                        tmem_ld_x32_sync(o_addr + ch * 32, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_x32(o_addr + ch * 32, o);
                    }
                    tmem_st_wait();
                }
            }
            const float off = m_ref == -INFINITY ? 0.f : -m_ref;       // a row that has seen nothing yet
            const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(off, off);
            float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int ch = 0; ch < BN / 32; ++ch) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float2 x = make_float2(__uint_as_float(sr[ch * 32 + c]), __uint_as_float(sr[ch * 32 + c + 1]));
                    x = __ffma2_rn(x, sc2, nm2);
                    const float2 pe = make_float2(ex2(x.x), ex2(x.y));
                    rs[(c >> 1) & 3] = __fadd2_rn(rs[(c >> 1) & 3], pe);
                    const __nv_bfloat162 pp = __floats2bfloat162_rn(pe.x, pe.y);
                    pk[c >> 1] = *reinterpret_cast<const uint32_t*>(&pp);
                }
                tmem_st_x16(s_addr + (FOLD ? sub * (BN / 2) : bf * BN) + ch * 16, pk);
            }
            if constexpr (FOLD) {
                uint32_t zero[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) zero[e] = 0u;
                tmem_st_x32(s_addr + (sub ^ 1) * (BN / 2), zero);
            }
            l += ((rs[0].x + rs[0].y) + (rs[1].x + rs[1].y)) + ((rs[2].x + rs[2].y) + (rs[3].x + rs[3].y));
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(bar(F::P_READY + 2 * t + bf));
        }
        if (ok && nh > 0) ok = wait_bar_warp(ctx, F::O_DONE + t, 0);
        if constexpr (FOLD) {
            // The four streams of a row (chain, half): maxima and sums, then the accumulators at the common maximum, meet in the ring, whose
            // stages are all read once both chains are done.
            constexpr int CH = HD / 4;          // 16-byte pieces of an accumulator's row
            float2* ml = reinterpret_cast<float2*>(smem + F::SMEM_RING);
            const uint32_t rows_at = base + F::SMEM_RING + 2048;
            static_assert(2048 + 4 * 64 * HD * 4 <= NST * F::STAGE, "the streams' rows fit the ring");
            tc_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            ml[t * BM + row] = make_float2(m_ref, l);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            ok = ok && !*ctx.abort;
            float m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x) m = fmaxf(m, ml[x * 64 + (row & 63)].x);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float2 v = ml[x * 64 + (row & 63)];
                if (v.x != -INFINITY) sum = fmaf(ex2(v.x - m), v.y, sum);
            }
            const bool direct = a.n_splits == 1;
            const float w = (m_ref == -INFINITY ? 0.f : ex2(m_ref - m)) * (direct ? 1.f / sum : 1.f);
            const uint4 hit = make_uint4(bad[0] & seen.x, bad[1] & seen.y, bad[2] & seen.z, bad[3] & seen.w);
            const bool mends = t == 0 && sub == 0 && (hit.x | hit.y | hit.z | hit.w) != 0u;
            if (ok) {
                tc_fence_after();
#pragma unroll
                for (int ch = 0; ch < HD / 32; ++ch) {
                    uint32_t o[32];
                    __syncwarp();
                    if (nh > 0) tmem_ld_x32_sync(o_addr + ch * 32, o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = nh > 0 && m_ref != -INFINITY ? __float_as_uint(__uint_as_float(o[e]) * w) : 0u;
                    if (mends) add_bad<HD>(a, table, kvh, prefix, n, hit, ch, o);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        sts128(rows_at + ((t * BM + row) * CH + ((ch * 8 + c) ^ (row & 15))) * 16, make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]));
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (ok) {
                const size_t rows = (size_t)a.B * a.Hkv * a.R, base_row = ((size_t)b * a.Hkv + kvh) * a.R;
                float* part = a.part + split * a.part_stride;
                for (int idx = tid - WARP_SOFTMAX * 32; idx < a.R * CH; idx += 256) {
                    const int rr = idx / CH, c = idx % CH, node_r = rr / a.G;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (ns > 0 && node_r < n) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint4 u = lds128(rows_at + ((x * 64 + rr) * CH + (c ^ (rr & 15))) * 16);
                            v.x += __uint_as_float(u.x); v.y += __uint_as_float(u.y); v.z += __uint_as_float(u.z); v.w += __uint_as_float(u.w);
                        }
                    }
                    if (direct) {
                        __nv_bfloat162 p0 = __floats2bfloat162_rn(v.x, v.y), p1 = __floats2bfloat162_rn(v.z, v.w);
                        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + node_r) * a.Hq + kvh * a.G + rr % a.G) * HD;
                        reinterpret_cast<uint2*>(out)[c] = make_uint2(*reinterpret_cast<uint32_t*>(&p0), *reinterpret_cast<uint32_t*>(&p1));
                    } else if (ns > 0 && node_r < n) {
                        reinterpret_cast<float4*>(part + (base_row + rr) * HD)[c] = v;
                    }
                }
                if (!direct && r < a.R && t == 0 && sub == 0)
                    *reinterpret_cast<float2*>(part + rows * HD + 2 * (base_row + r)) = live && ns > 0 ? make_float2(m, sum) : make_float2(-INFINITY, 0.f);
            }
        } else {
        float mine = 1.f, theirs = 0.f, m = m_ref;
        if constexpr (MODE == SPLIT) {
            // the other chain's maximum and sum, through the ring: both accumulators are final, so its stages are read
            float2* ml = reinterpret_cast<float2*>(smem + F::SMEM_RING);
            tc_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            ml[t * BM + row] = make_float2(m_ref, l);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float2 other = ml[(t ^ 1) * BM + row];
            ok = ok && !*ctx.abort;
            m = fmaxf(m_ref, other.x);
            mine = m_ref == -INFINITY ? 0.f : ex2(m_ref - m);
            theirs = other.x == -INFINITY ? 0.f : ex2(other.x - m);
            l = l * mine + other.y * theirs;
        }
        if (ok) {
            tc_fence_after();
            const bool direct = a.n_splits == 1;
            const float norm = direct ? 1.f / l : 1.f;
            const int steps1 = steps_of(1);
            const uint4 hit = make_uint4(bad[0] & seen.x, bad[1] & seen.y, bad[2] & seen.z, bad[3] & seen.w);
            const size_t rows = (size_t)a.B * a.Hkv * a.R, prow = ((size_t)b * a.Hkv + kvh) * a.R + r;
            float* part = a.part + split * a.part_stride;
            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + node) * a.Hq + kvh * a.G + r % a.G) * HD;
#pragma unroll
            for (int ch = 0; ch < HD / 32; ++ch) {
                if (!PAIR && ch / (HD / 64) != t) continue;         // SPLIT: each warpgroup writes half of the columns from both accumulators
                uint32_t o[32];
                __syncwarp();
                if (nh > 0 || (!PAIR && ns > 0)) {
                    if constexpr (PAIR) {
                        tmem_ld_x32_sync(o_addr + ch * 32, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * norm);
                    } else {
                        const float w0 = (t ? theirs : mine) * norm, w1 = (t ? mine : theirs) * norm;
                        tmem_ld_x32_sync(lane_addr + TMEM_O + ch * 32, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * w0);
                        if (steps1 > 0) {
                            uint32_t more[32];
                            tmem_ld_x32_sync(lane_addr + TMEM_CHAIN + TMEM_O + ch * 32, more);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(fmaf(__uint_as_float(more[e]), w1, __uint_as_float(o[e])));
                        }
                    }
                }
                if ((hit.x | hit.y | hit.z | hit.w) != 0u) add_bad<HD>(a, table, kvh, prefix, n, hit, ch, o);
                if (direct && r < a.R) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = live ? o[e] : 0u;
                    store32(out + ch * 32, o);
                } else if (live && ns > 0) {
                    store32(part + prow * HD + ch * 32, o);
                }
            }
            if (!direct && r < a.R && (PAIR || t == 0))
                *reinterpret_cast<float2*>(part + rows * HD + 2 * prow) = live && ns > 0 ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        }
        }
    }
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == WARP_MMA0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

// A pool as a 2-D bf16 tensor (rows = pages * Hkv * page tokens, head_dim columns); box = 64 columns x one page of one kv head.
static int make_pool_map(grl_device* dev, CUtensorMap* tm, const void* pool, const TreeArgs& a) {
    TmapKey k{};
    k.ptr = pool; k.rank = 2; k.swizzle_128b = 1;
    k.dims[0] = (uint64_t)a.D; k.dims[1] = (uint64_t)a.num_pages * a.Hkv * a.P;
    k.strides[0] = (uint64_t)a.D * 2;
    k.box[0] = 64; k.box[1] = (uint32_t)a.P;
    return get_tensor_map(dev, k, tm);
}

template <int HD, Mode MODE>
static int launch(grl_device* dev, const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a) {
    using F = Form<HD, MODE>;
    static bool attr_set[64] = {};
    if (!attr_set[dev->ordinal & 63]) {      // a function attribute belongs to the device that was current
        GRL_CUDA(cudaFuncSetAttribute(tree_sm100_kernel<HD, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::TOTAL));
        attr_set[dev->ordinal & 63] = true;
    }
    const int rows = MODE == PAIR ? 2 * BM : BM;
    dim3 grid(a.n_splits, a.Hkv * ((a.R + rows - 1) / rows), a.B);
    GRL_CUDA(launch_pdl(tree_sm100_kernel<HD, MODE>, grid, kThreads, F::TOTAL, dev->stream, tk, tv, a));
    GRL_LAUNCHED("tree_sm100_kernel");
    return GRL_OK;
}

}  // namespace tree

int tree_sm100_launch(grl_device* dev, const TreeArgs& a) {
    using namespace tree;
    CUtensorMap tk, tv;
    int rc = make_pool_map(dev, &tk, a.k_pages, a);
    if (!rc) rc = make_pool_map(dev, &tv, a.v_pages, a);
    if (rc) return rc;
    const Mode mode = a.R > BM ? PAIR : a.R > 64 ? SPLIT : FOLD;
    if (a.D == 128) return mode == PAIR ? launch<128, PAIR>(dev, tk, tv, a) : mode == SPLIT ? launch<128, SPLIT>(dev, tk, tv, a) : launch<128, FOLD>(dev, tk, tv, a);
    return mode == PAIR ? launch<64, PAIR>(dev, tk, tv, a) : mode == SPLIT ? launch<64, SPLIT>(dev, tk, tv, a) : launch<64, FOLD>(dev, tk, tv, a);
}

}  // namespace grl
