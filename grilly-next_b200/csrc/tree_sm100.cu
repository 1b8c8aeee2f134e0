// Attention of drafted trees over the bf16 cache on the tensor cores: head_dim 128 or 64, pages of 64, 32 or 16 tokens.
//
// The T * G rows (node, head of the group) of a (sequence, kv head) are the rows of the products, 128 to a tile; a CTA streams its
// share of the cached keys and values once, 64 tokens a stage, through a shared-memory ring filled by TMA:
//   warps 1, 3   TMA, the stages of one chain each (PAIR: every second one): the stage's pages (boxes of 64 columns, 128-byte swizzle) of K and V
//   warps 0, 2   one elected lane each issues tcgen05.mma:  S = Q K^T (64 keys) into TMEM,  O += P V  with P from TMEM
//   warps 4-7 / 8-11   softmax: a thread a row; S from TMEM, running maximum and sum in the exp2 domain, P back as bf16; the accumulator is
//                scaled only where a maximum grew by more than 2^8
// P is rounded to bf16, the type of V, since a product has operands of one type; each probability is off by half a step at most, 2^-8 of it, and an
// output by that of sum p |v|.  Scores, maxima, the sum (of the unrounded exponentials) and O are float32.
// The two chains of products and softmax (t = 0, 1) are
//   PAIR    two row tiles over the same stages, where there are more than 128 rows: a stage crosses shared memory once for 256 rows
//   SPLIT   the even and the odd stages of one row tile, joined in the epilogue
//   FOLD    up to 64 rows, twice in the tile: the first half of a chain's threads takes one stage of a pair, the second half the other.  P has zeros
//           where a half's rows meet the other's keys, so that one product sums both; four streams are joined in the epilogue
// A CTA takes one split of the stages of one (sequence, kv head, group of rows); the rows of several splits meet in tree_join_kernel.
// The predicate is applied to the last stages only, those with nodes in them: a row has one bit for each of 128 nodes.  There, rows
// of V past the sequence's end, which may hold anything, are cleared in shared memory ahead of the product, and so are elements
// that are no finite number; rows that see such an element get it added behind the epilogue, so that it reaches nobody else.  Among the
// cached tokens, which all rows see, infinities stay where they are; only FOLD, whose zeros in P meet them too, puts right what came out as NaN.
//
// Measured, from GPU to GPU: 32 x 8 heads x 4096 tokens, 64 rows 103 to 120 us (5.2 to 4.5 TB/s; HBM, and the ends of CTAs that have an SM to
// themselves), 1 x 8 x 131072, 244 rows 144 to 175 us (910 to 750 TFLOP/s; tensor pipe 48 % busy, exponentials 53 %, the chain between them),
// 1 x 8 x 1001, 20 rows 10.7 us (latency).
//
// Every mbarrier wait is bounded; on expiry the CTA records an error, and leaves when its copies and products in flight have ended, whichever
// warp's wait it was.
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
constexpr long long kDrainCycles = 200000000;       // 0.1 s: how long a CTA that gives up waits for its copies and products
// Behind the ring: barriers and flags.
struct Block {
    uint64_t bars[32];
    uint32_t tmem;
    int abort, bad_tree, nan_out;           // nan_out: FOLD, a result that is, or may be, NaN
    uint32_t bad[4];                        // nodes with elements of V that are no finite number
    int8_t up[GRL_MAX_TREE];                // parents
};
template <int HD, Mode MODE> struct Form {
    static constexpr int BOXES = HD / 64;
    static constexpr int SLAB = BOXES * KV_BOX;             // K (or V) of a stage
    static constexpr int STAGE = 2 * SLAB;
    static constexpr int Q_TILE = BOXES * Q_BOX;
    static constexpr int STREAMS = MODE == FOLD ? 4 : MODE == SPLIT ? 2 : 1;        // of a row
    static constexpr int ROWS = 256 / STREAMS;              // of a group
    static constexpr int Q_BYTES = MODE == PAIR ? 2 * Q_TILE : Q_TILE;
    static constexpr int OUT_BYTES = 256 * 32 * 4;          // 32 columns of 256 accumulator rows, where the queries were
    static constexpr int RING = Q_BYTES > OUT_BYTES ? Q_BYTES : OUT_BYTES;
    // PAIR: one ring that both chains read.  Else a ring for each chain: a phase of a slot's barrier is told by its parity, so whoever waits on it
    // has to have seen the phase before, which one of two chains that share out the stages of a ring may not have when copies come in late.
    static constexpr int FIT = (225 * 1024 - RING) / STAGE < 8 ? (225 * 1024 - RING) / STAGE : 8;
    static constexpr int NST = MODE == PAIR ? FIT : FIT / 2 * 2, SLOTS = MODE == PAIR ? NST : NST / 2;
    static constexpr int BLOCK = RING + NST * STAGE;
    static constexpr int TOTAL = BLOCK + (int)sizeof(Block) + 1024;     // + slack for 1024-byte alignment
    static_assert(TOTAL <= 227 * 1024, "shared memory");
    static constexpr size_t PART = (size_t)ROWS * (HD + 2);             // floats of a CTA in the workspace: O, then (m, l)
    // barriers
    static constexpr int FULL = 0, EMPTY = NST, S_FULL = 2 * NST, P_READY = S_FULL + 4, O_PREV = P_READY + 4, O_DONE = O_PREV + 2, Q_READY = O_DONE + 2,
                         DRAIN = Q_READY + 1, NUM = DRAIN + 2;
    static_assert(NUM <= 32, "barrier block");
};
struct Groups {
    uint32_t per_group;     // 2^32 / G rounded up: row / G is its product's upper half (rows and G below 2^15; 0: G is 1)
    int groups;             // of rows of a (sequence, kv head)
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
    if (mbar_test(addr, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (clock64() - t0 > c.limit) {
            *c.abort = 1;
            if (c.status && atomicCAS(c.status, 0, GRL_ERR_TIMEOUT) == 0) {
                c.status[1] = (7 << 28) | bar;
                c.status[2] = blockIdx.x;
                c.status[3] = blockIdx.y | (blockIdx.z << 16);
            }
            return false;
        }
        if (mbar_try_wait(addr, parity)) return true;
        if (*c.abort) return false;
    }
}
// The whole warp; it leaves converged, as the tensor-memory instructions behind it need.
__device__ __forceinline__ bool wait_bar_warp(const Ctx& c, int bar, uint32_t parity) {
    const bool ok = __all_sync(0xffffffffu, wait_bar(c, bar, parity));
    __syncwarp();
    return ok;
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


// Which of inf (1), -inf (2) and NaN (4) are among the cached values of tokens k0 .. k1 - 1, by column; the 256 softmax threads.
template <int HD>
__device__ __forceinline__ void find_infinities(const TreeArgs& a, int b, int kvh, int k0, int k1, uint32_t* columns, int st_id) {
    constexpr int CH = HD / 8;
#pragma unroll 1
    for (int idx = st_id; idx < (k1 - k0) * CH; idx += 256) {
        const int at = k0 + idx / CH, c = idx % CH, page = a.block_table[(size_t)b * a.max_pages + at / a.P];
        if ((unsigned)page >= (unsigned)a.num_pages) continue;
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.v_pages) +
                                                             (((size_t)page * a.Hkv + kvh) * a.P + at % a.P) * HD) + c);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t x = w[e >> 1] >> (e & 1) * 16 & 0xffffu;
            if ((x & 0x7f80u) == 0x7f80u) atomicOr(columns + 8 * c + e, x & 0x7fu ? 4u : x >> 15 ? 2u : 1u);
        }
    }
}

__device__ __forceinline__ int node_of(const Groups& sh, int r) { return sh.per_group ? (int)__umulhi((uint32_t)r, sh.per_group) : r; }

template <int HD, Mode MODE>
__global__ void __launch_bounds__(kThreads, 1)
tree_sm100_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeArgs a,
                  const __grid_constant__ Groups sh) {
    using F = Form<HD, MODE>;
    constexpr bool PAIR = MODE == tree::PAIR, FOLD = MODE == tree::FOLD;
    constexpr int NST = F::NST;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_addr);
    Block& blk = *reinterpret_cast<Block*>(smem + F::BLOCK);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Ctx ctx{base + F::BLOCK, &blk.abort, a.status, a.wait_limit};
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
            mbar_init(bar(F::DRAIN + t), 1);
        }
        mbar_init(bar(F::Q_READY), 256);
        blk.abort = blk.bad_tree = blk.nan_out = 0;
        blk.bad[0] = blk.bad[1] = blk.bad[2] = blk.bad[3] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == WARP_MMA0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&blk.tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // all of the above beside the tail of the kernel before this one, nothing below
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&blk.tmem);
    // nodes and length of the sequence (0, 0 where they do not fit); this CTA's stages
    const int b = blockIdx.z, kvh = blockIdx.y / sh.groups, r0 = blockIdx.y % sh.groups * F::ROWS;
    int cached;
    const int fits = tree_nodes(a, b, &cached, tid == 0), n = max(fits, 0), len = fits > 0 ? cached + fits : 0;
    const int stages = (len + BN - 1) / BN, per = (stages + a.n_splits - 1) / a.n_splits;
    const int st0 = min(stages, (int)blockIdx.x * per), ns = min(stages, ((int)blockIdx.x + 1) * per) - st0;
    // stages of chain t of ns, and its k-th one: all, or every second one, or every second pair
    auto count_of = [&](int t) { return PAIR ? ns : FOLD ? ns / 4 * 2 + max(0, min(2, ns % 4 - 2 * t)) : (ns - t + 1) / 2; };
    auto stage_of = [&](int t, int k) { return PAIR ? k : FOLD ? 4 * (k >> 1) + 2 * t + (k & 1) : 2 * k + t; };
    auto slot_of = [&](int t, int x) { return (PAIR ? 0 : t * F::SLOTS) + x % F::SLOTS; };        // of the x-th stage of a chain
    // steps of chain t over ns stages: one for each, or for two; a tile without rows takes none
    auto steps_of = [&](int t) { return PAIR ? (r0 + t * BM < a.R ? ns : 0) : FOLD ? ((ns + 1) / 2 - t + 1) / 2 : (ns - t + 1) / 2; };

    // every warp at its end; behind it nobody reads the shared or the tensor memory any more
    auto finish = [] {
        pdl_trigger();
        tc_fence_before();
        __syncwarp();
        asm volatile("bar.sync 2, %0;" ::"n"(kThreads) : "memory");
        tc_fence_after();
    };

    if (warp < WARP_SOFTMAX) {
      reg_dec<REGS_MISC>();
      if (warp == WARP_TMA0 || warp == WARP_TMA1) {
        // ------------------------------------------------------------------ TMA: a warp the stages of a chain (PAIR: the even or the odd ones)
        // A lane a copy: one lane's chain of waits and copies took some 1700 cycles a stage, longer than HBM takes to bring it.
        const int ppt = BN / a.P, t = uniform(warp == WARP_TMA1);
        int last = -1;          // the last stage this warp has asked for
        const int32_t* table = a.block_table + (size_t)b * a.max_pages;
        const int count = count_of(t);
        int first = st0 * ppt;
        int entry = table[min(first + lane, a.max_pages - 1)], next = table[min(first + 32 + lane, a.max_pages - 1)];
        for (int k = PAIR ? t : 0; k < count; k += PAIR ? 2 : 1) {
            const int p = st0 + stage_of(t, k), s = slot_of(t, k), it = k / F::SLOTS;
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
                tma_load_2d(base + F::RING + s * F::STAGE + v * F::SLAB + x * KV_BOX + j * a.P * 128, v ? &tmV : &tmK, x * 64,
                            (page * a.Hkv + kvh) * a.P, bar(F::FULL + s));
            }
            __syncwarp();
            last = k;
        }
        finish();
        // A wait ran out, maybe behind this warp's last look at the flag: copies in flight land before the shared memory is given back.
        if (*ctx.abort) {
            const long long t0 = clock64();
            for (int x = last; x >= 0 && x > last - F::SLOTS; x -= PAIR ? 2 : 1)
                while (!mbar_try_wait(bar(F::FULL + slot_of(t, x)), (x / F::SLOTS) & 1) && clock64() - t0 < kDrainCycles) {}
        }
      } else {
        // ------------------------------------------------------------------ products of chain t
        const int t = uniform(warp == WARP_MMA1);
        const uint32_t qa = desc_lo(base + (PAIR ? t * F::Q_TILE : 0), 16);
        const uint32_t k_lo = desc_lo(base + F::RING, 16), v_lo = desc_lo(base + F::RING + F::SLAB, KV_BOX);
        const uint32_t s_tmem = (uint32_t)uniform((int)tmem_base) + (uint32_t)t * TMEM_CHAIN, o_tmem = s_tmem + TMEM_O;
        const int steps = uniform(steps_of(t)), others = PAIR ? uniform(steps_of(t ^ 1)) : 1, mine = uniform(count_of(t));
        bool ok = true;
        // S of a step: 64 columns of the buffers in turn; FOLD: both buffers, a stage each
        auto issue_qk = [&](int i) -> bool {
#pragma unroll
            for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                const int k = FOLD ? 2 * i + half : i, s = slot_of(t, k);
                if (FOLD && k >= mine) break;
                if (!wait_bar_warp(ctx, F::FULL + s, (k / F::SLOTS) & 1)) return false;
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
        ok = wait_bar_warp(ctx, F::Q_READY, 0);
        if (ok) tc_fence_after();
        for (int i = 0; i < (FOLD ? 1 : 2) && i < steps && ok; ++i) ok = issue_qk(i);
        for (int i = 0; i < steps && ok; ++i) {
            ok = wait_bar_warp(ctx, F::P_READY + 2 * t + (FOLD ? 0 : i & 1), (FOLD ? i : i >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                const int k = FOLD ? 2 * i + half : i, s = slot_of(t, k);
                if (FOLD && k >= mine) break;
                const uint32_t p_tmem = s_tmem + (FOLD ? (uint32_t)half * (BN / 2) : (uint32_t)(i & 1) * BN), vb = v_lo + (uint32_t)s * (F::STAGE >> 4);
#pragma unroll
                for (int ks = 0; ks < BN / 16; ++ks)
                    mma_ts2(o_tmem, p_tmem + ks * 8, vb + (uint32_t)ks * (2048 >> 4), IdescPV<HD>::value, i > 0 || half > 0 || ks > 0);
                mma_commit(bar(F::EMPTY + s));
                // a stage that the other tile does not read is released for it too
                if (PAIR && others == 0) mma_commit(bar(F::EMPTY + s));
            }
            if (!FOLD && i + 2 == steps) mma_commit(bar(F::O_PREV + t));
            // overwrites the buffer of P(i): in order behind its product
            if (i + (FOLD ? 1 : 2) < steps) ok = issue_qk(i + (FOLD ? 1 : 2));
        }
        // for a chain without steps too
        if (ok) mma_commit(bar(F::O_DONE + t));
        finish();
        if (*ctx.abort) {       // and products in flight end before the tensor memory and the operands are
            mma_commit(bar(F::DRAIN + t));
            const long long t0 = clock64();
            while (!mbar_try_wait(bar(F::DRAIN + t), 0) && clock64() - t0 < kDrainCycles) {}
        }
      }
    } else {
        // ------------------------------------------------------------------ softmax and epilogue
        reg_inc<REGS_SOFTMAX>();
        const int t = (warp - WARP_SOFTMAX) >> 2, st_id = tid - WARP_SOFTMAX * 32;      // chain; thread of the 256
        const int row = tid & 127, sub = FOLD ? row >> 6 : 0;
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_addr + (uint32_t)t * TMEM_CHAIN, o_addr = s_addr + TMEM_O;
        constexpr int CH = HD / 8, PER = F::ROWS * CH / 256;     // 16-byte pieces of a query row, of a thread
        auto meet = [] {        // both warpgroups; the barrier is for converged warps
            __syncwarp();
            asm volatile("bar.sync 1, 256;" ::: "memory");
        };
        const int prefix = len - n;
        const bool whole = a.n_splits == 1;
        const int r = r0 + (PAIR ? t * BM : 0) + (FOLD ? row & 63 : row), node = node_of(sh, r);
        {   // query rows as the K-major operand, rows past the last one zero; parents
            const int up = a.parents && st_id < n ? a.parents[(size_t)b * a.T + st_id] : -1;
            const int c = st_id % CH, first = st_id / CH;
            const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + ((size_t)b * a.T * a.Hq + kvh * a.G) * HD) + c;
            uint4 v[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int g = r0 + first + e * (256 / CH), at = node_of(sh, g);
                v[e] = make_uint4(0u, 0u, 0u, 0u);
                if (g < a.R) v[e] = __ldg(q + (at * a.Hq + g - at * a.G) * CH);
            }
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int qr = first + e * (256 / CH);
                const uint32_t to = base + (qr >> 7) * F::Q_TILE + (c >> 3) * Q_BOX + (qr & 127) * 128 + (((c & 7) ^ (qr & 7)) << 4);
                sts128(to, v[e]);
                if (FOLD) sts128(to + 64 * 128, v[e]);
            }
            if (a.parents && st_id < n) {
                if (up < -1 || up >= st_id) blk.bad_tree = 1;
                blk.up[st_id] = (int8_t)up;
            }
        }
        fence_async_smem();
        mbar_arrive(bar(F::Q_READY));
        meet();
        const bool bad_tree = *reinterpret_cast<volatile int*>(&blk.bad_tree) != 0;
        if (bad_tree && st_id == 0) tree_fail(a.status, TREE_BAD_PARENT, b, n);
        const bool live = r < a.R && node < n && !bad_tree;
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (live) {
            if (!a.parents) seen = low_bits(node + 1);
            else
                for (int u = node; u >= 0; u = blk.up[u]) {         // up to the cached tokens: a tree's depth
                    const uint32_t bit = 1u << (u & 31);
                    seen.x |= u < 32 ? bit : 0u;
                    seen.y |= u >> 5 == 1 ? bit : 0u;
                    seen.z |= u >> 5 == 2 ? bit : 0u;
                    seen.w |= u >> 5 == 3 ? bit : 0u;
                }
        }
        __syncwarp();
        const int nh = steps_of(t), mine = count_of(t);
        float m_ref = -INFINITY, l = 0.f;
        bool ok = true;
        for (int i = 0; i < nh && ok; ++i) {
            const int bf = FOLD ? 0 : i & 1, own = FOLD ? 2 * i + sub : i, k0 = (st0 + stage_of(t, own)) * BN;
            const bool none = FOLD && own >= mine, nodes = none || k0 + BN > prefix;       // none: the pair's second stage is another CTA's, or past the end
            // stages with nodes in them: their values are there when their scores are
#pragma unroll
            for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                const int k = FOLD ? 2 * i + half : i, v0 = (st0 + stage_of(t, k)) * BN, s = slot_of(t, k);
                if (k < mine && v0 + BN > prefix) {
                    ok = ok && wait_bar_warp(ctx, F::FULL + s, (k / F::SLOTS) & 1);
                    if (!ok) break;
                    clean_values<HD>(base + F::RING + s * F::STAGE + F::SLAB, v0, prefix, len, blk.bad, row);
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
                    if constexpr (!FOLD)
                        ok = i + 1 < nh ? wait_bar_warp(ctx, F::S_FULL + 2 * t + (bf ^ 1), ((i + 1) >> 1) & 1)
                                        : wait_bar_warp(ctx, F::O_PREV + t, 0);
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
        if (ok) ok = wait_bar_warp(ctx, F::O_DONE + t, 0);

        // Epilogue.  The streams of a row meet at their common maximum; 32 columns at a time go through the queries' place, which both chains
        // have done with, so that rows leave in whole pieces.
        tc_fence_before();
        meet();
        ok = __all_sync(0xffffffffu, ok && !*ctx.abort);
        tc_fence_after();
        m_ref = tree_row_max(m_ref, l);
        float m = m_ref, sum = l;
        if constexpr (F::STREAMS > 1) {
            float2* ml = reinterpret_cast<float2*>(smem);
            ml[t * BM + row] = make_float2(m_ref, l);
            meet();
            m = -INFINITY;
            sum = 0.f;
#pragma unroll
            for (int x = 0; x < F::STREAMS; ++x) m = fmaxf(m, ml[x * F::ROWS + row % F::ROWS].x);
#pragma unroll
            for (int x = 0; x < F::STREAMS; ++x) {
                const float2 v = ml[x * F::ROWS + row % F::ROWS];
                if (v.x != -INFINITY) sum = fmaf(ex2(v.x - m), v.y, sum);
            }
            meet();
        }
        const float w = (m_ref == -INFINITY ? 0.f : ex2(m_ref - m)) * (whole ? 1.f / sum : 1.f);
        float* part = a.part + ((size_t)(b * gridDim.y + blockIdx.y) * a.n_splits + blockIdx.x) * F::PART;
        const int rows = min(F::ROWS, a.R - r0), live_nodes = bad_tree ? 0 : n;
        const bool full = ok && nh > 0 && m_ref != -INFINITY;
        const uint32_t empty = whole && live && sum == 0.f ? 0x7fc00000u : 0u;      // a node without any weight, scores of -inf only: NaN
        // a thread takes one 16-byte piece of every 32nd row
        constexpr int K = F::ROWS / 32;
        const int c = st_id & 7, rr0 = st_id >> 3;
        int at[K];                  // elements from the batch's, or the part's, first; below 0: nothing to write
        uint32_t alive = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int rg = r0 + rr0 + 32 * k, rn = node_of(sh, rg);
            const bool l_ = rn < live_nodes;
            alive |= (uint32_t)l_ << k;
            at[k] = rr0 + 32 * k >= rows || !ok || !(whole || l_) ? -1 : (whole ? (rn * a.Hq + rg - rn * a.G) * HD : (rr0 + 32 * k) * HD) + 4 * c;
        }
        __nv_bfloat16* out_at = reinterpret_cast<__nv_bfloat16*>(a.out) + ((size_t)b * a.T * a.Hq + kvh * a.G) * HD;
#pragma unroll 1
        for (int ch = 0; ch < HD / 32; ++ch) {
            uint32_t o[32];
            if (ok && nh > 0) tmem_ld_x32_sync(o_addr + ch * 32, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint4 v = make_uint4(__float_as_uint(__uint_as_float(o[4 * e]) * w), __float_as_uint(__uint_as_float(o[4 * e + 1]) * w),
                                           __float_as_uint(__uint_as_float(o[4 * e + 2]) * w), __float_as_uint(__uint_as_float(o[4 * e + 3]) * w));
                sts128(base + st_id * 128 + ((e ^ (st_id & 7)) << 4), full ? v : make_uint4(empty, empty, empty, empty));
            }
            meet();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (at[k] < 0) continue;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (alive >> k & 1u) {
#pragma unroll
                    for (int x = 0; x < F::STREAMS; ++x) {
                        const uint4 u = lds128(base + (x * F::ROWS + rr0 + 32 * k) * 128 + ((c ^ (rr0 & 7)) << 4));
                        v.x += __uint_as_float(u.x); v.y += __uint_as_float(u.y); v.z += __uint_as_float(u.z); v.w += __uint_as_float(u.w);
                    }
                    if (FOLD && isnan((v.x + v.y) + (v.z + v.w)))
                        *reinterpret_cast<volatile int*>(&blk.nan_out) = 1;
                }
                if (whole) {
                    const __nv_bfloat162 p0 = __floats2bfloat162_rn(v.x, v.y), p1 = __floats2bfloat162_rn(v.z, v.w);
                    *reinterpret_cast<uint2*>(out_at + at[k] + ch * 32) = make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
                } else {
                    *reinterpret_cast<float4*>(part + at[k] + ch * 32) = v;
                }
            }
            meet();
        }
        const bool owner = st_id < F::ROWS && st_id < rows;         // of row r in the results
        if (!whole && owner)
            reinterpret_cast<float2*>(part + (size_t)F::ROWS * HD)[st_id] =
                !live ? make_float2(-INFINITY, -1.f) : ok && ns > 0 ? make_float2(m, sum) : make_float2(-INFINITY, 0.f);
        if (FOLD && *reinterpret_cast<volatile int*>(&blk.nan_out)) {
            // rare: an infinity among the cached values times the zeros that a half's rows have for the other's keys.  A row that has a sum at all
            // has a weight for every cached token, so that its result is that infinity, or NaN where both are in the column, or a NaN.
            uint32_t* columns = reinterpret_cast<uint32_t*>(smem);
            if (st_id < HD) columns[st_id] = 0u;
            meet();
            find_infinities<HD>(a, b, kvh, min(prefix, st0 * BN), min(prefix, (st0 + ns) * BN), columns, st_id);
            meet();
            if (owner && live && ok && sum > 0.f)
#pragma unroll 1
                for (int d = 0; d < HD; ++d) {
                    if (columns[d] != 1u && columns[d] != 2u) continue;
                    const float x = columns[d] == 1u ? INFINITY : -INFINITY;
                    if (whole) reinterpret_cast<__nv_bfloat16*>(a.out)[(((size_t)b * a.T + node) * a.Hq + kvh * a.G + r - node * a.G) * HD + d] = __float2bfloat16_rn(x);
                    else part[(size_t)st_id * HD + d] = x;
                }
        }
        if ((blk.bad[0] | blk.bad[1] | blk.bad[2] | blk.bad[3]) != 0u) {         // rare: what is no finite number, for the rows that see it
            if (owner && live && ok)
                for (int u = 0; u < n; ++u) {
                    const uint32_t sees = u < 64 ? (u < 32 ? seen.x : seen.y) : (u < 96 ? seen.z : seen.w);
                    if (!(blk.bad[u >> 5] & sees & (1u << (u & 31)))) continue;
                    const int at = prefix + u, page = a.block_table[(size_t)b * a.max_pages + at / a.P];
                    if ((unsigned)page >= (unsigned)a.num_pages) continue;
                    const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(a.v_pages) + (((size_t)page * a.Hkv + kvh) * a.P + at % a.P) * HD;
                    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + node) * a.Hq + kvh * a.G + r % a.G) * HD;
                    for (int d = 0; d < HD; ++d) {
                        const float x = __bfloat162float(v[d]);
                        if (isfinite(x)) continue;
                        if (whole) out[d] = __float2bfloat16_rn(__bfloat162float(out[d]) + x);
                        else part[(size_t)st_id * HD + d] += x;
                    }
                }
        }
        finish();
    }
    if (*ctx.abort) __syncthreads();        // the whole CTA finds the flag as it is: no wait under the budget is left
    __syncwarp();
    if (warp == WARP_MMA0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

// Joins the parts of heads that several CTAs have worked on, a warp a row: the parts' sums at their common maximum, eight parts on
// their way at once.  Latency: two rows a warp, one behind the other, take 0.9 us longer behind 1 x 8 heads of 1001 tokens (11.5 / 10.6) and 2 us
// behind 131072 tokens of 244 rows (147.4 / 145.4).
constexpr int kJoinRows = 8;        // of a CTA
template <int HD>
__global__ void __launch_bounds__(32 * kJoinRows) tree_join_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ Groups sh, int part_rows) {
    const int hgs = a.Hkv * sh.groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x / hgs, hg = blockIdx.x % hgs;
    pdl_wait();                 // every CTA, or the kernel behind this one could start before the one ahead of it has ended
    pdl_trigger();
    constexpr int V = HD / 32;              // columns of a lane
    const size_t stride = (size_t)part_rows * (HD + 2);
    const float* first_part = a.part + (size_t)blockIdx.x * a.n_splits * stride;
    const int kvh = hg / sh.groups, r0 = hg % sh.groups * part_rows, rows = min(part_rows, a.R - r0);
    const int rr = blockIdx.y * kJoinRows + warp;
    if (rr >= rows) return;
    float m = -INFINITY, l = 0.f, acc[V];
    bool nobody = false;
#pragma unroll
    for (int c = 0; c < V; ++c) acc[c] = 0.f;
    for (int i0 = 0; i0 < a.n_splits; i0 += 8) {
        float2 ml[8];
        float o[8][V];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j;
            ml[j] = make_float2(-INFINITY, 0.f);
            if (i >= a.n_splits) continue;
            const float* p = first_part + (size_t)i * stride;
            ml[j] = __ldcg(reinterpret_cast<const float2*>(p + (size_t)part_rows * HD) + rr);
            if constexpr (V == 4) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(p + (size_t)rr * HD) + lane);
                o[j][0] = f.x; o[j][1] = f.y; o[j][2] = f.z; o[j][3] = f.w;
            } else {
                const float2 f = __ldcg(reinterpret_cast<const float2*>(p + (size_t)rr * HD) + lane);
                o[j][0] = f.x; o[j][1] = f.y;
            }
        }
        float m_new = m;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!(ml[j].y <= 0.f)) m_new = fmaxf(m_new, ml[j].x);
        const float f = m == -INFINITY ? 0.f : exp2f(m - m_new);
        l *= f;
#pragma unroll
        for (int c = 0; c < V; ++c) acc[c] *= f;
        m = m_new;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            nobody |= ml[j].y < 0.f;
            if (ml[j].y <= 0.f) continue;       // a part that has seen nothing has no O
            const float w = exp2f(ml[j].x - m);
            l = fmaf(w, ml[j].y, l);
#pragma unroll
            for (int c = 0; c < V; ++c) acc[c] = fmaf(w, o[j][c], acc[c]);
        }
    }
    const float inv = nobody ? 0.f : 1.f / l;
    const int r = r0 + rr, node = node_of(sh, r);
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + node) * a.Hq + kvh * a.G + r - node * a.G) * HD;
    if constexpr (V == 4) {
        const __nv_bfloat162 p0 = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv), p1 = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
        reinterpret_cast<uint2*>(out)[lane] = make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
    } else {
        reinterpret_cast<__nv_bfloat162*>(out)[lane] = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv);
    }
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

static int join(grl_device* dev, const TreeArgs& a, const Groups& sh, int part_rows) {
    const dim3 grid(a.B * a.Hkv * sh.groups, (min(part_rows, a.R) + kJoinRows - 1) / kJoinRows);
    GRL_CUDA(launch_pdl(a.D == 128 ? tree_join_kernel<128> : tree_join_kernel<64>, grid, 32 * kJoinRows, 0, dev->stream, a, sh, part_rows));
    GRL_LAUNCHED("tree_join_kernel");
    return GRL_OK;
}

template <int HD, Mode MODE>
static int launch(grl_device* dev, const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, const Groups& sh) {
    using F = Form<HD, MODE>;
    static bool attr_set[64] = {};
    if (!attr_set[dev->ordinal & 63]) {      // a function attribute belongs to the device that was current
        GRL_CUDA(cudaFuncSetAttribute(tree_sm100_kernel<HD, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::TOTAL));
        attr_set[dev->ordinal & 63] = true;
    }
    GRL_CUDA(launch_pdl(tree_sm100_kernel<HD, MODE>, dim3(a.n_splits, a.Hkv * sh.groups, a.B), kThreads, F::TOTAL, dev->stream, tk, tv, a, sh));
    GRL_LAUNCHED("tree_sm100_kernel");
    return a.n_splits == 1 ? GRL_OK : join(dev, a, sh, F::ROWS);
}

static Mode mode_of(int R) { return R > BM ? PAIR : R > 64 ? SPLIT : FOLD; }
static int rows_of(Mode m) { return m == PAIR ? 256 : m == SPLIT ? 128 : 64; }
static Groups groups_of(int G, int groups) { return {G == 1 ? 0u : (uint32_t)(((1ull << 32) + G - 1) / G), groups}; }

}  // namespace tree

int tree_join_launch(grl_device* dev, const TreeArgs& a, int rows) { return tree::join(dev, a, tree::groups_of(a.G, 1), rows); }

// The fewest stages of a split.  us, split into 1 / 2 / 3 / 4: 4 x 8 heads x 700 tokens, 124 rows 15.2 / 15.9 / 15.2 / 15.0, 64 rows 14.2 / 15.7 /
// 13.3 / 13.5; 1500 tokens, 64 rows 21.4 / 18.1 / - / 17.7.  More heads than SMs are not split: 20 x 8 x 4096, 124 rows 98.7 / 106 / 110, 64 rows
// 106 / 102 / 105, 20 x 8 x 1024 40.4 / 49.3 / 57.2, 24 x 8 x 4096 101 / 121.  Equal shares of all stages for every CTA, heads cut where they fall, are no
// faster anywhere: 4 x 8 x 1500 27.1 for 17.7, and in turn on one GPU 32 x 8 x 4096, 64 rows 130 for 120, 1 x 8 x 131072 of 244 rows 190 for 174.
constexpr int kSplitStages = 4;
// asked: the caller's number of splits, or 0.
TreeTensorPlan tree_sm100_plan(const grl_device* dev, int B, int Hkv, int R, int D, int longest, int asked) {
    using namespace tree;
    const int rows = rows_of(mode_of(R)), sms = dev->prop.multiProcessorCount;
    TreeTensorPlan p{};
    p.groups = (R + rows - 1) / rows;
    const long long heads = (long long)B * Hkv * p.groups, stages = (longest + BN - 1) / BN;
    long long s = asked > 0 ? asked : sms / heads;
    if (asked <= 0 && s > stages / kSplitStages) s = stages / kSplitStages;
    p.splits = (int)(s < 1 ? 1 : s);
    p.workspace = p.splits == 1 ? 0 : sizeof(float) * (size_t)rows * (D + 2) * heads * p.splits;
    return p;
}

int tree_sm100_launch(grl_device* dev, const TreeArgs& a, const TreeTensorPlan& plan) {
    using namespace tree;
    CUtensorMap tk, tv;
    int rc = make_pool_map(dev, &tk, a.k_pages, a);
    if (!rc) rc = make_pool_map(dev, &tv, a.v_pages, a);
    if (rc) return rc;
    const Groups sh = groups_of(a.G, plan.groups);
    const Mode mode = mode_of(a.R);
    if (a.D == 128)
        return mode == PAIR ? launch<128, PAIR>(dev, tk, tv, a, sh) : mode == SPLIT ? launch<128, SPLIT>(dev, tk, tv, a, sh) : launch<128, FOLD>(dev, tk, tv, a, sh);
    return mode == PAIR ? launch<64, PAIR>(dev, tk, tv, a, sh) : mode == SPLIT ? launch<64, SPLIT>(dev, tk, tv, a, sh) : launch<64, FOLD>(dev, tk, tv, a, sh);
}

}  // namespace grl
