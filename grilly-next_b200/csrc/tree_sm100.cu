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
// The work is a list of pieces, runs of stages of one (sequence, kv head, group of rows): one for every CTA of the grid where the caller names the
// number of splits or there are many sequences, else an equal share of all stages of the batch for every CTA, which may end one head, hold some
// whole and begin another.  Whole heads are written by their CTA, the parts of others meet in tree_join_kernel.  The loads of the next
// piece run under the epilogue of the one before.
// The predicate is applied to the last stages only, those with nodes in them: a row has one bit for each of 128 nodes.  There, rows
// of V past the sequence's end, which may hold anything, are cleared in shared memory ahead of the product, and so are elements
// that are no finite number; rows that see such an element get it added behind the epilogue, so that it reaches nobody else.
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
constexpr long long kDrainCycles = 200000000;       // 0.1 s: how long a CTA that gives up waits for its copies and products
constexpr int kMaxShared = 128;             // sequences of a batch that is cut into equal shares
// Behind the ring: barriers, flags and the lengths of the batch.
struct Block {
    uint64_t bars[32];
    uint32_t tmem;
    int abort, stop, bad_tree;
    uint32_t bad[4];                        // nodes with elements of V that are no finite number
    int8_t up[GRL_MAX_TREE];                // parents
    int before[kMaxShared + 1];             // stages of the sequences before each one (of one head and group)
    int len[kMaxShared];
    uint8_t nodes[kMaxShared];
};
template <int HD, Mode MODE> struct Form {
    static constexpr int BOXES = HD / 64;
    static constexpr int SLAB = BOXES * KV_BOX;             // K (or V) of a stage
    static constexpr int STAGE = 2 * SLAB;
    static constexpr int Q_TILE = BOXES * Q_BOX;
    static constexpr int STREAMS = MODE == FOLD ? 4 : MODE == SPLIT ? 2 : 1;        // of a row
    static constexpr int ROWS = 256 / STREAMS;              // of a piece
    static constexpr int Q_BYTES = MODE == PAIR ? 2 * Q_TILE : Q_TILE;
    static constexpr int OUT_BYTES = 256 * 32 * 4;          // 32 columns of 256 accumulator rows, where the queries were
    static constexpr int RING = Q_BYTES > OUT_BYTES ? Q_BYTES : OUT_BYTES;
    static constexpr int NST = (225 * 1024 - RING) / STAGE < 8 ? (225 * 1024 - RING) / STAGE : 8;
    static constexpr int BLOCK = RING + NST * STAGE;
    static constexpr int TOTAL = BLOCK + (int)sizeof(Block) + 1024;     // + slack for 1024-byte alignment
    static_assert(TOTAL <= 227 * 1024, "shared memory");
    static constexpr size_t PART = (size_t)ROWS * (HD + 2);             // floats of a piece in the workspace: O, then (m, l)
    // barriers
    static constexpr int FULL = 0, EMPTY = NST, S_FULL = 2 * NST, P_READY = S_FULL + 4, O_PREV = P_READY + 4, O_DONE = O_PREV + 2, Q_READY = O_DONE + 2,
                         DRAIN = Q_READY + 1, NUM = DRAIN + 2;
    static_assert(NUM <= 32, "barrier block");
};
struct Share {
    int ctas;               // > 0: equal shares of all stages; 0: one piece a CTA, grid (splits, Hkv * groups, B)
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


struct Piece {
    int b, hg, st0, ns;     // sequence, kv head * groups + group, first stage and stages
    bool whole;
    int part;               // where it goes in the workspace, where it is not whole
};

// Nodes and length of a sequence (0, 0 where they do not fit).
__device__ __forceinline__ int fitting(const TreeArgs& a, int b, int* n, bool tell) {
    int prefix;
    const int k = tree_nodes(a, b, &prefix, tell);
    *n = k < 0 ? 0 : k;
    return k > 0 ? prefix + k : 0;
}
// Stages of the sequences before each one, by one warp; four sequences a lane.
__device__ __forceinline__ void scan_batch(const TreeArgs& a, Block& k, bool tell) {
    const int lane = threadIdx.x & 31;
    int len[4], n[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        len[e] = n[e] = 0;
        if (4 * lane + e < a.B) len[e] = fitting(a, 4 * lane + e, &n[e], tell);
    }
    int at[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { at[e] = sum; sum += (len[e] + BN - 1) / BN; }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    before -= sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        k.before[4 * lane + e] = before + at[e];
        k.len[4 * lane + e] = len[e];
        k.nodes[4 * lane + e] = (uint8_t)n[e];
    }
    if (lane == 31) k.before[kMaxShared] = before + sum;
}
// The share of CTA `cta` of the stages of the batch, which are fewer than 2^31 (tree_sm100_plan).
__device__ __forceinline__ int share_begin(const Block& k, const TreeArgs& a, const Share& sh, int cta) {
    return (int)((long long)k.before[kMaxShared] * a.Hkv * sh.groups * cta / sh.ctas);
}
// The sequence of a stage of the batch.
__device__ __forceinline__ int sequence_at(const Block& k, int hgs, int stage) {
    int lo = 0, hi = kMaxShared;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (k.before[mid] * hgs <= stage) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Walks the pieces of a CTA; every role does so for itself.  32-bit arithmetic: a division of 64 bits is a call, and a called function may use more
// registers than the warps that have given theirs up still hold.
struct Pieces {
    int at, end;
    __device__ __forceinline__ void start(const Block& k, const TreeArgs& a, const Share& sh) {
        at = share_begin(k, a, sh, blockIdx.x);
        end = share_begin(k, a, sh, blockIdx.x + 1);
    }
    __device__ __forceinline__ bool take(const Block& k, const TreeArgs& a, const Share& sh, Piece* p) {
        if (at >= end) return false;
        const int hgs = a.Hkv * sh.groups;
        p->b = sequence_at(k, hgs, at);
        const int stages = k.before[p->b + 1] - k.before[p->b], rem = at - k.before[p->b] * hgs;
        p->hg = (int)((unsigned)rem / (unsigned)stages);
        p->st0 = rem - p->hg * stages;
        p->ns = min(stages - p->st0, end - at);
        p->whole = p->ns == stages;
        p->part = (int)blockIdx.x * 2 + (p->st0 == 0);       // a CTA goes on with one head at most, and begins one at most
        at += p->ns;
        return true;
    }
};

template <int HD, Mode MODE>
__global__ void __launch_bounds__(kThreads, 1)
tree_sm100_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeArgs a,
                  const __grid_constant__ Share sh) {
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
        blk.abort = blk.stop = blk.bad_tree = 0;
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
    if (sh.ctas && warp == WARP_TMA0) scan_batch(a, blk, blockIdx.x == 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&blk.tmem);
    // the piece of a CTA that has one only
    Piece only{};
    int only_len = 0, only_n = 0;
    if (!sh.ctas) {
        only.b = blockIdx.z;
        only.hg = blockIdx.y;
        only_len = fitting(a, only.b, &only_n, tid == 0);
        const int stages = (only_len + BN - 1) / BN, per = (stages + a.n_splits - 1) / a.n_splits;
        only.st0 = min(stages, (int)blockIdx.x * per);
        only.ns = min(stages, ((int)blockIdx.x + 1) * per) - only.st0;
        only.whole = a.n_splits == 1;
        only.part = (only.b * gridDim.y + only.hg) * a.n_splits + blockIdx.x;
    }
    Pieces pieces{};
    if (sh.ctas) pieces.start(blk, a, sh);
    bool taken = false;
    auto take = [&](Piece* p, int* len, int* n) -> bool {
        if (sh.ctas) {
            if (!pieces.take(blk, a, sh, p)) return false;
            *len = blk.len[p->b];
            *n = blk.nodes[p->b];
            return true;
        }
        if (taken) return false;
        taken = true;
        *p = only;
        *len = only_len;
        *n = only_n;
        return true;
    };
    // steps of chain t over ns stages: all, or every second one, or every second pair; a tile without rows takes none
    auto steps_of = [&](int t, int ns, int r0) { return PAIR ? (r0 + t * BM < a.R ? ns : 0) : FOLD ? ((ns + 1) / 2 - t + 1) / 2 : (ns - t + 1) / 2; };

    if (warp < WARP_SOFTMAX) {
      reg_dec<REGS_MISC>();
      if (warp == WARP_TMA0 || warp == WARP_TMA1) {
        // ------------------------------------------------------------------ TMA: a warp the even stages, a warp the odd ones
        // A lane a copy: one lane's chain of waits and copies took some 1700 cycles a stage, longer than HBM takes to bring it.
        const int ppt = BN / a.P, odd = uniform(warp == WARP_TMA1);
        int done = 0, last = -1, len, n;        // stages of earlier pieces; the last one this warp has asked for
        Piece pc;
        bool ok = true;
        while (ok && take(&pc, &len, &n)) {
            const int32_t* table = a.block_table + (size_t)pc.b * a.max_pages;
            const int kvh = pc.hg / sh.groups;
            int first = pc.st0 * ppt;
            int entry = table[min(first + lane, a.max_pages - 1)], next = table[min(first + 32 + lane, a.max_pages - 1)];
            for (int i = (done ^ odd) & 1; i < pc.ns; i += 2) {
                const int p = pc.st0 + i, s = (done + i) % NST, it = (done + i) / NST;
                if (p * ppt - first >= 32) {
                    first += 32;
                    entry = next;
                    next = table[min(first + 32 + lane, a.max_pages - 1)];
                }
                if (it > 0 && !wait_bar_warp(ctx, F::EMPTY + s, (it - 1) & 1)) { ok = false; break; }
                const int np = min(ppt, (len - p * BN + a.P - 1) / a.P);       // pages of the stage that hold tokens
                if (lane == 0) mbar_expect_tx(bar(F::FULL + s), (uint32_t)(np * a.P * HD * 4));
                __syncwarp();
                // lane: page j, then K or V, then the box
                constexpr int COPIES = 2 * F::BOXES;
                const int j = lane / COPIES, v = lane / F::BOXES & 1, x = lane % F::BOXES;
                int page = __shfl_sync(0xffffffffu, entry, (p * ppt - first + j) & 31);
                if (j < np) {
                    if ((unsigned)page >= (unsigned)a.num_pages) { tree_fail(a.status, TREE_BAD_PAGE, pc.b, page); page = 0; }
                    tma_load_2d(base + F::RING + s * F::STAGE + v * F::SLAB + x * KV_BOX + j * a.P * 128, v ? &tmV : &tmK, x * 64,
                                (page * a.Hkv + kvh) * a.P, bar(F::FULL + s));
                }
                __syncwarp();
                last = done + i;
            }
            if (ok) done += pc.ns;
        }
        if (*ctx.abort) {       // copies in flight land before the shared memory is given back
            const long long t0 = clock64();
            for (int x = last; x >= 0 && x > last - NST; x -= 2)
                while (!mbar_try_wait(bar(F::FULL + x % NST), (x / NST) & 1) && clock64() - t0 < kDrainCycles) {}
        }
      } else {
        // ------------------------------------------------------------------ products of chain t
        const int t = uniform(warp == WARP_MMA1);
        const uint32_t qa = desc_lo(base + (PAIR ? t * F::Q_TILE : 0), 16);
        const uint32_t k_lo = desc_lo(base + F::RING, 16), v_lo = desc_lo(base + F::RING + F::SLAB, KV_BOX);
        const uint32_t s_tmem = (uint32_t)uniform((int)tmem_base) + (uint32_t)t * TMEM_CHAIN, o_tmem = s_tmem + TMEM_O;
        int done = 0, steps_done = 0, count = 0, len, n;        // stages, this chain's steps and pieces so far
        Piece pc;
        bool ok = true;
        while (ok && take(&pc, &len, &n)) {
            const int ns = uniform(pc.ns), r0 = pc.hg % sh.groups * (PAIR ? 2 * BM : BM);
            const int steps = uniform(steps_of(t, ns, r0)), others = PAIR ? uniform(steps_of(t ^ 1, ns, r0)) : 1;
            auto stage_of = [&](int i) { return PAIR ? i : FOLD ? 4 * i + 2 * t : 2 * i + t; };
            // S of a step: 64 columns of the buffers in turn; FOLD: both buffers, a stage each
            auto issue_qk = [&](int i) -> bool {
                const int ci = steps_done + i;
#pragma unroll
                for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                    const int st = stage_of(i) + half, s = (done + st) % NST;
                    if (FOLD && st >= ns) break;
                    if (!wait_bar_warp(ctx, F::FULL + s, ((done + st) / NST) & 1)) return false;
                    tc_fence_after();
                    const uint32_t kb = k_lo + (uint32_t)s * (F::STAGE >> 4), d = s_tmem + (uint32_t)(FOLD ? half : ci & 1) * BN;
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        mma_ss2(d, qa + (uint32_t)(((ks >> 2) * Q_BOX + (ks & 3) * 32) >> 4), kb + (uint32_t)(((ks >> 2) * KV_BOX + (ks & 3) * 32) >> 4),
                                IDESC_QK, ks != 0);
                }
                mma_commit(bar(F::S_FULL + 2 * t + (FOLD ? 0 : ci & 1)));
                return true;
            };
            ok = wait_bar_warp(ctx, F::Q_READY, count & 1);
            if (ok) tc_fence_after();
            for (int i = 0; i < (FOLD ? 1 : 2) && i < steps && ok; ++i) ok = issue_qk(i);
            for (int i = 0; i < steps && ok; ++i) {
                const int ci = steps_done + i;
                ok = wait_bar_warp(ctx, F::P_READY + 2 * t + (FOLD ? 0 : ci & 1), (FOLD ? ci : ci >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                    const int st = stage_of(i) + half, s = (done + st) % NST;
                    if (FOLD && st >= ns) break;
                    const uint32_t p_tmem = s_tmem + (FOLD ? (uint32_t)half * (BN / 2) : (uint32_t)(ci & 1) * BN), vb = v_lo + (uint32_t)s * (F::STAGE >> 4);
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
            // for a chain without steps too, so that nobody falls two pieces behind
            if (ok) mma_commit(bar(F::O_DONE + t));
            done += ns;
            steps_done += steps;
            ++count;
        }
        if (!ok) {              // products in flight end before the tensor memory and the operands are given back
            mma_commit(bar(F::DRAIN + t));
            const long long t0 = clock64();
            while (!mbar_try_wait(bar(F::DRAIN + t), 0) && clock64() - t0 < kDrainCycles) {}
            __syncwarp();
        }
      }
    } else {
        // ------------------------------------------------------------------ softmax and epilogue
        reg_inc<REGS_SOFTMAX>();
        const int t = (warp - WARP_SOFTMAX) >> 2, st_id = tid - WARP_SOFTMAX * 32;      // chain; thread of the 256
        const int row = tid & 127, sub = FOLD ? row >> 6 : 0;
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_addr + (uint32_t)t * TMEM_CHAIN, o_addr = s_addr + TMEM_O;
        constexpr int CH = HD / 8, Q_ROWS = PAIR ? 2 * BM : BM, PER = Q_ROWS * CH / 256;    // 16-byte pieces of the query rows, of a thread
        int done = 0, steps_done = 0, count = 0, prevs = 0, len = 0, n = 0;
        Piece pc{};
        auto meet = [] {        // both warpgroups; the barrier is for converged warps
            __syncwarp();
            asm volatile("bar.sync 1, 256;" ::: "memory");
        };
        while (take(&pc, &len, &n)) {
            const int b = pc.b, kvh = pc.hg / sh.groups, r0 = pc.hg % sh.groups * (PAIR ? 2 * BM : BM), ns = pc.ns, st0 = pc.st0, now_len = len, now_n = n,
                      prefix = len - n;
            const bool whole = pc.whole;
            const int part_at = pc.part;
            const int r = r0 + (PAIR ? t * BM : 0) + (FOLD ? row & 63 : row), node = r / a.G;
            {   // query rows as the K-major operand, rows past the last one zero; parents
                const int up = a.parents && st_id < now_n ? a.parents[(size_t)b * a.T + st_id] : -1;
                uint4 v[PER];
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int idx = st_id + e * 256, qr = idx / CH, c = idx % CH, g = r0 + (FOLD ? qr & 63 : qr);
                    v[e] = make_uint4(0u, 0u, 0u, 0u);
                    if (g < a.R)
                        v[e] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) +
                                                                    (((size_t)b * a.T + g / a.G) * a.Hq + kvh * a.G + g % a.G) * HD) + c);
                }
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int idx = st_id + e * 256, qr = idx / CH, c = idx % CH;
                    sts128(base + (qr >> 7) * F::Q_TILE + (c >> 3) * Q_BOX + (qr & 127) * 128 + (((c & 7) ^ (qr & 7)) << 4), v[e]);
                }
                if (a.parents && st_id < now_n) {
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
            const int nh = steps_of(t, ns, r0);
            auto stage_of = [&](int i) { return PAIR ? i : FOLD ? 4 * i + 2 * t : 2 * i + t; };
            float m_ref = -INFINITY, l = 0.f;
            bool ok = true;
            for (int i = 0; i < nh && ok; ++i) {
                const int ci = steps_done + i, bf = FOLD ? 0 : ci & 1, st = stage_of(i) + sub, k0 = (st0 + st) * BN;
                const bool none = FOLD && st >= ns, nodes = none || k0 + BN > prefix;       // none: the pair's second stage is another CTA's, or past the end
                // stages with nodes in them: their values are there when their scores are
#pragma unroll
                for (int half = 0; half < (FOLD ? 2 : 1); ++half) {
                    const int vs = stage_of(i) + half, v0 = (st0 + vs) * BN;
                    if (vs < ns && v0 + BN > prefix) {
                        ok = ok && wait_bar_warp(ctx, F::FULL + (done + vs) % NST, ((done + vs) / NST) & 1);
                        if (!ok) break;
                        clean_values<HD>(base + F::RING + (done + vs) % NST * F::STAGE + F::SLAB, v0, prefix, now_len, blk.bad, row);
                        fence_async_smem();
                    }
                }
                if (!ok) break;
                ok = wait_bar_warp(ctx, F::S_FULL + 2 * t + bf, (FOLD ? ci : ci >> 1) & 1);
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
                            ok = i + 1 < nh ? wait_bar_warp(ctx, F::S_FULL + 2 * t + (bf ^ 1), ((ci + 1) >> 1) & 1)
                                            : wait_bar_warp(ctx, F::O_PREV + t, prevs & 1);
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
            if (ok) ok = wait_bar_warp(ctx, F::O_DONE + t, count & 1);
            done += ns;
            steps_done += nh;
            ++count;
            prevs += nh > 1;

            // Epilogue.  The streams of a row meet at their common maximum; 32 columns at a time go through the queries' place, which both chains
            // have done with, so that rows leave in whole pieces.
            tc_fence_before();
            meet();
            ok = __all_sync(0xffffffffu, ok && !*ctx.abort);
            tc_fence_after();
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
            float* part = a.part + (size_t)part_at * F::PART;
            const int rows = min(F::ROWS, a.R - r0), live_nodes = bad_tree ? 0 : now_n;
            const bool full = ok && nh > 0 && m_ref != -INFINITY;
#pragma unroll 1
            for (int ch = 0; ch < HD / 32; ++ch) {
                uint32_t o[32];
                if (ok && nh > 0) tmem_ld_x32_sync(o_addr + ch * 32, o);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 v = make_uint4(__float_as_uint(__uint_as_float(o[4 * c]) * w), __float_as_uint(__uint_as_float(o[4 * c + 1]) * w),
                                               __float_as_uint(__uint_as_float(o[4 * c + 2]) * w), __float_as_uint(__uint_as_float(o[4 * c + 3]) * w));
                    sts128(base + st_id * 128 + ((c ^ (st_id & 7)) << 4), full ? v : make_uint4(0u, 0u, 0u, 0u));
                }
                meet();
                if (ok)
                    for (int idx = st_id; idx < rows * 8; idx += 256) {
                        const int rr = idx >> 3, c = idx & 7, rg = r0 + rr, rnode = rg / a.G;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (rnode < live_nodes) {
#pragma unroll
                            for (int x = 0; x < F::STREAMS; ++x) {
                                const uint4 u = lds128(base + (x * F::ROWS + rr) * 128 + ((c ^ (rr & 7)) << 4));
                                v.x += __uint_as_float(u.x); v.y += __uint_as_float(u.y); v.z += __uint_as_float(u.z); v.w += __uint_as_float(u.w);
                            }
                        }
                        if (whole) {
                            const __nv_bfloat162 p0 = __floats2bfloat162_rn(v.x, v.y), p1 = __floats2bfloat162_rn(v.z, v.w);
                            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + rnode) * a.Hq + kvh * a.G + rg % a.G) * HD;
                            reinterpret_cast<uint2*>(out + ch * 32)[c] = make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
                        } else if (rnode < live_nodes) {
                            reinterpret_cast<float4*>(part + (size_t)rr * HD + ch * 32)[c] = v;
                        }
                    }
                meet();
            }
            const bool owner = st_id < F::ROWS && st_id < rows;         // of row r in the results
            if (!whole && owner)
                reinterpret_cast<float2*>(part + (size_t)F::ROWS * HD)[st_id] = live && ok && ns > 0 ? make_float2(m, sum) : make_float2(-INFINITY, 0.f);
            if ((blk.bad[0] | blk.bad[1] | blk.bad[2] | blk.bad[3]) != 0u) {         // rare: what is no finite number, for the rows that see it
                if (owner && live && ok)
                    for (int u = 0; u < now_n; ++u) {
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
                meet();
                if (st_id < 4) blk.bad[st_id] = 0u;
            }
            if (st_id == 0) {
                blk.bad_tree = 0;
                blk.stop = blk.abort;
            }
            meet();
            if (*reinterpret_cast<volatile int*>(&blk.stop)) break;
        }
    }
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    __syncwarp();
    if (warp == WARP_MMA0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

// Joins the parts of heads that several CTAs have worked on, a warp a row: their sums at their common maximum.  Rows of sequences
// without nodes are written here too where the batch is cut into shares.  grid (B * Hkv * groups, rows / 32)
template <int HD>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ Share sh, int piece_rows) {
    __shared__ Block blk;
    const int hgs = a.Hkv * sh.groups, b = blockIdx.x / hgs, hg = blockIdx.x % hgs, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_trigger();
    int c0 = 0, parts = a.n_splits;
    if (sh.ctas) {
        if (warp == 0) scan_batch(a, blk, false);
        __syncthreads();
        const int stages = blk.before[b + 1] - blk.before[b];
        const long long all = (long long)blk.before[kMaxShared] * hgs, first = (long long)blk.before[b] * hgs + hg * stages;
        parts = 0;
        if (stages > 0) {
            // the last CTA whose share begins at or before a stage has it
            c0 = (int)(((first + 1) * sh.ctas - 1) / all);
            parts = (int)(((first + stages) * sh.ctas - 1) / all) - c0 + 1;
            if (parts == 1) return;         // written by its CTA
        }
    }
    const size_t stride = (size_t)piece_rows * (HD + 2);
    constexpr int V = HD / 32;              // columns of a lane
    // part i: where, and whether there is one (a share may be empty where there are fewer stages than CTAs)
    auto part_of = [&](int i) -> const float* {
        if (!sh.ctas) return a.part + ((size_t)blockIdx.x * a.n_splits + i) * stride;
        if (share_begin(blk, a, sh, c0 + i) == share_begin(blk, a, sh, c0 + i + 1)) return nullptr;
        return a.part + ((size_t)(c0 + i) * 2 + (i == 0)) * stride;
    };
    for (int e = 0; e < 4; ++e) {
        const int rr = blockIdx.y * 32 + warp * 4 + e, r = hg % sh.groups * piece_rows + rr;
        if (rr >= piece_rows || r >= a.R) return;
        float m = -INFINITY;
        for (int i = lane; i < parts; i += 32) {
            const float* p = part_of(i);
            const float2 v = p ? __ldcg(reinterpret_cast<const float2*>(p + (size_t)piece_rows * HD) + rr) : make_float2(-INFINITY, 0.f);
            if (v.y != 0.f) m = fmaxf(m, v.x);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float l = 0.f, acc[V];
#pragma unroll
        for (int c = 0; c < V; ++c) acc[c] = 0.f;
        for (int i0 = 0; i0 < parts; i0 += 32) {
            const float* mine = i0 + lane < parts ? part_of(i0 + lane) : nullptr;
            const float2 v = mine ? __ldcg(reinterpret_cast<const float2*>(mine + (size_t)piece_rows * HD) + rr) : make_float2(-INFINITY, 0.f);
            const float w = v.y != 0.f ? exp2f(v.x - m) : 0.f;
            l = fmaf(w, v.y, l);
            uint32_t have = __ballot_sync(0xffffffffu, v.y != 0.f);         // a part that has seen nothing has no O
            while (have) {
                float x[4][V], ws[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = have ? __ffs(have) - 1 : 0;
                    ws[j] = __shfl_sync(0xffffffffu, w, i);
                    const float* p = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), i));
                    if (!have) ws[j] = 0.f;
#pragma unroll
                    for (int c = 0; c < V; ++c) x[j][c] = 0.f;
                    if (have) {
                        if constexpr (V == 4) {
                            const float4 f = __ldcg(reinterpret_cast<const float4*>(p + (size_t)rr * HD) + lane);
                            x[j][0] = f.x; x[j][1] = f.y; x[j][2] = f.z; x[j][3] = f.w;
                        } else {
                            const float2 f = __ldcg(reinterpret_cast<const float2*>(p + (size_t)rr * HD) + lane);
                            x[j][0] = f.x; x[j][1] = f.y;
                        }
                    }
                    have &= have - 1;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < V; ++c) acc[c] = fmaf(ws[j], x[j][c], acc[c]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const int kvh = hg / sh.groups;
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (((size_t)b * a.T + r / a.G) * a.Hq + kvh * a.G + r % a.G) * HD;
        if constexpr (V == 4) {
            const __nv_bfloat162 p0 = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv), p1 = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
            reinterpret_cast<uint2*>(out)[lane] = make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
        } else {
            reinterpret_cast<__nv_bfloat162*>(out)[lane] = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv);
        }
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

template <int HD, Mode MODE>
static int launch(grl_device* dev, const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, const Share& sh) {
    using F = Form<HD, MODE>;
    static bool attr_set[64] = {};
    if (!attr_set[dev->ordinal & 63]) {      // a function attribute belongs to the device that was current
        GRL_CUDA(cudaFuncSetAttribute(tree_sm100_kernel<HD, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::TOTAL));
        attr_set[dev->ordinal & 63] = true;
    }
    const dim3 grid = sh.ctas ? dim3(sh.ctas) : dim3(a.n_splits, a.Hkv * sh.groups, a.B);
    GRL_CUDA(launch_pdl(tree_sm100_kernel<HD, MODE>, grid, kThreads, F::TOTAL, dev->stream, tk, tv, a, sh));
    GRL_LAUNCHED("tree_sm100_kernel");
    if (!sh.ctas && a.n_splits == 1) return GRL_OK;
    GRL_CUDA(launch_pdl(tree_join_kernel<HD>, dim3(a.B * a.Hkv * sh.groups, (F::ROWS + 31) / 32), 256, 0, dev->stream, a, sh, F::ROWS));
    GRL_LAUNCHED("tree_join_kernel");
    return GRL_OK;
}

static Mode mode_of(int R) { return R > BM ? PAIR : R > 64 ? SPLIT : FOLD; }
static int piece_rows(Mode m) { return m == PAIR ? 256 : m == SPLIT ? 128 : 64; }

}  // namespace tree

// asked: the caller's number of splits, or 0.
TreeTensorPlan tree_sm100_plan(const grl_device* dev, int B, int Hkv, int R, int D, int longest, int capacity, int asked) {
    using namespace tree;
    const int rows = piece_rows(mode_of(R)), groups = (R + rows - 1) / rows, sms = dev->prop.multiProcessorCount;
    const long long heads = (long long)B * Hkv * groups, stages = (longest + BN - 1) / BN;
    TreeTensorPlan p{};
    p.groups = groups;
    const size_t part = sizeof(float) * (size_t)rows * (D + 2);
    if (asked > 0 || B > kMaxShared || heads * (capacity / BN + 1) >= (1LL << 31)) {
        long long s = asked > 0 ? asked : sms / heads;
        if (asked <= 0 && s > stages / 2) s = stages / 2;
        p.splits = (int)(s < 1 ? 1 : s > 4096 ? 4096 : s);
        p.workspace = p.splits == 1 ? 0 : part * heads * p.splits;
        return p;
    }
    // equal shares of at least two stages a CTA
    const long long ctas = (heads * stages + 1) / 2;
    p.splits = 1;
    p.ctas = (int)(ctas < 1 ? 1 : ctas < sms ? ctas : sms);
    p.workspace = part * 2 * p.ctas;
    return p;
}

int tree_sm100_launch(grl_device* dev, const TreeArgs& a, const TreeTensorPlan& plan) {
    using namespace tree;
    CUtensorMap tk, tv;
    int rc = make_pool_map(dev, &tk, a.k_pages, a);
    if (!rc) rc = make_pool_map(dev, &tv, a.v_pages, a);
    if (rc) return rc;
    const Share sh{plan.ctas, plan.groups};
    const Mode mode = mode_of(a.R);
    if (a.D == 128)
        return mode == PAIR ? launch<128, PAIR>(dev, tk, tv, a, sh) : mode == SPLIT ? launch<128, SPLIT>(dev, tk, tv, a, sh) : launch<128, FOLD>(dev, tk, tv, a, sh);
    return mode == PAIR ? launch<64, PAIR>(dev, tk, tv, a, sh) : mode == SPLIT ? launch<64, SPLIT>(dev, tk, tv, a, sh) : launch<64, FOLD>(dev, tk, tv, a, sh);
}

}  // namespace grl
