// A drafted step's rows in the paged cache: the append that normalises and rotates them on the way, and the keeping of the accepted path.
#include "qk_norm.cuh"
#include "tree.cuh"

namespace grl {

struct AppendNormArgs {
    void* k_pages;
    void* v_pages;
    const int32_t* block_table;
    int32_t* seq_lens;
    const void* k_new;
    const void* v_new;
    const void* q_in;
    void* q_out;
    long long ks, vs, qs;       // token strides in elements
    const float* q_weight;
    const float* k_weight;
    const int32_t* pos_offsets;
    const int32_t* parents;
    const int32_t* n_nodes;
    int32_t* status;
    int B, Hkv, Hq, D, P, max_pages, num_pages, n_new, pos_base, update_lens;
    float eps;
    RopeArgs rope;
};

// Whether sequence b's nodes fit; the whole CTA calls it.  Every CTA of a sequence comes to the same answer, before any row is stored.
__device__ __forceinline__ bool append_fits(const AppendNormArgs& a, int b, int len0, int n) {
    const bool tell = threadIdx.x == 0 && blockIdx.x == 0;
    if (n < 0 || n > a.n_new) {
        if (tell) tree_fail(a.status, TREE_BAD_COUNT, b, n);
        return false;
    }
    if (len0 < 0 || (long long)len0 + n > (long long)a.max_pages * a.P) {
        if (tell) tree_fail(a.status, TREE_BAD_LENGTH, b, len0);
        return false;
    }
    bool bad = false;
    if (n > 0)
        for (int i = len0 / a.P + threadIdx.x; i <= (len0 + n - 1) / a.P; i += blockDim.x)
            bad |= (unsigned)a.block_table[(size_t)b * a.max_pages + i] >= (unsigned)a.num_pages;
    if (__syncthreads_or(bad)) {
        if (tell) tree_fail(a.status, TREE_BAD_PAGE, b, len0);
        return false;
    }
    return true;
}

// The parent of node threadIdx.x, asked for beside the sequence's numbers.
__device__ __forceinline__ int parent_of(const AppendNormArgs& a, int b) {
    return a.parents && (int)threadIdx.x < a.n_new ? a.parents[(size_t)b * a.n_new + threadIdx.x] : -1;
}

// grid (CTAs of a sequence, B); a warp takes a row at a time: the Hkv keys, the Hkv values and the Hq queries of a node.  With update_lens
// there is one CTA a sequence.
template <typename TIn, typename TC, typename TQ>
__global__ void __launch_bounds__(256) append_norm_rows_kernel(const __grid_constant__ AppendNormArgs a) {
    __shared__ TreeMasks masks;
    const int b = blockIdx.y, lane = threadIdx.x & 31, pairs = a.D / 2;
    pdl_wait();
    pdl_trigger();
    const int len0 = a.seq_lens[b], n = tree_count(a.n_nodes, a.n_new, b), parent = parent_of(a, b);
    bool ok = append_fits(a, b, len0, n);
    if (ok && a.parents && !tree_masks(masks, parent, n)) {
        if (threadIdx.x == 0 && blockIdx.x == 0) tree_fail(a.status, TREE_BAD_PARENT, b, n);
        ok = false;
    }
    const int live = ok ? n : 0, pos0 = a.pos_base + (a.pos_offsets ? a.pos_offsets[b] : 0) + len0;
    const int rows = 2 * a.Hkv + (a.q_in ? a.Hq : 0), warps = gridDim.x * (blockDim.x >> 5);
    for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < (long long)a.n_new * rows; item += warps) {
        const int t = (int)(item / rows), hs = (int)(item % rows);
        const size_t tok = (size_t)b * a.n_new + t;
        const int kind = hs < a.Hkv ? 0 : hs < 2 * a.Hkv ? 1 : 2, h = kind == 0 ? hs : kind == 1 ? hs - a.Hkv : hs - 2 * a.Hkv;
        TQ* q_out = reinterpret_cast<TQ*>(a.q_out) + (tok * a.Hq + h) * a.D;
        if (t >= live) {
            if (kind == 2)
                for (int d = lane; d < a.D; d += 32) store_from_float<TQ>(q_out + d, 0.f);
            continue;
        }
        const int at = len0 + t;
        const size_t dst = kind == 2 ? 0 : (((size_t)a.block_table[(size_t)b * a.max_pages + at / a.P] * a.Hkv + h) * a.P + at % a.P) * a.D;
        const TIn* x = reinterpret_cast<const TIn*>(kind == 0 ? a.k_new : kind == 1 ? a.v_new : a.q_in) +
                       tok * (kind == 0 ? a.ks : kind == 1 ? a.vs : a.qs) + (size_t)h * a.D;
        if (kind == 1) {
            for (int d = lane; d < a.D; d += 32) store_from_float<TC>(reinterpret_cast<TC*>(a.v_pages) + dst + d, load_as_float<TIn>(x + d));
            continue;
        }
        const int pos = pos0 + (a.parents ? mask_depth(masks.seen[t]) : t);
        const float* w = kind ? a.q_weight : a.k_weight;
        float x0[4], x1[4], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = lane + 32 * e;
            x0[e] = x1[e] = 0.f;
            if (j < pairs) {
                int d0, d1;
                pair_place(a.rope, j, &d0, &d1);
                x0[e] = load_as_float<TIn>(x + d0);
                x1[e] = load_as_float<TIn>(x + d1);
            }
            sum = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], sum));
        }
        const float r = rsqrtf(warp_sum(sum) / (float)a.D + a.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = lane + 32 * e;
            if (j < pairs) {
                int d0, d1;
                float c, s;
                pair_place(a.rope, j, &d0, &d1);
                pair_angle(a.rope, j, pos, &c, &s);
                const float n0 = x0[e] * r * (w ? w[d0] : 1.f), n1 = x1[e] * r * (w ? w[d1] : 1.f);
                if (kind == 0) {
                    TC* kp = reinterpret_cast<TC*>(a.k_pages) + dst;
                    store_from_float<TC>(kp + d0, n0 * c - n1 * s);
                    store_from_float<TC>(kp + d1, n0 * s + n1 * c);
                } else {
                    store_from_float<TQ>(q_out + d0, n0 * c - n1 * s);
                    store_from_float<TQ>(q_out + d1, n0 * s + n1 * c);
                }
            }
        }
    }
    if (a.update_lens && ok) {
        __syncthreads();        // every thread has read the length
        if (threadIdx.x == 0) a.seq_lens[b] = len0 + n;
    }
}

// Rows of whole 8-element pieces on 16-byte boundaries: the form of qk_norm_kernel (qk_norm.cu).  A node's rows are its Hkv keys, Hkv values and
// Hq queries; a warp's first rows are on their way while the sequence's numbers are read and checked.
// 4 x 2048 tokens, 32 + 8 + 8 heads of 128: 41 us, HBM at 4.9 TB/s; 261 with a warp a row.  7 x 12 nodes: 5 us, latency.
template <typename T> constexpr int kRunOf = sizeof(T) == 2 ? 4 : 2;
template <typename TIn, typename TC, typename TQ, int LANES, bool HALF, bool FULL>
__global__ void __launch_bounds__(256, 3) append_norm_kernel(const __grid_constant__ AppendNormArgs a) {
    constexpr int RUN = kRunOf<TIn>, GPW = 32 / LANES;
    __shared__ TreeMasks masks;
    __shared__ __align__(16) RowTables tables;
    const int seq = blockIdx.y, l = threadIdx.x % LANES, g = (threadIdx.x & 31) / LANES, D = FULL ? 8 * LANES : a.D;
    const bool on = FULL || 8 * l < D;
    const float inv_d = 1.f / D;
    const RowPlace at = row_place<HALF>(l, FULL ? D : a.rope.rd);
    const int gap = FULL && HALF ? 4 * LANES : at.gap();
    const int slots = 2 * a.Hkv + a.Hq;
    const Share share((long long)a.n_new * slots, blockIdx.x, gridDim.x);
    int t = (int)(share.lo / slots), slot = (int)(share.lo - (long long)t * slots), left = share.items;
    RowRaw<TIn> raw[RUN];
    const TIn* in = nullptr;
    int kind = 0, h0 = 0, n = 0;        // the segment: keys, values or queries, its first head, its rows
    auto aim = [&] {
        kind = slot < a.Hkv ? 0 : slot < 2 * a.Hkv ? 1 : 2;
        h0 = slot - kind * a.Hkv;
        n = min(left, (kind == 2 ? a.Hq : a.Hkv) - h0);
        in = reinterpret_cast<const TIn*>(kind == 0 ? a.k_new : kind == 1 ? a.v_new : a.q_in) +
             (((long long)seq * a.n_new + t) * (kind == 0 ? a.ks : kind == 1 ? a.vs : a.qs) + (h0 + g) * D + at.o0);
#pragma unroll
        for (int h = 0; h < RUN; ++h)
            if (on && g + GPW * h < n) row_fetch<HALF>(in + GPW * h * D, gap, raw[h]);
            else row_zero(raw[h]);
    };
    pdl_wait();
    pdl_trigger();
    if (left > 0) aim();
    const int len0 = a.seq_lens[seq], count = tree_count(a.n_nodes, a.n_new, seq), offset = a.pos_offsets ? a.pos_offsets[seq] : 0, parent = parent_of(a, seq);
    row_tables(tables, a.rope, D, a.q_weight, a.k_weight);
    bool ok = append_fits(a, seq, len0, count);
    if (ok && a.parents && !tree_masks(masks, parent, count)) {
        if (threadIdx.x == 0 && blockIdx.x == 0) tree_fail(a.status, TREE_BAD_PARENT, seq, count);
        ok = false;
    }
    __syncthreads();
    const int nodes = ok ? count : 0, pos0 = a.pos_base + offset + len0;
    Pairs angle;
    bool fresh = true;
    size_t row = 0;         // of the node in the pools, for kv head 0
    for (bool first = true; left > 0; first = false) {
        if (!first) aim();
        const bool node = t < nodes;
        if (fresh && node) {
            const int place = len0 + t;
            row = ((size_t)a.block_table[(size_t)seq * a.max_pages + place / a.P] * a.Hkv * a.P + place % a.P) * D;
            angle = row_angles(tables, l, a.rope.gain, at.turned, pos0 + (a.parents ? mask_depth(masks.seen[t]) : t));
            fresh = false;
        }
        Turn turn;
        if (kind != 1) turn = weighted_turn(row_weights<HALF>(tables.w[kind != 2], at), angle);
        TQ* q_at = reinterpret_cast<TQ*>(a.q_out) + (((long long)seq * a.n_new + t) * a.Hq + h0 + g) * D + at.o0;
        TC* kv_at = reinterpret_cast<TC*>(kind ? a.v_pages : a.k_pages) + row + (long long)(h0 + g) * a.P * D + at.o0;
        const int kv_step = GPW * a.P * D;
        for (int i = g; i < n + g; i += GPW * RUN) {
            in += RUN * GPW * D;
#pragma unroll
            for (int h = 0; h < RUN; ++h) {
                Pairs x = row_pairs<HALF>(raw[h]);
                if (on && i + GPW * (RUN + h) < n) row_fetch<HALF>(in + GPW * h * D, gap, raw[h]);
                if (kind != 1) {
                    const float r = rsqrtf(row_sum<LANES>(squares(x)) * inv_d + a.eps);
                    turn_scaled(x, turn, r);
                }
                if (on && i + GPW * h < n) {
                    if (kind == 2) {
                        if (!node) x.f[0] = x.f[1] = x.g[0] = x.g[1] = make_float2(0.f, 0.f);
                        row_store<HALF>(q_at + GPW * h * D, gap, x);
                    } else if (node) {
                        row_store<HALF>(kv_at + (long long)h * kv_step, gap, x);
                    }
                }
            }
            q_at += RUN * GPW * D;
            kv_at += (long long)RUN * kv_step;
        }
        slot += n;
        left -= n;
        if (slot == slots) {
            slot = 0;
            ++t;
            fresh = true;
        }
    }
    if (a.update_lens && ok) {
        __syncthreads();        // every thread has read the length
        if (threadIdx.x == 0) a.seq_lens[seq] = len0 + count;
    }
}

template <typename TIn, typename TC, typename TQ, int LANES>
static void (*append_form_instance(bool half, bool full))(AppendNormArgs) {
    return half ? (full ? append_norm_kernel<TIn, TC, TQ, LANES, true, true> : append_norm_kernel<TIn, TC, TQ, LANES, true, false>)
                : (full ? append_norm_kernel<TIn, TC, TQ, LANES, false, true> : append_norm_kernel<TIn, TC, TQ, LANES, false, false>);
}
template <typename TIn, typename TC, typename TQ>
static void (*append_instance(bool fast, int D, int rd, bool half))(AppendNormArgs) {
    const bool full = row_full(D, rd);
    return !fast ? append_norm_rows_kernel<TIn, TC, TQ> : D <= 32 ? append_form_instance<TIn, TC, TQ, 4>(half, full)
         : D <= 64 ? append_form_instance<TIn, TC, TQ, 8>(half, full) : D <= 128 ? append_form_instance<TIn, TC, TQ, 16>(half, full)
                                                                                : append_form_instance<TIn, TC, TQ, 32>(half, full);
}
template <typename TIn>
static void (*append_norm_instance(bool cache32, bool q32, bool fast, int D, int rd, bool half))(AppendNormArgs) {
    return cache32 ? (q32 ? append_instance<TIn, float, float>(fast, D, rd, half) : append_instance<TIn, float, __nv_bfloat16>(fast, D, rd, half))
                   : (q32 ? append_instance<TIn, __nv_bfloat16, float>(fast, D, rd, half) : append_instance<TIn, __nv_bfloat16, __nv_bfloat16>(fast, D, rd, half));
}

struct CommitArgs {
    uint8_t* k_pages;
    uint8_t* v_pages;
    const int32_t* block_table;
    const int32_t* seq_lens;
    const int32_t* path;
    const int32_t* n_path;
    const int32_t* n_nodes;
    int32_t* lens_out;
    int32_t* status;
    float* cum_score;
    uint8_t* tombstone;
    float* relevance;
    int Hkv, P, max_pages, num_pages, max_path, n_tree, row_bytes, capacity;
};

// One CTA a sequence, its threads as groups of whole rows (key or value, kv head, piece).  Row i comes from row path[i] >= i, and later rows from further
// up: a round of rows is read into registers, then written, and no round reads what one before has written.  Latency-bound (the lengths, the path and the
// pages, then the rows), so that a round takes as many rows as its threads hold: 32 sequences
// of 24 nodes behind their append 16.7 us, 20 where a thread walked up its path a row at a time.
constexpr int kCommitThreads = 1024, kCommitHold = 8;
template <typename Piece>
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const __grid_constant__ CommitArgs a) {
    const int b = blockIdx.x, tid = threadIdx.x;
    pdl_wait();
    pdl_trigger();
    const int32_t* path = a.path + (size_t)b * a.max_path;
    const int32_t* table = a.block_table + (size_t)b * a.max_pages;
    const int mine = tid < a.max_path ? path[tid] : 0, before = tid > 0 && tid < a.max_path ? path[tid - 1] : -1;      // beside the sequence's numbers
    const int len = a.seq_lens[b], n = tree_count(a.n_nodes, a.n_tree, b), m = a.n_path[b], prefix = len - n;
    int what = 0;
    if (n < 0 || n > a.n_tree) what = TREE_BAD_COUNT;
    else if (prefix < 0 || len > a.max_pages * a.P) what = TREE_BAD_LENGTH;
    else if (m < 0 || m > n || m > a.max_path) what = TREE_BAD_PATH;
    if (!what) {
        bool bad = tid < m && (mine < 0 || mine >= n || before >= mine), lost = false;
        for (int i = tid + kCommitThreads; i < m; i += kCommitThreads) {
            const int t = path[i];
            bad |= t < 0 || t >= n || path[i - 1] >= t;
        }
        if (n > 0)
            for (int i = prefix / a.P + tid; i <= (len - 1) / a.P; i += kCommitThreads) lost |= (unsigned)table[i] >= (unsigned)a.num_pages;
        const int any_bad = __syncthreads_or(bad), any_lost = __syncthreads_or(lost);
        what = any_bad ? TREE_BAD_PATH : any_lost ? TREE_BAD_PAGE : 0;
    }
    if (what) {
        if (tid == 0) {
            tree_fail(a.status, what, b, what == TREE_BAD_COUNT ? n : what == TREE_BAD_PATH ? m : len);
            a.lens_out[b] = len;
        }
        return;
    }
    const int pieces = a.row_bytes / (int)sizeof(Piece), all = 2 * a.Hkv * pieces;
    for (int c0 = 0; c0 < all; c0 += kCommitThreads) {
        const int wide = min(kCommitThreads, all - c0), groups = kCommitThreads / wide, group = tid / wide, c = c0 + tid % wide;
        const int piece = c % pieces, h = c / pieces % a.Hkv;
        uint8_t* pool = c / pieces / a.Hkv ? a.v_pages : a.k_pages;
        const auto place = [&](int t) {
            const int at = prefix + t;
            return reinterpret_cast<Piece*>(pool + (((size_t)table[at / a.P] * a.Hkv + h) * a.P + at % a.P) * a.row_bytes) + piece;
        };
        for (int i0 = 0; i0 < m; i0 += groups * kCommitHold) {
            Piece held[kCommitHold];
            uint32_t moves = 0;
#pragma unroll
            for (int k = 0; k < kCommitHold; ++k) {
                const int i = i0 + k * groups + group;
                if (group < groups && i < m) {
                    const int from = path[i];
                    if (from != i) {
                        moves |= 1u << k;
                        held[k] = *place(from);
                    }
                }
            }
            if (groups > 1) __syncthreads();        // else a thread meets its own pieces only
#pragma unroll
            for (int k = 0; k < kCommitHold; ++k)
                if (moves >> k & 1u) *place(i0 + k * groups + group) = held[k];
        }
    }
    if (a.cum_score) {
        const size_t base = (size_t)b * a.capacity + prefix;
        for (int i0 = 0; i0 < n; i0 += kCommitThreads) {
            const int i = i0 + tid;
            const bool kept = i < m;
            const int from = kept ? path[i] : 0;
            const float cum = kept ? a.cum_score[base + from] : 0.f, rel = kept && a.relevance ? a.relevance[base + from] : 0.f;
            const uint8_t tomb = kept ? a.tombstone[base + from] : 0;
            __syncthreads();
            if (i < n) {
                a.cum_score[base + i] = cum;
                a.tombstone[base + i] = tomb;
                if (a.relevance) a.relevance[base + i] = rel;
            }
            __syncthreads();
        }
    }
    __syncthreads();
    if (tid == 0) a.lens_out[b] = prefix + m;
}

// seq_lens += nodes of the sequences that the append has taken: it raises no flag of its own, so the conditions are formed again.
__global__ void advance_nodes_kernel(const __grid_constant__ AppendNormArgs a) {
    __shared__ TreeMasks masks;
    const int b = blockIdx.x, len0 = a.seq_lens[b], n = tree_count(a.n_nodes, a.n_new, b);
    bool ok = append_fits(a, b, len0, n);
    if (ok && a.parents) ok = tree_masks(masks, parent_of(a, b), n);
    __syncthreads();
    if (ok && threadIdx.x == 0) a.seq_lens[b] = len0 + n;
}

static int check_append(const grl_append_norm_params* p, AppendNormArgs* a) {
    GRL_REQUIRE(p, "params is NULL");
    const grl_kv_layout& kv = p->kv;
    int rc = check_tree_layout(kv);
    if (rc) return rc;
    GRL_REQUIRE(p->k_new && p->v_new, "k_new / v_new is NULL");
    GRL_REQUIRE(!p->q_in || (p->q_out && p->num_q_heads > 0), "q_in given without q_out / num_q_heads");
    GRL_REQUIRE(p->in_dtype == GRL_F32 || p->in_dtype == GRL_BF16, "in_dtype must be GRL_F32 or GRL_BF16");
    GRL_REQUIRE(!p->q_in || p->q_out_dtype == GRL_F32 || p->q_out_dtype == GRL_BF16, "q_out_dtype must be GRL_F32 or GRL_BF16");
    GRL_REQUIRE(p->n_new > 0, "n_new must be positive");
    GRL_REQUIRE(!p->parents || p->n_new <= GRL_MAX_TREE, "a tree has at most %d nodes, got %d", GRL_MAX_TREE, p->n_new);
    GRL_REQUIRE(p->eps >= 0.f, "eps must not be negative");
    GRL_REQUIRE(p->k_token_stride >= 0 && p->v_token_stride >= 0 && p->q_token_stride >= 0, "strides must not be negative");
    rc = check_rope_spec(p->rope, kv.head_dim, &a->rope);
    if (rc) return rc;
    a->k_pages = kv.k_pages; a->v_pages = kv.v_pages; a->block_table = kv.block_table; a->seq_lens = kv.seq_lens;
    a->k_new = p->k_new; a->v_new = p->v_new; a->q_in = p->q_in; a->q_out = p->q_out;
    a->q_weight = p->q_weight; a->k_weight = p->k_weight;
    a->pos_offsets = p->pos_offsets; a->parents = p->parents; a->n_nodes = p->n_nodes;
    a->B = kv.batch; a->Hkv = kv.num_kv_heads; a->Hq = p->q_in ? p->num_q_heads : 0; a->D = kv.head_dim; a->P = kv.page_tokens;
    a->max_pages = kv.max_pages; a->num_pages = pool_pages(kv); a->n_new = p->n_new; a->pos_base = p->pos_base;
    a->ks = p->k_token_stride ? p->k_token_stride : (long long)a->Hkv * a->D;
    a->vs = p->v_token_stride ? p->v_token_stride : (long long)a->Hkv * a->D;
    a->qs = p->q_token_stride ? p->q_token_stride : (long long)a->Hq * a->D;
    a->eps = p->eps == 0.f ? 1e-6f : p->eps;
    return GRL_OK;
}

}  // namespace grl

using namespace grl;

extern "C" {

int grl_kv_append_norm(grl_device* dev, const grl_append_norm_params* p) {
    AppendNormArgs a{};
    int rc = check_append(p, &a);
    if (rc) return rc;
    GRL_REQUIRE(dev, "dev is NULL");
    DeviceGuard g(dev->ordinal);
    fill_rope_freq(dev, p->rope, &a.rope);
    a.status = dev->d_status;
    dev->status_dirty = true;
    const bool fast = a.D % 8 == 0 && a.rope.rd % 8 == 0 && a.P < (1 << 16) && row_aligned(a.k_new, p->in_dtype, &a.ks, 1) && row_aligned(a.v_new, p->in_dtype, &a.vs, 1) &&
                      (!a.q_in || row_aligned(a.q_in, p->in_dtype, &a.qs, 1)) &&
                      ((uintptr_t)a.q_out | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages) % 16 == 0;
    // a CTA for two rows of each of its groups (a row of each warp in the other form), as many as the SMs hold at once
    const long long rows = (long long)a.n_new * (2 * a.Hkv + a.Hq), per = fast ? 2 * 256 / row_lanes(a.D) : 8;
    const long long need = (rows + per - 1) / per, most = ((fast ? 3LL : 8LL) * dev->prop.multiProcessorCount + a.B - 1) / a.B;
    int ctas = (int)(need < most ? need : most);
    const bool fused = p->update_lens && ctas <= 4;
    if (fused) ctas = 1;
    a.update_lens = fused ? 1 : 0;
    const bool half = p->rope.mode == GRL_ROPE_HALF;
    auto kernel = p->in_dtype == GRL_F32 ? append_norm_instance<float>(p->kv.cache_dtype == GRL_F32, p->q_out_dtype == GRL_F32, fast, a.D, a.rope.rd, half)
                                         : append_norm_instance<__nv_bfloat16>(p->kv.cache_dtype == GRL_F32, p->q_out_dtype == GRL_F32, fast, a.D, a.rope.rd, half);
    GRL_CUDA(launch_pdl(kernel, dim3(ctas, a.B), 256, 0, dev->stream, a));
    GRL_LAUNCHED("append_norm_kernel");
    if (p->update_lens && !fused) {
        advance_nodes_kernel<<<a.B, GRL_MAX_TREE, 0, dev->stream>>>(a);
        GRL_LAUNCHED("advance_nodes_kernel");
    }
    return GRL_OK;
}

int grl_kv_commit(grl_device* dev, const grl_commit_params* p) {
    GRL_REQUIRE(p, "params is NULL");
    const grl_kv_layout& kv = p->kv;
    int rc = check_tree_layout(kv);
    if (rc) return rc;
    GRL_REQUIRE(p->path && p->n_path, "path or n_path is NULL");
    GRL_REQUIRE(p->max_path > 0 && p->n_tree > 0, "max_path and n_tree must be positive");
    CommitArgs a{};
    if (p->meta) {
        GRL_REQUIRE(p->meta->cum_score && p->meta->tombstone, "NULL metadata buffer");
        GRL_REQUIRE(p->meta->capacity >= kv.max_pages * kv.page_tokens, "metadata capacity %d below the cache's %d tokens", p->meta->capacity,
                    kv.max_pages * kv.page_tokens);
        a.cum_score = p->meta->cum_score; a.tombstone = p->meta->tombstone; a.relevance = p->meta->relevance;
        a.capacity = p->meta->capacity;
    }
    GRL_REQUIRE(dev, "dev is NULL");
    a.k_pages = static_cast<uint8_t*>(kv.k_pages); a.v_pages = static_cast<uint8_t*>(kv.v_pages);
    a.block_table = kv.block_table; a.seq_lens = kv.seq_lens;
    a.path = p->path; a.n_path = p->n_path; a.n_nodes = p->n_nodes;
    a.lens_out = p->lens_out ? p->lens_out : kv.seq_lens;
    a.status = dev->d_status;
    a.Hkv = kv.num_kv_heads; a.P = kv.page_tokens; a.max_pages = kv.max_pages; a.num_pages = pool_pages(kv);
    a.max_path = p->max_path; a.n_tree = p->n_tree;
    a.row_bytes = kv.head_dim * (kv.cache_dtype == GRL_BF16 ? 2 : 4);
    DeviceGuard g(dev->ordinal);
    dev->status_dirty = true;
    // 16-byte pieces where rows lie so, else 4-byte ones (head_dim is even)
    const bool wide = a.row_bytes % 16 == 0 && ((uintptr_t)a.k_pages | (uintptr_t)a.v_pages) % 16 == 0;
    GRL_REQUIRE(wide || ((uintptr_t)a.k_pages | (uintptr_t)a.v_pages) % 4 == 0, "page pools must be 4-byte aligned");
    GRL_CUDA(launch_pdl(wide ? commit_kernel<uint4> : commit_kernel<uint32_t>, dim3(kv.batch), kCommitThreads, 0, dev->stream, a));
    GRL_LAUNCHED("commit_kernel");
    return GRL_OK;
}

}  // extern "C"
