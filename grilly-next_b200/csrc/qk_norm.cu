// Query and key heads normalised (root mean square, learned weight) and rotated in one pass, and the gradients of that.
#include "qk_norm.cuh"

namespace grl {

struct NormSide {
    const void* x;
    void* y;            // forward: the result; backward: the gradient of the inputs
    const void* dy;     // backward: the gradient of the result
    const float* w;
    float* dw;
    long long xs[3], ys[3], dys[3];     // strides in elements: sequence, token, head
    int H;
};
struct NormArgs {
    NormSide q, k;
    int B, S, D;
    float eps;
    const int32_t* positions;
    int pos_base;
    float* part;        // backward: weight gradients of every CTA, [CTA][q, k][D]
    RopeArgs rope;
};

constexpr int kPairs = 4;       // pairs of a row that a lane holds: head_dim up to 256

__device__ __forceinline__ int position_of(const NormArgs& a, int b, int s) {
    return a.pos_base + (a.positions ? a.positions[(size_t)b * a.S + s] : s);
}

// Any head_dim, stride and alignment: a warp a row.
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(256) qk_norm_rows_kernel(const __grid_constant__ NormArgs a) {
    const int lane = threadIdx.x & 31, pairs = a.D / 2;
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    const int heads = a.q.H + a.k.H;
    const long long rows = (long long)a.B * a.S * heads;
    for (long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); row < rows; row += warps) {
        const int hs = (int)(row % heads);
        const long long tok = row / heads;
        const int s = (int)(tok % a.S), b = (int)(tok / a.S);
        const bool is_k = hs >= a.q.H;
        const NormSide& side = is_k ? a.k : a.q;
        const int h = is_k ? hs - a.q.H : hs;
        const TIn* x = reinterpret_cast<const TIn*>(side.x) + b * side.xs[0] + s * side.xs[1] + h * side.xs[2];
        TOut* y = reinterpret_cast<TOut*>(side.y) + b * side.ys[0] + s * side.ys[1] + h * side.ys[2];
        const int pos = position_of(a, b, s);
        float x0[kPairs], x1[kPairs], sum = 0.f;
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
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
        for (int e = 0; e < kPairs; ++e) {
            const int j = lane + 32 * e;
            if (j < pairs) {
                int d0, d1;
                float c, sn;
                pair_place(a.rope, j, &d0, &d1);
                pair_angle(a.rope, j, pos, &c, &sn);
                const float n0 = x0[e] * r * (side.w ? side.w[d0] : 1.f), n1 = x1[e] * r * (side.w ? side.w[d1] : 1.f);
                store_from_float<TOut>(y + d0, n0 * c - n1 * sn);
                store_from_float<TOut>(y + d1, n0 * sn + n1 * c);
            }
        }
    }
}

// Rows of whole 8-element pieces on 16-byte boundaries: LANES threads a row, eight elements each (threads past the row's end idle).  Bound by HBM, each element read and
// written once.  A thread group keeps its places in the rows, walks the heads of a token in runs, the next run's loads on their
// way under the present one, and forms a token's angles (double precision) once for all of them; every group has an equal,
// contiguous share of all runs, and steps from run to run without dividing.
template <typename T> constexpr int kRunOf = sizeof(T) == 2 ? 4 : 2;      // rows of a run
struct RunWalk {
    int b, s, run;
    __device__ __forceinline__ void start(long long item, int S, int runs) {
        const long long tok = item / runs;
        run = (int)(item - tok * runs);
        b = (int)(tok / S);
        s = (int)(tok - (long long)b * S);
    }
    __device__ __forceinline__ void step(int S, int runs) {
        if (++run < runs) return;
        run = 0;
        if (++s < S) return;
        s = 0;
        ++b;
    }
};
template <typename TIn, typename TOut, int LANES, bool HALF>
__global__ void __launch_bounds__(256, 3) qk_norm_kernel(const __grid_constant__ NormArgs a) {
    constexpr int RUN = kRunOf<TIn>;
    __shared__ __align__(16) RowTables tables;
    const int l = threadIdx.x % LANES, D = a.D;
    const bool on = 8 * l < D;
    const float inv_d = 1.f / D;
    const RowPlace at = row_place<HALF>(l, a.rope.rd);
    const int q_runs = (a.q.H + RUN - 1) / RUN, runs = q_runs + (a.k.H + RUN - 1) / RUN;
    const long long total = (long long)a.B * a.S * runs, all = (long long)gridDim.x * (256 / LANES), mine = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const long long lo = mine * total / all;
    const int items = (int)((mine + 1) * total / all - lo), most = (int)((total + all - 1) / all);      // of the group; of any group: the
                                                                        // groups of a warp take the same trips, for the shuffles
    pdl_wait();
    pdl_trigger();
    RunWalk at_run;
    at_run.start(items > 0 ? lo : 0, a.S, runs);
    RowRaw<TIn> raw[RUN];
    auto fetch = [&](const RunWalk& w, bool live) {
        const bool is_k = w.run >= q_runs;
        const NormSide& side = is_k ? a.k : a.q;
        const int h0 = (is_k ? w.run - q_runs : w.run) * RUN, heads = live && on ? min(RUN, side.H - h0) : 0;
        const TIn* in = reinterpret_cast<const TIn*>(side.x) + w.b * side.xs[0] + w.s * side.xs[1] + h0 * side.xs[2];
#pragma unroll
        for (int h = 0; h < RUN; ++h)
            if (h < heads) row_fetch<HALF>(in + h * side.xs[2], at, raw[h]);
            else row_zero(raw[h]);
    };
    fetch(at_run, items > 0);
    row_tables<HALF>(tables, a.rope, D, a.q.w, a.k.w);
    __syncthreads();
    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
    bool fresh = true;          // a token whose angles are not formed yet
    for (int i = 0; i < most; ++i) {
        const RunWalk now = at_run;
        RowRaw<TIn> x_raw[RUN];
#pragma unroll
        for (int h = 0; h < RUN; ++h) x_raw[h] = raw[h];
        const bool live = i < items;
        at_run.step(a.S, runs);
        if (i + 1 < most) fetch(at_run, i + 1 < items);
        if (live && fresh) row_angles(tables, l, a.rope.gain, at.turned, position_of(a, now.b, now.s), c, s);
        fresh = at_run.run == 0;
        const bool is_k = now.run >= q_runs;
        const NormSide& side = is_k ? a.k : a.q;
        const int h0 = (is_k ? now.run - q_runs : now.run) * RUN, heads = live && on ? min(RUN, side.H - h0) : 0;
        TOut* out = reinterpret_cast<TOut*>(side.y) + now.b * side.ys[0] + now.s * side.ys[1] + h0 * side.ys[2];
        float w[8];
        row_weights(tables.w[is_k], at, w);
#pragma unroll
        for (int h = 0; h < RUN; ++h) {
            float x[8], sum = 0.f;
            row_unpack(x_raw[h], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
            const float r = rsqrtf(row_sum<LANES>(sum) * inv_d + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
            row_turn<HALF, false>(x, c, s, at.turned);
            if (h < heads) row_store<HALF>(out + h * side.ys[2], at, x);
        }
    }
}

// The backward pass in the same form, the queries and then the keys; a group keeps its share of the weight's gradient in registers, the CTA adds
// them in order of its groups.
template <typename T> constexpr int kGradRunOf = sizeof(T) == 2 ? 2 : 1;
template <typename TIn, typename TOut, int LANES, bool HALF>
__global__ void __launch_bounds__(256, 3) qk_norm_backward_kernel(const __grid_constant__ NormArgs a) {
    constexpr int GROUPS = 256 / LANES, RUN = kGradRunOf<TIn>;
    __shared__ __align__(16) RowTables tables;
    __shared__ __align__(16) float sm[GROUPS][8 * LANES];
    const int l = threadIdx.x % LANES, group = threadIdx.x / LANES, D = a.D;
    const bool on = 8 * l < D;
    const float inv_d = 1.f / D;
    const RowPlace at = row_place<HALF>(l, a.rope.rd);
    const long long all = (long long)gridDim.x * GROUPS, mine = (long long)blockIdx.x * GROUPS + group;
    pdl_wait();
    row_tables<HALF>(tables, a.rope, D, a.q.w, a.k.w);
    __syncthreads();
#pragma unroll 1
    for (int side_i = 0; side_i < 2; ++side_i) {
        const NormSide& side = side_i ? a.k : a.q;
        const int runs = (side.H + RUN - 1) / RUN;
        const long long total = (long long)a.B * a.S * runs, lo = mine * total / all;
        const int items = (int)((mine + 1) * total / all - lo), most = (int)((total + all - 1) / all);
        RunWalk at_run{0, 0, 0};
        if (items > 0) at_run.start(lo, a.S, runs);
        RowRaw<TIn> xr[RUN];
        RowRaw<TOut> gr[RUN];
        auto fetch = [&](const RunWalk& w, bool live) {
            const int h0 = w.run * RUN, heads = live && on ? min(RUN, side.H - h0) : 0;
            const TIn* in = reinterpret_cast<const TIn*>(side.x) + w.b * side.xs[0] + w.s * side.xs[1] + h0 * side.xs[2];
            const TOut* dy = reinterpret_cast<const TOut*>(side.dy) + w.b * side.dys[0] + w.s * side.dys[1] + h0 * side.dys[2];
#pragma unroll
            for (int h = 0; h < RUN; ++h)
                if (h < heads) {
                    row_fetch<HALF>(in + h * side.xs[2], at, xr[h]);
                    row_fetch<HALF>(dy + h * side.dys[2], at, gr[h]);
                } else {
                    row_zero(xr[h]);
                    row_zero(gr[h]);
                }
        };
        if (most > 0) fetch(at_run, items > 0);
        float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f}, acc[8], w[8];
        row_weights(tables.w[side_i], at, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        bool fresh = true;
        for (int i = 0; i < most; ++i) {
            const RunWalk now = at_run;
            RowRaw<TIn> xn[RUN];
            RowRaw<TOut> gn[RUN];
#pragma unroll
            for (int h = 0; h < RUN; ++h) { xn[h] = xr[h]; gn[h] = gr[h]; }
            const bool live = i < items;
            at_run.step(a.S, runs);
            if (i + 1 < most) fetch(at_run, i + 1 < items);
            if (live && fresh) row_angles(tables, l, a.rope.gain, at.turned, position_of(a, now.b, now.s), c, s);
            fresh = at_run.run == 0;
            const int h0 = now.run * RUN, heads = live && on ? min(RUN, side.H - h0) : 0;
            TIn* dx = reinterpret_cast<TIn*>(side.y) + now.b * side.ys[0] + now.s * side.ys[1] + h0 * side.ys[2];
#pragma unroll
            for (int h = 0; h < RUN; ++h) {
                float x[8], g[8], sum = 0.f, dot = 0.f;
                row_unpack(xn[h], x);
                row_unpack(gn[h], g);
                row_turn<HALF, true>(g, c, s, at.turned);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sum = fmaf(x[e], x[e], sum);
                    dot = fmaf(g[e] * w[e], x[e], dot);
                }
                const float r = rsqrtf(row_sum<LANES>(sum) * inv_d + a.eps), f = row_sum<LANES>(dot) * inv_d * r * r;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    acc[e] = fmaf(g[e], x[e] * r, acc[e]);
                    x[e] = r * (g[e] * w[e] - x[e] * f);
                }
                if (h < heads) row_store<HALF>(dx + h * side.ys[2], at, x);
            }
        }
        if (side_i == 1) pdl_trigger();
        if (!a.part) continue;
        if (on) row_store<HALF>(sm[group], at, acc);
        __syncthreads();
        if (threadIdx.x < D) {
            float sum = 0.f;
#pragma unroll 8
            for (int j = 0; j < GROUPS; ++j) sum += sm[j][threadIdx.x];
            a.part[((size_t)blockIdx.x * 2 + side_i) * D + threadIdx.x] = sum;
        }
        __syncthreads();
    }
}

template <typename TIn, typename TOut, bool BACK>
static void (*lane_instance(int D, bool half))(NormArgs) {
    if constexpr (BACK) {
        return D <= 32 ? (half ? qk_norm_backward_kernel<TIn, TOut, 4, true> : qk_norm_backward_kernel<TIn, TOut, 4, false>)
             : D <= 64 ? (half ? qk_norm_backward_kernel<TIn, TOut, 8, true> : qk_norm_backward_kernel<TIn, TOut, 8, false>)
             : D <= 128 ? (half ? qk_norm_backward_kernel<TIn, TOut, 16, true> : qk_norm_backward_kernel<TIn, TOut, 16, false>)
                        : (half ? qk_norm_backward_kernel<TIn, TOut, 32, true> : qk_norm_backward_kernel<TIn, TOut, 32, false>);
    } else {
        return D <= 32 ? (half ? qk_norm_kernel<TIn, TOut, 4, true> : qk_norm_kernel<TIn, TOut, 4, false>)
             : D <= 64 ? (half ? qk_norm_kernel<TIn, TOut, 8, true> : qk_norm_kernel<TIn, TOut, 8, false>)
             : D <= 128 ? (half ? qk_norm_kernel<TIn, TOut, 16, true> : qk_norm_kernel<TIn, TOut, 16, false>)
                        : (half ? qk_norm_kernel<TIn, TOut, 32, true> : qk_norm_kernel<TIn, TOut, 32, false>);
    }
}
template <bool BACK>
static void (*instance(const grl_qk_norm_params& f))(NormArgs) {
    const bool in32 = f.in_dtype == GRL_F32, out32 = f.out_dtype == GRL_F32, half = f.rope.mode == GRL_ROPE_HALF;
    return in32 ? (out32 ? lane_instance<float, float, BACK>(f.head_dim, half) : lane_instance<float, __nv_bfloat16, BACK>(f.head_dim, half))
                : (out32 ? lane_instance<__nv_bfloat16, float, BACK>(f.head_dim, half) : lane_instance<__nv_bfloat16, __nv_bfloat16, BACK>(f.head_dim, half));
}

// Backward, a warp a row:  g = R^T dy,  dw += g * x r,  dx = r (w g - x r^2 mean(w g x)).
// A warp keeps its share of both weight gradients in registers; the CTA's sum goes to the workspace, and
// qk_norm_weight_kernel adds the CTAs' in order.
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(256) qk_norm_rows_backward_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float sm[256];
    const int lane = threadIdx.x & 31, pairs = a.D / 2;
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    float acc[2][kPairs][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < kPairs; ++e) acc[i][e][0] = acc[i][e][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const NormSide& side = i ? a.k : a.q;
        const long long rows = (long long)a.B * a.S * side.H;
        for (long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); row < rows; row += warps) {
            const int h = (int)(row % side.H);
            const long long tok = row / side.H;
            const int s = (int)(tok % a.S), b = (int)(tok / a.S);
            const TIn* x = reinterpret_cast<const TIn*>(side.x) + b * side.xs[0] + s * side.xs[1] + h * side.xs[2];
            const TOut* dy = reinterpret_cast<const TOut*>(side.dy) + b * side.dys[0] + s * side.dys[1] + h * side.dys[2];
            TIn* dx = reinterpret_cast<TIn*>(side.y) + b * side.ys[0] + s * side.ys[1] + h * side.ys[2];
            const int pos = position_of(a, b, s);
            float x0[kPairs], x1[kPairs], g0[kPairs], g1[kPairs], sum = 0.f, dot = 0.f;
#pragma unroll
            for (int e = 0; e < kPairs; ++e) {
                const int j = lane + 32 * e;
                x0[e] = x1[e] = g0[e] = g1[e] = 0.f;
                if (j < pairs) {
                    int d0, d1;
                    float c, sn;
                    pair_place(a.rope, j, &d0, &d1);
                    pair_angle(a.rope, j, pos, &c, &sn);
                    x0[e] = load_as_float<TIn>(x + d0);
                    x1[e] = load_as_float<TIn>(x + d1);
                    const float y0 = load_as_float<TOut>(dy + d0), y1 = load_as_float<TOut>(dy + d1);
                    g0[e] = y0 * c + y1 * sn;
                    g1[e] = y1 * c - y0 * sn;
                }
                sum = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], sum));
            }
            const float r = rsqrtf(warp_sum(sum) / (float)a.D + a.eps);
#pragma unroll
            for (int e = 0; e < kPairs; ++e) {
                const int j = lane + 32 * e;
                acc[i][e][0] = fmaf(g0[e], x0[e] * r, acc[i][e][0]);
                acc[i][e][1] = fmaf(g1[e], x1[e] * r, acc[i][e][1]);
                if (j < pairs && side.w) {
                    int d0, d1;
                    pair_place(a.rope, j, &d0, &d1);
                    g0[e] *= side.w[d0];
                    g1[e] *= side.w[d1];
                }
                dot = fmaf(g0[e], x0[e], fmaf(g1[e], x1[e], dot));
            }
            const float f = warp_sum(dot) / (float)a.D * r * r;
#pragma unroll
            for (int e = 0; e < kPairs; ++e) {
                const int j = lane + 32 * e;
                if (j < pairs) {
                    int d0, d1;
                    pair_place(a.rope, j, &d0, &d1);
                    store_from_float<TIn>(dx + d0, r * (g0[e] - x0[e] * f));
                    store_from_float<TIn>(dx + d1, r * (g1[e] - x1[e] * f));
                }
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int w = 0; w < 8; ++w) {       // the warps of the CTA add in order
            if ((int)(threadIdx.x >> 5) == w) {
#pragma unroll
                for (int e = 0; e < kPairs; ++e) {
                    const int j = lane + 32 * e;
                    if (j < pairs) {
                        int d0, d1;
                        pair_place(a.rope, j, &d0, &d1);
                        sm[d0] = (w ? sm[d0] : 0.f) + acc[i][e][0];
                        sm[d1] = (w ? sm[d1] : 0.f) + acc[i][e][1];
                    }
                }
            }
            __syncthreads();
        }
        if ((int)threadIdx.x < a.D) a.part[((size_t)blockIdx.x * 2 + i) * a.D + threadIdx.x] = sm[threadIdx.x];
        __syncthreads();
    }
}

// dw[d] = sum over the CTAs of part[CTA][side][d], in order of the CTAs for every thread group; in double, which costs nothing here.
__global__ void __launch_bounds__(1024) qk_norm_weight_kernel(const float* __restrict__ part, int ctas, int D, float* dq, float* dk) {
    __shared__ double sm[32][33];
    float* out = blockIdx.y ? dk : dq;
    pdl_wait();
    pdl_trigger();
    if (!out) return;
    const int d = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    double sum = 0.0;
    if (d < D)
        for (int c = g; c < ctas; c += 32) sum += (double)part[((size_t)c * 2 + blockIdx.y) * D + d];
    sm[g][threadIdx.x & 31] = sum;
    __syncthreads();
    if (g == 0 && d < D) {
        double t = 0.0;
        for (int i = 0; i < 32; ++i) t += sm[i][threadIdx.x];
        out[d] = (float)t;
    }
}

// CTAs of the backward pass: what the GPU holds at once, or a warp a row.
static int backward_ctas(grl_device* dev, const grl_qk_norm_params& f) {
    const long long rows = (long long)f.batch * f.seq_len * f.num_q_heads, most = 3LL * dev->prop.multiProcessorCount;
    const long long ctas = (rows + 7) / 8;
    return (int)(ctas < most ? ctas : most);
}

int check_rope_spec(const grl_rope_spec& r, int head_dim, RopeArgs* out) {
    GRL_REQUIRE(r.mode >= GRL_ROPE_NONE && r.mode <= GRL_ROPE_HALF, "unknown rope mode");
    const int rd = r.rotary_dim ? r.rotary_dim : head_dim;
    GRL_REQUIRE(rd > 0 && rd % 2 == 0 && rd <= head_dim, "rotary_dim must be even and at most head_dim (%d), got %d", head_dim, r.rotary_dim);
    GRL_REQUIRE(r.mode == GRL_ROPE_NONE || r.inv_freq || r.theta > 0.f, "theta must be positive");
    GRL_REQUIRE(r.scaling >= 0.f && r.gain >= 0.f, "scaling and gain must not be negative");
    out->mode = r.mode;
    out->rd = r.mode == GRL_ROPE_NONE ? 0 : rd;
    out->gain = r.gain == 0.f ? 1.f : r.gain;
    out->inv_freq = r.inv_freq;
    return GRL_OK;
}

void fill_rope_freq(grl_device* dev, const grl_rope_spec& r, RopeArgs* out) {
    if (out->mode != GRL_ROPE_NONE && !r.inv_freq) out->freq = cached_rope_freq(dev, out->rd, r.theta, r.scaling);
}

// Strides as given, or those of contiguous (B,S,H,D).
static void strides_of(const int64_t (&given)[3], int S, int H, int D, long long (&out)[3]) {
    const bool none = !given[0] && !given[1] && !given[2];
    out[0] = none ? (long long)S * H * D : given[0];
    out[1] = none ? (long long)H * D : given[1];
    out[2] = none ? D : given[2];
}

// Whether no two rows of a written tensor share an element: in order of their strides, every dimension steps over all that lies inside it.
static bool rows_apart(const long long (&st)[3], int B, int S, int H, int D) {
    struct Dim { long long step, n; } d[3] = {{st[0], B}, {st[1], S}, {st[2], H}};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (d[j].step < d[i].step) { const Dim t = d[i]; d[i] = d[j]; d[j] = t; }
    long long inside = D;
    for (int i = 0; i < 3; ++i) {
        if (d[i].n == 1) continue;
        if (d[i].step < inside) return false;
        inside = d[i].step * (d[i].n - 1) + inside;
    }
    return true;
}

static int side_args(const grl_qk_norm_params& f, bool key, NormSide* s) {
    s->x = key ? f.k : f.q;
    s->w = key ? f.k_weight : f.q_weight;
    s->H = key ? (f.k ? f.num_kv_heads : 0) : f.num_q_heads;
    const int H = s->H ? s->H : 1;
    strides_of(key ? f.k_strides : f.q_strides, f.seq_len, H, f.head_dim, s->xs);
    for (long long v : s->xs) GRL_REQUIRE(v >= 0, "strides must not be negative");
    return GRL_OK;
}

static int check_norm(const grl_qk_norm_params& f, NormArgs* a) {
    GRL_REQUIRE(f.q, "q is NULL");
    GRL_REQUIRE(f.in_dtype == GRL_F32 || f.in_dtype == GRL_BF16, "in_dtype must be GRL_F32 or GRL_BF16");
    GRL_REQUIRE(f.out_dtype == GRL_F32 || f.out_dtype == GRL_BF16, "out_dtype must be GRL_F32 or GRL_BF16");
    GRL_REQUIRE(f.batch > 0 && f.seq_len > 0 && f.num_q_heads > 0 && (!f.k || f.num_kv_heads > 0), "bad shape");
    GRL_REQUIRE(f.head_dim > 0 && f.head_dim % 2 == 0 && f.head_dim <= 256, "head_dim must be even and <= 256");
    GRL_REQUIRE(f.eps >= 0.f, "eps must not be negative");
    GRL_REQUIRE((long long)f.batch * f.seq_len < (1LL << 31), "more than 2^31 tokens");
    int rc = side_args(f, false, &a->q);
    if (!rc) rc = side_args(f, true, &a->k);
    if (!rc) rc = check_rope_spec(f.rope, f.head_dim, &a->rope);
    if (rc) return rc;
    a->B = f.batch; a->S = f.seq_len; a->D = f.head_dim;
    a->eps = f.eps == 0.f ? 1e-6f : f.eps;
    a->positions = f.positions; a->pos_base = f.pos_base;
    return GRL_OK;
}

static int check_grad(const grl_qk_norm_grad_params* p, NormArgs* a) {
    GRL_REQUIRE(p, "params is NULL");
    const grl_qk_norm_params& f = p->fwd;
    int rc = check_norm(f, a);
    if (rc) return rc;
    GRL_REQUIRE(p->q_out_grad && p->q_grad, "q_out_grad or q_grad is NULL");
    GRL_REQUIRE(!f.k || (p->k_out_grad && p->k_grad), "k given without k_out_grad and k_grad");
    GRL_REQUIRE(f.k || !p->k_weight_grad, "k_weight_grad without k");
    for (int i = 0; i < (f.k ? 2 : 1); ++i) {
        NormSide& s = i ? a->k : a->q;
        s.dy = i ? p->k_out_grad : p->q_out_grad;
        s.y = i ? p->k_grad : p->q_grad;
        s.dw = i ? p->k_weight_grad : p->q_weight_grad;
        strides_of(i ? f.k_out_strides : f.q_out_strides, f.seq_len, s.H, f.head_dim, s.dys);
        strides_of(i ? p->k_grad_strides : p->q_grad_strides, f.seq_len, s.H, f.head_dim, s.ys);
        for (long long v : s.dys) GRL_REQUIRE(v >= 0, "strides must not be negative");
        GRL_REQUIRE(rows_apart(s.ys, f.batch, f.seq_len, s.H, f.head_dim), "rows of %s overlap: every gradient needs a place of its own",
                    i ? "k_grad" : "q_grad");
    }
    return GRL_OK;
}

}  // namespace grl

using namespace grl;

extern "C" {

int grl_qk_norm_rope(grl_device* dev, const grl_qk_norm_params* p) {
    GRL_REQUIRE(p, "params is NULL");
    NormArgs a{};
    int rc = check_norm(*p, &a);
    if (rc) return rc;
    GRL_REQUIRE(p->q_out && (!p->k || p->k_out), "q_out or k_out is NULL");
    a.q.y = p->q_out; a.k.y = p->k_out;
    strides_of(p->q_out_strides, p->seq_len, a.q.H, p->head_dim, a.q.ys);
    strides_of(p->k_out_strides, p->seq_len, a.k.H ? a.k.H : 1, p->head_dim, a.k.ys);
    GRL_REQUIRE(rows_apart(a.q.ys, p->batch, p->seq_len, a.q.H, p->head_dim) &&
                    (!p->k || rows_apart(a.k.ys, p->batch, p->seq_len, a.k.H, p->head_dim)),
                "rows of q_out or k_out overlap: every result needs a place of its own");
    GRL_REQUIRE(dev, "dev is NULL");
    DeviceGuard g(dev->ordinal);
    fill_rope_freq(dev, p->rope, &a.rope);
    const long long rows = (long long)a.B * a.S * (a.q.H + a.k.H), most = 8LL * dev->prop.multiProcessorCount;
    bool fast = a.D % 8 == 0 && a.rope.rd % 8 == 0;
    for (const NormSide* s : {&a.q, &a.k})
        if (s->H) fast = fast && row_aligned(s->x, p->in_dtype, s->xs, 3) && row_aligned(s->y, p->out_dtype, s->ys, 3);
    if (fast) {
        const int run = p->in_dtype == GRL_BF16 ? kRunOf<__nv_bfloat16> : kRunOf<float>;
        const long long runs = (long long)a.B * a.S * ((a.q.H + run - 1) / run + (a.k.H + run - 1) / run), groups = 256 / row_lanes(a.D);
        const long long need = (runs + groups - 1) / groups, held = 3LL * dev->prop.multiProcessorCount;
        GRL_CUDA(launch_pdl(instance<false>(*p), dim3((unsigned)(need < held ? need : held)), 256, 0, dev->stream, a));
        GRL_LAUNCHED("qk_norm_kernel");
        return GRL_OK;
    }
    const int ctas = (int)((rows + 7) / 8 < most ? (rows + 7) / 8 : most);
    const bool in32 = p->in_dtype == GRL_F32, out32 = p->out_dtype == GRL_F32;
    auto kernel = in32 ? (out32 ? qk_norm_rows_kernel<float, float> : qk_norm_rows_kernel<float, __nv_bfloat16>)
                       : (out32 ? qk_norm_rows_kernel<__nv_bfloat16, float> : qk_norm_rows_kernel<__nv_bfloat16, __nv_bfloat16>);
    kernel<<<ctas, 256, 0, dev->stream>>>(a);
    GRL_LAUNCHED("qk_norm_rows_kernel");
    return GRL_OK;
}

int grl_qk_norm_rope_backward_workspace_bytes(grl_device* dev, const grl_qk_norm_grad_params* p, size_t* bytes) {
    NormArgs a{};
    int rc = check_grad(p, &a);
    if (rc) return rc;
    GRL_REQUIRE(dev && bytes, "NULL argument");
    *bytes = a.q.dw || a.k.dw ? (size_t)backward_ctas(dev, p->fwd) * 2 * a.D * sizeof(float) : 0;
    return GRL_OK;
}

int grl_qk_norm_rope_backward(grl_device* dev, const grl_qk_norm_grad_params* p) {
    NormArgs a{};
    int rc = check_grad(p, &a);
    if (rc) return rc;
    GRL_REQUIRE(dev, "dev is NULL");
    const int ctas = backward_ctas(dev, p->fwd);
    if (a.q.dw || a.k.dw) {
        const size_t need = (size_t)ctas * 2 * a.D * sizeof(float);
        GRL_REQUIRE(p->workspace && p->workspace_bytes >= need, "workspace too small: %zu < %zu", p->workspace ? p->workspace_bytes : 0, need);
        GRL_REQUIRE((uintptr_t)p->workspace % 16 == 0, "workspace must be 16-byte aligned");
        a.part = static_cast<float*>(p->workspace);
    }
    DeviceGuard g(dev->ordinal);
    fill_rope_freq(dev, p->fwd.rope, &a.rope);
    bool fast = a.D % 8 == 0 && a.rope.rd % 8 == 0;
    for (const NormSide* s : {&a.q, &a.k})
        if (s->H)
            fast = fast && row_aligned(s->x, p->fwd.in_dtype, s->xs, 3) && row_aligned(s->y, p->fwd.in_dtype, s->ys, 3) &&
                   row_aligned(s->dy, p->fwd.out_dtype, s->dys, 3);
    const bool in32 = p->fwd.in_dtype == GRL_F32, out32 = p->fwd.out_dtype == GRL_F32;
    auto kernel = fast ? instance<true>(p->fwd)
                : in32 ? (out32 ? qk_norm_rows_backward_kernel<float, float> : qk_norm_rows_backward_kernel<float, __nv_bfloat16>)
                       : (out32 ? qk_norm_rows_backward_kernel<__nv_bfloat16, float> : qk_norm_rows_backward_kernel<__nv_bfloat16, __nv_bfloat16>);
    if (fast) GRL_CUDA(launch_pdl(kernel, dim3(ctas), 256, 0, dev->stream, a));
    else kernel<<<ctas, 256, 0, dev->stream>>>(a);
    GRL_LAUNCHED("qk_norm_backward_kernel");
    if (a.part) {
        GRL_CUDA(launch_pdl(qk_norm_weight_kernel, dim3((a.D + 31) / 32, 2), 1024, 0, dev->stream, (const float*)a.part, ctas, a.D, a.q.dw, a.k.dw));
        GRL_LAUNCHED("qk_norm_weight_kernel");
    }
    return GRL_OK;
}

}  // extern "C"
