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
    float* part;        // backward: weight gradients of every CTA, [CTA][D]
    int q_ctas;         // backward: the first CTAs take the queries, the others the keys
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

// Rows of whole 8-element pieces on 16-byte boundaries: LANES threads a row, eight elements each (threads past the row's end idle).  Bound by
// HBM as to bytes, and nearly as much by instructions, so those are few: two elements an operation; weight, rotation and angle as four
// factors for all heads of a token; addresses a step from head to head.  Every warp has an equal, contiguous share of the rows (token, head)
// and walks it in segments, heads of one token and one side: its groups take the heads in turn, RUN rows of each in flight, the next one
// asked for as soon as its registers are free.
// 4 x 2048 tokens, 32 + 8 heads of 128, bf16: 34 us (4.9 TB/s); a warp a row 229, without packed operations 69, without segments 36.
template <typename T> constexpr int kRunOf = sizeof(T) == 2 ? 4 : 2;
template <typename TIn, typename TOut, int LANES, bool HALF, bool FULL>
__global__ void __launch_bounds__(256, 3) qk_norm_kernel(const __grid_constant__ NormArgs a) {
    constexpr int RUN = kRunOf<TIn>, GPW = 32 / LANES;
    __shared__ __align__(16) RowTables tables;
    const int l = threadIdx.x % LANES, g = (threadIdx.x & 31) / LANES, D = FULL ? 8 * LANES : a.D;
    const bool on = FULL || 8 * l < D;
    const float inv_d = 1.f / D;
    const RowPlace at = row_place<HALF>(l, FULL ? D : a.rope.rd);
    const int gap = FULL && HALF ? 4 * LANES : at.gap();
    const int hq = a.q.H, slots = hq + a.k.H;
    const Share share((long long)a.B * a.S * slots, blockIdx.x, gridDim.x);
    const long long tok = share.lo / slots;
    int slot = (int)(share.lo - tok * slots), b = (int)(tok / a.S), s = (int)(tok - (long long)b * a.S), left = share.items;
    pdl_wait();
    pdl_trigger();
    row_tables(tables, a.rope, D, a.q.w, a.k.w);
    __syncthreads();
    Pairs angle;
    bool fresh = true;              // a token whose angles are not formed yet
    while (left > 0) {
        const bool is_k = slot >= hq;
        const int n = min(left, (is_k ? slots : hq) - slot), h0 = is_k ? slot - hq : slot;
        const long long* xs = is_k ? a.k.xs : a.q.xs;
        const long long* ys = is_k ? a.k.ys : a.q.ys;
        const int x_step = (int)xs[2] * GPW, y_step = (int)ys[2] * GPW;
        const TIn* in = reinterpret_cast<const TIn*>(is_k ? a.k.x : a.q.x) + (b * xs[0] + s * xs[1] + (h0 + g) * xs[2] + at.o0);
        TOut* out = reinterpret_cast<TOut*>(is_k ? a.k.y : a.q.y) + (b * ys[0] + s * ys[1] + (h0 + g) * ys[2] + at.o0);
        RowRaw<TIn> raw[RUN];
#pragma unroll
        for (int h = 0; h < RUN; ++h)
            if (on && g + GPW * h < n) row_fetch<HALF>(in + (long long)h * x_step, gap, raw[h]);
            else row_zero(raw[h]);
        if (fresh) {
            angle = row_angles(tables, l, a.rope.gain, at.turned, position_of(a, b, s));
            fresh = false;
        }
        const Turn turn = weighted_turn(row_weights<HALF>(tables.w[is_k], at), angle);
        for (int i = g; i < n + g; i += GPW * RUN) {
            in += (long long)RUN * x_step;
#pragma unroll
            for (int h = 0; h < RUN; ++h) {
                Pairs x = row_pairs<HALF>(raw[h]);
                if (on && i + GPW * (RUN + h) < n) row_fetch<HALF>(in + (long long)h * x_step, gap, raw[h]);
                const float r = rsqrtf(row_sum<LANES>(squares(x)) * inv_d + a.eps);
                turn_scaled(x, turn, r);
                if (on && i + GPW * h < n) row_store<HALF>(out + (long long)h * y_step, gap, x);
            }
            out += (long long)RUN * y_step;
        }
        slot += n;
        left -= n;
        if (slot == slots) {
            slot = 0;
            fresh = true;
            if (++s == a.S) { s = 0; ++b; }
        }
    }
}

// The backward pass in the same form.  A CTA takes the queries or the keys, as many CTAs each as they have rows; a group keeps its share of the
// weight's gradient in registers, the CTA adds them in order of its groups.
// 2 x 2048 tokens, 32 + 8 heads of 128, bf16: 31.7 us with the launch that adds the parts; a warp a row 199, both sides in every CTA 35.
template <typename T> constexpr int kGradRunOf = sizeof(T) == 2 ? 4 : 2;
template <typename TIn, typename TOut, int LANES, bool HALF, bool FULL>
__global__ void __launch_bounds__(256, 2) qk_norm_backward_kernel(const __grid_constant__ NormArgs a) {
    constexpr int GROUPS = 256 / LANES, RUN = kGradRunOf<TIn>, GPW = 32 / LANES;
    __shared__ __align__(16) RowTables tables;
    __shared__ __align__(16) float sm[GROUPS][8 * LANES];
    const int l = threadIdx.x % LANES, g = (threadIdx.x & 31) / LANES, D = FULL ? 8 * LANES : a.D;
    const bool on = FULL || 8 * l < D;
    const float inv_d = 1.f / D;
    const RowPlace at = row_place<HALF>(l, FULL ? D : a.rope.rd);
    const int gap = FULL && HALF ? 4 * LANES : at.gap();
    pdl_wait();
    row_tables(tables, a.rope, D, a.q.w, a.k.w);
    __syncthreads();
    const bool is_k = (int)blockIdx.x >= a.q_ctas;
    const NormSide& side = is_k ? a.k : a.q;
    const int H = side.H;
    const int x_step = (int)side.xs[2] * GPW, dy_step = (int)side.dys[2] * GPW, dx_step = (int)side.ys[2] * GPW;
    const Share share((long long)a.B * a.S * H, is_k ? blockIdx.x - a.q_ctas : blockIdx.x, is_k ? gridDim.x - a.q_ctas : a.q_ctas);
    const long long tok = share.lo / H;
    int h0 = (int)(share.lo - tok * H), b = (int)(tok / a.S), s = (int)(tok - (long long)b * a.S), left = share.items;
    const Pairs w = row_weights<HALF>(tables.w[is_k], at);
    Pairs acc;
    acc.f[0] = acc.f[1] = acc.g[0] = acc.g[1] = make_float2(0.f, 0.f);
    while (left > 0) {
        const int n = min(left, H - h0);
        const TIn* x_at = reinterpret_cast<const TIn*>(side.x) + (b * side.xs[0] + s * side.xs[1] + (h0 + g) * side.xs[2] + at.o0);
        const TOut* dy_at = reinterpret_cast<const TOut*>(side.dy) + (b * side.dys[0] + s * side.dys[1] + (h0 + g) * side.dys[2] + at.o0);
        TIn* dx_at = reinterpret_cast<TIn*>(side.y) + (b * side.ys[0] + s * side.ys[1] + (h0 + g) * side.ys[2] + at.o0);
        RowRaw<TIn> x_raw[RUN];
        RowRaw<TOut> dy_raw[RUN];
        auto ask = [&](int i, int h) {
            if (on && i + GPW * h < n) {
                row_fetch<HALF>(x_at + (long long)h * x_step, gap, x_raw[h]);
                row_fetch<HALF>(dy_at + (long long)h * dy_step, gap, dy_raw[h]);
            } else {
                row_zero(x_raw[h]);
                row_zero(dy_raw[h]);
            }
        };
#pragma unroll
        for (int h = 0; h < RUN; ++h) ask(g, h);
        const Pairs angle = row_angles(tables, l, a.rope.gain, at.turned, position_of(a, b, s));
        for (int i = g; i < n + g; i += GPW * RUN) {
            x_at += (long long)RUN * x_step;
            dy_at += (long long)RUN * dy_step;
#pragma unroll
            for (int h = 0; h < RUN; ++h) {
                Pairs x = row_pairs<HALF>(x_raw[h]);
                const Pairs y = row_pairs<HALF>(dy_raw[h]);
                ask(i + GPW * RUN, h);
                Pairs gr, wg;
                float2 dot = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    gr.f[e] = __ffma2_rn(y.g[e], angle.g[e], __fmul2_rn(y.f[e], angle.f[e]));
                    gr.g[e] = __ffma2_rn(neg2(y.f[e]), angle.g[e], __fmul2_rn(y.g[e], angle.f[e]));
                    wg.f[e] = __fmul2_rn(gr.f[e], w.f[e]);
                    wg.g[e] = __fmul2_rn(gr.g[e], w.g[e]);
                    dot = __ffma2_rn(wg.f[e], x.f[e], dot);
                    dot = __ffma2_rn(wg.g[e], x.g[e], dot);
                }
                const float r = rsqrtf(row_sum<LANES>(squares(x)) * inv_d + a.eps);
                const float2 rr = twice(r), back = twice(-row_sum<LANES>(dot.x + dot.y) * inv_d * r * r);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    acc.f[e] = __ffma2_rn(gr.f[e], __fmul2_rn(x.f[e], rr), acc.f[e]);
                    acc.g[e] = __ffma2_rn(gr.g[e], __fmul2_rn(x.g[e], rr), acc.g[e]);
                    x.f[e] = __fmul2_rn(__ffma2_rn(x.f[e], back, wg.f[e]), rr);
                    x.g[e] = __fmul2_rn(__ffma2_rn(x.g[e], back, wg.g[e]), rr);
                }
                if (on && i + GPW * h < n) row_store<HALF>(dx_at + (long long)h * dx_step, gap, x);
            }
            dx_at += (long long)RUN * dx_step;
        }
        left -= n;
        h0 = 0;
        if (++s == a.S) { s = 0; ++b; }
    }
    pdl_trigger();
    if (!a.part) return;
    if (on) row_store<HALF>(sm[threadIdx.x / LANES] + at.o0, gap, acc);
    __syncthreads();
    if (threadIdx.x < D) {
        float sum = 0.f;
#pragma unroll 8
        for (int j = 0; j < GROUPS; ++j) sum += sm[j][threadIdx.x];
        a.part[(size_t)blockIdx.x * D + threadIdx.x] = sum;
    }
}

template <typename TIn, typename TOut, bool BACK, int LANES>
static void (*form_instance(bool half, bool full))(NormArgs) {
    if constexpr (BACK)
        return half ? (full ? qk_norm_backward_kernel<TIn, TOut, LANES, true, true> : qk_norm_backward_kernel<TIn, TOut, LANES, true, false>)
                    : (full ? qk_norm_backward_kernel<TIn, TOut, LANES, false, true> : qk_norm_backward_kernel<TIn, TOut, LANES, false, false>);
    else
        return half ? (full ? qk_norm_kernel<TIn, TOut, LANES, true, true> : qk_norm_kernel<TIn, TOut, LANES, true, false>)
                    : (full ? qk_norm_kernel<TIn, TOut, LANES, false, true> : qk_norm_kernel<TIn, TOut, LANES, false, false>);
}
template <typename TIn, typename TOut, bool BACK>
static void (*lane_instance(int D, int rd, bool half))(NormArgs) {
    const bool full = row_full(D, rd);
    return D <= 32 ? form_instance<TIn, TOut, BACK, 4>(half, full) : D <= 64 ? form_instance<TIn, TOut, BACK, 8>(half, full)
         : D <= 128 ? form_instance<TIn, TOut, BACK, 16>(half, full) : form_instance<TIn, TOut, BACK, 32>(half, full);
}
template <bool BACK>
static void (*instance(const grl_qk_norm_params& f, int rd))(NormArgs) {
    const bool in32 = f.in_dtype == GRL_F32, out32 = f.out_dtype == GRL_F32, half = f.rope.mode == GRL_ROPE_HALF;
    return in32 ? (out32 ? lane_instance<float, float, BACK>(f.head_dim, rd, half) : lane_instance<float, __nv_bfloat16, BACK>(f.head_dim, rd, half))
                : (out32 ? lane_instance<__nv_bfloat16, float, BACK>(f.head_dim, rd, half) : lane_instance<__nv_bfloat16, __nv_bfloat16, BACK>(f.head_dim, rd, half));
}

// Backward, a warp a row:  g = R^T dy,  dw += g * x r,  dx = r (w g - x r^2 mean(w g x)).
// A warp keeps its share of both weight gradients in registers; the CTA's sum goes to the workspace, and
// qk_norm_weight_kernel adds the CTAs' in order.
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(256) qk_norm_rows_backward_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float sm[256];
    const int lane = threadIdx.x & 31, pairs = a.D / 2;
    const bool is_k = (int)blockIdx.x >= a.q_ctas;
    const NormSide& side = is_k ? a.k : a.q;
    const int cta = is_k ? blockIdx.x - a.q_ctas : blockIdx.x, ctas = is_k ? gridDim.x - a.q_ctas : a.q_ctas;
    float acc[kPairs][2];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) acc[e][0] = acc[e][1] = 0.f;
    {
        const long long rows = (long long)a.B * a.S * side.H;
        for (long long row = (long long)cta * 8 + (threadIdx.x >> 5); row < rows; row += 8LL * ctas) {
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
                acc[e][0] = fmaf(g0[e], x0[e] * r, acc[e][0]);
                acc[e][1] = fmaf(g1[e], x1[e] * r, acc[e][1]);
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
    for (int w = 0; w < 8; ++w) {       // the warps of the CTA add in order
        if ((int)(threadIdx.x >> 5) == w) {
#pragma unroll
            for (int e = 0; e < kPairs; ++e) {
                const int j = lane + 32 * e;
                if (j < pairs) {
                    int d0, d1;
                    pair_place(a.rope, j, &d0, &d1);
                    sm[d0] = (w ? sm[d0] : 0.f) + acc[e][0];
                    sm[d1] = (w ? sm[d1] : 0.f) + acc[e][1];
                }
            }
        }
        __syncthreads();
    }
    if ((int)threadIdx.x < a.D) a.part[(size_t)blockIdx.x * a.D + threadIdx.x] = sm[threadIdx.x];
}

// dw[d] = sum of part[CTA][d] over the CTAs of a side, in the same order every time; in double, which costs nothing here.
__global__ void __launch_bounds__(1024) qk_norm_weight_kernel(const float* __restrict__ part, int q_ctas, int ctas, int D, float* dq, float* dk) {
    __shared__ double sm[32][33];
    float* out = blockIdx.y ? dk : dq;
    pdl_wait();
    pdl_trigger();
    if (!out) return;
    const int d = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5, first = blockIdx.y ? q_ctas : 0, end = blockIdx.y ? ctas : q_ctas;
    double sum = 0.0;
    if (d < D)
        for (int c0 = first + g; c0 < end; c0 += 32 * 8) {         // eight loads in flight
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c0 + 32 * j < end ? __ldcg(part + (size_t)(c0 + 32 * j) * D + d) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += (double)v[j];
        }
    sm[g][threadIdx.x & 31] = sum;
    __syncthreads();
    if (g == 0 && d < D) {
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sm[i][threadIdx.x];
        out[d] = (float)t;
    }
}

// CTAs of the backward pass: for two rows of each warp, as many as the SMs hold at once; the sides share them by their rows.
static int backward_ctas(grl_device* dev, const grl_qk_norm_params& f, int* q_ctas) {
    const long long tokens = (long long)f.batch * f.seq_len, heads = f.num_q_heads + (f.k ? f.num_kv_heads : 0);
    const long long need = (tokens * heads + 15) / 16, most = 2LL * dev->prop.multiProcessorCount;
    const int ctas = (int)(need < 2 ? 2 : need < most ? need : most);
    const int q = (int)((ctas * (long long)f.num_q_heads + heads / 2) / heads);
    *q_ctas = !f.k ? ctas : q < 1 ? 1 : q > ctas - 1 ? ctas - 1 : q;
    return ctas;
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
// Whether a side's rows serve the eight-element form.
static bool side_fits(const NormSide& s, int in_dtype, int x_dtype, int out_dtype, bool back) {
    const auto near = [](const long long* st) { return st[2] < (1LL << 27); };      // steps of eight heads fit 32 bits
    return !s.H || (row_aligned(s.x, in_dtype, s.xs, 3) && near(s.xs) && row_aligned(s.y, x_dtype, s.ys, 3) && near(s.ys) &&
                    (!back || (row_aligned(s.dy, out_dtype, s.dys, 3) && near(s.dys))));
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
    const bool fast = a.D % 8 == 0 && a.rope.rd % 8 == 0 && side_fits(a.q, p->in_dtype, p->out_dtype, 0, false) &&
                      side_fits(a.k, p->in_dtype, p->out_dtype, 0, false);
    if (fast) {
        // a CTA for two rows of each of its groups, as many as the SMs hold at once
        const long long two = 2 * 256 / row_lanes(a.D), need = (rows + two - 1) / two, held = 3LL * dev->prop.multiProcessorCount;
        GRL_CUDA(launch_pdl(instance<false>(*p, a.rope.rd), dim3((unsigned)(need < held ? need : held)), 256, 0, dev->stream, a));
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
    int q_ctas;
    *bytes = a.q.dw || a.k.dw ? (size_t)backward_ctas(dev, p->fwd, &q_ctas) * a.D * sizeof(float) : 0;
    return GRL_OK;
}

int grl_qk_norm_rope_backward(grl_device* dev, const grl_qk_norm_grad_params* p) {
    NormArgs a{};
    int rc = check_grad(p, &a);
    if (rc) return rc;
    GRL_REQUIRE(dev, "dev is NULL");
    const int ctas = backward_ctas(dev, p->fwd, &a.q_ctas);
    if (a.q.dw || a.k.dw) {
        const size_t need = (size_t)ctas * a.D * sizeof(float);
        GRL_REQUIRE(p->workspace && p->workspace_bytes >= need, "workspace too small: %zu < %zu", p->workspace ? p->workspace_bytes : 0, need);
        GRL_REQUIRE((uintptr_t)p->workspace % 16 == 0, "workspace must be 16-byte aligned");
        a.part = static_cast<float*>(p->workspace);
    }
    DeviceGuard g(dev->ordinal);
    fill_rope_freq(dev, p->fwd.rope, &a.rope);
    const bool fast = a.D % 8 == 0 && a.rope.rd % 8 == 0 && side_fits(a.q, p->fwd.in_dtype, p->fwd.in_dtype, p->fwd.out_dtype, true) &&
                      side_fits(a.k, p->fwd.in_dtype, p->fwd.in_dtype, p->fwd.out_dtype, true);
    const bool in32 = p->fwd.in_dtype == GRL_F32, out32 = p->fwd.out_dtype == GRL_F32;
    auto kernel = fast ? instance<true>(p->fwd, a.rope.rd)
                : in32 ? (out32 ? qk_norm_rows_backward_kernel<float, float> : qk_norm_rows_backward_kernel<float, __nv_bfloat16>)
                       : (out32 ? qk_norm_rows_backward_kernel<__nv_bfloat16, float> : qk_norm_rows_backward_kernel<__nv_bfloat16, __nv_bfloat16>);
    if (fast) GRL_CUDA(launch_pdl(kernel, dim3(ctas), 256, 0, dev->stream, a));
    else kernel<<<ctas, 256, 0, dev->stream>>>(a);
    GRL_LAUNCHED("qk_norm_backward_kernel");
    if (a.part) {
        GRL_CUDA(launch_pdl(qk_norm_weight_kernel, dim3((a.D + 31) / 32, 2), 1024, 0, dev->stream, (const float*)a.part, a.q_ctas, ctas, a.D, a.q.dw, a.k.dw));
        GRL_LAUNCHED("qk_norm_weight_kernel");
    }
    return GRL_OK;
}

}  // extern "C"
