// Normalised and rotated heads: what the stand-alone operator, its backward pass and the append into the paged cache share.
//   y = R(pos) (w * x * r),  r = 1 / sqrt(mean(x^2) + eps)
// A row is the head_dim elements of one (sequence, token, head).
#pragma once
#include "common.cuh"

namespace grl {

struct RopeArgs {
    int mode, rd;               // rd: elements of a head that the rotation turns
    float gain;
    const float* inv_freq;      // given frequencies, or NULL: freq
    RopeFreq freq;
};

// Checks of a grl_rope_spec and the kernel's form of it; freq is filled in by the caller, who has a device.
int check_rope_spec(const grl_rope_spec& r, int head_dim, RopeArgs* out);
// The frequencies of a spec that names none.
void fill_rope_freq(grl_device* dev, const grl_rope_spec& r, RopeArgs* out);

// Whether rows that start at p and lie `strides` apart serve the eight-element form.
inline bool row_aligned(const void* p, int dtype, const long long* strides, int n) {
    const long long unit = 16 / (dtype == GRL_BF16 ? 2 : 4);        // elements of 16 bytes
    bool ok = (uintptr_t)p % 16 == 0;
    for (int i = 0; i < n; ++i) ok = ok && strides[i] % unit == 0;
    return ok;
}
// FULL: every thread of a row has elements and all of them are turned, so that the gap is known to the compiler.
inline bool row_full(int D, int rd) { return rd == D && (D == 32 || D == 64 || D == 128 || D == 256); }
inline int row_lanes(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }      // threads of a row

#ifdef __CUDACC__
// Element places of pair j of a row: the rotated pairs first, then the elements that are left as they are, in neighbours.
__device__ __forceinline__ void pair_place(const RopeArgs& r, int j, int* d0, int* d1) {
    const int half = r.rd / 2;
    if (j >= half) { *d0 = r.rd + 2 * (j - half); *d1 = *d0 + 1; }
    else if (r.mode == GRL_ROPE_HALF) { *d0 = j; *d1 = j + half; }
    else { *d0 = 2 * j; *d1 = 2 * j + 1; }
}
__device__ __forceinline__ void pair_angle(const RopeArgs& r, int j, int pos, float* c, float* s) {
    if (j >= r.rd / 2) { *c = 1.f; *s = 0.f; return; }
    rope_sincos(pos, r.inv_freq ? (double)r.inv_freq[j] : r.freq.inv_freq[j], c, s);
    *c *= r.gain;
    *s *= r.gain;
}
// ---- rows of up to 8 * LANES elements held by LANES neighbouring threads, eight elements each: x[0..3] at o0 and x[4..7] at o1.  Rotated in
// halves, element e and e + 4 of a thread are a pair (o1 = o0 + rd / 2); else neighbours are, and o1 = o0 + 4.  The threads behind the
// rotated part hold the elements that are left as they are.  Needs D % 8 == 0 and rd % 8 == 0, and rows on boundaries of four elements
// (eight where o1 = o0 + 4).
struct RowPlace {
    int o0, o1;
    bool turned;
    __device__ __forceinline__ int gap() const { return o1 - o0; }
};
template <bool HALF>
__device__ __forceinline__ RowPlace row_place(int l, int rd) {
    RowPlace p;
    p.turned = 8 * l < rd;
    p.o0 = HALF && p.turned ? 4 * l : 8 * l;
    p.o1 = HALF && p.turned ? p.o0 + rd / 2 : p.o0 + 4;
    return p;
}
// A thread's part of a row as it lies in memory: what is on its way for later rows takes no more registers than that.
template <typename T> struct RowRaw {
    uint32_t w[sizeof(T) * 2];
};
// p: the thread's o0 in the row, gap: o1 - o0
template <bool HALF>
__device__ __forceinline__ void row_fetch(const float* p, int gap, RowRaw<float>& r) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p)), b = __ldcs(reinterpret_cast<const uint4*>(p + (HALF ? gap : 4)));
    r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
}
template <bool HALF>
__device__ __forceinline__ void row_fetch(const __nv_bfloat16* p, int gap, RowRaw<__nv_bfloat16>& r) {
    if constexpr (HALF) {
        const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p)), b = __ldcs(reinterpret_cast<const uint2*>(p + gap));
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = b.x; r.w[3] = b.y;
    } else {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    }
}
template <typename T>
__device__ __forceinline__ void row_zero(RowRaw<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 2; ++i) r.w[i] = 0u;
}
// The pairs of a thread's eight elements, two to a packed operation: f the first ones, g the second ones (f and g lie side by side
// where neighbours are turned, in the two halves where halves are).
struct Pairs {
    float2 f[2], g[2];
};
__device__ __forceinline__ float2 both(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 lows(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a << 16), __uint_as_float(b << 16)); }
__device__ __forceinline__ float2 highs(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)); }
template <bool HALF>
__device__ __forceinline__ Pairs row_pairs(const RowRaw<__nv_bfloat16>& r) {
    Pairs p;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        p.f[i] = HALF ? both(r.w[i]) : lows(r.w[2 * i], r.w[2 * i + 1]);
        p.g[i] = HALF ? both(r.w[2 + i]) : highs(r.w[2 * i], r.w[2 * i + 1]);
    }
    return p;
}
template <bool HALF>
__device__ __forceinline__ Pairs pairs_of(const float (&x)[8]) {
    Pairs p;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        p.f[i] = HALF ? make_float2(x[2 * i], x[2 * i + 1]) : make_float2(x[4 * i], x[4 * i + 2]);
        p.g[i] = HALF ? make_float2(x[4 + 2 * i], x[5 + 2 * i]) : make_float2(x[4 * i + 1], x[4 * i + 3]);
    }
    return p;
}
template <bool HALF>
__device__ __forceinline__ Pairs row_pairs(const RowRaw<float>& r) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(r.w[e]);
    return pairs_of<HALF>(x);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool HALF>
__device__ __forceinline__ void row_store(float* p, int gap, const Pairs& y) {
    if constexpr (HALF) {
        *reinterpret_cast<float4*>(p) = make_float4(y.f[0].x, y.f[0].y, y.f[1].x, y.f[1].y);
        *reinterpret_cast<float4*>(p + gap) = make_float4(y.g[0].x, y.g[0].y, y.g[1].x, y.g[1].y);
    } else {
        *reinterpret_cast<float4*>(p) = make_float4(y.f[0].x, y.g[0].x, y.f[0].y, y.g[0].y);
        *reinterpret_cast<float4*>(p + 4) = make_float4(y.f[1].x, y.g[1].x, y.f[1].y, y.g[1].y);
    }
}
template <bool HALF>
__device__ __forceinline__ void row_store(__nv_bfloat16* p, int gap, const Pairs& y) {
    if constexpr (HALF) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(y.f[0].x, y.f[0].y), pack_bf16x2(y.f[1].x, y.f[1].y));
        *reinterpret_cast<uint2*>(p + gap) = make_uint2(pack_bf16x2(y.g[0].x, y.g[0].y), pack_bf16x2(y.g[1].x, y.g[1].y));
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(y.f[0].x, y.g[0].x), pack_bf16x2(y.f[0].y, y.g[0].y),
                                                  pack_bf16x2(y.f[1].x, y.g[1].x), pack_bf16x2(y.f[1].y, y.g[1].y));
    }
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, LANES);
    return v;
}
// Turns per position (frequency / pi) of the pairs and the weights of both sides, in shared memory: read once for a token's heads.
struct RowTables {
    double turns[128];
    float w[2][256];
};
__device__ __forceinline__ void row_tables(RowTables& t, const RopeArgs& r, int D, const float* w0, const float* w1) {
    for (int i = threadIdx.x; i < 256; i += blockDim.x) {
        // zeros behind the row: threads without elements take part in its sums
        t.w[0][i] = i >= D ? 0.f : w0 ? __ldg(w0 + i) : 1.f;
        t.w[1][i] = i >= D ? 0.f : w1 ? __ldg(w1 + i) : 1.f;
        if (2 * i < r.rd) t.turns[i] = (r.inv_freq ? (double)__ldg(r.inv_freq + i) : r.freq.inv_freq[i]) * 0.31830988618379067;     // 1 / pi
    }
}
template <bool HALF>
__device__ __forceinline__ Pairs row_weights(const float* w, const RowPlace& at) {
    const float4 a = *reinterpret_cast<const float4*>(w + at.o0), b = *reinterpret_cast<const float4*>(w + at.o1);
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return pairs_of<HALF>(x);
}
// Cosine (f) and sine (g) of a thread's four pairs at a position, times the gain; 1 and 0 where nothing turns.  The angle in units of pi is
// formed and reduced to [-1, 1] in double, so that positions up to 2^24 keep some 1e-7 of a turn.
__device__ __forceinline__ Pairs row_angles(const RowTables& t, int l, float gain, bool turned, int pos) {
    Pairs a;
    a.f[0] = a.f[1] = make_float2(1.f, 1.f);
    a.g[0] = a.g[1] = make_float2(0.f, 0.f);
    if (turned) {
        float c[4], s[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double x = (double)pos * t.turns[4 * l + e];
            sincospif((float)fma(-2.0, rint(0.5 * x), x), &s[e], &c[e]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a.f[i] = make_float2(c[2 * i] * gain, c[2 * i + 1] * gain);
            a.g[i] = make_float2(s[2 * i] * gain, s[2 * i + 1] * gain);
        }
    }
    return a;
}
// A warp's equal, contiguous share of the `total` rows that `ctas` CTAs have.
struct Share {
    long long lo;
    int items;
    __device__ __forceinline__ Share(long long total, int cta, int ctas) {
        const long long warps = (long long)ctas * (blockDim.x >> 5), mine = (long long)cta * (blockDim.x >> 5) + (threadIdx.x >> 5);
        lo = mine * total / warps;
        items = (int)((mine + 1) * total / warps - lo);
    }
};
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }
__device__ __forceinline__ float2 twice(float a) { return make_float2(a, a); }
__device__ __forceinline__ float squares(const Pairs& x) {
    float2 s = __fmul2_rn(x.f[0], x.f[0]);
    s = __ffma2_rn(x.f[1], x.f[1], s);
    s = __ffma2_rn(x.g[0], x.g[0], s);
    s = __ffma2_rn(x.g[1], x.g[1], s);
    return s.x + s.y;
}
// Weight and rotation of a token's heads together: y_f = f ff + g fg, y_g = f gf + g gg.
struct Turn {
    float2 ff[2], fg[2], gf[2], gg[2];
};
__device__ __forceinline__ Turn weighted_turn(const Pairs& w, const Pairs& a) {
    Turn t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        t.ff[i] = __fmul2_rn(w.f[i], a.f[i]);
        t.fg[i] = neg2(__fmul2_rn(w.g[i], a.g[i]));
        t.gf[i] = __fmul2_rn(w.f[i], a.g[i]);
        t.gg[i] = __fmul2_rn(w.g[i], a.f[i]);
    }
    return t;
}
__device__ __forceinline__ void turn_scaled(Pairs& x, const Turn& t, float r) {
    const float2 rr = twice(r);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 f = __fmul2_rn(__ffma2_rn(x.g[i], t.fg[i], __fmul2_rn(x.f[i], t.ff[i])), rr);
        x.g[i] = __fmul2_rn(__ffma2_rn(x.g[i], t.gg[i], __fmul2_rn(x.f[i], t.gf[i])), rr);
        x.f[i] = f;
    }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
#endif

}  // namespace grl
