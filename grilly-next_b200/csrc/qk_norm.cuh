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
};
template <bool HALF>
__device__ __forceinline__ RowPlace row_place(int l, int rd) {
    RowPlace p;
    p.turned = 8 * l < rd;
    p.o0 = HALF && p.turned ? 4 * l : 8 * l;
    p.o1 = HALF && p.turned ? p.o0 + rd / 2 : p.o0 + 4;
    return p;
}
__device__ __forceinline__ void unpack_bf16(uint32_t w, float& a, float& b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// A thread's part of a row as it lies in memory: what is on its way for later rows takes no more registers than that.
template <typename T> struct RowRaw {
    uint32_t w[sizeof(T) * 2];
};
template <bool HALF>
__device__ __forceinline__ void row_fetch(const float* p, const RowPlace& at, RowRaw<float>& r) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p + at.o0)), b = __ldcs(reinterpret_cast<const uint4*>(p + at.o1));
    r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
}
template <bool HALF>
__device__ __forceinline__ void row_fetch(const __nv_bfloat16* p, const RowPlace& at, RowRaw<__nv_bfloat16>& r) {
    if constexpr (HALF) {
        const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p + at.o0)), b = __ldcs(reinterpret_cast<const uint2*>(p + at.o1));
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = b.x; r.w[3] = b.y;
    } else {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p + at.o0));
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    }
}
template <typename T>
__device__ __forceinline__ void row_zero(RowRaw<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 2; ++i) r.w[i] = 0u;
}
__device__ __forceinline__ void row_unpack(const RowRaw<float>& r, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(r.w[e]);
}
__device__ __forceinline__ void row_unpack(const RowRaw<__nv_bfloat16>& r, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) unpack_bf16(r.w[e], x[2 * e], x[2 * e + 1]);
}
template <bool HALF>
__device__ __forceinline__ void row_store(float* p, const RowPlace& at, const float (&y)[8]) {
    *reinterpret_cast<float4*>(p + at.o0) = make_float4(y[0], y[1], y[2], y[3]);
    *reinterpret_cast<float4*>(p + at.o1) = make_float4(y[4], y[5], y[6], y[7]);
}
template <bool HALF>
__device__ __forceinline__ void row_store(__nv_bfloat16* p, const RowPlace& at, const float (&y)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(y[2 * e], y[2 * e + 1]);
    if constexpr (HALF) {
        *reinterpret_cast<uint2*>(p + at.o0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(p + at.o1) = make_uint2(w[2], w[3]);
    } else {
        *reinterpret_cast<uint4*>(p + at.o0) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, LANES);
    return v;
}
// Frequencies of the pairs and the weights of both sides, in shared memory: a thread's own are read where they are used.
struct RowTables {
    double freq[128];
    float w[2][256];
};
template <bool HALF>
__device__ __forceinline__ void row_tables(RowTables& t, const RopeArgs& r, int D, const float* w0, const float* w1) {
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        t.w[0][i] = w0 ? __ldg(w0 + i) : 1.f;
        t.w[1][i] = w1 ? __ldg(w1 + i) : 1.f;
        if (2 * i < r.rd) t.freq[i] = r.inv_freq ? (double)__ldg(r.inv_freq + i) : r.freq.inv_freq[i];
    }
}
__device__ __forceinline__ void row_weights(const float* w, const RowPlace& at, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(w + at.o0), b = *reinterpret_cast<const float4*>(w + at.o1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
// cosine and sine of a thread's four pairs at a position; 1 and 0 where nothing turns
__device__ __forceinline__ void row_angles(const RowTables& t, int l, float gain, bool turned, int pos, float (&c)[4], float (&s)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        c[e] = 1.f;
        s[e] = 0.f;
        if (turned) {
            rope_sincos(pos, t.freq[4 * l + e], &c[e], &s[e]);
            c[e] *= gain;
            s[e] *= gain;
        }
    }
}
// The rotation of a thread's pairs; BACK: its transpose.
template <bool HALF, bool BACK>
__device__ __forceinline__ void row_turn(float (&x)[8], const float (&c)[4], const float (&s)[4], bool turned) {
    if (!turned) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = HALF ? e : 2 * e, j = HALF ? e + 4 : 2 * e + 1;
        const float sn = BACK ? -s[e] : s[e], a = x[i] * c[e] - x[j] * sn, b = x[i] * sn + x[j] * c[e];
        x[i] = a;
        x[j] = b;
    }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
#endif

}  // namespace grl
