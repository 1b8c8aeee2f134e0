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
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
#endif

}  // namespace grl
