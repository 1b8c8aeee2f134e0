#pragma once
// Standalone RoPE and attention-mask ops with the push-constant contracts of
// shaders/rope.glsl:32-40 and shaders/attention-mask.glsl:18-24 (the reference ships the shaders
// without a C++ dispatcher; these follow its op-layer conventions).
#include <cstdint>
#include <stdexcept>

#include "grilly/buffer_pool.h"
#include "grilly/command_batch.h"
#include "grilly/ops/attention.h"
#include "grilly/pipeline_cache.h"

namespace grilly {
namespace ops {

/// x, y: (B,S,H,D) float32 host arrays.  cosTable/sinTable: nullptr or (>=S, D/2) float32.
void rope(CommandBatch& batch, BufferPool& pool, PipelineCache& cache, const float* x, float* y, uint32_t batchSize,
          uint32_t seqLen, uint32_t numHeads, uint32_t headDim, float base = 10000.0f, float scaling = 1.0f,
          RopeMode mode = RopeMode::Half, const float* cosTable = nullptr, const float* sinTable = nullptr);

/// The rotation of normalised heads: the first rotaryDim elements (0: all), angles position * theta^(-2j/rotaryDim) / scaling, cosine
/// and sine times gain.  scaling and gain must be positive: the C structure reads 0 as 1.
struct HeadRope {
    RopeMode mode = RopeMode::Interleaved;
    uint32_t rotaryDim = 0;
    float theta = 10000.0f, scaling = 1.0f, gain = 1.0f;
    grl_rope_spec spec() const {
        if (!(scaling > 0.0f) || !(gain > 0.0f)) throw std::runtime_error("rope scaling and gain must be positive");
        grl_rope_spec s{};
        s.mode = int(mode); s.rotary_dim = int(rotaryDim); s.theta = theta; s.scaling = scaling; s.gain = gain;
        return s;
    }
};
/// The weights of normalised query and key heads: device float32 (headDim), or invalid buffers for ones.  eps must be positive: the C structures
/// read 0 as 1e-6.
struct HeadNorm {
    GrillyBuffer qWeight, kWeight;
    float eps = 1e-6f;
    float epsilon() const {
        if (!(eps > 0.0f)) throw std::runtime_error("eps must be positive");
        return eps;
    }
};

/// Queries and keys of a layer normalised by head and rotated; q, qOut (B,S,Hq,D), k, kOut (B,S,Hkv,D) device buffers of `dtype`, k may be
/// invalid; positions: device int32 (B,S), or invalid for 0 .. S-1.  Asynchronous on the context stream.
struct HeadShape { uint32_t batch, seqLen, numQHeads, numKvHeads, headDim; };
void qkNormRopeDevice(BufferPool& pool, PipelineCache& cache, const GrillyBuffer& q, const GrillyBuffer& k, GrillyBuffer& qOut,
                      GrillyBuffer& kOut, int dtype, const HeadShape& shape, const HeadNorm& norm, const HeadRope& rope,
                      const GrillyBuffer& positions, int32_t posBase = 0);
/// Its gradients: of q and k (of `dtype`), and of the weights (float32, where the buffers are valid).  `ws` receives the pooled workspace, to
/// be released by the caller behind the launch.
void qkNormRopeBackwardDevice(BufferPool& pool, PipelineCache& cache, const GrillyBuffer& qOutGrad, const GrillyBuffer& kOutGrad,
                              const GrillyBuffer& q, const GrillyBuffer& k, GrillyBuffer& qGrad, GrillyBuffer& kGrad,
                              GrillyBuffer& qWeightGrad, GrillyBuffer& kWeightGrad, int dtype, const HeadShape& shape,
                              const HeadNorm& norm, const HeadRope& rope, const GrillyBuffer& positions, int32_t posBase, GrillyBuffer& ws);

/// scores: (B,H,S,S) float32 host array, modified in place.  keyMask: (B,S) or nullptr with causal.
void attentionMask(CommandBatch& batch, BufferPool& pool, PipelineCache& cache, float* scores, const float* keyMask,
                   uint32_t batchSize, uint32_t numHeads, uint32_t seqLen, bool causal, float maskValue = -1e9f);

}  // namespace ops
}  // namespace grilly
