// sampling.cuh -- parameters and launcher of the token sampler (sampling.cu).
#pragma once

#include "pma_common.cuh"

namespace pma {

// A setting of the call: one value, or one per row.
template <typename T> struct PerRow {
    const T *rows;
    T value;
    __device__ __forceinline__ T at(int b) const { return rows ? rows[b] : value; }
};

struct SampleParams {
    int B, V;
    const void *logits;  // [B, V], V contiguous
    int64_t stride;
    const float *u;      // [B]
    PerRow<float> temperature, top_p, min_p;
    PerRow<int> top_k;
    int64_t *token;      // [B]
    float *logprob;      // [B] or nullptr
    int range;           // tokens of a warp's range (set by the launcher)
    int lists;           // there is shared memory for lists of candidates (set by the launcher)
};

constexpr int SAMPLE_MAX_V = 360448;  // 8 CTAs of 176 KB of float32 logits
cudaError_t launch_sample(SampleParams p, int dtype, int sms, cudaStream_t st);

}  // namespace pma
