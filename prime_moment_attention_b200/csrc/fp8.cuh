// fp8.cuh -- parameters and launchers of the block-scaled e4m3 product (fp8.cu).
#pragma once

#include "pma_common.cuh"

namespace pma {

constexpr int FP8_BLOCK = 128;  // elements of K (and, for weights, rows) under one scale

struct Fp8Rows {           // [rows, K] e4m3
    const uint8_t *q;
    int64_t stride;        // bytes, a multiple of 16
    const float *scale;    // scale of (row or row block i, K block j): scale[i * si + j * sj]
    int64_t si, sj;
};

struct Fp8Params {
    int M, N, K;
    Fp8Rows x, w;          // x: a scale per row and 128 of K; w: per 128 rows and 128 of K
    void *y;               // [M, N], row stride ys elements
    int64_t ys;
    int y_f32;
    int tiles_a, tiles_b;  // tiles along the 128-row operand and along the other
    int blocks;            // K blocks
    int *fault;
    unsigned long long test_wait_ns;
};

cudaError_t launch_fp8_quantize(const void *x, int64_t xs, int dtype, int M, int K, uint8_t *q, int64_t qs,
                                float *scale, int64_t si, int64_t sj, int sms, cudaStream_t st);
cudaError_t launch_fp8_quantize_weight(const void *w, int64_t ws, int dtype, int N, int K, uint8_t *q, int64_t qs,
                                       float *scale, cudaStream_t st);
// after_quantize: the last kernel in the stream is launch_fp8_quantize's, with which it may overlap.
cudaError_t launch_fp8_matmul(Fp8Params p, int sms, bool after_quantize, cudaStream_t st);

}  // namespace pma
