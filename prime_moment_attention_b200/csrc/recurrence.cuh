// recurrence.cuh -- parameters and launchers of the gated linear recurrence (recurrence.cu).
#pragma once

#include "pma_common.cuh"

namespace pma {

// A [B, L, C] device tensor: element strides on B and L, C contiguous.
struct Blc {
    void *p;
    int64_t sb, sl;
};

struct ScanParams {
    int B, L, C;
    int chunks, ctiles;       // tiles along L and along C
    Blc x, f, gate;           // gate.p == nullptr: y = h
    const float *bias;        // [C] or nullptr
    const float *h0;          // [B, C] or nullptr (zero)
    const uint8_t *reset;     // [B, L] or nullptr: nonzero cuts the state before that token
    Blc y;                    // forward
    float *h_last;            // [B, C] or nullptr
    Blc dy, dx, df, dgate;    // backward
    const float *dh_last;     // [B, C] or nullptr
    float *dh0;               // [B, C] or nullptr
    float *dbias_part;        // [B * chunks, C] or nullptr
    const uint32_t *states;   // backward: the forward pass's chunk-end states [B, chunks, C]
    // Workspace words, set to all ones before the launch: a word is unwritten until it is not.
    int *counter;             // [0] next tile, [1] abort flag
    uint32_t *incl;           // [B, chunks, C] state (or carry) leaving a tile
    unsigned long long *agg;  // [B, chunks, C] a tile's (Q, H)
    int *fault;
    unsigned long long wait_ns, test_wait_ns;
};

constexpr int SCAN_ROWS = 128;  // tokens in a tile
inline int scan_chunks(int L) { return (int)(((int64_t)L + SCAN_ROWS - 1) / SCAN_ROWS); }

// One cluster a sequence: the launch needs no words set up.
bool scan_by_cluster(int B, int L, int C, int dtype, int sms);
cudaError_t launch_gated_scan(ScanParams p, int dtype, int sms, cudaStream_t st);
cudaError_t launch_gated_scan_backward(ScanParams p, int dtype, float *dbias, int sms, cudaStream_t st);

struct ScanStepParams {
    int N, C;
    Blc x, f, gate, y;        // sl unused
    const float *bias;
    const float *h_in;        // [rows, C]
    float *h_out;             // may be h_in
    const int32_t *rows;      // nullable: state row of batch row n
    int pool_rows;
};
cudaError_t launch_gated_scan_step(const ScanStepParams &p, int dtype, cudaStream_t st);

}  // namespace pma
