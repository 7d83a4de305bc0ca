// Token sampling with temperature, top-k, top-p and min-p (sd_sample.hip).
#pragma once
#include "sd_kernels.hpp"

namespace sd {

constexpr int kSmpSlice = 8192;       // entries of a slice: one workgroup of the first launch
constexpr int kSmpBins = 1024;        // histogram bins of a slice
constexpr int kSmpMaxVocab = 262144;  // token indices take 18 bits

struct SampleParams {
    const float *logits;
    int64_t ld;
    int V, rows;
    float temperature;  // 0: the first maximum
    int top_k;          // 0: off
    float top_p;        // 1: off
    float min_p;        // 0: off
    const float *u;     // [rows] in [0, 1)
    int *tokens;        // [rows]; -1 for a row without a distribution
    float *probs;       // [rows][V] or null
    void *ws;           // sample_ws_bytes
};
size_t sample_ws_bytes(int V, int rows);
void launch_sample(const SampleParams &p, hipStream_t st);

}  // namespace sd
