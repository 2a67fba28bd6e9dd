// Host interface of the weight gradient from an 8-bit checkpoint (act8_wgrad.cu).
#pragma once
#include <cstdint>

#include "norm.h"

namespace psb {

struct Act8WgradArgs {
    const void* dy = nullptr;        // bf16 [tokens][N], rows on 16-byte boundaries
    int64_t lddy = 0;
    Act8View x;                      // [tokens][K]
    float* out = nullptr;            // [N][K] = dy^T x
    int64_t ldo = 0;
    int accumulate = 0;
    // The operand is x * weight + bias (a layer norm's output rebuilt from its normalised rows); bf16 [K], and the column sums
    // of dy, fp32 [N], where bias is given. Null: x itself.
    const void* weight = nullptr;
    const void* bias = nullptr;
    const float* dy_sum = nullptr;
    int64_t tokens = 0;
    int N = 0, K = 0;
    void* scratch = nullptr;         // act8_wgrad_scratch() bytes; null: the checkpoint is converted tile by tile
    void* workspace = nullptr;       // as of linear_fused()
    unsigned* err_flag = nullptr;
    double wait_limit_s = 2.0;
};

// Returns 0, a cudaError_t, -2 (alignment or an argument that is not supported) or -3 (tensor map).
int act8_wgrad(const Act8WgradArgs& args, void* stream);
// Bytes of `scratch` for the faster of the two ways for these sizes (0: none).
int64_t act8_wgrad_scratch(int64_t tokens, int N, int K);

}  // namespace psb
