// Host interface of dropout (dropout.cu). Device pointers; leading dimensions in elements; `dtype`: 0 = bf16, 1 = fp32.
#pragma once
#include <cstdint>

namespace psb {

struct DropoutArgs {
    uint32_t keys[20] = {};           // of the generator's rounds, from the seed
    const void* seed_ptr = nullptr;   // device int64, read when the kernel runs; `keys` are not used then
    uint64_t offset = 0;
    uint32_t threshold = 0;           // values whose word is below are dropped
    float scale = 1.f;                // of the others
};

// The keys of the rounds, two each, for a seed
void dropout_keys(uint64_t seed, uint32_t* keys);

// out = x * scale where kept, 0 elsewhere, + residual (optional). out may be x or residual itself.
// Returns 0, a cudaError_t, or -2 (a shape or dtype that is not supported).
int dropout(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldres, void* out, int64_t ldo, int64_t rows, int64_t cols,
            const DropoutArgs& drop, void* stream);

}  // namespace psb
