// Host interface of rotary positions (rotary.cu). Device pointers; strides in elements; `dtype`: 0 = bf16, 1 = fp32.
#pragma once
#include <cstdint>

namespace psb {

// Heads of queries or keys: [batch][tokens][heads][dim] with these strides, values of a head side by side.
struct RotaryHeads {
    const void* x = nullptr;
    int64_t xb = 0, xt = 0, xh = 0;
    void* out = nullptr;
    int64_t ob = 0, ot = 0, oh = 0;
    int heads = 0;
};

struct RotaryArgs {
    RotaryHeads q, k;                 // k may have no heads
    int64_t batch = 0, tokens = 0;
    int dim = 0, pairs = 0;           // the first 2 * pairs values of a head turn, the others are copied (in place: left)
    int interleaved = 0;              // pairs are neighbours, or `pairs` apart
    const double* freqs = nullptr;    // [pairs], radians per position
    const void* positions = nullptr;  // int64, or int32 with positions32; null: offset + token
    int positions32 = 0;
    int64_t pb = 0, pt = 0;
    int64_t offset = 0;
    float scale = 1.f;
    int backward = 0;                 // turn back
};

// Returns 0, a cudaError_t, or -2 (a shape or dtype that is not supported).
int rotary(int dtype, const RotaryArgs& args, void* stream);

}  // namespace psb
