// Dropout masks that are never stored: what a value at (row, column) of a call has drawn is a function of its place, the call's offset
// and the seed, so that the backward pass forms the same mask again.
//
// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two
// 32 x 32 -> 64 bit products over a counter of four words under a key of two. Counter (column / 4, row, offset low, offset high), key
// (seed low, seed high); word `column % 4` belongs to the value. It is kept where the word is at least `threshold` = round(p 2^32), and
// grows by `scale` = 2^32 / (2^32 - threshold), the inverse of the exact share of words that keep a value.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "dropout.h"

namespace psb {

namespace {

struct DropKey {
    uint32_t k0, k1, o0, o1;
};
__device__ __forceinline__ DropKey drop_key(const DropoutArgs& d) {
    const uint64_t seed = d.seed_ptr != nullptr ? (uint64_t)*(const volatile int64_t*)d.seed_ptr : d.seed;
    return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)d.offset, (uint32_t)(d.offset >> 32)};
}
// The words of columns 4 group .. 4 group + 3 of a row
__device__ __forceinline__ uint4 drop_words(const DropKey& key, uint32_t row, uint32_t group) {
    uint32_t c0 = group, c1 = row, c2 = key.o0, c3 = key.o1, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
// Four neighbours after dropout. What is dropped is 0, whatever it was.
__device__ __forceinline__ void drop4(const DropKey& key, uint32_t threshold, float scale, uint32_t row, uint32_t group, float* f) {
    const uint4 w = drop_words(key, row, group);
    f[0] = w.x >= threshold ? f[0] * scale : 0.f;
    f[1] = w.y >= threshold ? f[1] * scale : 0.f;
    f[2] = w.z >= threshold ? f[2] * scale : 0.f;
    f[3] = w.w >= threshold ? f[3] * scale : 0.f;
}

}  // namespace

}  // namespace psb
