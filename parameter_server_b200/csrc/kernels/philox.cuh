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

__host__ __device__ __forceinline__ void drop_keys(uint64_t seed, uint32_t* keys) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        keys[2 * r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
        keys[2 * r + 1] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
    }
}
// The keys of the rounds: operands from constant memory where the seed came with the call (formed in every thread they were a fifth of the
// instructions), in registers where it lies in memory.
template <bool IN_MEMORY>
struct DropKeys {
    uint32_t k[20];
    __device__ __forceinline__ explicit DropKeys(const DropoutArgs& d) { drop_keys((uint64_t)*(const volatile int64_t*)d.seed_ptr, k); }
    __device__ __forceinline__ uint32_t operator[](int i) const { return k[i]; }
};
template <>
struct DropKeys<false> {
    const DropoutArgs& d;
    __device__ __forceinline__ explicit DropKeys(const DropoutArgs& args) : d(args) {}
    __device__ __forceinline__ uint32_t operator[](int i) const { return d.keys[i]; }
};
// The words of columns 4 group .. 4 group + 3 of a row
template <typename Keys>
__device__ __forceinline__ uint4 drop_words(const Keys& key, uint64_t offset, uint32_t row, uint32_t group) {
    uint32_t c0 = group, c1 = row, c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ key[2 * r];
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ key[2 * r + 1];
        c3 = (uint32_t)a;
    }
    return make_uint4(c0, c1, c2, c3);
}
// Four neighbours after dropout. What is dropped is 0, whatever it was.
template <typename Keys>
__device__ __forceinline__ void drop4(const Keys& key, const DropoutArgs& d, uint32_t row, uint32_t group, float* f) {
    const uint4 w = drop_words(key, d.offset, row, group);
    f[0] = w.x >= d.threshold ? f[0] * d.scale : 0.f;
    f[1] = w.y >= d.threshold ? f[1] * d.scale : 0.f;
    f[2] = w.z >= d.threshold ? f[2] * d.scale : 0.f;
    f[3] = w.w >= d.threshold ? f[3] * d.scale : 0.f;
}

}  // namespace

}  // namespace psb
