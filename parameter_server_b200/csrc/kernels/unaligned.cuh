// Rows that do not start on 16-byte boundaries, read and written by aligned blocks of 16 bytes all the same.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace psb {

namespace {

// 16 bytes of 32, from byte `past` (a multiple of W, below 16) on
template <int W>
__device__ __forceinline__ uint4 from_byte(uint32_t* w, uint32_t past) {
    if (past & 8u) {
#pragma unroll
        for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
    }
    if constexpr (W <= 4) {
        if (past & 4u) {
#pragma unroll
            for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
        }
    }
    if constexpr (W == 2) {
        const uint32_t shift = (past & 2u) * 8u;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], shift);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// 16 bytes of a row, of which `n` (one at least) exist, out of the two aligned blocks that they lie in (the second only where the row has
// bytes in it). Aligned blocks never reach past an allocation; what lies in them beside the row is not used.
template <int W>
__device__ __forceinline__ uint4 load_across(const char* p, int n) {
    const uint32_t past = (uint32_t)(uintptr_t)p & 15u;
    const char* block = p - past;
    const uint4 a = *(const uint4*)block;
    uint4 b = make_uint4(0, 0, 0, 0);
    if ((int)past + n > 16) b = *(const uint4*)(block + 16);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return from_byte<W>(w, past);
}
// The values in bytes [from, to) of 32, one by one
template <typename T>
__device__ __forceinline__ void store_some(char* p, const uint32_t* w, int from, int to) {
#pragma unroll
    for (int b = 0; b < 32; b += (int)sizeof(T)) {
        if (b < from || b >= to) continue;
        if constexpr (sizeof(T) == 4) *(uint32_t*)(p + b) = w[b / 4];
        else *(unsigned short*)(p + b) = (unsigned short)(w[b / 4] >> (8 * (b % 4)));
    }
}

}  // namespace

}  // namespace psb
