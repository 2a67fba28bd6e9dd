// Activation checkpoints in 8 bits: 32 neighbours of a row share one power of two, each value is a whole number of
// -127..127 steps. With m the largest magnitude of a block,
//     e    = the smallest exponent (1..249) at which m / 2^(e-127) rounds to at most 127,
//     q_i  = round-to-nearest-even(x_i / 2^(e-127)),          x_i is rebuilt as q_i * 2^(e-127).
// The error of a value is at most half a step, a step is between m / 127.5 and m / 63.7 (from m = 127.5 * 2^121 = 3.39e38 on, bf16's
// largest number, q is 64 and its value 2^128, infinity: rounding to nearest beyond the largest number, as everywhere). A step is a power of two, so that
// scaling never rounds: q * 2^(e-127) has at most 7 significant bits and is exact in bf16, which is what lets the weight
// gradient feed rebuilt values to the bf16 tensor cores without a second rounding. A block that holds an infinity or NaN is
// stored as e = 255 with q = 0 (0 * 2^128 = NaN): a training step that has gone wrong shows it in its gradients.
// (Blocks of 32 with a shared power of two are the layout of the published microscaling formats; the rule for e, which uses
// the whole range of q, and the mark for blocks that are not finite are this file's.)
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace psb {

namespace {

constexpr int kAct8Block = 32;

// The exponent byte for a block whose largest magnitude has these bits (compared as integers, NaN is above infinity is
// above every number, so a maximum over the bits carries both). Adding 2^16 carries into the exponent exactly when the
// mantissa is at least 127.5 / 64.
__device__ __forceinline__ uint32_t act8_exponent(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return 255u;
    const int e = (int)((amax_bits + 0x10000u) >> 23) - 6;
    return (uint32_t)(e < 1 ? 1 : e);
}
// 2^(127-e), and 0 for e = 255
__device__ __forceinline__ float act8_inverse_step(uint32_t e) { return e == 255u ? 0.f : __uint_as_float((254u - e) << 23); }
// 2^(e-127), and infinity for e = 255
__device__ __forceinline__ float act8_step(uint32_t e) { return __uint_as_float(e << 23); }
// (the conversion takes NaN = infinity * 0 to 0)
__device__ __forceinline__ int act8_quantise(float x, float inverse_step) { return __float2int_rn(x * inverse_step); }
// The larger magnitude of a and b, NaN if one of them is
__device__ __forceinline__ float abs_max(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
    return m;
}
// Four values as bytes: adding 1.5 * 2^23 leaves the rounded number in the low bits (one multiply-add per value where a
// conversion instruction has a quarter of its rate). Only for finite blocks.
__device__ __forceinline__ uint32_t act8_quantise4(float a, float b, float c, float d, float inverse_step) {
    const float magic = 12582912.f;
    const uint32_t x = __float_as_uint(fmaf(a, inverse_step, magic)), y = __float_as_uint(fmaf(b, inverse_step, magic));
    const uint32_t z = __float_as_uint(fmaf(c, inverse_step, magic)), w = __float_as_uint(fmaf(d, inverse_step, magic));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}
// Byte i of `biased` (four numbers with their sign bits flipped) as a float: byte b in the second byte of 0x4700bb00 is 32768 + b
template <int I>
__device__ __forceinline__ float s8_of_biased(uint32_t biased) {
    return __uint_as_float(__byte_perm(biased, 0x47000000u, 0x7404 | (I << 4))) - 32896.f;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

}  // namespace

}  // namespace psb
