// Rotary positions: pair i of a head's values turns by position * freqs[i],
//   x' = s (x cos - y sin),  y' = s (x sin + y cos),  and backward by the negative angle.
// The angle's product and its reduction to a turn are in 64 bits (position 2^20 times one radian is off by 0.06 in 32).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "launch.cuh"
#include "rotary.h"

namespace psb {

namespace {

constexpr int kRotThreads = 256;

__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t b, int64_t t) {
    if (a.positions == nullptr) return a.offset + t;
    const int64_t at = b * a.pb + t * a.pt;
    return a.offset + (a.positions32 ? (int64_t)((const int32_t*)a.positions)[at] : ((const int64_t*)a.positions)[at]);
}
// cosine and sine of position * freq
__device__ __forceinline__ void turn_of(double position, double freq, float* c, float* s) {
    const double turns = position * (freq * 0.15915494309189533577);
    sincospif(2.f * (float)(turns - rint(turns)), s, c);
}

// One thread has a pair of one token, and all heads of it
template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    wait_predecessor();
    allow_successor();
    const int units = a.pairs + a.dim - 2 * a.pairs;
    const int64_t total = a.batch * a.tokens * units;
    for (int64_t i = (int64_t)blockIdx.x * kRotThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kRotThreads) {
        const int64_t row = i / units, b = row / a.tokens, t = row - b * a.tokens;
        const int u = (int)(i - row * units);
        const bool turns = u < a.pairs;
        const int lo = !turns ? a.pairs + u : a.interleaved ? 2 * u : u, hi = a.interleaved ? lo + 1 : lo + a.pairs;
        float c = 1.f, s = 0.f;
        if (turns) {
            turn_of((double)position_of(a, b, t), a.freqs[u], &c, &s);
            c *= a.scale;
            s *= a.backward ? -a.scale : a.scale;
        }
        for (int h = 0; h < a.q.heads + a.k.heads; ++h) {
            const RotaryHeads& x = h < a.q.heads ? a.q : a.k;
            const int hh = h < a.q.heads ? h : h - a.q.heads;
            const T* from = (const T*)x.x + b * x.xb + t * x.xt + hh * x.xh;
            T* to = (T*)x.out + b * x.ob + t * x.ot + hh * x.oh;
            if (turns) {
                const float v = as_float(from[lo]), w = as_float(from[hi]);
                put(to + lo, v * c - w * s);
                put(to + hi, v * s + w * c);
            } else {
                to[lo] = from[lo];
            }
        }
    }
}

}  // namespace

int rotary(int dtype, const RotaryArgs& a, void* stream) {
    if (a.batch <= 0 || a.tokens <= 0 || a.dim <= 0 || a.q.heads + a.k.heads <= 0) return 0;
    if (dtype < 0 || dtype > 1 || a.pairs < 0 || 2 * a.pairs > a.dim || (a.pairs > 0 && a.freqs == nullptr)) return -2;
    const int64_t blocks = (a.batch * a.tokens * (a.dim - a.pairs) + kRotThreads - 1) / kRotThreads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8));
    cfg.blockDim = dim3(kRotThreads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1] = {start_early()};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)(dtype == 0 ? cudaLaunchKernelEx(&cfg, rotary_kernel<__nv_bfloat16>, a) : cudaLaunchKernelEx(&cfg, rotary_kernel<float>, a));
}

}  // namespace psb
