// Dropout with a mask that is never stored, on its way into the residual stream: out = mask(x) + residual, and its backward pass, which is
// the same without a residual. One thread has four neighbouring columns, the values of one block of random words.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "dropout.h"
#include "launch.cuh"
#include "philox.cuh"

namespace psb {

namespace {

constexpr int kDropThreads = 256;

struct DropParams {
    const void* x;
    int64_t ldx;
    const void* res;
    int64_t ldres;
    void* out;
    int64_t ldo;
    int64_t rows, cols, units;   // blocks of four columns in a row
    DropoutArgs drop;
};

__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

template <typename T>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const __grid_constant__ DropParams p) {
    wait_predecessor();
    allow_successor();
    const DropKey key = drop_key(p.drop);
    const int64_t total = p.rows * p.units;
    for (int64_t i = (int64_t)blockIdx.x * kDropThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kDropThreads) {
        const int64_t row = i / p.units, unit = i - row * p.units, n = p.cols - 4 * unit;
        const T* x = (const T*)p.x + row * p.ldx + 4 * unit;
        const T* res = (const T*)p.res + row * p.ldres + 4 * unit;
        T* out = (T*)p.out + row * p.ldo + 4 * unit;
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = j < n ? as_float(x[j]) : 0.f;
        drop4(key, p.drop.threshold, p.drop.scale, (uint32_t)row, (uint32_t)unit, f);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) put(out + j, p.res == nullptr ? f[j] : f[j] + as_float(res[j]));
    }
}

}  // namespace

int dropout(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldres, void* out, int64_t ldo, int64_t rows, int64_t cols,
            const DropoutArgs& drop, void* stream) {
    if (rows <= 0 || cols <= 0) return 0;
    if (dtype < 0 || dtype > 1 || rows > 0xFFFFFFFFll || cols > 4 * 0xFFFFFFFFll) return -2;   // the generator's counter words
    const DropParams p = {x, ldx, residual, ldres, out, ldo, rows, cols, (cols + 3) / 4, drop};
    const int64_t blocks = (rows * p.units + kDropThreads - 1) / kDropThreads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8));
    cfg.blockDim = dim3(kDropThreads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute a[1] = {start_early()};
    cfg.attrs = a;
    cfg.numAttrs = 1;
    return (int)(dtype == 0 ? cudaLaunchKernelEx(&cfg, dropout_kernel<__nv_bfloat16>, p) : cudaLaunchKernelEx(&cfg, dropout_kernel<float>, p));
}

}  // namespace psb
