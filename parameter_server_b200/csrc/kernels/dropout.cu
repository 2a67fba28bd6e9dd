// Dropout with a mask that is never stored, on its way into the residual stream: out = mask(x) + residual, and its backward pass, which is
// the same without a residual.
//
// 6 bytes a value in bf16 (4 backward) beside ten rounds of the generator for four of them: twenty wide products and as many three-way XORs, which
// take the integer pipes about as long as the bytes take HBM. A thread has units of 16 bytes, whose columns are whole blocks of four random words, one
// at a time; as many warps as an SM holds hide its way through memory (a second unit on its way, or four, took registers and with them warps:
// 38 to 46 us). 16384 x 2048: bf16 36.5 us (5.5 TB/s; a plain copy 6.5), backward 32.5 (the integer pipes); fp32 64.5 (6.2).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "dropout.h"
#include "launch.cuh"
#include "philox.cuh"
#include "unaligned.cuh"

namespace psb {

namespace {

constexpr int kDropThreads = 256;
constexpr int kDropBlocks = 8;     // of an SM

struct DropParams {
    const char* x;
    int64_t ldx;                   // bytes between rows
    const char* res;
    int64_t ldres;
    char* out;
    int64_t ldo;
    int64_t rows;
    int64_t width;                 // bytes of a row
    int64_t units;                 // of a row
    int64_t row_step, unit_step;   // from one unit of a thread to its next
    int64_t x_step, x_wrap, res_step, res_wrap, out_step, out_wrap;   // the same in bytes, and where that passes the end of a row
    DropoutArgs drop;
};

// 16 bytes of a row, of which `n` exist
template <int W>
__device__ __forceinline__ uint4 load_unit(const char* p, int n) {
    if constexpr (W == 16) return *(const uint4*)p;
    else return load_across<W>(p, n);
}
// A warp's units, side by side in their rows. Rows on boundaries of 8 and 4 bytes take that many at a time (4099 x 1001 in fp32: 8.2 us, as below
// 10.1). Where they start on 2, a lane writes the aligned block that begins inside its unit, with the first bytes of the next lane's, and what no
// such block takes goes value by value (20000 x 1501 in bf16: 56.5 us, with 2 bytes of every lane at a time 77). `first`: the lane before this one
// has not the unit before this one; `next`: the lane behind has the one behind.
template <typename T, int W>
__device__ __forceinline__ void store_unit(char* p, uint4 v, int n, bool there, bool first, bool next, int n_next) {
    if constexpr (W == 16) {
        const uint32_t w[8] = {v.x, v.y, v.z, v.w, 0, 0, 0, 0};
        if (there && n >= 16) *(uint4*)p = v;
        else if (there) store_some<T>(p, w, 0, n);
    } else if constexpr (W == 8) {
        const uint32_t w[8] = {v.x, v.y, v.z, v.w, 0, 0, 0, 0};
        if (there && n >= 16) {
            *(uint2*)p = make_uint2(v.x, v.y);
            *(uint2*)(p + 8) = make_uint2(v.z, v.w);
        } else if (there) {
            store_some<T>(p, w, 0, n);
        }
    } else if constexpr (W == 4) {
        const uint32_t w[8] = {v.x, v.y, v.z, v.w, 0, 0, 0, 0};
        if (there && n >= 16) store_some<uint32_t>(p, w, 0, 16);
        else if (there) store_some<T>(p, w, 0, n);
    } else {
        uint32_t w[8] = {v.x, v.y, v.z, v.w, 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 + j] = __shfl_down_sync(0xFFFFFFFFu, w[j], 1);
        if (!there) return;
        const int ahead = (16 - (int)((uintptr_t)p & 15u)) & 15;   // bytes ahead of the first aligned block
        if (first) store_some<T>(p, w, 0, min(ahead, n));
        const int end = next ? 16 + min(ahead, n_next) : n;
        if (end - ahead >= 16) *(uint4*)(p + ahead) = from_byte<W>(w, (uint32_t)ahead);
        else store_some<T>(p, w, ahead, end);
    }
}
template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
            f[j] = __uint_as_float(w[j]);
        } else {
            f[2 * j] = __uint_as_float(w[j] << 16);
            f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float* f) {
    uint4 v;
    if constexpr (sizeof(T) == 4) {
        v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    } else {
        __nv_bfloat162* h = (__nv_bfloat162*)&v;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    }
    return v;
}

template <typename T, int W, bool RES, bool IN_MEMORY>
__global__ void __launch_bounds__(kDropThreads, kDropBlocks) dropout_kernel(const __grid_constant__ DropParams p) {
    constexpr int kColumns = 16 / (int)sizeof(T);   // of a unit
    wait_predecessor();
    allow_successor();
    const DropKeys<IN_MEMORY> key(p.drop);
    const int64_t first = (int64_t)blockIdx.x * kDropThreads + threadIdx.x;
    uint32_t row = (uint32_t)(first / p.units), unit = (uint32_t)(first - (int64_t)row * p.units);
    const uint32_t rows = (uint32_t)p.rows, row_step = (uint32_t)p.row_step, unit_step = (uint32_t)p.unit_step, per_row = (uint32_t)p.units;
    const int tail = (int)(p.width - (p.units - 1) * 16);   // bytes of a row's last unit
    const char* x = p.x + row * p.ldx + (int64_t)unit * 16;
    const char* res = RES ? p.res + row * p.ldres + (int64_t)unit * 16 : nullptr;
    char* out = p.out + row * p.ldo + (int64_t)unit * 16;
    bool there = first / p.units < p.rows;
    while (__any_sync(0xFFFFFFFFu, there)) {
        const int n = unit + 1 == per_row ? tail : 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there) {
            float f[kColumns];
            v = load_unit<W>(x, n);
            [[maybe_unused]] uint4 r;
            if constexpr (RES) r = load_unit<W>(res, n);
            unpack<T>(v, f);
#pragma unroll
            for (int j = 0; j < kColumns; j += 4) drop4(key, p.drop, row, unit * (kColumns / 4) + j / 4, f + j);
            if constexpr (RES) {
                float add[kColumns];
                unpack<T>(r, add);
#pragma unroll
                for (int j = 0; j < kColumns; ++j) f[j] += add[j];
            }
            v = pack<T>(f);
        }
        const bool ends = unit + 1 == per_row;
        store_unit<T, W>(out, v, n, there, unit == 0 || (threadIdx.x & 31) == 0, !ends && (threadIdx.x & 31) != 31, unit + 2 == per_row ? tail : 16);
        const bool wraps = unit >= per_row - unit_step;   // (unit_step < per_row)
        const uint32_t down = row_step + (wraps ? 1u : 0u);
        there = there && rows - row > down;
        row += down;
        unit = wraps ? unit - (per_row - unit_step) : unit + unit_step;
        x += wraps ? p.x_wrap : p.x_step;
        if constexpr (RES) res += wraps ? p.res_wrap : p.res_step;
        out += wraps ? p.out_wrap : p.out_step;
    }
}

template <typename T, int W>
int launch(DropParams& p, cudaStream_t s) {
    const int64_t blocks = std::min<int64_t>((p.rows * p.units + kDropThreads - 1) / kDropThreads, 148 * kDropBlocks);
    const int64_t step = blocks * kDropThreads;
    p.row_step = step / p.units;
    p.unit_step = step % p.units;
    auto steps = [&](int64_t ld, int64_t* within, int64_t* wrap) {
        *within = p.row_step * ld + p.unit_step * 16;
        *wrap = *within + ld - p.units * 16;
    };
    steps(p.ldx, &p.x_step, &p.x_wrap);
    steps(p.ldres, &p.res_step, &p.res_wrap);
    steps(p.ldo, &p.out_step, &p.out_wrap);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kDropThreads);
    cfg.stream = s;
    cudaLaunchAttribute a[1] = {start_early()};
    cfg.attrs = a;
    cfg.numAttrs = 1;
    if (p.drop.seed_ptr != nullptr)
        return (int)(p.res != nullptr ? cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, true, true>, p) : cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, false, true>, p));
    return (int)(p.res != nullptr ? cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, true, false>, p) : cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, false, false>, p));
}

}  // namespace

void dropout_keys(uint64_t seed, uint32_t* keys) { drop_keys(seed, keys); }

int dropout(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldres, void* out, int64_t ldo, int64_t rows, int64_t cols,
            const DropoutArgs& drop, void* stream) {
    if (rows <= 0 || cols <= 0) return 0;
    if (dtype < 0 || dtype > 1 || rows > 0xFFFFFFFFll || cols > 4 * 0xFFFFFFFFll) return -2;   // the generator's counter words
    const int64_t size = dtype == 0 ? 2 : 4;
    DropParams p = {(const char*)x, ldx * size, (const char*)residual, ldres * size, (char*)out, ldo * size, rows, cols * size, (cols * size + 15) / 16, 0, 0, 0, 0, 0, 0, 0, 0, drop};
    uint64_t low = (uint64_t)p.x | (uint64_t)p.out | (uint64_t)p.res;
    if (rows > 1) low |= (uint64_t)p.ldx | (uint64_t)p.ldo | (p.res != nullptr ? (uint64_t)p.ldres : 0);
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == 0) {
        if (low % 16 == 0) return launch<__nv_bfloat16, 16>(p, s);
        if (low % 8 == 0) return launch<__nv_bfloat16, 8>(p, s);
        if (low % 4 == 0) return launch<__nv_bfloat16, 4>(p, s);
        return launch<__nv_bfloat16, 2>(p, s);
    }
    if (low % 16 == 0) return launch<float, 16>(p, s);
    if (low % 8 == 0) return launch<float, 8>(p, s);
    return launch<float, 4>(p, s);
}

}  // namespace psb
