// Dropout with a mask that is never stored, on its way into the residual stream: out = mask(x) + residual, and its backward pass, which is
// the same without a residual.
//
// 6 bytes a value in bf16 (4 backward) beside ten rounds of the generator for four of them: twenty wide products and as many three-way XORs, which
// take about as long as the bytes take HBM: the half of the FMA pipe that has the wide products is busy 72 % of the time (76 % backward), the ALU,
// which has the XORs, 58 %, HBM 61 % (34 %). A thread has units of 16 bytes, whose columns are whole blocks of four random words; in
// bf16, where there are many, of 32: their four blocks share what hangs on the row alone, and are four chains side by side. 16384 x 2048: bf16 31 us
// (6.5 TB/s, as a plain copy; 16 bytes at a time 36), backward 28 (33: the wide products); fp32 59 (6.8). A second unit on its way while one is worked
// on, or four, took registers and with them warps: 38 to 46 us.
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
constexpr int kDropBlocksWide = 4; // with 32 bytes of a thread at a time
constexpr int kDropRuns = 4;       // units of a thread where there are many
constexpr int64_t kDropMany = 148ll * kDropBlocks * kDropThreads * 32;   // bytes

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

// U times 16 bytes of a row, of which `n` exist, by aligned blocks, which never reach past an allocation. (Of rows on 16-byte boundaries two only
// where they hold whole ones.)
template <int W, int U>
__device__ __forceinline__ void load_unit(const char* p, int n, uint4* v) {
    if constexpr (W == 16) {
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = *(const uint4*)(p + 16 * i);
    } else {
        const int past = (int)((uintptr_t)p & 15u);
        uint4 blocks[U + 1];
#pragma unroll
        for (int i = 0; i <= U; ++i) blocks[i] = 16 * i < past + n ? *(const uint4*)(p - past + 16 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            uint32_t w[8] = {blocks[i].x, blocks[i].y, blocks[i].z, blocks[i].w, blocks[i + 1].x, blocks[i + 1].y, blocks[i + 1].z, blocks[i + 1].w};
            v[i] = from_byte<W>(w, (uint32_t)past);
        }
    }
}
// A warp's units, side by side in their rows. Rows on boundaries of 8 and 4 bytes take that many at a time (4099 x 1001 in fp32: 8.2 us, as below
// 10.1). Where they start on 2, a lane writes the aligned blocks that begin inside its unit, the last of them with the first bytes of the next lane's,
// and what no such block takes goes value by value (20000 x 1501 in bf16 by 2 bytes of every lane at a time: 77 us for 56, and with 32 bytes to a thread 50). `first`: the lane before
// this one has not the unit before this one; `next`: the lane behind has the one behind, of which `n_next` bytes exist.
template <typename T, int W, int U>
__device__ __forceinline__ void store_unit(char* p, const uint4* v, int n, bool there, bool first, bool next, int n_next) {
    if constexpr (W > 2) {
        if (!there) return;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t w[8] = {v[i].x, v[i].y, v[i].z, v[i].w, 0, 0, 0, 0};
            char* to = p + 16 * i;
            const int have = W == 16 && U > 1 ? 16 : n - 16 * i;
            if (have < 16) {
                store_some<T>(to, w, 0, have);
            } else if constexpr (W == 16) {
                *(uint4*)to = v[i];
            } else if constexpr (W == 8) {
                *(uint2*)to = make_uint2(v[i].x, v[i].y);
                *(uint2*)(to + 8) = make_uint2(v[i].z, v[i].w);
            } else {
                store_some<uint32_t>(to, w, 0, 16);
            }
        }
    } else {
        uint32_t w[4 * U + 4];
#pragma unroll
        for (int i = 0; i < U; ++i) { w[4 * i] = v[i].x; w[4 * i + 1] = v[i].y; w[4 * i + 2] = v[i].z; w[4 * i + 3] = v[i].w; }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * U + j] = __shfl_down_sync(0xFFFFFFFFu, w[j], 1);
        if (!there) return;
        const int ahead = (16 - (int)((uintptr_t)p & 15u)) & 15;   // bytes ahead of the first aligned block
        if (first) store_some<T>(p, w, 0, min(ahead, n));
        const int end = next ? 16 * U + min(ahead, n_next) : n;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (end - 16 * i - ahead >= 16) {
                uint32_t t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = w[4 * i + j];
                *(uint4*)(p + 16 * i + ahead) = from_byte<W>(t, (uint32_t)ahead);
            } else {
                store_some<T>(p + 16 * i, w + 4 * i, ahead, end - 16 * i);
            }
        }
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

template <typename T, int W, int U, bool RES, bool IN_MEMORY>
__global__ void __launch_bounds__(kDropThreads, U == 1 ? kDropBlocks : kDropBlocksWide) dropout_kernel(const __grid_constant__ DropParams p) {
    constexpr int kColumns = 16 / (int)sizeof(T), kBytes = 16 * U;   // of 16 bytes; of a unit
    wait_predecessor();
    allow_successor();
    const DropKeys<IN_MEMORY> key(p.drop);
    const int64_t first = (int64_t)blockIdx.x * kDropThreads + threadIdx.x;
    uint32_t row = (uint32_t)(first / p.units), unit = (uint32_t)(first - (int64_t)row * p.units);
    const uint32_t rows = (uint32_t)p.rows, row_step = (uint32_t)p.row_step, unit_step = (uint32_t)p.unit_step, per_row = (uint32_t)p.units;
    const int tail = (int)(p.width - (p.units - 1) * kBytes);   // bytes of a row's last unit
    const char* x = p.x + row * p.ldx + (int64_t)unit * kBytes;
    const char* res = RES ? p.res + row * p.ldres + (int64_t)unit * kBytes : nullptr;
    char* out = p.out + row * p.ldo + (int64_t)unit * kBytes;
    bool there = first / p.units < p.rows;
    while (W == 2 ? __any_sync(0xFFFFFFFFu, there) : there) {   // (stores on 2-byte boundaries are a warp's)
        const bool ends = unit + 1 == per_row;
        const int n = ends ? tail : kBytes;
        uint4 v[U];
        if (there) {
            [[maybe_unused]] uint4 r[U];
            load_unit<W, U>(x, n, v);
            if constexpr (RES) load_unit<W, U>(res, n, r);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float f[kColumns];
                unpack<T>(v[i], f);
#pragma unroll
                for (int j = 0; j < kColumns; j += 4) drop4(key, p.drop, row, (unit * U + i) * (kColumns / 4) + j / 4, f + j);
                if constexpr (RES) {
                    float add[kColumns];
                    unpack<T>(r[i], add);
#pragma unroll
                    for (int j = 0; j < kColumns; ++j) f[j] += add[j];
                }
                v[i] = pack<T>(f);
            }
        }
        store_unit<T, W, U>(out, v, n, there, unit == 0 || (threadIdx.x & 31) == 0, !ends && (threadIdx.x & 31) != 31, unit + 2 == per_row ? tail : kBytes);
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

template <typename T, int W, int U>
int launch(DropParams& p, cudaStream_t s) {
    p.units = (p.width + 16 * U - 1) / (16 * U);
    // as many blocks as run at once, or more with kDropRuns units to a thread: blocks that are dealt out as others end
    const int64_t need = (p.rows * p.units + kDropThreads - 1) / kDropThreads;
    const int64_t blocks = std::min(need, std::max<int64_t>(148 * kDropBlocks, (need + kDropRuns - 1) / kDropRuns));
    if (blocks > 0x7FFFFFFF) return -2;
    const int64_t step = blocks * kDropThreads;
    p.row_step = step / p.units;
    p.unit_step = step % p.units;
    auto steps = [&](int64_t ld, int64_t* within, int64_t* wrap) {
        *within = p.row_step * ld + p.unit_step * (16 * U);
        *wrap = *within + ld - p.units * (16 * U);
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
        return (int)(p.res != nullptr ? cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, U, true, true>, p) : cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, U, false, true>, p));
    return (int)(p.res != nullptr ? cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, U, true, false>, p) : cudaLaunchKernelEx(&cfg, dropout_kernel<T, W, U, false, false>, p));
}

}  // namespace

void dropout_keys(uint64_t seed, uint32_t* keys) { drop_keys(seed, keys); }

int dropout(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldres, void* out, int64_t ldo, int64_t rows, int64_t cols,
            const DropoutArgs& drop, void* stream) {
    if (rows <= 0 || cols <= 0) return 0;
    if (dtype < 0 || dtype > 1 || rows > 0xFFFFFFFFll || cols > 4 * 0xFFFFFFFFll) return -2;   // the generator's counter words
    const int64_t size = dtype == 0 ? 2 : 4;
    DropParams p = {(const char*)x, ldx * size, (const char*)residual, ldres * size, (char*)out, ldo * size, rows, cols * size, 0, 0, 0, 0, 0, 0, 0, 0, 0, drop};
    uint64_t low = (uint64_t)p.x | (uint64_t)p.out | (uint64_t)p.res;
    if (rows > 1) low |= (uint64_t)p.ldx | (uint64_t)p.ldo | (p.res != nullptr ? (uint64_t)p.ldres : 0);
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == 0) {
        const bool many = p.rows * p.width >= kDropMany;
        if (low % 16 == 0) return many && p.width % 32 == 0 ? launch<__nv_bfloat16, 16, 2>(p, s) : launch<__nv_bfloat16, 16, 1>(p, s);
        if (low % 8 == 0) return many ? launch<__nv_bfloat16, 8, 2>(p, s) : launch<__nv_bfloat16, 8, 1>(p, s);
        if (low % 4 == 0) return many ? launch<__nv_bfloat16, 4, 2>(p, s) : launch<__nv_bfloat16, 4, 1>(p, s);
        return many ? launch<__nv_bfloat16, 2, 2>(p, s) : launch<__nv_bfloat16, 2, 1>(p, s);
    }
    if (low % 16 == 0) return launch<float, 16, 1>(p, s);
    if (low % 8 == 0) return launch<float, 8, 1>(p, s);
    return launch<float, 4, 1>(p, s);
}

}  // namespace psb
