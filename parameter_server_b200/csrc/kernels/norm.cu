// Layer norm forward and backward, 8-bit checkpoints of rows, and column sums with a fixed order: the memory-bound
// operators of a decoder block (the consumer of dense tables; the reference is a storage service and has no model code).
//
//   forward   mean = sum(x) / d,  rstd = 1 / sqrt(sum((x - mean)^2) / d + eps),  y = xhat * weight + bias
//   backward  p = dy * weight:  dx = rstd * (p - sum(p) / d - xhat * sum(p * xhat) / d)  (+ the residual branch's gradient)
//             dweight = sum_rows dy * xhat,  dbias = sum_rows dy
//
// All of it is bound by HBM: a row is read once, kept in registers between the statistics and the output (the squared
// distances are taken from the mean, not as a difference of sums), and written once. Sums and statistics are fp32.
// 16384 x 2048 in bf16, back to back in a graph: forward 24 us (5.6 TB/s), with the 8-bit rows 32 us (5.3), backward 37 us (5.4; 47
// with a residual gradient, 5.7), from 8-bit rows 42 us (4.0: conversions take their share), column sums 10 us (L2), packing and
// unpacking 17 us (5.9). A plain copy reaches 6.5 TB/s. 16 rows: 3 us forward, 4.5 backward, most of it the launch.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "act8.cuh"
#include "launch.cuh"
#include "norm.h"

namespace psb {

namespace {

constexpr int kMaxTeam = 512;        // threads that share one row
constexpr int kBwdThreads = 512;
constexpr int kBwdElems = 16;        // columns per thread of the backward kernel: two fp32 sums each stay in registers
constexpr int kSms = 148;

// VEC consecutive values of a row as fp32: one 16-byte access, two bf16 (rows on 4-byte boundaries), or one element.
template <typename T, int VEC>
struct Io;
template <>
struct Io<__nv_bfloat16, 8> {
    using Raw = uint4;
    static __device__ __forceinline__ Raw load(const __nv_bfloat16* p) { return *(const uint4*)p; }
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) {
        uint4 r;
        __nv_bfloat162* h = (__nv_bfloat162*)&r;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        *(uint4*)p = r;
    }
    static __device__ __forceinline__ Raw zero() { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ Raw one() { return make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u); }
};
template <>
struct Io<float, 4> {
    using Raw = float4;
    static __device__ __forceinline__ Raw load(const float* p) { return *(const float4*)p; }
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w; }
    static __device__ __forceinline__ void store(float* p, const float* f) { *(float4*)p = make_float4(f[0], f[1], f[2], f[3]); }
    static __device__ __forceinline__ Raw zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
    static __device__ __forceinline__ Raw one() { return make_float4(1.f, 1.f, 1.f, 1.f); }
};
template <>
struct Io<__nv_bfloat16, 2> {
    using Raw = uint32_t;
    static __device__ __forceinline__ Raw load(const __nv_bfloat16* p) { return *(const uint32_t*)p; }
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
        f[0] = __uint_as_float(r << 16);
        f[1] = __uint_as_float(r & 0xFFFF0000u);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) { *(__nv_bfloat162*)p = __floats2bfloat162_rn(f[0], f[1]); }
    static __device__ __forceinline__ Raw zero() { return 0u; }
    static __device__ __forceinline__ Raw one() { return 0x3F803F80u; }
};
template <>
struct Io<__nv_bfloat16, 1> {
    using Raw = __nv_bfloat16;
    static __device__ __forceinline__ Raw load(const __nv_bfloat16* p) { return *p; }
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = __bfloat162float(r); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) { *p = __float2bfloat16_rn(f[0]); }
    static __device__ __forceinline__ Raw zero() { return __float2bfloat16_rn(0.f); }
    static __device__ __forceinline__ Raw one() { return __float2bfloat16_rn(1.f); }
};
template <>
struct Io<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ Raw load(const float* p) { return *p; }
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = r; }
    static __device__ __forceinline__ void store(float* p, const float* f) { *p = f[0]; }
    static __device__ __forceinline__ Raw zero() { return 0.f; }
    static __device__ __forceinline__ Raw one() { return 1.f; }
};

// VEC consecutive whole numbers of a checkpoint row
template <int VEC>
struct Q8;
__device__ __forceinline__ void unpack_word(uint32_t w, float step, float* f) {
    const uint32_t biased = w ^ 0x80808080u;
    f[0] = s8_of_biased<0>(biased) * step;
    f[1] = s8_of_biased<1>(biased) * step;
    f[2] = s8_of_biased<2>(biased) * step;
    f[3] = s8_of_biased<3>(biased) * step;
}
__device__ __forceinline__ uint32_t pack_word(const float* f, uint32_t e, float inverse_step) {
    return e == 255u ? 0u : act8_quantise4(f[0], f[1], f[2], f[3], inverse_step);
}
template <>
struct Q8<8> {
    using Raw = uint2;
    static __device__ __forceinline__ Raw load(const int8_t* p) { return *(const uint2*)p; }
    static __device__ __forceinline__ Raw zero() { return make_uint2(0, 0); }
    static __device__ __forceinline__ void unpack(const Raw& r, float step, float* f) {
        unpack_word(r.x, step, f);
        unpack_word(r.y, step, f + 4);
    }
    static __device__ __forceinline__ void store(int8_t* p, const float* f, uint32_t e, float inv) {
        *(uint2*)p = make_uint2(pack_word(f, e, inv), pack_word(f + 4, e, inv));
    }
};
template <>
struct Q8<4> {
    using Raw = uint32_t;
    static __device__ __forceinline__ Raw load(const int8_t* p) { return *(const uint32_t*)p; }
    static __device__ __forceinline__ Raw zero() { return 0u; }
    static __device__ __forceinline__ void unpack(const Raw& r, float step, float* f) { unpack_word(r, step, f); }
    static __device__ __forceinline__ void store(int8_t* p, const float* f, uint32_t e, float inv) { *(uint32_t*)p = pack_word(f, e, inv); }
};
template <>
struct Q8<2> {
    using Raw = uint16_t;
    static __device__ __forceinline__ Raw zero() { return 0; }
    static __device__ __forceinline__ void store(int8_t* p, const float* f, uint32_t, float inv) {
        *(uint16_t*)p = (uint16_t)((act8_quantise(f[0], inv) & 255) | (act8_quantise(f[1], inv) & 255) << 8);
    }
};
template <>
struct Q8<1> {
    using Raw = int8_t;
    static __device__ __forceinline__ Raw load(const int8_t* p) { return *p; }
    static __device__ __forceinline__ Raw zero() { return 0; }
    static __device__ __forceinline__ void unpack(const Raw& r, float step, float* f) { f[0] = (float)r * step; }
    static __device__ __forceinline__ void store(int8_t* p, const float* f, uint32_t, float inv) { *p = (int8_t)act8_quantise(f[0], inv); }
};

// Copies of a thread's own 4, 8 or 16 bytes from global to shared memory, any number in flight; a group is what was issued since
// the group before.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
template <typename V>
__device__ __forceinline__ V from_shared(uint32_t addr) { return *(const V*)__cvta_shared_to_generic(addr); }
__device__ __forceinline__ void close_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void wait_groups() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Eight bf16 of a row on any 2-byte boundary ("loose"), beside eight whole numbers of a checkpoint: the aligned words that hold them,
// five at most, on their way and in shared memory (a stride of five words: no bank conflicts), shifted by half a word where the row
// starts on one. `m` of the eight exist. 16384 x 1001, one value at a time and so, us: backward from 8-bit rows 90, 39; from x one at a
// time is faster, since its accesses lie side by side: 29, 42.
constexpr int kLooseBytes = 20;
__device__ __forceinline__ uint32_t half_of(const void* p) { return (uint32_t)(uintptr_t)p & 2u; }
__device__ __forceinline__ void loose_copy(uint32_t dst, const __nv_bfloat16* p, int m) {
    const uint32_t odd = half_of(p);
    const char* w = (const char*)p - odd;
    const int words = ((int)odd + 2 * m + 3) / 4;
#pragma unroll
    for (int k = 0; k < 5; ++k)
        if (k < words) copy_async<4>(dst + 4 * k, w + 4 * k);
}
__device__ __forceinline__ uint4 loose_read(uint32_t src, uint32_t odd, int m) {
    uint32_t w[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = from_shared<uint32_t>(src + 4 * k);
    const uint32_t shift = odd * 8;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], shift);
    if (m < 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = 2 * k >= m ? 0u : 2 * k + 1 >= m ? w[k] & 0xFFFFu : w[k];
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 loose_load(const __nv_bfloat16* p, int m) {   // straight from memory: once per kernel
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < m) w[j / 2] |= (uint32_t)((const unsigned short*)p)[j] << (16 * (j & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void loose_store(__nv_bfloat16* p, const float* f, int m) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
        w[k] = *(const uint32_t*)&h;
    }
    unsigned short* o = (unsigned short*)p;
    if (m < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < m) o[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
    } else if (half_of(p) == 0u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) *(uint32_t*)(o + 2 * k) = w[k];
    } else {
        o[0] = (unsigned short)w[0];
#pragma unroll
        for (int k = 0; k < 3; ++k) *(uint32_t*)(o + 2 * k + 1) = __funnelshift_r(w[k], w[k + 1], 16);
        o[7] = (unsigned short)(w[3] >> 16);
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
// exponent of the block of 32 columns that 32 / VEC neighbouring lanes share (all lanes of the warp call)
template <int VEC>
__device__ __forceinline__ uint32_t block_exponent(const float* f, bool valid) {
    float m = 0.f;
    if (valid) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = abs_max(m, f[j]);
    }
    uint32_t v = abs_bits(m);
    if constexpr (VEC == 1) {
        v = __reduce_max_sync(0xFFFFFFFFu, v);
    } else {
#pragma unroll
        for (int o = kAct8Block / VEC / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    }
    return act8_exponent(v);
}

// Quantises the VEC values of this thread (col = first column; all lanes of the warp call, `valid` false past the row).
template <int VEC>
__device__ __forceinline__ void keep8(const float* f, bool valid, int8_t* qrow, uint8_t* erow, int col) {
    const uint32_t e = block_exponent<VEC>(f, valid);
    if (!valid) return;
    Q8<VEC>::store(qrow + col, f, e, act8_inverse_step(e));
    if (col % kAct8Block == 0) erow[col / kAct8Block] = (uint8_t)e;
}

// ---- forward ---------------------------------------------------------------------------------------------------------
// `tpr` threads (a power of two, 32..512) hold one row in registers, NV vectors each: thread t has the columns
// (i * tpr + t) * VEC, and its part of weight and bias, packed, over all rows. (A warp per row up to d = 2048 needs no barrier,
// but its 64 values a lane leave no registers for the weight, and 4 warps per scheduler do not hide its loads: 39 us.)
// With few rows a row is spread over as many threads as have a vector each, since then the latency of one row is the time.
// CTAs are persistent, and a thread copies its part of the next two rows to shared memory while it works on this one (only
// the thread itself reads it, so no barrier is involved): with loads straight into registers a row's arithmetic and the next
// row's latency add up (16384 x 2048: 35 us). bf16 rows on 4-byte boundaries go in pairs (10923 x 2086: 29 us, one by one 47); on
// none (VEC 1; a copy has 4 bytes at least) they are read straight into registers all the same.
constexpr int kFwdSlots = 3;
template <typename T, int VEC>
constexpr bool copies_ahead() { return VEC * sizeof(T) >= 4; }
// TPR: `tpr` known to the compiler, so that a thread's places in the row and in the ring are constants; 0 = `tpr_arg` (few rows).
template <typename T, int VEC, int NV, bool OUT8, int TPR>
__global__ void __launch_bounds__(TPR == 0 ? kMaxTeam : TPR == 32 ? 128 : TPR)
layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ weight, const T* __restrict__ bias, T* __restrict__ y,
                      int64_t ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out, int8_t* q, int64_t ldq, uint8_t* e,
                      int64_t lde, int64_t rows, int d, float eps, int tpr_arg) {
    allow_successor();
    const int tpr = TPR > 0 ? TPR : tpr_arg, threads = TPR == 0 ? (int)blockDim.x : TPR == 32 ? 128 : TPR;
    constexpr bool kAsync = copies_ahead<T, VEC>();
    constexpr int kVecBytes = VEC * (int)sizeof(T);
    using IO = Io<T, VEC>;
    extern __shared__ uint4 ring[];   // [kFwdSlots][NV][threads] vectors
    __shared__ float red[2][kMaxTeam / 32];
    const int team = threadIdx.x / tpr, t = threadIdx.x % tpr, teams = threads / tpr;
    const int warps = tpr / 32, w0 = team * warps;
    const int nv = t * VEC < d ? min(NV, (d - t * VEC + tpr * VEC - 1) / (tpr * VEC)) : 0;   // this thread's vectors that exist
    const int64_t step = (int64_t)gridDim.x * teams, first = (int64_t)blockIdx.x * teams;
    typename IO::Raw graw[NV], braw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * tpr + t) * VEC;
        graw[i] = weight != nullptr && col < d ? IO::load(weight + col) : IO::one();
        braw[i] = bias != nullptr && col < d ? IO::load(bias + col) : IO::zero();
    }
    // running positions: a row's overhead is shared by 32 values only
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * kVecBytes, vec_stride = threads * kVecBytes, slot_stride = NV * vec_stride;
    const T* ahead = x + (first + team) * ldx + t * VEC;
    int64_t ahead_row = first + team;
    auto request = [&](int slot) {   // the next row that has not been asked for
        if (ahead_row < rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < nv) copy_async<kAsync ? kVecBytes : 4>(mine + slot * slot_stride + i * vec_stride, ahead + i * tpr * VEC);
        }
        close_group();   // (an empty group where there is no such row: the count of groups stays the same)
        ahead += step * ldx;
        ahead_row += step;
    };
    int slot = 0;
    if constexpr (kAsync) {
#pragma unroll
        for (int k = 0; k < kFwdSlots - 1; ++k) request(k);
    }
    for (int64_t base = first; base < rows; base += step) {
        const int64_t row = base + team;
        const bool live = row < rows;
        float v[NV * VEC];
        if constexpr (kAsync) {
            request(slot == 0 ? kFwdSlots - 1 : slot - 1);
            wait_groups<kFwdSlots - 1>();
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + t) * VEC;
            typename IO::Raw raw = IO::zero();
            if (live && i < nv) {
                if constexpr (kAsync) raw = from_shared<typename IO::Raw>(mine + slot * slot_stride + i * vec_stride);
                else raw = IO::load(x + row * ldx + col);
            }
            IO::unpack(raw, v + i * VEC);
        }
        slot = slot + 1 == kFwdSlots ? 0 : slot + 1;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) s += v[i];
        auto team_sum = [&](float part, int k) -> float {
            part = warp_sum(part);
            if (warps == 1) return part;
            if ((threadIdx.x & 31) == 0) red[k][threadIdx.x >> 5] = part;
            __syncthreads();
            float all = 0.f;
            for (int w = 0; w < warps; ++w) all += red[k][w0 + w];
            return all;
        };
        const float mean = team_sum(s, 0) / (float)d;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = i < nv;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i * VEC + j] -= mean;
                if (in) s += v[i * VEC + j] * v[i * VEC + j];
            }
        }
        const float rstd = __frsqrt_rn(team_sum(s, 1) / (float)d + eps);
        if (live && t == 0) {
            if (mean_out != nullptr) mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + t) * VEC;
            const bool in = live && i < nv;
            float* f = v + i * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] *= rstd;
            if constexpr (OUT8) keep8<VEC>(f, in, q + (live ? row : 0) * ldq, e + (live ? row : 0) * lde, col);
            if (!in) continue;
            float g[VEC], b[VEC];
            IO::unpack(graw[i], g);
            IO::unpack(braw[i], b);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j], g[j], b[j]);
            IO::store(y + row * ldy + col, f);
        }
    }
}

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float all = 0.f;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) all += red[w];
    return all;
}

// Rows longer than registers hold: a CTA per row, the row is read again (from L2) for each statistic, an element at a time:
// 2048 x 32768 in bf16 233 us (1.15 TB/s), where 4096 x 16384 takes 48.
template <typename T, bool OUT8>
__global__ void __launch_bounds__(512)
layer_norm_fwd_long_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ weight, const T* __restrict__ bias,
                           T* __restrict__ y, int64_t ldy, float* mean_out, float* rstd_out, int8_t* q, int64_t ldq, uint8_t* e,
                           int64_t lde, int d, float eps) {
    allow_successor();
    __shared__ float red[16];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    float s = 0.f, f;
    for (int c = threadIdx.x; c < d; c += blockDim.x) { Io<T, 1>::unpack(xr[c], &f); s += f; }
    const float mean = block_sum(s, red) / (float)d;
    s = 0.f;
    for (int c = threadIdx.x; c < d; c += blockDim.x) { Io<T, 1>::unpack(xr[c], &f); s += (f - mean) * (f - mean); }
    const float rstd = __frsqrt_rn(block_sum(s, red) / (float)d + eps);
    if (threadIdx.x == 0) {
        if (mean_out != nullptr) mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    for (int c0 = 0; c0 < d; c0 += blockDim.x) {
        const int c = c0 + threadIdx.x;
        float h = 0.f, g = 1.f, b = 0.f;
        if (c < d) {
            Io<T, 1>::unpack(xr[c], &f);
            h = (f - mean) * rstd;
            if (weight != nullptr) Io<T, 1>::unpack(weight[c], &g);
            if (bias != nullptr) Io<T, 1>::unpack(bias[c], &b);
            const float o = h * g + b;
            Io<T, 1>::store(y + row * ldy + c, &o);
        }
        if constexpr (OUT8) keep8<1>(&h, c < d, q + row * ldq, e + row * lde, c);
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------
// Persistent CTAs (one per SM) of blockDim / tpr teams; a team walks rows and thread t keeps the sums of its 16 columns'
// dweight and dbias in registers over all of them, so that the weight's gradient costs no second pass over dy and x. The
// next rows are copied to shared memory meanwhile, every thread its own part (see the forward kernel; loads into registers
// left room for one row in flight and took 67 us for 16384 x 2048 with a residual gradient). The two row sums cross the
// team's warps through shared memory with one barrier per row. At the end the teams' sums are added in a tree and leave
// as one partial row per CTA, which column_reduce_kernel adds in CTA order: the result does not depend on timing. (More CTAs
// per SM would write and read more partial rows: 2 * d floats each.)
template <typename T, int VEC, bool SRC8, bool LOOSE>
struct BwdRing {
    static constexpr int kVecs = kBwdElems / VEC, kVecBytes = LOOSE ? kLooseBytes : VEC * (int)sizeof(T);
    static constexpr bool kAsync = LOOSE || copies_ahead<T, VEC>() && (VEC >= 4 || !SRC8);   // (a vector of q has VEC bytes)
    static constexpr int kSlots = sizeof(T) == 2 ? 3 : 2;
    // per thread and slot: dy, the residual's gradient, and x or (8 or 4 bytes a vector) q with a word of exponents
    static constexpr int kRowBytes = SRC8 ? kVecs * (2 * kVecBytes + VEC + 4) : kVecs * 3 * kVecBytes;
    static constexpr int kBytes = kAsync ? kSlots * kRowBytes * kBwdThreads : 0;
};

// TPR: threads that share a row, known to the compiler, so that a thread's places in the row and in the ring are constants (with
// a run-time value an element took twice the instructions); 0 = `tpr_arg` (8-bit rows beside fp32 ones that are not aligned).
template <typename T, int VEC, bool SRC8, int TPR, bool LOOSE>
__global__ void __launch_bounds__(kBwdThreads, 1)
layer_norm_bwd_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, const int8_t* __restrict__ q,
                      int64_t ldq, const uint8_t* __restrict__ e, int64_t lde, const T* __restrict__ weight,
                      const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const T* __restrict__ join, int64_t ldjoin,
                      T* __restrict__ dx, int64_t lddx, float* __restrict__ partial, int64_t rows, int d, int tpr_arg) {
    allow_successor();
    constexpr int NV = kBwdElems / VEC;
    const int tpr = TPR > 0 ? TPR : tpr_arg;
    using IO = Io<T, VEC>;
    using Ring = BwdRing<T, VEC, SRC8, LOOSE>;
    constexpr bool kAsync = Ring::kAsync;
    constexpr int kVecBytes = Ring::kVecBytes, kCopy = kAsync && !LOOSE ? kVecBytes : 4, kCopyQ = kAsync && SRC8 ? VEC : 4;
    extern __shared__ uint4 ring_raw[];         // the ring; at the end sums of the teams
    __shared__ float red[2][kBwdThreads / 32][2];
    const int team = threadIdx.x / tpr, t = threadIdx.x % tpr, teams = blockDim.x / tpr;
    const int warps = tpr / 32, w0 = team * warps, lane = threadIdx.x & 31;
    float dg[kBwdElems], db[kBwdElems];
    typename IO::Raw graw[NV];
#pragma unroll
    for (int i = 0; i < kBwdElems; ++i) dg[i] = db[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * tpr + t) * VEC;
        if constexpr (LOOSE) graw[i] = weight != nullptr ? loose_load(weight + col, d - col) : IO::one();
        else graw[i] = weight != nullptr && col < d ? IO::load(weight + col) : IO::one();
    }
    const float inv_d = 1.f / (float)d;
    // Running positions: a row's overhead is shared by 16 values only. In a slot the thread's vectors of dy, of the residual's
    // gradient, and of x (or of q and the exponents' words) follow one another with `n` threads between them.
    constexpr uint32_t n = kBwdThreads;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring_raw);
    const uint32_t my_y = base + threadIdx.x * kVecBytes;
    const uint32_t ring2 = base + Ring::kSlots * 2 * NV * n * kVecBytes;
    const uint32_t my_q = ring2 + threadIdx.x * VEC, my_e = ring2 + Ring::kSlots * NV * n * VEC + threadIdx.x * 4;
    auto at_y = [&](int s, int i) { return my_y + (uint32_t)((s * 2 + 0) * NV + i) * n * kVecBytes; };
    auto at_j = [&](int s, int i) { return my_y + (uint32_t)((s * 2 + 1) * NV + i) * n * kVecBytes; };
    auto at_x = [&](int s, int i) { return my_y + (uint32_t)(Ring::kSlots * 2 * NV + s * NV + i) * n * kVecBytes; };
    auto at_q = [&](int s, int i) { return my_q + (uint32_t)(s * NV + i) * n * VEC; };
    auto at_e = [&](int s, int i) { return my_e + (uint32_t)(s * NV + i) * n * 4; };
    const int64_t step = (int64_t)gridDim.x * teams, first = (int64_t)blockIdx.x * teams + team;
    const int c0 = t * VEC;
    const int nv = c0 < d ? min(NV, (d - c0 + tpr * VEC - 1) / (tpr * VEC)) : 0;   // this thread's vectors that exist
    const T *ahead_y = dy + first * lddy + c0, *ahead_x = SRC8 ? nullptr : x + first * ldx + c0, *ahead_j = join != nullptr ? join + first * ldjoin + c0 : nullptr;
    const int8_t* ahead_q = SRC8 ? q + first * ldq + c0 : nullptr;
    const uint8_t* ahead_e = SRC8 ? e + first * lde : nullptr;
    int64_t ahead_row = first;
    auto copy = [&](uint32_t to, const T* from, int i) {
        if constexpr (LOOSE) loose_copy(to, from, min(VEC, d - c0 - i * tpr * VEC));
        else copy_async<kCopy>(to, from);
    };
    auto fetched = [&](uint32_t at, const T* row_start, int i) -> typename IO::Raw {
        if constexpr (LOOSE) return loose_read(at, half_of(row_start), d - c0 - i * tpr * VEC);
        else return from_shared<typename IO::Raw>(at);
    };
    auto request = [&](int s) {   // the next row that has not been asked for
        if constexpr (kAsync) {
            if (ahead_row < rows) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int off = i * tpr * VEC;
                    if (i >= nv) continue;
                    copy(at_y(s, i), ahead_y + off, i);
                    if (join != nullptr) copy(at_j(s, i), ahead_j + off, i);
                    if constexpr (SRC8) {
                        copy_async<kCopyQ>(at_q(s, i), ahead_q + off);
                        copy_async<4>(at_e(s, i), ahead_e + (c0 + off) / (4 * kAct8Block) * 4);   // the exponents of 128 columns
                    } else {
                        copy(at_x(s, i), ahead_x + off, i);
                    }
                }
            }
            close_group();
            ahead_row += step;
            ahead_y += step * lddy;
            if constexpr (SRC8) {
                ahead_q += step * ldq;
                ahead_e += step * lde;
            } else {
                ahead_x += step * ldx;
            }
            if (join != nullptr) ahead_j += step * ldjoin;
        }
    };
#pragma unroll
    for (int k = 0; k < Ring::kSlots - 1; ++k) request(k);
    T* dx_row = dx + first * lddx + c0;
    float next_rstd = first < rows ? rstd_in[first] : 0.f, next_mean = !SRC8 && first < rows ? mean_in[first] : 0.f;
    int buf = 0, slot = 0;
    for (int64_t row = first; row < rows; row += step, buf ^= 1) {
        request(slot == 0 ? Ring::kSlots - 1 : slot - 1);
        const float rstd = next_rstd, mean = next_mean;
        if (row + step < rows) {
            next_rstd = rstd_in[row + step];
            if constexpr (!SRC8) next_mean = mean_in[row + step];
        }
        if constexpr (kAsync) wait_groups<Ring::kSlots - 1>();
        typename IO::Raw ry[NV], rx[NV];
        typename Q8<VEC>::Raw rq[NV];
        float rs[NV];
        // one value at a time: the residual's gradient is requested with the rest of its row, and kept in pairs
        constexpr bool kPairs = !kAsync && sizeof(T) == 2;
        uint32_t rj[kPairs ? kBwdElems / 2 : 1];
        if constexpr (kPairs) {
            if (join != nullptr) {
                const unsigned short* j = (const unsigned short*)(join + row * ldjoin + c0);
#pragma unroll
                for (int i = 0; i < NV; i += 2)
                    rj[i / 2] = (i < nv ? (uint32_t)j[i * tpr] : 0u) | (i + 1 < nv ? (uint32_t)j[(i + 1) * tpr] << 16 : 0u);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + t) * VEC;
            const bool in = i < nv;
            if constexpr (kAsync) ry[i] = in ? fetched(at_y(slot, i), dy + row * lddy, i) : IO::zero();
            else ry[i] = in ? IO::load(dy + row * lddy + col) : IO::zero();
            if constexpr (SRC8) {
                if constexpr (kAsync) {
                    rq[i] = in ? from_shared<typename Q8<VEC>::Raw>(at_q(slot, i)) : Q8<VEC>::zero();
                    rs[i] = in ? act8_step((from_shared<uint32_t>(at_e(slot, i)) >> (8 * ((col / kAct8Block) & 3))) & 255u) : 0.f;
                } else {
                    rq[i] = in ? Q8<VEC>::load(q + row * ldq + col) : Q8<VEC>::zero();
                    rs[i] = in ? act8_step(e[row * lde + col / kAct8Block]) : 0.f;
                }
            } else {
                if constexpr (kAsync) rx[i] = in ? fetched(at_x(slot, i), x + row * ldx, i) : IO::zero();
                else rx[i] = in ? IO::load(x + row * ldx + col) : IO::zero();
            }
        }
        float p[kBwdElems], xh[kBwdElems];   // dy * weight and the normalised values (past the row's end the gradient is 0)
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float fy[VEC], g[VEC], *fh = xh + i * VEC;
            IO::unpack(ry[i], fy);
            if constexpr (SRC8) {
                Q8<VEC>::unpack(rq[i], rs[i], fh);
            } else {
                IO::unpack(rx[i], fh);
#pragma unroll
                for (int j = 0; j < VEC; ++j) fh[j] = (fh[j] - mean) * rstd;
            }
            IO::unpack(graw[i], g);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = i * VEC + j;
                p[c] = fy[j] * g[j];
                dg[c] = fmaf(fy[j], fh[j], dg[c]);
                db[c] += fy[j];
                s1 += p[c];
                s2 = fmaf(p[c], fh[j], s2);
            }
        }
        s1 = warp_sum(s1);
        s2 = warp_sum(s2);
        if (warps > 1) {
            if (lane == 0) {
                red[buf][threadIdx.x >> 5][0] = s1;
                red[buf][threadIdx.x >> 5][1] = s2;
            }
            asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(tpr) : "memory");
            s1 = s2 = 0.f;
            for (int w = 0; w < warps; ++w) {
                s1 += red[buf][w0 + w][0];
                s2 += red[buf][w0 + w][1];
            }
        }
        const float a1 = s1 * inv_d, a2 = s2 * inv_d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i >= nv) continue;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = rstd * (p[i * VEC + j] - fmaf(xh[i * VEC + j], a2, a1));
            if (join != nullptr) {
                float fj[VEC];
                if constexpr (kAsync) IO::unpack(fetched(at_j(slot, i), join + row * ldjoin, i), fj);
                else if constexpr (kPairs) fj[0] = __uint_as_float(i & 1 ? rj[i / 2] & 0xFFFF0000u : rj[i / 2] << 16);
                else IO::unpack(IO::load(join + row * ldjoin + c0 + i * tpr * VEC), fj);
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] += fj[j];
            }
            if constexpr (LOOSE) loose_store(dx_row + i * tpr * VEC, o, d - c0 - i * tpr * VEC);
            else IO::store(dx_row + i * tpr * VEC, o);
        }
        dx_row += step * lddx;
        slot = slot + 1 == Ring::kSlots ? 0 : slot + 1;
    }
    if (partial == nullptr) return;
    // The teams' sums in a tree (the same one every time): the upper half hands its sums over, [16 + 16 sums][threads], and leaves.
    float* comb = (float*)ring_raw;
    if constexpr (kAsync) wait_groups<0>();
    __syncthreads();   // the ring is free
    for (int half = teams / 2; half > 0; half /= 2) {
        float* place = comb + (int64_t)(team - (team >= half ? half : 0)) * 2 * kBwdElems * tpr + t;
        if (team >= half && team < 2 * half) {
#pragma unroll
            for (int c = 0; c < kBwdElems; ++c) {
                place[c * tpr] = dg[c];
                place[(kBwdElems + c) * tpr] = db[c];
            }
        }
        __syncthreads();
        if (team < half) {
#pragma unroll
            for (int c = 0; c < kBwdElems; ++c) {
                dg[c] += place[c * tpr];
                db[c] += place[(kBwdElems + c) * tpr];
            }
        }
        __syncthreads();
    }
    if (team != 0) return;
    float* out = partial + (int64_t)blockIdx.x * 2 * d + c0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i >= nv) continue;
        if constexpr (LOOSE) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (c0 + i * tpr * VEC + j >= d) continue;
                out[i * tpr * VEC + j] = dg[i * VEC + j];
                out[d + i * tpr * VEC + j] = db[i * VEC + j];
            }
        } else if constexpr (VEC >= 4) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const int c = i * VEC + j;
                *(float4*)(out + i * tpr * VEC + j) = make_float4(dg[c], dg[c + 1], dg[c + 2], dg[c + 3]);
                *(float4*)(out + d + i * tpr * VEC + j) = make_float4(db[c], db[c + 1], db[c + 2], db[c + 3]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                out[i * tpr * VEC + j] = dg[i * VEC + j];
                out[d + i * tpr * VEC + j] = db[i * VEC + j];
            }
        }
    }
}

// Rows longer than 8192 columns: dx with a CTA per row that reads it twice, and the weight's gradient by columns. An element at a
// time: 4096 x 16384 in bf16 321 us (1.25 TB/s), where 8192 x 8192 takes 100.
template <typename T, bool SRC8>
__device__ __forceinline__ float xhat_at(const T* x, int64_t ldx, const int8_t* q, int64_t ldq, const uint8_t* e, int64_t lde, int64_t row,
                                         int c, float mean, float rstd) {
    if constexpr (SRC8) return (float)q[row * ldq + c] * act8_step(e[row * lde + c / kAct8Block]);
    float f;
    Io<T, 1>::unpack(x[row * ldx + c], &f);
    return (f - mean) * rstd;
}
template <typename T, bool SRC8>
__global__ void __launch_bounds__(512)
layer_norm_bwd_long_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, const int8_t* q, int64_t ldq,
                           const uint8_t* e, int64_t lde, const T* __restrict__ weight, const float* mean_in, const float* rstd_in,
                           const T* join, int64_t ldjoin, T* __restrict__ dx, int64_t lddx, int d) {
    allow_successor();
    __shared__ float red[16];
    const int64_t row = blockIdx.x;
    const float rstd = rstd_in[row], mean = SRC8 ? 0.f : mean_in[row];
    auto p_at = [&](int c) {
        float f, g = 1.f;
        Io<T, 1>::unpack(dy[row * lddy + c], &f);
        if (weight != nullptr) Io<T, 1>::unpack(weight[c], &g);
        return f * g;
    };
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
        const float p = p_at(c);
        s1 += p;
        s2 += p * xhat_at<T, SRC8>(x, ldx, q, ldq, e, lde, row, c, mean, rstd);
    }
    s1 = block_sum(s1, red) / (float)d;
    s2 = block_sum(s2, red) / (float)d;
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
        float o = rstd * (p_at(c) - s1 - xhat_at<T, SRC8>(x, ldx, q, ldq, e, lde, row, c, mean, rstd) * s2), j = 0.f;
        if (join != nullptr) Io<T, 1>::unpack(join[row * ldjoin + c], &j);
        o += j;
        Io<T, 1>::store(dx + row * lddx + c, &o);
    }
}
template <typename T, bool SRC8>
__global__ void __launch_bounds__(256)
layer_norm_dw_long_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, const int8_t* q, int64_t ldq,
                          const uint8_t* e, int64_t lde, const float* mean_in, const float* rstd_in, float* partial, int64_t rows, int d) {
    allow_successor();
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= d) return;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r1 = min(rows, (int64_t)(blockIdx.y + 1) * per);
    float g = 0.f, b = 0.f, f;
    for (int64_t row = (int64_t)blockIdx.y * per; row < r1; ++row) {
        Io<T, 1>::unpack(dy[row * lddy + c], &f);
        g += f * xhat_at<T, SRC8>(x, ldx, q, ldq, e, lde, row, c, SRC8 ? 0.f : mean_in[row], rstd_in[row]);
        b += f;
    }
    partial[(int64_t)blockIdx.y * 2 * d + c] = g;
    partial[(int64_t)blockIdx.y * 2 * d + d + c] = b;
}

// out[c] (+)= sum over the partial rows, eight interleaved sums per column that are then added in a fixed order. Column c
// of the partials goes to out0[c], or to out1[c - split] from `split` on; either may be null.
__global__ void __launch_bounds__(256)
column_reduce_kernel(const float* partial, int n, int64_t width, int64_t split, float* out0, float* out1, int accumulate) {
    __shared__ float part[8][33];
    wait_predecessor();   // launched ahead of the end of the kernel that writes the partials (and not __restrict__: nothing is read before)
    allow_successor();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    float s = 0.f;
    if (c < width) {
#pragma unroll 8
        for (int r = ty; r < n; r += 8) s += partial[(int64_t)r * width + c];
    }
    part[ty][tx] = s;
    __syncthreads();
    if (ty != 0 || c >= width) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += part[k][tx];
    float* o = c < split ? (out0 != nullptr ? out0 + c : nullptr) : (out1 != nullptr ? out1 + (c - split) : nullptr);
    if (o != nullptr) *o = accumulate ? *o + s : s;
}

// ---- column sums -----------------------------------------------------------------------------------------------------
// A CTA sums a slab of rows for 128 columns (16 lanes of 8, or 4 bytes wide where rows are not aligned): four rows requested
// before the first is added, then one partial row per slab.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
column_sum_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols, float* __restrict__ partial) {
    allow_successor();
    constexpr int TX = 128 / VEC, TY = 256 / TX > 0 ? 256 / TX : 1;
    __shared__ float part[TY][128 + 4];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = (int64_t)blockIdx.x * 128 + tx * VEC;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r1 = min(rows, (int64_t)(blockIdx.y + 1) * per);
    float s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = 0.f;
    if (col < cols) {
        const T* p = x + col;
        int64_t r = (int64_t)blockIdx.y * per + ty;
        for (; r + 3 * TY < r1; r += 4 * TY) {
            typename Io<T, VEC>::Raw raw[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) raw[k] = Io<T, VEC>::load(p + (r + k * TY) * ldx);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[VEC];
                Io<T, VEC>::unpack(raw[k], f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[j] += f[j];
            }
        }
        for (; r < r1; r += TY) {
            float f[VEC];
            Io<T, VEC>::unpack(Io<T, VEC>::load(p + r * ldx), f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j] += f[j];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) part[ty][tx * VEC + j] = s[j];
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (threadIdx.x < 128 && c < cols) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < TY; ++k) a += part[k][threadIdx.x];
        partial[(int64_t)blockIdx.y * cols + c] = a;
    }
}

// ---- 8-bit checkpoints of rows ---------------------------------------------------------------------------------------
// A warp takes U vectors of a row per lane, all requested before the first is used.
template <typename T, int VEC, int U>
__global__ void __launch_bounds__(256)
act8_pack_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ e, int64_t lde, int64_t rows,
                 int64_t cols, int64_t per_row) {
    allow_successor();
    const int lane = threadIdx.x & 31;
    const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t row = task / per_row, c0 = (task - row * per_row) * (32 * VEC * U) + lane * VEC;
    if (row >= rows) return;   // a whole warp
    typename Io<T, VEC>::Raw raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t col = c0 + i * 32 * VEC;
        raw[i] = col < cols ? Io<T, VEC>::load(x + row * ldx + col) : Io<T, VEC>::zero();
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t col = c0 + i * 32 * VEC;
        float f[VEC];
        Io<T, VEC>::unpack(raw[i], f);
        const uint32_t ex = block_exponent<VEC>(f, true);   // (lanes past the row hold zeros)
        if (col >= cols) continue;
        Q8<VEC>::store(q + row * ldq + col, f, ex, act8_inverse_step(ex));
        if (col % kAct8Block == 0) e[row * lde + col / kAct8Block] = (uint8_t)ex;
    }
}
template <typename T, int VEC, int U>
__global__ void __launch_bounds__(256)
act8_unpack_kernel(const int8_t* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ e, int64_t lde, T* __restrict__ x, int64_t ldx,
                   int64_t rows, int64_t cols, int64_t per_row) {
    allow_successor();
    const int lane = threadIdx.x & 31;
    const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t row = task / per_row, c0 = (task - row * per_row) * (32 * VEC * U) + lane * VEC;
    if (row >= rows) return;
    typename Q8<VEC>::Raw raw[U];
    uint32_t ex[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t col = c0 + i * 32 * VEC;
        raw[i] = col < cols ? Q8<VEC>::load(q + row * ldq + col) : Q8<VEC>::zero();
        ex[i] = col < cols ? e[row * lde + col / kAct8Block] : 0u;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t col = c0 + i * 32 * VEC;
        if (col >= cols) continue;
        float f[VEC];
        Q8<VEC>::unpack(raw[i], act8_step(ex[i]), f);
        Io<T, VEC>::store(x + row * ldx + col, f);
    }
}

// ---- bf16 rows onto 16-byte boundaries, which is what loads by tensor map ask for ------------------------------------------
// A thread writes one block of 16 bytes: the two aligned blocks of the source row that hold its values (the second is the
// neighbour's first, and comes from L1), shifted by what the row starts past a boundary. A block that is read holds a value of the row.
__global__ void __launch_bounds__(256)
pad_rows_kernel(const __nv_bfloat16* __restrict__ src, int64_t ld, __nv_bfloat16* __restrict__ dst, int64_t ldp, int64_t total, int64_t cols, uint32_t per_row) {
    allow_successor();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t row = total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / per_row) : i / per_row;
    const int64_t j = i - row * per_row;
    const uintptr_t start = (uintptr_t)(src + row * ld), past = start & 15, end = start + 2 * cols;
    const uintptr_t block = start - past + 16 * j;
    const uint4 a = *(const uint4*)block;
    uint4 b = make_uint4(0, 0, 0, 0);
    if (past != 0 && block + 16 < end) b = *(const uint4*)(block + 16);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (past & 8) {
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
    }
    if (past & 4) {
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
    }
    const uint32_t shift = (uint32_t)(past & 2) * 8;
    *(uint4*)(dst + row * ldp + 8 * j) = make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift),
                                                    __funnelshift_r(w[2], w[3], shift), __funnelshift_r(w[3], w[4], shift));
}

// ---- host ------------------------------------------------------------------------------------------------------------
int pow2_at_least(int64_t v, int lo, int hi) {
    int p = lo;
    while (p < v && p < hi) p <<= 1;
    return p;
}
template <typename T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }
// Whether accesses of `bytes` fit: every row of every tensor starts on such a boundary and holds whole vectors.
template <typename T>
bool aligned(int64_t d, std::initializer_list<std::pair<const void*, int64_t>> rows, int bytes = 16) {
    const int vec = bytes / (int)sizeof(T);
    if (d % vec) return false;
    for (const auto& r : rows)
        if (r.first != nullptr && (((uintptr_t)r.first % bytes) || (r.second % vec))) return false;
    return true;
}
bool kept_ok(const Act8View& k) { return ((uintptr_t)k.q % 16) == 0 && (k.ldq % 16) == 0 && ((uintptr_t)k.e % 4) == 0 && (k.lde % 4) == 0; }

template <auto kern>
struct Kernel {
    static constexpr auto value = kern;
};
// CTAs of `threads` (32 << i) and `smem` bytes that an SM holds; also allows the kernel that much shared memory. Asked once per
// kernel, device and shape: the driver's answer costs more than a small launch.
template <auto kern>
cudaError_t ctas_per_sm(int threads, int smem, int* count) {
    static int known[16][8] = {}, bytes[16][8] = {};
    int dev = 0;
    cudaError_t rc = cudaGetDevice(&dev);
    if (rc != cudaSuccess) return rc;
    int i = 0;
    while ((32 << i) < threads && i < 7) ++i;
    const bool keep = dev >= 0 && dev < 16;
    if (keep && known[dev][i] != 0 && bytes[dev][i] == smem) {
        *count = known[dev][i];
        return cudaSuccess;
    }
    if (smem > 40 * 1024) {   // with the static part more than a launch gets by default; the largest shape so far sets it
        static int allowed[16] = {};
        if (!keep || allowed[dev] < smem) {
            rc = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (rc != cudaSuccess) return rc;
            if (keep) allowed[dev] = smem;
        }
    }
    rc = cudaOccupancyMaxActiveBlocksPerMultiprocessor(count, kern, threads, smem);
    if (rc != cudaSuccess) return rc;
    if (*count < 1) return cudaErrorLaunchOutOfResources;
    if (keep) {
        known[dev][i] = *count;
        bytes[dev][i] = smem;
    }
    return cudaSuccess;
}

template <typename T, int VEC, int NV, int TPR>
int launch_fwd(const T* x, int64_t ldx, const T* w, const T* b, T* y, int64_t ldy, float* mean, float* rstd, const Act8View& keep,
               int64_t rows, int d, float eps, int tpr, cudaStream_t s) {
    // a CTA per row where a row takes several warps, so that a barrier stops nobody else
    const int threads = tpr == 32 ? 128 : tpr, teams = threads / tpr;
    const int64_t need = (rows + teams - 1) / teams;
    const int smem = copies_ahead<T, VEC>() ? kFwdSlots * NV * threads * VEC * (int)sizeof(T) : 0;
    auto go = [&](auto instance) -> int {
        constexpr auto kern = decltype(instance)::value;
        int per_sm = 0;
        const cudaError_t rc = ctas_per_sm<kern>(threads, smem, &per_sm);
        if (rc != cudaSuccess) return (int)rc;
        const unsigned grid = (unsigned)std::min<int64_t>(need, (int64_t)per_sm * kSms);   // one wave of CTAs at most
        kern<<<grid, threads, smem, s>>>(x, ldx, w, b, y, ldy, mean, rstd, (int8_t*)keep.q, keep.ldq, (uint8_t*)keep.e, keep.lde, rows, d, eps, tpr);
        return (int)cudaGetLastError();
    };
    return keep.q != nullptr ? go(Kernel<layer_norm_fwd_kernel<T, VEC, NV, true, TPR>>{}) : go(Kernel<layer_norm_fwd_kernel<T, VEC, NV, false, TPR>>{});
}

template <typename T, int VEC>
int fwd_vec(const T* x, int64_t ldx, const T* w, const T* b, T* y, int64_t ldy, float* mean, float* rstd, const Act8View& keep, int64_t rows,
            int d, float eps, cudaStream_t s) {
    constexpr int NV = VEC <= 2 ? 16 : VEC == 4 ? 8 : 4;   // 32 values (16 where they are read one by one)
    const int64_t vecs = (d + VEC - 1) / VEC;
    // fewer rows than SMs x 4: one vector per thread if 512 threads have the row (with two values a thread the meeting of sixteen
    // warps costs more than it saves: 300 x 1002, 5.2 us for 3.2)
    if (rows <= 4 * kSms && vecs <= (VEC == 2 ? kMaxTeam / 2 : kMaxTeam))
        return launch_fwd<T, VEC, 1, 0>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, pow2_at_least(vecs, 32, kMaxTeam), s);
    if (vecs <= 64) return launch_fwd<T, VEC, 2, 32>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, 32, s);
    if (vecs <= (int64_t)kMaxTeam * NV) {
        const int tpr = pow2_at_least((vecs + NV - 1) / NV, 32, kMaxTeam);
        switch (tpr) {
            case 32: return launch_fwd<T, VEC, NV, 32>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, tpr, s);
            case 64: return launch_fwd<T, VEC, NV, 64>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, tpr, s);
            case 128: return launch_fwd<T, VEC, NV, 128>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, tpr, s);
            case 256: return launch_fwd<T, VEC, NV, 256>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, tpr, s);
            default: return launch_fwd<T, VEC, NV, 512>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, d, eps, tpr, s);
        }
    }
    if (rows > 0x7FFFFFFF) return -2;
    if (keep.q != nullptr)
        layer_norm_fwd_long_kernel<T, true><<<(unsigned)rows, 512, 0, s>>>(x, ldx, w, b, y, ldy, mean, rstd, (int8_t*)keep.q, keep.ldq,
                                                                          (uint8_t*)keep.e, keep.lde, d, eps);
    else
        layer_norm_fwd_long_kernel<T, false><<<(unsigned)rows, 512, 0, s>>>(x, ldx, w, b, y, ldy, mean, rstd, nullptr, 0, nullptr, 0, d, eps);
    return (int)cudaGetLastError();
}

template <typename T>
int fwd_typed(const T* x, int64_t ldx, const T* w, const T* b, T* y, int64_t ldy, float* mean, float* rstd, const Act8View& keep, int64_t rows,
              int64_t d, float eps, cudaStream_t s) {
    constexpr int V = vec_of<T>();
    if (aligned<T>(d, {{x, ldx}, {y, ldy}, {w, 0}, {b, 0}}) && (keep.q == nullptr || kept_ok(keep)))
        return fwd_vec<T, V>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, (int)d, eps, s);
    if constexpr (sizeof(T) == 2) {
        if (aligned<T>(d, {{x, ldx}, {y, ldy}, {w, 0}, {b, 0}}, 4) && (keep.q == nullptr || kept_ok(keep)))
            return fwd_vec<T, 2>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, (int)d, eps, s);
    }
    return fwd_vec<T, 1>(x, ldx, w, b, y, ldy, mean, rstd, keep, rows, (int)d, eps, s);
}

struct BwdPlan {
    bool fits;     // the row fits one team's registers
    int tpr, threads, grid;
};
BwdPlan bwd_plan(int64_t rows, int64_t d) {
    BwdPlan p;
    p.fits = d <= (int64_t)kBwdThreads * kBwdElems;
    p.tpr = pow2_at_least((d + kBwdElems - 1) / kBwdElems, 32, kBwdThreads);
    // few rows: one team per CTA until every SM has one
    const int teams = (int)std::max<int64_t>(1, std::min<int64_t>(kBwdThreads / p.tpr, (rows + kSms - 1) / kSms));
    p.threads = p.tpr * pow2_at_least(teams, 1, kBwdThreads / p.tpr);
    const int64_t need = (rows + p.threads / p.tpr - 1) / (p.threads / p.tpr);
    p.grid = p.fits ? (int)std::max<int64_t>(1, std::min<int64_t>(kSms, need))
                    : (int)std::max<int64_t>(1, std::min<int64_t>(64, (rows + 63) / 64));
    return p;
}

int reduce_partials(const float* partial, int n, int64_t width, int64_t split, float* out0, float* out1, int accumulate, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((width + 31) / 32));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute a[1] = {start_early()};
    cfg.attrs = a;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, column_reduce_kernel, partial, n, width, split, out0, out1, accumulate);
}

template <typename T, int VEC, bool SRC8, bool LOOSE = false>
int launch_bwd(const T* dy, int64_t lddy, const T* x, int64_t ldx, const Act8View& k, const T* w, const float* mean, const float* rstd,
               const T* join, int64_t ldjoin, T* dx, int64_t lddx, float* partial, int64_t rows, int d, const BwdPlan& p, cudaStream_t s) {
    using Ring = BwdRing<T, VEC, SRC8, LOOSE>;
    // the ring, or half the teams' sums
    const int smem = std::max(Ring::kBytes, p.threads > p.tpr ? p.threads / 2 * 2 * kBwdElems * (int)sizeof(float) : 0);
    auto go = [&](auto instance) -> int {
        constexpr auto kern = decltype(instance)::value;
        int per_sm = 0;
        const cudaError_t rc = ctas_per_sm<kern>(p.threads, smem, &per_sm);
        if (rc != cudaSuccess) return (int)rc;
        kern<<<p.grid, p.threads, smem, s>>>(dy, lddy, x, ldx, (const int8_t*)k.q, k.ldq, (const uint8_t*)k.e, k.lde, w, mean, rstd, join, ldjoin,
                                             dx, lddx, partial, rows, d, p.tpr);
        return (int)cudaGetLastError();
    };
    if constexpr (SRC8 && VEC == 1) {
        return go(Kernel<layer_norm_bwd_kernel<T, VEC, SRC8, 0, LOOSE>>{});
    } else {
        switch (p.tpr) {
            case 32: return go(Kernel<layer_norm_bwd_kernel<T, VEC, SRC8, 32, LOOSE>>{});
            case 64: return go(Kernel<layer_norm_bwd_kernel<T, VEC, SRC8, 64, LOOSE>>{});
            case 128: return go(Kernel<layer_norm_bwd_kernel<T, VEC, SRC8, 128, LOOSE>>{});
            case 256: return go(Kernel<layer_norm_bwd_kernel<T, VEC, SRC8, 256, LOOSE>>{});
            default: return go(Kernel<layer_norm_bwd_kernel<T, VEC, SRC8, 512, LOOSE>>{});
        }
    }
}

template <typename T, bool SRC8>
int bwd_typed(const T* dy, int64_t lddy, const T* x, int64_t ldx, const Act8View& k, const T* w, const float* mean, const float* rstd,
              const T* join, int64_t ldjoin, T* dx, int64_t lddx, float* dweight, float* dbias, int accumulate, float* partial, int64_t rows,
              int64_t d, cudaStream_t s) {
    const BwdPlan p = bwd_plan(rows, d);
    const bool want = dweight != nullptr || dbias != nullptr;
    float* part = want ? partial : nullptr;
    int rc;
    if (p.fits) {
        const bool vec = aligned<T>(d, {{dy, lddy}, {x, ldx}, {dx, lddx}, {join, ldjoin}, {w, 0}}) && (!SRC8 || kept_ok(k));
        constexpr bool kLoose = sizeof(T) == 2 && SRC8;   // unaligned rows otherwise: one value at a time
        if (kLoose && !kept_ok(k)) return -2;
        auto go = [&](auto vec_c, auto loose_c) {
            return launch_bwd<T, decltype(vec_c)::value, SRC8, decltype(loose_c)::value>(dy, lddy, x, ldx, k, w, mean, rstd, join, ldjoin, dx, lddx, part,
                                                                                        rows, (int)d, p, s);
        };
        using No = std::false_type;
        auto go_unaligned = [&]() -> int {
            if constexpr (sizeof(T) == 2 && !SRC8) {   // (beside 8-bit rows bf16 ones are loose)
                if (aligned<T>(d, {{dy, lddy}, {x, ldx}, {dx, lddx}, {join, ldjoin}, {w, 0}}, 4)) return go(std::integral_constant<int, 2>{}, No{});
            }
            return go(std::integral_constant<int, kLoose ? 8 : 1>{}, std::bool_constant<kLoose>{});
        };
        rc = vec ? go(std::integral_constant<int, vec_of<T>()>{}, No{}) : go_unaligned();
    } else {
        if (rows > 0x7FFFFFFF) return -2;
        layer_norm_bwd_long_kernel<T, SRC8><<<(unsigned)rows, 512, 0, s>>>(dy, lddy, x, ldx, (const int8_t*)k.q, k.ldq, (const uint8_t*)k.e, k.lde,
                                                                          w, mean, rstd, join, ldjoin, dx, lddx, (int)d);
        rc = (int)cudaGetLastError();
        if (rc == 0 && want) {
            layer_norm_dw_long_kernel<T, SRC8><<<dim3((unsigned)((d + 255) / 256), p.grid), 256, 0, s>>>(
                dy, lddy, x, ldx, (const int8_t*)k.q, k.ldq, (const uint8_t*)k.e, k.lde, mean, rstd, part, rows, (int)d);
            rc = (int)cudaGetLastError();
        }
    }
    if (rc != 0 || !want) return rc;
    return reduce_partials(part, p.grid, 2 * d, d, dweight, dbias, accumulate, s);
}

int column_slabs(int64_t rows, int64_t cols) {
    if (cols <= 0) return 1;
    const int64_t gx = (cols + 127) / 128;
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 63) / 64, (kSms * 8 + gx - 1) / gx));
}

constexpr int64_t kMaxCols = 1 << 30;   // column indices are 32-bit

}  // namespace

int layer_norm_fwd(int dtype, const void* x, int64_t ldx, const void* weight, const void* bias, void* y, int64_t ldy, float* mean,
                   float* rstd, const Act8View& keep, int64_t rows, int64_t d, float eps, void* stream) {
    if (rows <= 0 || d <= 0) return 0;
    if (d > kMaxCols) return -2;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == 0)
        return fwd_typed<__nv_bfloat16>((const __nv_bfloat16*)x, ldx, (const __nv_bfloat16*)weight, (const __nv_bfloat16*)bias, (__nv_bfloat16*)y,
                                        ldy, mean, rstd, keep, rows, d, eps, s);
    if (dtype == 1)
        return fwd_typed<float>((const float*)x, ldx, (const float*)weight, (const float*)bias, (float*)y, ldy, mean, rstd, keep, rows, d, eps, s);
    return -2;
}

int64_t layer_norm_bwd_scratch(int64_t rows, int64_t d) { return (int64_t)bwd_plan(rows, d).grid * 2 * d; }

int layer_norm_bwd(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, const Act8View& kept, const void* weight,
                   const float* mean, const float* rstd, const void* join, int64_t ldjoin, void* dx, int64_t lddx, float* dweight,
                   float* dbias, int accumulate, float* partial, int64_t rows, int64_t d, void* stream) {
    cudaStream_t s = (cudaStream_t)stream;
    if (d <= 0) return 0;
    if (d > kMaxCols) return -2;
    if (rows <= 0) {   // sums over no rows
        cudaError_t rc = cudaSuccess;
        if (!accumulate && dweight != nullptr) rc = cudaMemsetAsync(dweight, 0, (size_t)d * 4, s);
        if (rc == cudaSuccess && !accumulate && dbias != nullptr) rc = cudaMemsetAsync(dbias, 0, (size_t)d * 4, s);
        return (int)rc;
    }
#define PSB_BWD(T, SRC8)                                                                                                              \
    bwd_typed<T, SRC8>((const T*)dy, lddy, (const T*)x, ldx, kept, (const T*)weight, mean, rstd, (const T*)join, ldjoin, (T*)dx, lddx, dweight, \
                       dbias, accumulate, partial, rows, d, s)
    if (dtype == 0) return kept.q != nullptr ? PSB_BWD(__nv_bfloat16, true) : PSB_BWD(__nv_bfloat16, false);
    if (dtype == 1) return kept.q != nullptr ? PSB_BWD(float, true) : PSB_BWD(float, false);
#undef PSB_BWD
    return -2;
}

namespace {
template <typename T, int VEC, int U, bool PACK>
int launch_act8(void* x, int64_t ldx, const Act8View& k, int64_t rows, int64_t cols, cudaStream_t s) {
    const int64_t per_row = (cols + 32 * VEC * U - 1) / (32 * VEC * U);
    const int64_t grid = (rows * per_row + 7) / 8;
    if (grid > 0x7FFFFFFF) return -2;
    if (PACK)
        act8_pack_kernel<T, VEC, U><<<(unsigned)grid, 256, 0, s>>>((const T*)x, ldx, (int8_t*)k.q, k.ldq, (uint8_t*)k.e, k.lde, rows, cols, per_row);
    else
        act8_unpack_kernel<T, VEC, U><<<(unsigned)grid, 256, 0, s>>>((const int8_t*)k.q, k.ldq, (const uint8_t*)k.e, k.lde, (T*)x, ldx, rows, cols,
                                                                    per_row);
    return (int)cudaGetLastError();
}
template <typename T, bool PACK>
int act8_typed(void* x, int64_t ldx, const Act8View& k, int64_t rows, int64_t cols, cudaStream_t s) {
    constexpr int V = vec_of<T>();
    if (aligned<T>(cols, {{x, ldx}}) && kept_ok(k))
        return cols > 32 * V ? launch_act8<T, V, 4, PACK>(x, ldx, k, rows, cols, s) : launch_act8<T, V, 1, PACK>(x, ldx, k, rows, cols, s);
    return launch_act8<T, 1, 4, PACK>(x, ldx, k, rows, cols, s);
}
}  // namespace

int act8_pack(int dtype, const void* x, int64_t ldx, const Act8View& out, int64_t rows, int64_t cols, void* stream) {
    if (rows <= 0 || cols <= 0) return 0;
    if (dtype == 0) return act8_typed<__nv_bfloat16, true>((void*)x, ldx, out, rows, cols, (cudaStream_t)stream);
    if (dtype == 1) return act8_typed<float, true>((void*)x, ldx, out, rows, cols, (cudaStream_t)stream);
    return -2;
}
int act8_unpack(int dtype, const Act8View& in, void* x, int64_t ldx, int64_t rows, int64_t cols, void* stream) {
    if (rows <= 0 || cols <= 0) return 0;
    if (dtype == 0) return act8_typed<__nv_bfloat16, false>(x, ldx, in, rows, cols, (cudaStream_t)stream);
    if (dtype == 1) return act8_typed<float, false>(x, ldx, in, rows, cols, (cudaStream_t)stream);
    return -2;
}

int64_t column_sum_scratch(int64_t rows, int64_t cols) { return (int64_t)column_slabs(rows, cols) * cols; }

namespace {
template <typename T>
int column_sum_typed(const T* x, int64_t ldx, int64_t rows, int64_t cols, float* out, int accumulate, float* partial, cudaStream_t s) {
    const int slabs = column_slabs(rows, cols);
    const int64_t gx = (cols + 127) / 128;
    if (gx > 0x7FFFFFFF) return -2;
    dim3 grid((unsigned)gx, (unsigned)slabs);
    if (aligned<T>(cols, {{x, ldx}})) column_sum_kernel<T, vec_of<T>()><<<grid, 256, 0, s>>>(x, ldx, rows, cols, partial);
    else column_sum_kernel<T, 1><<<grid, 256, 0, s>>>(x, ldx, rows, cols, partial);
    const int rc = (int)cudaGetLastError();
    return rc != 0 ? rc : reduce_partials(partial, slabs, cols, cols, out, nullptr, accumulate, s);
}
}  // namespace

int column_sum(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, float* out, int accumulate, float* partial, void* stream) {
    cudaStream_t s = (cudaStream_t)stream;
    if (cols <= 0) return 0;
    if (rows <= 0) return accumulate ? 0 : (int)cudaMemsetAsync(out, 0, (size_t)cols * 4, s);
    if (dtype == 0) return column_sum_typed<__nv_bfloat16>((const __nv_bfloat16*)x, ldx, rows, cols, out, accumulate, partial, s);
    if (dtype == 1) return column_sum_typed<float>((const float*)x, ldx, rows, cols, out, accumulate, partial, s);
    return -2;
}

int pad_rows(const void* src, int64_t ld, void* dst, int64_t ldp, int64_t rows, int64_t cols, void* stream) {
    if (rows <= 0 || cols <= 0) return 0;
    const int64_t per_row = (cols + 7) / 8, total = rows * per_row;
    if ((uintptr_t)dst % 16 || ldp % 8 || ldp < per_row * 8 || (uintptr_t)src % 2 || per_row > 0x7FFFFFFF || (total + 255) / 256 > 0x7FFFFFFF) return -2;
    pad_rows_kernel<<<(unsigned)((total + 255) / 256), 256, 0, (cudaStream_t)stream>>>((const __nv_bfloat16*)src, ld, (__nv_bfloat16*)dst, ldp, total,
                                                                                     cols, (uint32_t)per_row);
    return (int)cudaGetLastError();
}

}  // namespace psb
