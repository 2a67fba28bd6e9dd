// Rotary positions: pair i of a head's values turns by position * freqs[i],
//   x' = s (x cos - y sin),  y' = s (x sin + y cos),  and backward by the negative angle.
// The angle's product and its reduction to a turn are in 64 bits (position 2^20 times one radian is off by 0.06 in 32), sine and cosine of
// the fraction of a turn in 32, the values in 32 with one rounding at the end.
//
// Bound by HBM: every value is read and written once. A thread has a unit of P pairs (16 bytes from each half of a head, or 32 of
// neighbours; fewer where rows, heads or halves lie on smaller boundaries) of one token in up to eight heads, so that its P sines and cosines are
// used again. Loads of four heads are on their way before the first is turned. 16384 tokens, 32 heads of 128 in bf16: 42.8 us (6.3 TB/s; a plain
// copy 6.5), fp32 81 (6.6); halves of 25 pairs, two bytes at a time, 93 (2.2). One token: 2.3 us, the launch.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "launch.cuh"
#include "rotary.h"

namespace psb {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotHeads = 4;        // of a thread at a time
constexpr int kRotShared = 8;       // heads that a thread turns with its sines and cosines
constexpr int kRotBusy = 148 * 1024;   // threads that keep the GPU busy

struct RotParams {
    RotaryArgs a;
    int turning, units;     // units of a head that turn, and with those that are only copied
    int lanes;              // threads that share a unit's heads
    int rows;               // tokens of a block
    int64_t total;          // tokens
};

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t b, int64_t t) {
    if (a.positions == nullptr) return a.offset + t;
    const int64_t at = b * a.pb + t * a.pt;
    return a.offset + (a.positions32 ? (int64_t)((const int32_t*)a.positions)[at] : ((const int64_t*)a.positions)[at]);
}
// Cosine and sine of position * freq. The angle in quarter turns, in 64 bits; adding 1.5 * 2^52 leaves the nearest whole number in the low
// bits. What is left of it, an eighth of a turn at most either way, goes into the Taylor series of both, whose first terms left out are 2^-29.1 (sine)
// and 2^-33 (cosine), and the whole quarters swap them and turn their signs. With the rounding of what is left to fp32 and those of the series' steps
// they are off by 2^-23.2 and 2^-23.6 at most. (sincospif took four times the instructions, and they were the kernel's time.)
__device__ __forceinline__ void turn_of(double position, double freq, float* c, float* s) {
    constexpr double kMagic = 6755399441055744.0;
    const double quarters = position * (freq * 0.63661977236758134308), shifted = quarters + kMagic;
    const uint32_t n = (uint32_t)__double2loint(shifted);
    const float f = (float)(quarters - (shifted - kMagic)), w = f * f;
    // (pi/2)^k / k!
    const float sine = f * fmaf(w, fmaf(w, fmaf(w, fmaf(w, 1.6044118478735983e-4f, -4.6817541353186881e-3f), 7.9692626246167046e-2f), -0.64596409750624625f), 1.5707963267948966f);
    const float cosine = fmaf(w, fmaf(w, fmaf(w, fmaf(w, fmaf(w, -2.5202042373060605e-5f, 9.1926027483942659e-4f), -2.0863480763352961e-2f), 0.25366950790104802f), -1.2337005501361698f), 1.f);
    const bool odd = (n & 1u) != 0u;
    *s = __uint_as_float(__float_as_uint(odd ? cosine : sine) ^ (n & 2u) << 30);
    *c = __uint_as_float(__float_as_uint(odd ? sine : cosine) ^ ((n + 1u) & 2u) << 30);
}

// P neighbours of a head as they lie in memory, and as floats
template <int BYTES>
using Block = std::conditional_t<BYTES == 16, uint4, std::conditional_t<BYTES == 8, uint2, std::conditional_t<BYTES == 4, uint32_t, unsigned short>>>;
__device__ __forceinline__ void words(uint4 v, uint32_t* w) { w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
__device__ __forceinline__ void words(uint2 v, uint32_t* w) { w[0] = v.x; w[1] = v.y; }
__device__ __forceinline__ void words(uint32_t v, uint32_t* w) { w[0] = v; }
__device__ __forceinline__ void words(unsigned short v, uint32_t* w) { w[0] = v; }
__device__ __forceinline__ void block(const uint32_t* w, uint4& v) { v = make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ void block(const uint32_t* w, uint2& v) { v = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void block(const uint32_t* w, uint32_t& v) { v = w[0]; }
__device__ __forceinline__ void block(const uint32_t* w, unsigned short& v) { v = (unsigned short)w[0]; }
template <typename T, int P, typename B>
__device__ __forceinline__ void unpack(B raw, float* f) {
    uint32_t w[4];
    words(raw, w);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        if constexpr (sizeof(T) == 4) f[j] = __uint_as_float(w[j]);
        else f[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
    }
}
template <typename T, int P, typename B>
__device__ __forceinline__ void pack(const float* f, B& raw) {
    uint32_t w[4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < P; ++j) w[j] = __float_as_uint(f[j]);
    } else {
#pragma unroll
        for (int j = 0; j < (P + 1) / 2; ++j) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(f[2 * j], 2 * j + 1 < P ? f[2 * j + 1] : 0.f);
            w[j] = *(const uint32_t*)&two;
        }
    }
    block(w, raw);
}

template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads, 3) rotary_kernel(const __grid_constant__ RotParams p) {
    wait_predecessor();
    allow_successor();
    const RotaryArgs& a = p.a;
    using Raw = Block<P * (int)sizeof(T)>;
    const int heads = a.q.heads + a.k.heads;
    const uint32_t per_token = (uint32_t)p.units * (uint32_t)p.lanes, work = per_token * (uint32_t)p.rows;
    for (uint32_t w = threadIdx.x; w < work; w += kRotThreads) {
        const uint32_t row = w / per_token, in = w - row * per_token, lane = in / (uint32_t)p.units, u = in - lane * (uint32_t)p.units;
        const int64_t token = (int64_t)blockIdx.x * p.rows + row;
        if (token >= p.total) break;
        const int64_t b = p.total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)token / (uint32_t)a.tokens) : token / a.tokens, t = token - b * a.tokens;
        const bool turns = (int)u < p.turning;
        // places of the unit's two blocks in a head: the pairs' first and second values, 2 P neighbours, or 2 P values that stay
        const int lo = !turns ? 2 * a.pairs + ((int)u - p.turning) * 2 * P : INTERLEAVED ? (int)u * 2 * P : (int)u * P;
        const int hi = !turns || INTERLEAVED ? lo + P : lo + a.pairs;
        const int there = turns ? 2 * P : a.dim - lo;   // values of the unit that exist
        const T* q = (const T*)a.q.x + b * a.q.xb + t * a.q.xt;
        const T* k = (const T*)a.k.x + b * a.k.xb + t * a.k.xt;
        T* oq = (T*)a.q.out + b * a.q.ob + t * a.q.ot;
        T* ok = (T*)a.k.out + b * a.k.ob + t * a.k.ot;
        auto from = [&](int h) { return h < a.q.heads ? q + h * a.q.xh : k + (h - a.q.heads) * a.k.xh; };
        auto to = [&](int h) { return h < a.q.heads ? oq + h * a.q.oh : ok + (h - a.q.heads) * a.k.oh; };
        if (there < 2 * P) {   // the end of a head whose last values stay
            for (int h = (int)lane; h < heads; h += p.lanes)
                for (int j = 0; j < there; ++j) to(h)[lo + j] = from(h)[lo + j];
            continue;
        }
        Raw x[kRotHeads], y[kRotHeads];
        auto load = [&](int h0) {
#pragma unroll
            for (int i = 0; i < kRotHeads; ++i) {
                const int h = h0 + i * p.lanes;
                if (h >= heads) break;
                const T* src = from(h);
                x[i] = *(const Raw*)(src + lo);
                y[i] = *(const Raw*)(src + hi);
            }
        };
        load((int)lane);
        float c[P], s[P];
        if (turns) {
            const double position = (double)position_of(a, b, t);
            const float scale = a.scale, back = a.backward ? -scale : scale;
#pragma unroll
            for (int j = 0; j < P; ++j) {
                turn_of(position, a.freqs[u * P + j], &c[j], &s[j]);
                c[j] *= scale;
                s[j] *= back;
            }
        }
        for (int h0 = (int)lane; h0 < heads; h0 += kRotHeads * p.lanes) {
            if (h0 != (int)lane) load(h0);
#pragma unroll
            for (int i = 0; i < kRotHeads; ++i) {
                const int h = h0 + i * p.lanes;
                if (h >= heads) break;
                if (turns) {
                    float f[2 * P];
                    unpack<T, P>(x[i], f);
                    unpack<T, P>(y[i], f + P);
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        float &first = f[INTERLEAVED ? 2 * j : j], &second = f[INTERLEAVED ? 2 * j + 1 : P + j];
                        const float v = first;
                        first = v * c[j] - second * s[j];
                        second = v * s[j] + second * c[j];
                    }
                    pack<T, P>(f, x[i]);
                    pack<T, P>(f + P, y[i]);
                }
                T* dst = to(h);
                *(Raw*)(dst + lo) = x[i];
                *(Raw*)(dst + hi) = y[i];
            }
        }
    }
}

// Whether blocks of `values` fit: every head of every tensor starts on such a boundary
bool fits(const RotaryArgs& a, int values, int size) {
    auto ok = [&](const void* p, int64_t b, int64_t t, int64_t h, int heads) {
        return (uintptr_t)p % (uintptr_t)(values * size) == 0 && (a.batch == 1 || b % values == 0) && (a.tokens == 1 || t % values == 0) && (heads == 1 || h % values == 0);
    };
    if (a.pairs % values) return false;
    for (const RotaryHeads* x : {&a.q, &a.k})
        if (x->heads > 0 && !(ok(x->x, x->xb, x->xt, x->xh, x->heads) && ok(x->out, x->ob, x->ot, x->oh, x->heads))) return false;
    return true;
}
bool in_place(const RotaryHeads& x) { return x.heads == 0 || (x.x == x.out && x.xb == x.ob && x.xt == x.ot && x.xh == x.oh); }

template <typename T, int P>
int launch(const RotaryArgs& a, cudaStream_t s) {
    RotParams p;
    p.a = a;
    p.turning = a.pairs / P;
    const int rest = in_place(a.q) && in_place(a.k) ? 0 : a.dim - 2 * a.pairs;
    p.units = p.turning + (rest + 2 * P - 1) / (2 * P);
    if (p.units == 0) return 0;
    p.total = a.batch * a.tokens;
    const int heads = a.q.heads + a.k.heads;
    // one head to a thread where there are few, eight where that keeps the GPU busy (16384 tokens, 32 heads of 128 in bf16: two 55 us, four 44)
    const int at_once = p.total * p.units * ((heads + kRotShared - 1) / kRotShared) >= kRotBusy ? kRotShared : 1;
    p.lanes = (heads + at_once - 1) / at_once;
    const int64_t per_token = (int64_t)p.units * p.lanes;
    if (per_token > 0x7FFFFFFF) return -2;
    p.rows = per_token >= kRotThreads ? 1 : (int)(kRotThreads / per_token);
    const int64_t blocks = (p.total + p.rows - 1) / p.rows;
    if (blocks > 0x7FFFFFFF) return -2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kRotThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1] = {start_early()};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)(a.interleaved ? cudaLaunchKernelEx(&cfg, rotary_kernel<T, P, true>, p) : cudaLaunchKernelEx(&cfg, rotary_kernel<T, P, false>, p));
}

}  // namespace

int rotary(int dtype, const RotaryArgs& a, void* stream) {
    if (a.batch <= 0 || a.tokens <= 0 || a.dim <= 0 || a.q.heads + a.k.heads <= 0) return 0;
    if (dtype < 0 || dtype > 1 || a.pairs < 0 || 2 * a.pairs > a.dim || (a.pairs > 0 && a.freqs == nullptr)) return -2;
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == 0) {
        if (fits(a, 8, 2)) return launch<__nv_bfloat16, 8>(a, s);
        if (fits(a, 4, 2)) return launch<__nv_bfloat16, 4>(a, s);
        if (fits(a, 2, 2)) return launch<__nv_bfloat16, 2>(a, s);
        return launch<__nv_bfloat16, 1>(a, s);
    }
    if (fits(a, 4, 4)) return launch<float, 4>(a, s);
    if (fits(a, 2, 4)) return launch<float, 2>(a, s);
    return launch<float, 1>(a, s);
}

}  // namespace psb
