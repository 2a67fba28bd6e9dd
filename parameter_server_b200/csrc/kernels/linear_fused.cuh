// Linear layers of a decoder block on the 5th-generation tensor cores, with their neighbours in the epilogue:
//
//   forward   h = x w^T + b,   y = act(h) + residual,   h kept for the backward pass in bf16 or in 8 bits
//   dgrad     dh = (dy w) * act'(h),   and act(h) again, for the weight gradient of the layer that dy belongs to
//
// and in the gated form, with w the gate's rows and those of the second factor behind them:
//
//   forward   g = x wg^T + bg, u = x wu^T + bu,   y = act(g) * u,   g and u kept
//   dgrad     da = dy w:   dg = da * u * act'(g) and du = da * act(g) side by side,   and act(g) * u again
//
// bf16 operands, fp32 accumulation in TMEM; everything in the epilogue is fp32 and rounded once per output. (The tensor core cuts
// its sums off instead of rounding them, 1e-9 of the sum per product: 9e-6 at K = 8192, far below the rounding of a bf16 output.)
// Fusing the neighbours saves their passes over M x N values through HBM; the product itself is bound by the tensor cores and by
// the operand feed from L2 (see the tile shape below), and over many launches by the power limit.
// Measured back to back in a graph, us: 16384 tokens, 2048 -> 8192: 363 (1510 TFLOP/s; a plain library product 358 to 412 as the
// clock goes), with gelu and h kept in bf16 406, in 8 bits 390; dgrad with act(h) 447, from 8 bits 441. 8192 -> 2048 with a residual
// 360. 1024 tokens, 2048 -> 8192: 28.5 (library 26), gelu 30.4, h kept 32.5, dgrad with act(h) 35: two waves of tiles for 1.73, and
// the second's epilogue (3 to 5 us) with nothing beside it. Gated, 2048 -> 2 x 5504, silu: 16384 tokens 469 (1577 TFLOP/s; a library product of
// 2048 -> 11008 487), h kept 515; dgrad with act(g) u 345; 1024 tokens 39.5 and 31.6. 2048 -> 2048 with a residual 99, with dropout 113.
//
// One persistent launch of CTA pairs (cta_group::2), one pair per two SMs. A pair works on a 256 x BN tile: each CTA loads
// its 128 rows of A and half of the B tile per k-step of 64 (32 KB for 512 cycles of MMA, which is what an SM's port to L2
// delivers; a single-CTA tile would need half as much again), the leader issues the MMAs for both, and each CTA drains its
// own 128 rows. Warps: 0 TMA producer, 1 MMA issuer and TMEM owner, 2-3 idle, 4-11 epilogue (a warp has one 32-lane quarter
// of TMEM and half of the tile's columns; the first warpgroup's registers go to them). The accumulator is double-buffered in
// TMEM, so the epilogue of a tile runs beside the MMAs of the next. Tiles are dealt out as tile_walk.cuh says. Every wait is
// bounded; on a time-out the CTA records where, lets what it has under way land, frees its TMEM and returns.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "act8.cuh"
#include "gemm_tcgen05.h"
#include "linear_fused.h"
#include "philox.cuh"
#include "tcgen05.cuh"
#include "tile_walk.cuh"
#include "unaligned.cuh"

namespace psb {

namespace {

// What the epilogue is of: one product, a gated pair of them, or one with dropout behind its activation (its seed in the call or in memory)
constexpr int kLinPlain = 0, kLinGated = 1, kLinDropout = 2, kLinDropoutSeed = 3;
constexpr int kLinEpilogueWarps = 8;
constexpr int kLinThreads = 32 * (4 + kLinEpilogueWarps);
constexpr int kLinRegsIssue = 56, kLinRegsEpilogue = 224;   // 56 + 2 * 224 = 3 * 168, the launch's share
static_assert(kLinRegsIssue + 2 * kLinRegsEpilogue == 3 * (65536 / kLinThreads / 8 * 8), "setmaxnreg would wait for registers that the launch does not have");

template <int BN, bool GATED_DGRAD = false>
struct LinSmem {
    static constexpr int kABytes = BM * BK * 2;
    static constexpr int kBBytes = BN / 2 * BK * 2;          // a CTA of a pair holds half of the B tile
    static constexpr int kStageBytes = kABytes + kBBytes;
    // k-steps that share a stage and its barriers: half as much for the MMA issuer to do between two MMAs, which counts where
    // the epilogue keeps the same schedulers busy (dgrad with an 8-bit h: 397 us with one, 383 us with two)
    static constexpr int kSub = 2;
    static constexpr int kStages = BN == 256 ? 3 : 4;
    static constexpr int kTileBytes = kStages * kSub * kStageBytes;
    static constexpr int kBarBytes = 256;
    static constexpr int kBiasBytes = GATED_DGRAD ? 0 : 2 * BN * 4;   // double-buffered with the accumulator
    static constexpr int kWarpBytes = GATED_DGRAD ? 4096 : 2048;      // a warp's [32 rows][64 bytes] on the way out; gated dgrad: 32 x 32 sums
    static constexpr int kOutBytes = kLinEpilogueWarps * kWarpBytes;
    static constexpr int kTotal = kTileBytes + kBarBytes + kBiasBytes + kOutBytes + 1024;   // + alignment slack
};

struct LinParams {
    CUtensorMap map_a, map_b;
    TileGrid grid;
    int M, N;
    int b_blocked;                    // MN-major B comes in with one 3-D load per stage
    const __nv_bfloat16* bias;
    const float* bias32;
    const __nv_bfloat16* res;
    int64_t ldres;
    __nv_bfloat16* out;
    int64_t ldo;
    __nv_bfloat16* out2;
    int64_t ldo2;
    __nv_bfloat16* pre;
    int64_t ldpre;
    int8_t* q;
    int64_t ldq;
    uint8_t* e;
    int64_t lde;
    int aux_width, pre_width, out_width, out2_width;   // rows of residual (forward) / pre / out / out2 start on multiples of 16, 8, 4 or 2
    float* partial;                   // shared tiles: [pair][2 places][cta][warp][BN / 64 pieces][8][32 lanes][4]
    unsigned* arrived;                // [shared tile][cta][warp]
    // gated: the second factor's columns of pre, of the checkpoint and (dgrad) of out
    __nv_bfloat16* pre_up;
    __nv_bfloat16* out_up;
    int pre_up_width, out_up_width;
    int8_t* q_up;
    int64_t ldq_up;
    uint8_t* e_up;
    int64_t lde_up;
    DropoutArgs drop;
    unsigned* err_flag;
    unsigned long long limit_ns;
};

// ---- activations -----------------------------------------------------------------------------------------------------
// gelu_tanh(h) = h / 2 * (1 + tanh(u)) = h * s(2u) with s(z) = 1 / (1 + exp(-z)) and u = sqrt(2/pi) (h + 0.044715 h^3): no
// cancellation in the tails, two special-function operations per value. Its slope is s + h s (1 - s) d(2u)/dh.
constexpr float kGeluC = 1.5957691216057308f;             // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 1.5957691216057308f * 0.044715f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int ACT>
__device__ __forceinline__ float act_of(float h) {
    if constexpr (ACT == kActRelu) return h > 0.f ? h : (h != h ? h : 0.f);
    if constexpr (ACT == kActGelu) return 0.5f * h * (1.f + erff(h * 0.70710678118654752f));
    if constexpr (ACT == kActGeluTanh) return h * reciprocal_fast(1.f + exp2_fast(h * fmaf(-kGeluC3 * kLog2e, h * h, -kGeluC * kLog2e)));
    if constexpr (ACT == kActSilu) return h * reciprocal_fast(1.f + exp2_fast(h * -kLog2e));
    return h;
}
// act(h) and act'(h). The square in the slope stops at 400 (|h| = 20), where s has long reached 0 or 1: further out the
// products would meet infinity * 0.
template <int ACT>
__device__ __forceinline__ float act_slope(float h, float* value) {
    if constexpr (ACT == kActRelu) {
        *value = act_of<kActRelu>(h);
        return h > 0.f ? 1.f : (h != h ? h : 0.f);
    }
    if constexpr (ACT == kActGelu) {
        const float cdf = 0.5f * (1.f + erff(h * 0.70710678118654752f));
        *value = h * cdf;
        return fmaf(h, 0.3989422804014327f * exp2_fast(fminf(h * h, 400.f) * (-0.5f * kLog2e)), cdf);
    }
    if constexpr (ACT == kActGeluTanh) {
        const float w = fminf(h * h, 400.f);
        const float s = reciprocal_fast(1.f + exp2_fast(h * fmaf(-kGeluC3 * kLog2e, w, -kGeluC * kLog2e)));
        *value = h * s;
        return fmaf(*value * (1.f - s), fmaf(3.f * kGeluC3, w, kGeluC), s);
    }
    if constexpr (ACT == kActSilu) {
        const float s = reciprocal_fast(1.f + exp2_fast(h * -kLog2e));
        *value = h * s;
        return fmaf(*value, 1.f - s, s);
    }
    *value = h;
    return 1.f;
}

// ---- epilogue: memory side -------------------------------------------------------------------------------------------
// 32 values of a bf16 row on a 16-byte boundary: four wide loads, or one by one where the tensor's edge cuts it off
__device__ __forceinline__ void load32(const __nv_bfloat16* p, int n, uint4* raw) {
    if (n >= 32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = ld_global_v4(p + 8 * j);
    } else {
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t lo = 2 * j < n ? (uint32_t)__bfloat16_as_ushort(p[2 * j]) : 0u;
            const uint32_t hi = 2 * j + 1 < n ? (uint32_t)__bfloat16_as_ushort(p[2 * j + 1]) : 0u;
            w[j] = lo | (hi << 16);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
}
__device__ __forceinline__ float bf16_at(const uint4* raw, int j) {   // j is a constant after unrolling
    const uint4 v = raw[j / 8];
    const uint32_t w = (j / 2) % 4 == 0 ? v.x : (j / 2) % 4 == 1 ? v.y : (j / 2) % 4 == 2 ? v.z : v.w;
    return __uint_as_float((j & 1) ? (w & 0xFFFF0000u) : (w << 16));
}
// Value j of 32 whole numbers of a checkpoint
__device__ __forceinline__ float s8_at(const uint4* raw, int j) {   // j is a constant after unrolling
    const uint4 v = raw[j / 16];
    const uint32_t w = ((j / 4) % 4 == 0 ? v.x : (j / 4) % 4 == 1 ? v.y : (j / 4) % 4 == 2 ? v.z : v.w) ^ 0x80808080u;
    return j % 4 == 0 ? s8_of_biased<0>(w) : j % 4 == 1 ? s8_of_biased<1>(w) : j % 4 == 2 ? s8_of_biased<2>(w) : s8_of_biased<3>(w);
}
// Eight neighbours into a bf16 row on a 16-byte boundary, of which `n` (one at least) have a place there
__device__ __forceinline__ void store8(__nv_bfloat16* p, int n, uint4 v) {
    if (n >= 8) {
        *(uint4*)p = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < n) ((unsigned short*)p)[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
}
__device__ __forceinline__ uint4 pack8(const float* f) {
    uint4 v;
    __nv_bfloat162* h = (__nv_bfloat162*)&v;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    return v;
}
// Four rows' pieces of 64 bytes, four lanes to a row with eight neighbours each (`d`), in rows that start on no 16-byte boundary: a lane writes the
// aligned block that ends among its values, with the last ones of the lane before it, the first lane of a row with those of the piece before
// (`carry`). Only a row's ends go value by value. `at` + i * step: where the lane's values of row i go; `rows`: how many of the four exist;
// `n`: how many of a lane's values exist (any number). All lanes of the warp come here.
__device__ __forceinline__ void put_joined(const uint4* d, uint4* carry, char* at, int64_t step, int rows, int n, int lane, bool first, bool last) {
    const bool opens = (lane & 3) == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[8] = {0, 0, 0, 0, d[i].x, d[i].y, d[i].z, d[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __shfl_up_sync(0xFFFFFFFFu, w[4 + j], 1);
        if (opens) {
            w[0] = carry[i].x; w[1] = carry[i].y; w[2] = carry[i].z; w[3] = carry[i].w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) (&carry[i].x)[j] = __shfl_sync(0xFFFFFFFFu, w[4 + j], lane | 3);
        char* p = at + i * step;
        const int past = (int)((uintptr_t)p & 15u), own = 2 * min(max(n, 0), 8);   // bytes behind a boundary; bytes that exist
        if (i >= rows || n <= -8) continue;
        // of the 32 bytes from p - 16 on: the block [16 - past, 32 - past), and what of it exists
        const int from = (opens && first) ? 16 : 16 - past, to = 16 + min(own, 16 - past);
        if (to - from == 16) {
            uint32_t t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = w[j];
            *(uint4*)(p - past) = past == 0 ? d[i] : from_byte<2>(t, (uint32_t)(16 - past));
        } else if (n > 0) {
            store_some<unsigned short>(p - 16, w, from, to);
        } else {   // nothing of its own: the end of the lane's before it
            store_some<unsigned short>(p - 16, w, 16 - past, 16 + 2 * n);
        }
        if (last && (lane & 3) == 3 && own > 16 - past) store_some<unsigned short>(p - 16, w, 32 - past, 16 + own);
    }
}
// Where in the warp's 2 KB the bytes [16 j, 16 j + 16) of row r of a [32 rows][64 bytes] piece lie
__device__ __forceinline__ uint32_t in_piece(uint32_t stage, int r, int byte) {
    return stage + (uint32_t)(r * 64 + (((byte >> 4) ^ ((r >> 1) & 3)) << 4) + (byte & 15));
}
// The pieces of rows that do not start on 16-byte boundaries, W bytes at a time (8, 4 or 2: what all of them start on): the lanes
// cover a row side by side, so that an access is a few whole row segments. (One lane's 2 bytes at a time at a stride of 16, as a
// row's wide blocks lie, took ten times as long: 12837 x 7860 with h kept, 888 us.) Out of line: most calls never come here.
template <int W, typename V>
__device__ __forceinline__ void put_narrow_of(uint32_t stage, int lane, char* out, int64_t ld_bytes, int rows, int bytes) {
    constexpr int kLanes = 64 / W, kRows = 32 / kLanes;
    const int byte = lane % kLanes * W;
#pragma unroll 4
    for (int i = 0; i < 32 / kRows; ++i) {
        const int r = i * kRows + lane / kLanes;
        const uint32_t at = in_piece(stage, r, byte);
        char* o = out + r * ld_bytes + byte;
        if (r >= rows) continue;
        if (byte + W <= bytes) {
            *(V*)o = *(const V*)__cvta_shared_to_generic(at);
        } else {
            for (int b = 0; byte + b < bytes; b += 2) *(unsigned short*)(o + b) = *(const unsigned short*)__cvta_shared_to_generic(at + b);
        }
    }
}
__device__ __noinline__ void put_narrow(uint32_t stage, int lane, void* out, int64_t ld_bytes, int rows, int bytes, int width) {
    if (width == 8) put_narrow_of<8, uint2>(stage, lane, (char*)out, ld_bytes, rows, bytes);
    else if (width == 4) put_narrow_of<4, uint32_t>(stage, lane, (char*)out, ld_bytes, rows, bytes);
    else put_narrow_of<2, unsigned short>(stage, lane, (char*)out, ld_bytes, rows, bytes);
}
template <int W, typename V>
__device__ __forceinline__ void get_narrow_of(uint32_t stage, int lane, const char* src, int64_t ld_bytes, int rows, int bytes) {
    constexpr int kLanes = 64 / W, kRows = 32 / kLanes, kBatch = 8;
    const int byte = lane % kLanes * W;
#pragma unroll 1
    for (int i = 0; i < 32 / kRows; i += kBatch) {
        V v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int r = (i + k) * kRows + lane / kLanes;
            const char* p = src + r * ld_bytes + byte;
            v[k] = V{};
            if (r >= rows) continue;
            if (byte + W <= bytes) {
                v[k] = *(const V*)p;
            } else {
                for (int b = 0; byte + b < bytes; b += 2) ((unsigned short*)&v[k])[b / 2] = *(const unsigned short*)(p + b);
            }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) *(V*)__cvta_shared_to_generic(in_piece(stage, (i + k) * kRows + lane / kLanes, byte)) = v[k];
    }
}
__device__ __noinline__ void get_narrow(uint32_t stage, int lane, const void* src, int64_t ld_bytes, int rows, int bytes, int width) {
    __syncwarp();   // the reads of the piece before are done
    if (width == 8) get_narrow_of<8, uint2>(stage, lane, (const char*)src, ld_bytes, rows, bytes);
    else if (width == 4) get_narrow_of<4, uint32_t>(stage, lane, (const char*)src, ld_bytes, rows, bytes);
    else get_narrow_of<2, unsigned short>(stage, lane, (const char*)src, ld_bytes, rows, bytes);
    __syncwarp();
}
// A warp's [32 rows][32 columns] of bf16 results, one row per lane, through the warp's 2 KB of shared memory so that every
// store instruction writes 8 whole 64-byte row segments instead of 16 bytes in each of 32 rows. The 16-byte blocks of a row
// are XOR-swizzled by (row / 2) % 4: neither side has bank conflicts.
__device__ __forceinline__ void store_piece(uint32_t stage, int lane, const float* f, __nv_bfloat16* out, int64_t ldo, int row0, int col0, int M,
                                            int N, int width) {
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        __nv_bfloat162* h = (__nv_bfloat162*)&raw[j];
#pragma unroll
        for (int t = 0; t < 4; ++t) h[t] = __floats2bfloat162_rn(f[8 * j + 2 * t], f[8 * j + 2 * t + 1]);
    }
    __syncwarp();   // the reads of the piece before are done
    const uint32_t mine = stage + (uint32_t)lane * 64;
    const int sw = (lane >> 1) & 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) st_smem_v4(mine + (uint32_t)((j ^ sw) << 4), raw[j]);
    __syncwarp();
    if (width != 16) {
        put_narrow(stage, lane, out + (int64_t)row0 * ldo + col0, ldo * 2, min(32, M - row0), 2 * min(32, N - col0), width);
        return;
    }
    const int cb = lane & 3, r0 = lane >> 2, col = col0 + cb * 8;
    uint4 d[4];   // rows r0 + 8 i
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = ld_smem_v4(stage + (uint32_t)(i * 512 + r0 * 64 + ((cb ^ ((r0 >> 1) & 3)) << 4)));
    __nv_bfloat16* op = out + (int64_t)(row0 + r0) * ldo + col;
    if (col + 8 <= N) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row0 + r0 + 8 * i < M) *(uint4*)(op + 8 * i * ldo) = d[i];
    } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            if (row0 + r0 + 8 * i >= M) break;
            const uint4 x = i == 0 ? d[0] : i == 1 ? d[1] : i == 2 ? d[2] : d[3];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (col + t < N) ((unsigned short*)(op + 8 * i * ldo))[t] = (unsigned short)(w[t / 2] >> (16 * (t & 1)));
        }
    }
}
// 32 values of this lane's row into the 8-bit checkpoint; returns the exponent. (Columns past N carry zeros here, and the
// padding of a row takes them.)
__device__ __forceinline__ uint32_t keep_row32(const float* f, int8_t* qp, int n, bool live) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) m = abs_max(m, f[j]);
    const uint32_t e = act8_exponent(__float_as_uint(m));
    const float inv = act8_inverse_step(e);
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = e == 255u ? 0u : act8_quantise4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3], inv);
    if (live) {
        *(uint4*)qp = make_uint4(w[0], w[1], w[2], w[3]);
        if (n > 16) *(uint4*)(qp + 16) = make_uint4(w[4], w[5], w[6], w[7]);
    }
    return e;
}

// ---- gated dgrad: the epilogue ---------------------------------------------------------------------------------------
// Two neighbours of a sum come in and three go out, twice what the other epilogues move. So the sums change places once, 32 rows and 32 columns at
// a time through the warp's 4 KB, and a lane then has eight columns of four rows, eight apart, of everything: loads and stores of whole 16-byte
// blocks, four lanes to a row, none of which goes through shared memory (16384 tokens, 5504 x 2048, silu: 439 us with a row to a lane, 376 so; sixteen
// warps with 16 columns at a time, two lanes to a row, 510). Whole tiles need no checks, and ask for the neighbours of the next unit, also of the
// next tile's first, while one is worked on: 350. The accumulator is given back with the last read; what is written leaves L2 first: 345.
// Without these loads 300, without these stores 300, with neither 240, which is 20 waves of MMAs: 64 x 22 tiles, the last column's half padding, on 74
// pairs, where the values fill 18.6. What the rest waits for is not known: nothing is full (4096 tokens, from bf16 / from 8 bits: the tensor pipe busy 64 %
// of the time, L1 64 and 65 %, L2 42 and 40 %, HBM 34 and 25 %, issue slots 28 and 41 %).
template <int ACT, int BN>
__device__ __forceinline__ void gated_dgrad_epilogue(const LinParams& p, uint32_t tmem_base, uint64_t* tfull_bar, uint64_t* tempty_bar, uint32_t* tmem_slot,
                                                     uint32_t stage, int pair, int cr, int ew, int lane) {
    constexpr int kColumns = BN / 2, kUnits = kColumns / 32;   // of a warp
    const int quarter = ew & 3, cbase = (ew >> 2) * kColumns;
    const int qrow = lane >> 2, qcol = (lane & 3) * 8;          // a lane's place in a unit: rows qrow, qrow + 8, ..., eight columns
    const bool kept8 = p.q != nullptr;
    const bool wide = (kept8 || (p.pre_width == 16 && p.pre_up_width == 16)) && p.out_up_width == 16;   // (out and out2 always are)
    const unsigned long long limit_ns = p.limit_ns;
    auto first_row = [&](const Tile& t) { return t.m * 2 * BM + cr * BM + quarter * 32; };
    auto first_column = [&](const Tile& t) { return t.n * BN + cbase; };
    // whole tiles on 16-byte boundaries: nothing to check, and the neighbours of the next tile's first unit are asked for in this one's last
    auto whole = [&](const Tile& t) { return wide && t.runs == 1 && first_row(t) + 32 <= p.M && first_column(t) + kColumns <= p.N; };
    // where four sums of a unit lie: the 16-byte blocks of a row are XOR-swizzled by it, neither side has bank conflicts
    auto in_unit = [&](int r, int j) { return stage + (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4)); };
    auto lay_down = [&](const uint32_t* v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) st_smem_v4(in_unit(lane, j), make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
    };
    auto unpack16 = [&](uint4 g, uint4 u, float* vg, float* vu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            vg[j] = bf16_at(&g, j);
            vu[j] = bf16_at(&u, j);
        }
    };
    auto unpack8 = [&](uint4 g, uint4 u, uint32_t eg, uint32_t eu, float* vg, float* vu) {
        const float step = act8_step(eg & 255u), step_up = act8_step(eu & 255u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            vg[j] = s8_at(&g, j) * step;
            vu[j] = s8_at(&u, j) * step_up;
        }
    };
    // eight columns of row qrow + 8 i: the gradients of g (in vg to begin with) and u (in vu), and act(g) u
    auto turn = [&](int i, float* vg, float* vu, float* va) {
        const uint4 lo = ld_smem_v4(in_unit(8 * i + qrow, qcol / 4)), hi = ld_smem_v4(in_unit(8 * i + qrow, qcol / 4 + 1));
        const uint32_t da[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = __uint_as_float(da[j]);
            float value;
            const float slope = act_slope<ACT>(vg[j], &value);
            va[j] = value * vu[j];
            vg[j] = d * vu[j] * slope;
            vu[j] = d * value;
        }
    };
    auto exponents = [&](const uint8_t* e) -> uint32_t {   // a byte for 32 columns; rows of e are padded to 16
        return kUnits == 4 ? *(const uint32_t*)e : (uint32_t)*(const uint16_t*)e;
    };
    uint4 g[4], u[4];
    uint32_t eg[4], eu[4];
    // the neighbours of a whole tile's unit `c`, in rows qrow + 8 i
    auto place = [&](const Tile& t, int c, const char** at, const char** at_up) {
        const int64_t r = first_row(t) + qrow;
        const int col = first_column(t) + c * 32 + qcol;
        *at = kept8 ? (const char*)(p.q + r * p.ldq + col) : (const char*)(p.pre + r * p.ldpre + col);
        *at_up = kept8 ? (const char*)(p.q_up + r * p.ldq_up + col) : (const char*)(p.pre_up + r * p.ldpre + col);
    };
    const int64_t step = kept8 ? 8 * p.ldq : 16 * p.ldpre, step_up = kept8 ? 8 * p.ldq_up : 16 * p.ldpre;   // bytes between rows qrow + 8 i
    auto load = [&](int i, const char* at, const char* at_up) {
        if (kept8) {
            const uint2 a = *(const uint2*)(at + i * step), b = *(const uint2*)(at_up + i * step_up);
            g[i] = make_uint4(a.x, a.y, 0, 0);
            u[i] = make_uint4(b.x, b.y, 0, 0);
        } else {
            g[i] = ld_global_v4(at + i * step);
            u[i] = ld_global_v4(at_up + i * step_up);
        }
    };
    auto load_exponents = [&](const Tile& t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = first_row(t) + 8 * i + qrow;
            const bool there = kept8 && r < p.M && first_column(t) < p.N;
            eg[i] = there ? exponents(p.e + r * p.lde + first_column(t) / 32) : 0u;
            eu[i] = there ? exponents(p.e_up + r * p.lde_up + first_column(t) / 32) : 0u;
        }
    };
    TileWalk walk(p.grid, pair);
    Tile t, coming = {};
    uint32_t tc = 0;
    bool loaded = false;
    for (bool more = walk.next(p.grid, t); more; t = coming, ++tc) {
        more = walk.next(p.grid, coming);
        const uint32_t buf = tc & 1u;
        const int row0 = first_row(t), colw = first_column(t);
        const bool is_whole = whole(t);
        if (is_whole && !loaded) {
            const char *at, *at_up;
            place(t, 0, &at, &at_up);
#pragma unroll
            for (int i = 0; i < 4; ++i) load(i, at, at_up);
        }
        if (!loaded) load_exponents(t);
        loaded = false;
        const bool waited = ew != 0 || mbar_wait(&tfull_bar[buf], (tc >> 1) & 1u, limit_ns * 4);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        if (!meet_all(1, 32 * kLinEpilogueWarps, waited)) {
            if (!waited && lane == 0) give_up_pair(p.err_flag, 23u, tmem_slot);
            break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * (uint32_t)BN + (uint32_t)cbase;
        auto release = [&]() {   // this warp has read the accumulator
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_pair(mapa_cluster(smem_u32(&tempty_bar[buf]), 0));
        };
        uint32_t v[32];
        if (is_whole) {
            const char *at, *at_up;
            const int64_t place_out = (int64_t)(row0 + qrow) * p.ldo + colw + qcol;
            char *o = (char*)(p.out + place_out), *o_up = (char*)(p.out_up + place_out);
            char* o2 = p.out2 == nullptr ? nullptr : (char*)(p.out2 + (int64_t)(row0 + qrow) * p.ldo2 + colw + qcol);
            const int64_t ostep = 16 * p.ldo, ostep2 = 16 * p.ldo2;
            loaded = more && whole(coming);
            tmem_ld32_issue(taddr, v);
#pragma unroll 1
            for (int c = 0; c < kUnits; ++c) {
                const bool last = c + 1 == kUnits, ahead = !last || loaded;
                if (last) place(coming, 0, &at, &at_up);
                else place(t, c + 1, &at, &at_up);
                tmem_wait_ld(v);
                __syncwarp();   // what was in the warp's memory has been read
                lay_down(v);
                if (!last) tmem_ld32_issue(taddr + (uint32_t)(c + 1) * 32u, v);
                else release();
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float vg[8], vu[8], va[8];
                    if (kept8) unpack8(g[i], u[i], eg[i] >> (8 * c), eu[i] >> (8 * c), vg, vu);
                    else unpack16(g[i], u[i], vg, vu);
                    if (ahead) load(i, at, at_up);
                    turn(i, vg, vu, va);
                    __stcs((uint4*)(o + i * ostep), pack8(vg));
                    __stcs((uint4*)(o_up + i * ostep), pack8(vu));
                    if (o2 != nullptr) __stcs((uint4*)(o2 + i * ostep2), pack8(va));
                }
                o += 64;
                o_up += 64;
                if (o2 != nullptr) o2 += 64;
            }
            if (loaded) load_exponents(coming);
            continue;
        }
        // a tile with edges, with rows on smaller boundaries, or in parts: one unit with its sums in v, a row to a lane
        uint4 carry[4];
        auto finish = [&](int c) {
            const int col = colw + c * 32, n = p.N - col - qcol;   // columns of this lane that exist
            auto get = [&](const __nv_bfloat16* pre, const int8_t* q, int64_t ldq, uint4* to) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t r = row0 + 8 * i + qrow;
                    to[i] = make_uint4(0, 0, 0, 0);
                    if (r >= p.M || n <= 0) continue;
                    if (kept8) {
                        const uint2 b = *(const uint2*)(q + r * ldq + col + qcol);   // (rows are padded to 16 bytes)
                        to[i] = make_uint4(b.x, b.y, 0, 0);
                    } else {
                        to[i] = load_across<2>((const char*)(pre + r * p.ldpre + col + qcol), 2 * min(n, 8));
                    }
                }
            };
            auto put = [&](const uint4* d, __nv_bfloat16* out, int64_t ldo) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t r = row0 + 8 * i + qrow;
                    if (r < p.M && n > 0) store8(out + r * ldo + col + qcol, n, d[i]);
                }
            };
            get(p.pre, p.q, p.ldq, g);
            get(p.pre_up, p.q_up, p.ldq_up, u);
            __syncwarp();   // what was in the warp's memory has been read
            lay_down(v);
            __syncwarp();
            uint4 a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float vg[8], vu[8], va[8];
                if (kept8) unpack8(g[i], u[i], eg[i] >> (8 * c), eu[i] >> (8 * c), vg, vu);
                else unpack16(g[i], u[i], vg, vu);
                turn(i, vg, vu, va);
                g[i] = pack8(vg);
                u[i] = pack8(vu);
                a[i] = pack8(va);
            }
            put(g, p.out, p.ldo);
            if (p.out2 != nullptr) put(a, p.out2, p.ldo2);
            if (p.out_up_width == 16) {
                put(u, p.out_up, p.ldo);
            } else {
                const int r = row0 + qrow;
                put_joined(u, carry, (char*)(p.out_up + (int64_t)r * p.ldo + col + qcol), 16 * p.ldo, r >= p.M ? 0 : min(4, (p.M - r + 7) / 8), n, lane, c == 0,
                           c + 1 == kUnits || col + 32 >= p.N);
            }
        };
        if (row0 >= p.M) {   // nothing of this warp's 32 rows exists
            release();
            continue;
        }
        if (t.runs == 1) {
#pragma unroll 1
            for (int c = 0; c < kUnits; ++c) {
                if (colw + c * 32 >= p.N) break;   // warp-uniform
                tmem_ld32_issue(taddr + (uint32_t)c * 32u, v);
                tmem_wait_ld(v);
                finish(c);
            }
            release();
            continue;
        }
        // shared tile: see the other epilogue
        constexpr int64_t kWarpFloats = kUnits * 1024;
        auto part_of = [&](int worker, int slot) {
            return p.partial + ((((int64_t)worker * 2 + slot) * 2 + cr) * kLinEpilogueWarps + ew) * kWarpFloats + lane * 4;
        };
        float* mine = part_of(pair, t.slot);
#pragma unroll 1
        for (int c = 0; c < kUnits; ++c) {
            if (colw + c * 32 >= p.N) break;
            tmem_ld32_issue(taddr + (uint32_t)c * 32u, v);
            tmem_wait_ld(v);
#pragma unroll
            for (int j = 0; j < 8; ++j) *(uint4*)(mine + c * 1024 + j * 128) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
        release();
        __threadfence();
        __syncwarp();
        unsigned last = 0;
        unsigned* count = p.arrived + ((int64_t)t.index * 2 + cr) * kLinEpilogueWarps + ew;
        if (lane == 0) last = atomicAdd(count, 1u) == (unsigned)(t.runs - 1) ? 1u : 0u;
        if (__shfl_sync(0xFFFFFFFFu, last, 0) == 0u) continue;
        __threadfence();
        if (lane == 0) *count = 0u;   // at rest for the next launch
#pragma unroll 1
        for (int c = 0; c < kUnits; ++c) {
            if (colw + c * 32 >= p.N) break;
            float f[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = 0.f;
#pragma unroll 1
            for (int r = 0; r < t.runs; ++r) {
                const float* src = part_of(t.first + r, TileWalk::slot_of(p.grid, t, r)) + c * 1024;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float4 x = __ldcg((const float4*)(src + j * 128));
                    f[4 * j] += x.x; f[4 * j + 1] += x.y; f[4 * j + 2] += x.z; f[4 * j + 3] += x.w;
                }
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(f[j]);
            finish(c);
        }
    }
}

// ---- the kernel ------------------------------------------------------------------------------------------------------
template <bool DGRAD, int ACT, int BN, int KIND>
__global__ void __launch_bounds__(kLinThreads, 1) linear_fused_kernel(const __grid_constant__ LinParams p) {
    constexpr bool GATED_FWD = KIND == kLinGated && !DGRAD, GATED_DGRAD = KIND == kLinGated && DGRAD;
    using L = LinSmem<BN, GATED_DGRAD>;
    constexpr int kWide = GATED_FWD ? BN / 2 : BN;   // output columns of a tile: of a gated one's BN products, half are the gate's
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full_bar = (uint64_t*)(smem + L::kTileBytes);
    uint64_t* empty_bar = full_bar + L::kStages;
    uint64_t* tfull_bar = empty_bar + L::kStages;   // [2] accumulator complete
    uint64_t* tempty_bar = tfull_bar + 2;           // [2] accumulator drained
    uint32_t* tmem_slot = (uint32_t*)(tempty_bar + 2);
    float* bias_smem = (float*)(smem + L::kTileBytes + L::kBarBytes);
    uint8_t* stage_out = smem + L::kTileBytes + L::kBarBytes + L::kBiasBytes;

    const int cr = (int)cluster_ctarank();
    const bool leader = cr == 0;
    const int pair = (int)blockIdx.x / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned long long limit_ns = p.limit_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull_bar[b], 1);
            mbar_init(&tempty_bar[b], 2 * kLinEpilogueWarps);   // the epilogue warps of both CTAs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_arrive_all();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)(2 * BN))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    cluster_wait_all();   // the peer's barriers must exist before anything is signalled on them
    wait_predecessor();
    uint32_t tmem_base = 0;
    if (warp == 1 || warp >= 4) {   // (the loads need no TMEM and do not wait for it)
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        meet_named(2, 32 * (1 + kLinEpilogueWarps));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_base = tmem_address(tmem_slot);
        allow_successor();
    }

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLinRegsIssue));
        if (warp == 0) {
            // ---- TMA producer ----
            if (lane == 0) {
                asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_a) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_b) : "memory");
                TileWalk walk(p.grid, pair);
                Tile t;
                uint32_t it = 0;
                bool ok = true;
                while (ok && walk.next(p.grid, t)) {
                    // (gated: the leader has the gate's rows of w, the other CTA the rows behind them)
                    const int m0 = t.m * 2 * BM + cr * BM, n0 = t.n * kWide + cr * (GATED_FWD ? p.N : BN / 2);
                    for (int k = 0; k < t.nk; k += L::kSub, ++it) {
                        const int s = it % L::kStages;
                        const int n = min(L::kSub, t.nk - k);
                        if (!mbar_wait(&empty_bar[s], ((it / L::kStages) & 1u) ^ 1u, limit_ns)) {
                            give_up_pair(p.err_flag, 21u, tmem_slot);
                            ok = false;
                            break;
                        }
                        if (leader) mbar_expect_tx(&full_bar[s], 2u * (uint32_t)(L::kStageBytes * n));   // both CTAs' bytes
                        const uint32_t fb = mapa_cluster(smem_u32(&full_bar[s]), 0);
                        for (int u = 0; u < n; ++u) {
                            uint8_t* sa = smem + (s * L::kSub + u) * L::kStageBytes;
                            uint8_t* sb = sa + L::kABytes;
                            const int k0 = (t.k0 + k + u) * BK;
                            tma_load_2d_pair(sa, &p.map_a, fb, k0, m0);   // [128 rows][64 k]
                            if constexpr (!DGRAD) {
                                tma_load_2d_pair(sb, &p.map_b, fb, k0, n0);   // [BN / 2 rows][64 k]
                            } else if (p.b_blocked) {
                                tma_load_3d_pair(sb, &p.map_b, fb, 0, k0, n0 / 64);   // [BN / 128 blocks][64 k][64 n]
                            } else {
#pragma unroll
                                for (int j = 0; j < BN / 128; ++j) tma_load_2d_pair(sb + j * 64 * 128, &p.map_b, fb, n0 + 64 * j, k0);
                            }
                        }
                    }
                }
            }
        } else if (warp == 1) {
            // ---- MMA issuer ----
            if (lane == 0 && leader) {
                const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((DGRAD ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
                                       ((uint32_t)((2 * BM) >> 4) << 24);
                // The issue of an MMA blocks while the tensor core's queue is full, and the queue is short: what this thread does
                // between two k-steps is time in which it may run dry. So the next k-step's barrier is asked while the current one's
                // MMAs are issued, and descriptors and ring positions are kept as running values.
                // K-major: 8-row groups 1024 B apart, 16 k are 32 B inside the swizzle span; MN-major: 64-column blocks 8192 B
                // apart, 16 k-rows are 2048 B. (Descriptors count in 16 bytes.)
                constexpr uint32_t kNextB = DGRAD ? 2048 >> 4 : 32 >> 4;
                const uint64_t desc_a = make_desc(smem_u32(smem), 16, 1024);
                const uint64_t desc_b = DGRAD ? make_desc(smem_u32(smem + L::kABytes), 8192, 1024) : make_desc(smem_u32(smem + L::kABytes), 16, 1024);
                TileWalk walk(p.grid, pair);
                Tile t;
                uint32_t s = 0, ph = 0, tc = 0;
                bool ok = true, have = false;
                while (ok && walk.next(p.grid, t)) {
                    const uint32_t buf = tc & 1u;
                    if (!mbar_wait(&tempty_bar[buf], ((tc >> 1) & 1u) ^ 1u, limit_ns)) {
                        give_up_pair(p.err_flag, 24u, tmem_slot);
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t tmem_d = tmem_base + buf * (uint32_t)BN;
                    for (int k = 0; k < t.nk; k += L::kSub) {
                        // consumers wait longer than producers, so that the wait that reports is the one at the root
                        if (!have && !mbar_wait(&full_bar[s], ph, limit_ns * 2)) {
                            give_up_pair(p.err_flag, 22u, tmem_slot);
                            ok = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t next = s + 1 == L::kStages ? 0 : s + 1, next_ph = next == 0 ? ph ^ 1u : ph;
                        const uint64_t da = desc_a + s * (uint32_t)(L::kSub * L::kStageBytes >> 4), db = desc_b + s * (uint32_t)(L::kSub * L::kStageBytes >> 4);
                        umma_bf16_pair(tmem_d, da, db, idesc, k ? 1u : 0u);
#pragma unroll
                        for (int u = 1; u < BK / UMMA_K; ++u) umma_bf16_pair(tmem_d, da + u * 2, db + u * kNextB, idesc, 1u);
                        have = mbar_try_wait(&full_bar[next], next_ph);
                        if (k + 1 < t.nk) {
#pragma unroll
                            for (int u = 0; u < BK / UMMA_K; ++u)
                                umma_bf16_pair(tmem_d, da + (L::kStageBytes >> 4) + u * 2, db + (L::kStageBytes >> 4) + u * kNextB, idesc, 1u);
                        }
                        umma_commit_pair(&empty_bar[s]);   // frees the stage in both CTAs when these MMAs have read it
                        s = next;
                        ph = next_ph;
                    }
                    umma_commit_pair(&tfull_bar[buf]);     // (also on error, so that the epilogue moves on)
                    ++tc;
                }
            }
        }
    } else if constexpr (GATED_DGRAD) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLinRegsEpilogue));
        gated_dgrad_epilogue<ACT, BN>(p, tmem_base, tfull_bar, tempty_bar, tmem_slot, smem_u32(stage_out) + (uint32_t)((warp - 4) * L::kWarpBytes), pair, cr,
                                      warp - 4, lane);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLinRegsEpilogue));
        // ---- epilogue ----
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2, etid = ew * 32 + lane;
        constexpr int kPieces = kWide / 64;   // 32-column pieces of a warp
        const uint32_t stage = smem_u32(stage_out) + (uint32_t)ew * 2048;
        TileWalk walk(p.grid, pair);
        Tile t;
        uint32_t tc = 0;
        [[maybe_unused]] const DropKeys<KIND == kLinDropoutSeed> key(p.drop);
        while (walk.next(p.grid, t)) {
            const uint32_t buf = tc & 1u;
            const int tile_n = t.n * kWide, row0 = t.m * 2 * BM + cr * BM + quarter * 32, row = row0 + lane;
            const int cbase = half * (kWide / 2), colw = tile_n + cbase;   // first column of this warp
            const bool live = row < p.M;
            const uint32_t bs = smem_u32(bias_smem) + buf * (uint32_t)(BN * 4);
            if constexpr (!DGRAD) {
                if (etid < BN) {   // (BN = 128: the first four warps)
                    const int col = tile_n + etid % kWide, at = GATED_FWD && etid >= kWide ? p.N + col : col;
                    float v = 0.f;
                    if (col < p.N) v = p.bias32 != nullptr ? p.bias32[at] : p.bias != nullptr ? __bfloat162float(p.bias[at]) : 0.f;
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(bs + (uint32_t)etid * 4), "f"(v) : "memory");
                }
            }
            // What a piece needs from memory (residual, or h) is requested before the piece ahead of it is worked on, the first
            // one before the wait for the accumulator.
            uint4 aux[4], coming[4];
            uint32_t ex = 0;
            const __nv_bfloat16* aux_row = DGRAD ? p.pre : p.res;
            const int64_t aux_ld = DGRAD ? p.ldpre : p.ldres;
            const int aux_width = DGRAD ? p.pre_width : p.aux_width;
            const bool kept8 = DGRAD && p.q != nullptr;
            auto fetch = [&](int c) {
                const int col = colw + c * 32;
                if (c >= kPieces || col >= p.N) return;   // warp-uniform
                if (!kept8 && aux_row != nullptr && aux_width != 16) {
                    get_narrow(stage, lane, aux_row + (int64_t)row0 * aux_ld + col, aux_ld * 2, min(32, p.M - row0), 2 * min(32, p.N - col), aux_width);
#pragma unroll
                    for (int j = 0; j < 4; ++j) coming[j] = ld_smem_v4(in_piece(stage, lane, j * 16));
                    return;
                }
                if (!live) return;
                if (kept8) {
                    const int8_t* qp = p.q + (int64_t)row * p.ldq + col;
                    coming[0] = ld_global_v4(qp);
                    if (col + 16 < p.N) coming[1] = ld_global_v4(qp + 16);
                } else if (aux_row != nullptr) {
                    load32(aux_row + (int64_t)row * aux_ld + col, p.N - col, coming);
                }
            };
#pragma unroll
            for (int j = 0; j < 4; ++j) coming[j] = make_uint4(0, 0, 0, 0);
            if (t.runs == 1) fetch(0);
            if (kept8 && live && colw < p.N) {   // one byte per piece; rows of e are padded to 16
                if constexpr (kPieces == 4) ex = *(const uint32_t*)(p.e + (int64_t)row * p.lde + colw / 32);
                else ex = *(const uint16_t*)(p.e + (int64_t)row * p.lde + colw / 32);
            }
            // One barrier of the epilogue warps per tile: publishes the bias, and makes the decision to give up uniform. One warp
            // asks for the accumulator, the others sleep at this barrier (asking takes issue slots from the MMAs' thread).
            const bool waited = ew != 0 || mbar_wait(&tfull_bar[buf], (tc >> 1) & 1u, limit_ns * 4);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (!meet_all(1, 32 * kLinEpilogueWarps, waited)) {
                if (!waited && lane == 0) give_up_pair(p.err_flag, 23u, tmem_slot);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * (uint32_t)BN + (uint32_t)cbase;
            auto release = [&]() {   // this warp has read the accumulator
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_cluster(smem_u32(&tempty_bar[buf]), 0));
            };
            // one 32-column piece with its values in f (gated: the activated gate in f, the other factor in u)
            uint32_t ewrite = 0;
            [[maybe_unused]] uint32_t ewrite_up = 0;
            auto add_bias = [&](float* f, int at) {
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const uint4 b = ld_smem_v4(bs + (uint32_t)(at + j) * 4);
                    f[j] += __uint_as_float(b.x); f[j + 1] += __uint_as_float(b.y);
                    f[j + 2] += __uint_as_float(b.z); f[j + 3] += __uint_as_float(b.w);
                }
            };
            // gated: the gate's piece first, to its activation
            [[maybe_unused]] auto finish_gate = [&](float* f, int c) {
                const int col = colw + c * 32;
                add_bias(f, cbase + c * 32);
                if (p.pre != nullptr) store_piece(stage, lane, f, p.pre, p.ldpre, row0, col, p.M, p.N, p.pre_width);
                if (p.q != nullptr) {
                    if (col + 32 > p.N) {   // behind the gate's last row of w, the tile has the other factor's first
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] = col + j < p.N ? f[j] : 0.f;
                    }
                    ewrite |= keep_row32(f, p.q + (int64_t)row * p.ldq + col, p.N - col, live) << (8 * c);
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) f[j] = act_of<ACT>(f[j]);
            };
            auto finish = [&](float* f, [[maybe_unused]] float* u, int c) {
                const int col = colw + c * 32;
#pragma unroll
                for (int j = 0; j < 4; ++j) aux[j] = coming[j];
                fetch(c + 1);
                if constexpr (GATED_FWD) {
                    add_bias(u, kWide + cbase + c * 32);
                    if (p.pre != nullptr) store_piece(stage, lane, u, p.pre_up, p.ldpre, row0, col, p.M, p.N, p.pre_up_width);
                    if (p.q != nullptr) ewrite_up |= keep_row32(u, p.q_up + (int64_t)row * p.ldq_up + col, p.N - col, live) << (8 * c);
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] *= u[j];
                } else if constexpr (!DGRAD) {
                    add_bias(f, cbase + c * 32);
                    if (p.pre != nullptr) store_piece(stage, lane, f, p.pre, p.ldpre, row0, col, p.M, p.N, p.pre_width);
                    if (p.q != nullptr) ewrite |= keep_row32(f, p.q + (int64_t)row * p.ldq + col, p.N - col, live) << (8 * c);
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] = act_of<ACT>(f[j]);
                    if constexpr (KIND >= kLinDropout) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) drop4(key, p.drop, (uint32_t)row, (uint32_t)(col + j) / 4, f + j);
                    }
                    if (p.res != nullptr) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] += bf16_at(aux, j);
                    }
                } else {
                    float a[32];
                    if (kept8) {
                        const float step = act8_step((ex >> (8 * c)) & 255u);
                        const uint32_t w[8] = {aux[0].x, aux[0].y, aux[0].z, aux[0].w, aux[1].x, aux[1].y, aux[1].z, aux[1].w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t biased = w[j] ^ 0x80808080u;
                            f[4 * j] *= act_slope<ACT>(s8_of_biased<0>(biased) * step, &a[4 * j]);
                            f[4 * j + 1] *= act_slope<ACT>(s8_of_biased<1>(biased) * step, &a[4 * j + 1]);
                            f[4 * j + 2] *= act_slope<ACT>(s8_of_biased<2>(biased) * step, &a[4 * j + 2]);
                            f[4 * j + 3] *= act_slope<ACT>(s8_of_biased<3>(biased) * step, &a[4 * j + 3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] *= act_slope<ACT>(bf16_at(aux, j), &a[j]);
                    }
                    if (p.out2 != nullptr) store_piece(stage, lane, a, p.out2, p.ldo2, row0, col, p.M, p.N, p.out2_width);
                }
                store_piece(stage, lane, f, p.out, p.ldo, row0, col, p.M, p.N, p.out_width);
            };
            if (row0 >= p.M) {   // nothing of this warp's 32 rows exists (few rows, or the last tile's second half)
                release();
                ++tc;
                continue;
            }
            uint32_t v[32];
            if constexpr (GATED_FWD) {
                if (t.runs == 1) {
                    // the next sums are on their way while these are worked on, and the accumulator is given back with the last
                    if (colw < p.N) tmem_ld32_issue(taddr, v);
#pragma unroll 1
                    for (int c = 0; c < kPieces; ++c) {
                        if (colw + c * 32 >= p.N) break;   // warp-uniform
                        float f[32], u[32];
                        tmem_wait_ld(v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
                        tmem_ld32_issue(taddr + (uint32_t)(kWide + c * 32), v);
                        finish_gate(f, c);
                        tmem_wait_ld(v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) u[j] = __uint_as_float(v[j]);
                        if (c + 1 < kPieces && colw + c * 32 + 32 < p.N) tmem_ld32_issue(taddr + (uint32_t)(c + 1) * 32u, v);
                        else release();
                        finish(f, u, c);
                    }
                    if (colw >= p.N) release();
                }
            } else if (t.runs == 1) {
                if (colw < p.N) tmem_ld32_issue(taddr, v);
#pragma unroll 1
                for (int c = 0; c < kPieces; ++c) {
                    if (colw + c * 32 >= p.N) break;   // warp-uniform
                    tmem_wait_ld(v);
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
                    if (c + 1 < kPieces && colw + c * 32 + 32 < p.N) tmem_ld32_issue(taddr + (uint32_t)(c + 1) * 32u, v);
                    finish(f, nullptr, c);
                }
                release();
            }
            if (t.runs > 1) {
                // shared tile: this pair's part goes to memory; the last one to arrive adds all parts in run order
                constexpr int kParts = BN / 64;   // (gated: the gate's pieces, then the other factor's)
                constexpr int64_t kWarpFloats = kParts * 1024;
                auto part_of = [&](int worker, int slot) {
                    return p.partial + ((((int64_t)worker * 2 + slot) * 2 + cr) * kLinEpilogueWarps + ew) * kWarpFloats + lane * 4;
                };
                float* mine = part_of(pair, t.slot);
#pragma unroll 1
                for (int c = 0; c < kParts; ++c) {
                    if (colw + c % kPieces * 32 >= p.N) continue;
                    tmem_ld32_issue(taddr + (uint32_t)(c / kPieces * kWide + c % kPieces * 32), v);
                    tmem_wait_ld(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        *(uint4*)(mine + c * 1024 + j * 128) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                }
                release();
                __threadfence();
                __syncwarp();
                unsigned last = 0;
                unsigned* count = p.arrived + ((int64_t)t.index * 2 + cr) * kLinEpilogueWarps + ew;
                if (lane == 0) last = atomicAdd(count, 1u) == (unsigned)(t.runs - 1) ? 1u : 0u;
                if (__shfl_sync(0xFFFFFFFFu, last, 0) != 0u) {
                    __threadfence();
                    if (lane == 0) *count = 0u;   // at rest for the next launch
                    fetch(0);
#pragma unroll 1
                    for (int c = 0; c < kPieces; ++c) {
                        if (colw + c * 32 >= p.N) break;
                        auto joined = [&](float* f, int part) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) f[j] = 0.f;
#pragma unroll 1
                            for (int r = 0; r < t.runs; ++r) {
                                const float* src = part_of(t.first + r, TileWalk::slot_of(p.grid, t, r)) + part * 1024;
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float4 x = __ldcg((const float4*)(src + j * 128));
                                    f[4 * j] += x.x; f[4 * j + 1] += x.y; f[4 * j + 2] += x.z; f[4 * j + 3] += x.w;
                                }
                            }
                        };
                        float f[32];
                        joined(f, c);
                        if constexpr (GATED_FWD) {
                            float u[32];
                            finish_gate(f, c);
                            joined(u, kPieces + c);
                            finish(f, u, c);
                        } else {
                            finish(f, nullptr, c);
                        }
                    }
                } else {
                    ++tc;
                    continue;
                }
            }
            if constexpr (!DGRAD) {
                if (p.q != nullptr && live && colw < p.N) {
                    if constexpr (kPieces == 4) *(uint32_t*)(p.e + (int64_t)row * p.lde + colw / 32) = ewrite;
                    else *(uint16_t*)(p.e + (int64_t)row * p.lde + colw / 32) = (uint16_t)ewrite;
                    if constexpr (GATED_FWD) *(uint16_t*)(p.e_up + (int64_t)row * p.lde_up + colw / 32) = (uint16_t)ewrite_up;
                }
            }
            ++tc;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();   // until here the peer may signal this CTA's barriers or read its shared memory
    if (warp == 1) {
        if (gave_up(tmem_slot)) let_copies_land();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)(2 * BN)) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
constexpr int64_t kArrivedWords = (int64_t)kMaxPairs * 2 * kLinEpilogueWarps;
constexpr int64_t kPartialFloats = (int64_t)kMaxPairs * 2 * 2 * kLinEpilogueWarps * 4 * 1024;

// How many CTA pairs of this kernel the device holds at once, within gemm_set_cta_limit().
template <auto kern>
cudaError_t pairs_of(int threads, int smem, int* pairs) {
    static int cached[64] = {};   // per kernel and device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    int n = dev >= 0 && dev < 64 ? cached[dev] : 0;
    if (n == 0) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t q = {};
        q.gridDim = dim3(2);
        q.blockDim = dim3(threads);
        q.dynamicSmemBytes = smem;
        cudaLaunchAttribute a[1] = {in_clusters(2)};
        q.attrs = a;
        q.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&n, kern, &q);
        if (e != cudaSuccess) return e;
        if (n <= 0) return cudaErrorLaunchOutOfResources;
        if (dev >= 0 && dev < 64) cached[dev] = n;
    }
    if (gemm_cta_limit() > 0) n = std::min(n, std::max(1, gemm_cta_limit() / 2));
    *pairs = std::min(n, kMaxPairs);
    return cudaSuccess;
}
// How many of `n` launch attributes hold, the last of which is start_early(): under gemm_set_cta_limit() it does not. A launch that
// starts beside its predecessor's tail has its CTAs wait on SMs of their own, and those would be the ones that were to stay free.
inline int overlap_attrs(int n) { return gemm_cta_limit() > 0 ? n - 1 : n; }
template <typename Kernel, typename Params>
cudaError_t launch_pairs(Kernel kern, int threads, int smem, int pairs, const Params& p, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute a[2] = {in_clusters(2), start_early()};
    cfg.attrs = a;
    cfg.numAttrs = overlap_attrs(2);
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <bool DGRAD, int ACT, int BN, int KIND>
int launch_linear(LinParams& p, int k_steps, cudaStream_t s) {
    constexpr auto kern = linear_fused_kernel<DGRAD, ACT, BN, KIND>;
    const int rows_of_w = KIND == kLinGated && !DGRAD ? 2 * p.N : p.N, wide = KIND == kLinGated && !DGRAD ? BN / 2 : BN;
    int pairs = 0;
    constexpr bool GATED_DGRAD = KIND == kLinGated && DGRAD;
    constexpr int kSmem = LinSmem<BN, GATED_DGRAD>::kTotal;
    static_assert(kSmem <= 227 * 1024, "more shared memory than a CTA may have");
    cudaError_t e = pairs_of<kern>(kLinThreads, kSmem, &pairs);
    if (e != cudaSuccess) return (int)e;
    // A weight that L2 holds beside the stream of activations is walked along n (16384 x 2048 x 8192 with a residual, sustained:
    // 429 us, in groups of 8 rows 441); a larger one in blocks (8192^3: 844 us, along n 923).
    const int group = (int64_t)rows_of_w * k_steps * BK * 2 <= (48ll << 20) ? 1 : 8;
    // Joining a cut tile takes 10 to 20 us (its parts are read one after the other, eight 16-byte loads in flight per thread).
    p.grid = plan_tiles((p.M + 2 * BM - 1) / (2 * BM), (p.N + wide - 1) / wide, k_steps, pairs, 64, group);
    if (p.grid.shared > 0 && p.arrived == nullptr) return kNeedsWorkspace;
    return (int)launch_pairs(kern, kLinThreads, kSmem, p.grid.pairs, p, s);
}

template <bool DGRAD, int BN, int KIND>
int launch_act(int act, LinParams& p, int k_steps, cudaStream_t s) {
    switch (act) {
        case kActNone: return launch_linear<DGRAD, kActNone, BN, KIND>(p, k_steps, s);
        case kActRelu: return launch_linear<DGRAD, kActRelu, BN, KIND>(p, k_steps, s);
        case kActGelu: return launch_linear<DGRAD, kActGelu, BN, KIND>(p, k_steps, s);
        case kActGeluTanh: return launch_linear<DGRAD, kActGeluTanh, BN, KIND>(p, k_steps, s);
        case kActSilu: return launch_linear<DGRAD, kActSilu, BN, KIND>(p, k_steps, s);
    }
    return -2;
}

// the largest of 16, 8, 4 and 2 bytes that every row of a bf16 matrix starts on
int width_of(const void* p, int64_t ld) {
    const uint64_t both = (uint64_t)(uintptr_t)p | (uint64_t)(ld * 2) | 16u;
    return (int)(both & (~both + 1));
}
bool rows16(const void* p, int64_t ld) { return ((uintptr_t)p % 16) == 0 && (ld % 8) == 0; }

template <bool DGRAD, int KIND>
int linear_typed(const LinearArgs& a, cudaStream_t s) {
    constexpr bool GATED_FWD = KIND == kLinGated && !DGRAD;
    // tiles 128 wide only where 256 would be more than half padding: they need twice the operand bytes per flop
    const int BN = a.N > 128 || GATED_FWD ? 256 : 128;
    LinParams p;
    p.M = a.M;
    p.N = a.N;
    p.b_blocked = DGRAD && a.N % 64 == 0 && a.N >= BN ? 1 : 0;
    if (!make_map(&p.map_a, a.a, (uint64_t)a.M, (uint64_t)a.K, (uint64_t)a.lda, BM)) return -3;
    const bool ok = !DGRAD ? make_map(&p.map_b, a.w, (uint64_t)a.N * (GATED_FWD ? 2 : 1), (uint64_t)a.K, (uint64_t)a.ldw, BN / 2)
                   : p.b_blocked ? make_map_blocked(&p.map_b, a.w, (uint64_t)a.K, (uint64_t)a.N, (uint64_t)a.ldw, BN / 128)
                                 : make_map(&p.map_b, a.w, (uint64_t)a.K, (uint64_t)a.N, (uint64_t)a.ldw, 64);
    if (!ok) return -3;
    p.bias = a.bias_f32 ? nullptr : (const __nv_bfloat16*)a.bias;
    p.bias32 = a.bias_f32 ? (const float*)a.bias : nullptr;
    p.res = (const __nv_bfloat16*)a.residual;
    p.ldres = a.ldres;
    p.out = (__nv_bfloat16*)a.out;
    p.ldo = a.ldo;
    p.out2 = (__nv_bfloat16*)a.out2;
    p.ldo2 = a.ldo2;
    p.pre = (__nv_bfloat16*)a.pre;
    p.ldpre = a.ldpre;
    p.q = (int8_t*)a.q;
    p.ldq = a.ldq;
    p.e = (uint8_t*)a.e;
    p.lde = a.lde;
    p.aux_width = width_of(a.residual, a.ldres);
    p.pre_width = width_of(a.pre, a.ldpre);
    p.out_width = width_of(a.out, a.ldo);
    p.out2_width = width_of(a.out2, a.ldo2);
    p.drop = a.drop;
    if constexpr (KIND == kLinGated) {
        p.pre_up = p.pre == nullptr ? nullptr : p.pre + a.N;
        p.out_up = p.out + a.N;
        p.q_up = (int8_t*)a.q_up;
        p.ldq_up = a.ldq_up;
        p.e_up = (uint8_t*)a.e_up;
        p.lde_up = a.lde_up;
        p.pre_up_width = width_of(p.pre_up, a.ldpre);
        p.out_up_width = width_of(p.out_up, a.ldo);
    }
    p.arrived = (unsigned*)a.workspace;
    p.partial = a.workspace == nullptr ? nullptr : (float*)((uint8_t*)a.workspace + linear_workspace_zeros());
    p.err_flag = a.err_flag;
    p.limit_ns = (unsigned long long)(a.wait_limit_s * 1e9);
    const int k_steps = (a.K + BK - 1) / BK;
    if constexpr (GATED_FWD) return launch_act<false, 256, KIND>(a.act, p, k_steps, s);
    else return BN == 256 ? launch_act<DGRAD, 256, KIND>(a.act, p, k_steps, s) : launch_act<DGRAD, 128, KIND>(a.act, p, k_steps, s);
}

}  // namespace

int linear_fused_fwd(const LinearArgs& a, cudaStream_t s);
int linear_fused_dgrad(const LinearArgs& a, cudaStream_t s);
int linear_gated_fwd(const LinearArgs& a, cudaStream_t s);
int linear_gated_dgrad(const LinearArgs& a, cudaStream_t s);
int linear_dropout_fwd(const LinearArgs& a, cudaStream_t s);
int linear_dropout_seed_fwd(const LinearArgs& a, cudaStream_t s);

}  // namespace psb
