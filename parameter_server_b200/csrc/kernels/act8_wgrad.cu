// Weight gradient of a linear layer whose input was kept in 8 bits:
//
//   dw[n][k] = sum_t dy[t][n] * x[t][k],     x = q * 2^(e-127)                              (act8.cuh)
//   norm form: the layer's input was xhat * g + b, and xhat is what was kept:
//   dw[n][k] = g[k] * sum_t dy[t][n] * xhat[t][k] + b[k] * sum_t dy[t][n]
//
// The checkpoint is read as it is (a byte and a 32nd per value instead of two) and becomes bf16 on its way to the tensor
// cores, in shared memory; q * 2^(e-127) is exact in bf16, so the products are those of the values that were kept. Unpacking
// in a pass of its own would move five bytes per value through HBM. The norm form is applied to the fp32 sums, where it
// needs no rounding of x.
//
// CTA pairs on 256 x 256 tiles of dw as in linear_fused.cuh, both operands MN-major, with two more roles per CTA: four warps
// convert the pair's half of the checkpoint tile ([64 tokens][128 columns], 8 KB) into the swizzled bf16 tile that the MMA
// reads (5 integer / packed-bf16 instructions per two values, about a third of the issue slots of the 512 cycles that a
// k-step's MMAs take), and the eight epilogue warps keep the tile's sums in registers: the tensor core adds to its fp32
// accumulator with truncation, which loses 1e-9 of the sum per token (2e-5 at 16384, all towards zero), so a chain in TMEM
// ends after 512 tokens and the chains are added in round-to-nearest by the epilogue warps, one TMEM buffer behind the MMAs.
// Registers move from the producer and converter warps to them (setmaxnreg).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "act8_wgrad.h"
#include "linear_fused.cuh"

namespace psb {

namespace {

constexpr int kWgThreads = 512;          // warpgroups: 0 producer / MMA, 1 converters, 2 and 3 epilogue
constexpr int kWgChain = 8;              // k-steps (of 64 tokens) that are added inside TMEM
constexpr int kWgBN = 256;
constexpr int kRegsIssue = 40, kRegsConvert = 56, kRegsEpilogue = 208;   // 40 + 56 + 2 * 208 = 4 * 128, the launch's share
static_assert(kRegsIssue + kRegsConvert + 2 * kRegsEpilogue == 4 * (65536 / kWgThreads), "setmaxnreg would wait for registers that the launch does not have");

struct WgSmem {
    static constexpr int kABytes = BM * BK * 2;       // dy: 2 blocks of [64 tokens][64 n]
    static constexpr int kBBytes = 128 * BK * 2;      // converted x: the same of the CTA's 128 columns
    static constexpr int kRawBytes = BK * 128;        // q: [64 tokens][128]
    static constexpr int kExpBytes = BK * 16;         // e: [64 tokens][16], four of them ours
    static constexpr int kStageBytes = kABytes + kBBytes + kRawBytes + kExpBytes;
    static constexpr int kStages = 5;
    static constexpr int kTileBytes = kStages * kStageBytes;
    static constexpr int kBarBytes = 256;
    static constexpr int kOutBytes = kLinEpilogueWarps * 2048;
    static constexpr int kTotal = kTileBytes + kBarBytes + kOutBytes + 1024;
};

struct WgParams {
    CUtensorMap map_a, map_q, map_e;
    TileGrid grid;
    int N, K;             // rows and columns of dw
    int a_blocked;
    float* out;
    int64_t ldo;
    int accumulate, out_vec;
    const __nv_bfloat16* weight;
    const __nv_bfloat16* bias;
    const float* dy_sum;
    float* partial;
    unsigned* arrived;
    unsigned* err_flag;
    unsigned long long limit_ns;
};

// Two bytes of `w` (selector 0x4140: bytes 0 and 1, 0x4342: bytes 2 and 3) as bf16 times `step`: 128 + the low seven bits,
// less 128 or, where the sign bit is set, 256 (it is the lowest exponent bit of the subtrahend); both steps are exact.
__device__ __forceinline__ uint32_t convert2(uint32_t w, uint32_t selector, __nv_bfloat162 step) {
    const uint32_t t = __byte_perm(w, 0u, selector);
    uint32_t m = (t & 0x007F007Fu) | 0x43004300u, c = (t & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hmul2(__hsub2(*(__nv_bfloat162*)&m, *(__nv_bfloat162*)&c), step);
    return *(const uint32_t*)&v;
}

__global__ void __launch_bounds__(kWgThreads, 1) act8_wgrad_kernel(const __grid_constant__ WgParams p) {
    using L = WgSmem;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full_bar = (uint64_t*)(smem + L::kTileBytes);   // leader: dy of both CTAs
    uint64_t* raw_bar = full_bar + L::kStages;                // this CTA's q and e
    uint64_t* conv_bar = raw_bar + L::kStages;                // leader: both CTAs' converters
    uint64_t* empty_bar = conv_bar + L::kStages;
    uint64_t* tfull_bar = empty_bar + L::kStages;
    uint64_t* tempty_bar = tfull_bar + 2;
    uint32_t* tmem_slot = (uint32_t*)(tempty_bar + 2);
    uint8_t* stage_out = smem + L::kTileBytes + L::kBarBytes;
    static_assert((4 * L::kStages + 4) * 8 + 4 <= L::kBarBytes, "barriers");

    const int cr = (int)cluster_ctarank();
    const bool leader = cr == 0;
    const int pair = (int)blockIdx.x / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned long long limit_ns = p.limit_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&raw_bar[s], 1);
            mbar_init(&conv_bar[s], 8);   // four converter warps of each CTA
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull_bar[b], 1);
            mbar_init(&tempty_bar[b], 2 * kLinEpilogueWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)(2 * kWgBN))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *((volatile uint32_t*)tmem_slot);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        if (warp == 0 && lane == 0) {
            // ---- TMA producer ----
            asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_q) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_e) : "memory");
            TileWalk walk(p.grid, pair);
            Tile t;
            uint32_t it = 0;
            bool ok = true;
            while (ok && walk.next(p.grid, t)) {
                const int m0 = t.m * 2 * BM + cr * BM, n0 = t.n * kWgBN + cr * 128;
                for (int k = 0; k < t.nk; ++k, ++it) {
                    const int s = it % L::kStages;
                    if (!mbar_wait(&empty_bar[s], ((it / L::kStages) & 1u) ^ 1u, limit_ns)) {
                        atomicCAS(p.err_flag, 0u, 31u);
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + s * L::kStageBytes;
                    uint8_t* sq = sa + L::kABytes + L::kBBytes;
                    const int t0 = (t.k0 + k) * BK;   // first token
                    mbar_expect_tx(&raw_bar[s], (uint32_t)(L::kRawBytes + L::kExpBytes));
                    tma_load_2d(sq, &p.map_q, &raw_bar[s], n0, t0);
                    tma_load_2d(sq + L::kRawBytes, &p.map_e, &raw_bar[s], (n0 / kAct8Block) & ~15, t0);   // x is a multiple of 16 bytes
                    if (leader) mbar_expect_tx(&full_bar[s], 2u * (uint32_t)L::kABytes);
                    const uint32_t fb = mapa_cluster(smem_u32(&full_bar[s]), 0);
                    if (p.a_blocked) {
                        tma_load_3d_pair(sa, &p.map_a, fb, 0, t0, m0 / 64);
                    } else {
                        tma_load_2d_pair(sa, &p.map_a, fb, m0, t0);
                        tma_load_2d_pair(sa + 64 * 128, &p.map_a, fb, m0 + 64, t0);
                    }
                }
            }
        } else if (warp == 1 && lane == 0 && leader) {
            // ---- MMA issuer ----
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(kWgBN >> 3) << 17) |
                                   ((uint32_t)((2 * BM) >> 4) << 24);
            TileWalk walk(p.grid, pair);
            Tile t;
            uint32_t it = 0, tc = 0;
            bool ok = true;
            while (ok && walk.next(p.grid, t)) {
                for (int k = 0; ok && k < t.nk; ++tc) {
                    const uint32_t buf = tc & 1u;
                    if (!mbar_wait(&tempty_bar[buf], ((tc >> 1) & 1u) ^ 1u, limit_ns)) {
                        atomicCAS(p.err_flag, 0u, 34u);
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t tmem_d = tmem_base + buf * (uint32_t)kWgBN;
                    const int lim = min(t.nk, k + kWgChain);
                    for (bool fresh = true; k < lim; ++k, ++it) {
                        const int s = it % L::kStages;
                        const uint32_t ph = (it / L::kStages) & 1u;
                        if (!mbar_wait(&full_bar[s], ph, limit_ns * 2) || !mbar_wait(&conv_bar[s], ph, limit_ns * 2)) {
                            atomicCAS(p.err_flag, 0u, 32u);
                            ok = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t sa = smem_u32(smem + s * L::kStageBytes), sb = sa + L::kABytes;
#pragma unroll
                        for (int u = 0; u < BK / UMMA_K; ++u) {
                            umma_bf16_pair(tmem_d, make_desc(sa + u * 2048, 8192, 1024), make_desc(sb + u * 2048, 8192, 1024), idesc, fresh ? 0u : 1u);
                            fresh = false;
                        }
                        umma_commit_pair(&empty_bar[s]);
                    }
                    umma_commit_pair(&tfull_bar[buf]);   // (also on error, so that the epilogue moves on)
                }
            }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        // ---- converters: thread = 16 columns of rows r0, r0 + 16, ... of the 64 x 128 tile ----
        const int ct = threadIdx.x - 128, g = ct & 7, r0 = ct >> 3;
        const int chunk = (g & 3) * 2;   // 16-byte chunks of the row's 128-byte span in block g / 4
        TileWalk walk(p.grid, pair);
        Tile t;
        uint32_t it = 0;
        bool ok = true;
        while (ok && walk.next(p.grid, t)) {
            const int eb = (((t.n * kWgBN + cr * 128) / kAct8Block) & 15) + g / 2;
            for (int k = 0; k < t.nk; ++k, ++it) {
                const int s = it % L::kStages;
                if (!mbar_wait(&raw_bar[s], (it / L::kStages) & 1u, limit_ns * 2)) {
                    atomicCAS(p.err_flag, 0u, 35u);
                    ok = false;
                    break;
                }
                uint8_t* sb = smem + s * L::kStageBytes + L::kABytes + (g >> 2) * 8192;
                const uint8_t* sq = smem + s * L::kStageBytes + L::kABytes + L::kBBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = r0 + 16 * i;
                    const uint4 raw = *(const uint4*)(sq + r * 128 + g * 16);
                    const uint32_t e = sq[L::kRawBytes + r * 16 + eb];
                    const uint32_t e2 = (e << 7) | (e << 23);
                    const __nv_bfloat162 step = *(const __nv_bfloat162*)&e2;
                    uint4 lo, hi;
                    lo.x = convert2(raw.x, 0x4140, step); lo.y = convert2(raw.x, 0x4342, step);
                    lo.z = convert2(raw.y, 0x4140, step); lo.w = convert2(raw.y, 0x4342, step);
                    hi.x = convert2(raw.z, 0x4140, step); hi.y = convert2(raw.z, 0x4342, step);
                    hi.z = convert2(raw.w, 0x4140, step); hi.w = convert2(raw.w, 0x4342, step);
                    uint8_t* row = sb + r * 128;
                    uint8_t *p0 = row + ((chunk ^ (r & 7)) << 4), *p1 = row + (((chunk + 1) ^ (r & 7)) << 4);
                    // the eight lanes of a row write eight different chunk positions: block 1 starts with its odd ones
                    if (g < 4) { *(uint4*)p0 = lo; *(uint4*)p1 = hi; }
                    else { *(uint4*)p1 = hi; *(uint4*)p0 = lo; }
                }
                fence_async_smem();   // the MMAs read through the async proxy
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_cluster(smem_u32(&conv_bar[s]), 0));
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue));
        // ---- epilogue ----
        const int ew = warp - 8, quarter = warp & 3, half = ew >> 2;
        uint8_t* stage = stage_out + ew * 2048;
        TileWalk walk(p.grid, pair);
        Tile t;
        uint32_t tc = 0;
        bool ok = true;
        while (ok && walk.next(p.grid, t)) {
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.f;
            for (int k = 0; k < t.nk; k += kWgChain, ++tc) {
                const uint32_t buf = tc & 1u;
                if (!mbar_wait(&tfull_bar[buf], (tc >> 1) & 1u, limit_ns * 4)) {
                    atomicCAS(p.err_flag, 0u, 33u);
                    ok = false;
                    break;
                }
                __syncwarp();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * (uint32_t)kWgBN + (uint32_t)(half * 128);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld32_issue(taddr + (uint32_t)c * 32u, v);
                    tmem_wait_ld(v);
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c * 32 + j] += __uint_as_float(v[j]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_cluster(smem_u32(&tempty_bar[buf]), 0));
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            if (t.runs > 1) {
                constexpr int64_t kWarpFloats = 4 * 1024;
                auto part_of = [&](int worker, int slot) {
                    return p.partial + ((((int64_t)worker * 2 + slot) * 2 + cr) * kLinEpilogueWarps + ew) * kWarpFloats + lane * 4;
                };
                float* mine = part_of(pair, t.slot);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    *(float4*)(mine + j * 128) = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
                __threadfence();
                __syncwarp();
                unsigned last = 0;
                unsigned* count = p.arrived + ((int64_t)t.index * 2 + cr) * kLinEpilogueWarps + ew;
                if (lane == 0) last = atomicAdd(count, 1u) == (unsigned)(t.runs - 1) ? 1u : 0u;
                if (__shfl_sync(0xFFFFFFFFu, last, 0) == 0u) continue;
                __threadfence();
                if (lane == 0) *count = 0u;
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] = 0.f;
#pragma unroll 1
                for (int r = 0; r < t.runs; ++r) {
                    const float* src = part_of(t.first + r, TileWalk::slot_of(p.grid, t, r));
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float4 x = __ldcg((const float4*)(src + j * 128));
                        acc[4 * j] += x.x; acc[4 * j + 1] += x.y; acc[4 * j + 2] += x.z; acc[4 * j + 3] += x.w;
                        if (j % 8 == 7) asm volatile("" ::: "memory");   // eight loads in flight: more would not fit the registers
                    }
                }
            }
            const int row0 = t.m * 2 * BM + cr * BM + quarter * 32, colw = t.n * kWgBN + half * 128;
            const bool affine = p.weight != nullptr || p.bias != nullptr;
            const float sum = p.dy_sum != nullptr && row0 + lane < p.N ? p.dy_sum[row0 + lane] : 0.f;
            // 16 columns at a time through the warp's 2 KB, so that stores (and the loads of a gradient that is added to)
            // cover 64-byte row segments; swizzled as in linear_fused.cuh
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (colw + c * 16 < p.K) {   // warp-uniform
                    if (affine) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int col = min(colw + c * 16 + j, p.K - 1);   // the same for all lanes
                            const float w = p.weight != nullptr ? __bfloat162float(p.weight[col]) : 1.f;
                            const float b = p.bias != nullptr ? __bfloat162float(p.bias[col]) : 0.f;
                            acc[c * 16 + j] = acc[c * 16 + j] * w + sum * b;
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *(float4*)(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                            make_float4(acc[c * 16 + 4 * j], acc[c * 16 + 4 * j + 1], acc[c * 16 + 4 * j + 2], acc[c * 16 + 4 * j + 3]);
                    __syncwarp();
                    const int cb = lane & 3, col = colw + c * 16 + cb * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = i * 8 + (lane >> 2);
                        if (row0 + r >= p.N) continue;
                        float4 d = *(const float4*)(stage + r * 64 + ((cb ^ ((r >> 1) & 3)) << 4));
                        float* op = p.out + (int64_t)(row0 + r) * p.ldo + col;
                        if (p.out_vec && col + 4 <= p.K) {
                            if (p.accumulate) {
                                const float4 o = *(const float4*)op;
                                d.x += o.x; d.y += o.y; d.z += o.z; d.w += o.w;
                            }
                            *(float4*)op = d;
                        } else {
                            const float x[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (col + k < p.K) op[k] = p.accumulate ? op[k] + x[k] : x[k];
                        }
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)(2 * kWgBN)) : "memory");
    }
}

// 2-D byte matrix [rows][cols] with `box_cols` x 64 boxes, no swizzle
bool make_byte_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols) {
    EncodeFn enc = get_encode();
    if (!enc) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {ld};
    cuuint32_t box[2] = {box_cols, (cuuint32_t)BK};
    cuuint32_t estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

int act8_wgrad(const Act8WgradArgs& a, void* stream) {
    if (a.N <= 0 || a.K <= 0) return 0;
    if (a.tokens <= 0 || a.tokens > 0x7FFFFFFFll - 64 || a.workspace == nullptr || a.err_flag == nullptr || a.out == nullptr) return -2;
    if (a.bias != nullptr && a.dy_sum == nullptr) return -2;
    if (!rows16(a.dy, a.lddy) || ((uintptr_t)a.x.q % 16) || (a.x.ldq % 16) || ((uintptr_t)a.x.e % 16) || (a.x.lde % 16)) return -2;
    WgParams p;
    p.N = a.N;
    p.K = a.K;
    p.a_blocked = a.N % 64 == 0 && a.N >= BM ? 1 : 0;
    const uint64_t tokens = (uint64_t)a.tokens, blocks = (uint64_t)(a.K + kAct8Block - 1) / kAct8Block;
    const bool ok = (p.a_blocked ? make_map_blocked(&p.map_a, a.dy, tokens, (uint64_t)a.N, (uint64_t)a.lddy, BM / 64)
                                 : make_map(&p.map_a, a.dy, tokens, (uint64_t)a.N, (uint64_t)a.lddy, 64)) &&
                    make_byte_map(&p.map_q, a.x.q, tokens, (uint64_t)a.K, (uint64_t)a.x.ldq, 128) &&
                    make_byte_map(&p.map_e, a.x.e, tokens, blocks, (uint64_t)a.x.lde, 16);
    if (!ok) return -3;
    p.out = a.out;
    p.ldo = a.ldo;
    p.accumulate = a.accumulate;
    p.out_vec = ((uintptr_t)a.out % 16) == 0 && a.ldo % 4 == 0;
    p.weight = (const __nv_bfloat16*)a.weight;
    p.bias = (const __nv_bfloat16*)a.bias;
    p.dy_sum = a.dy_sum;
    p.arrived = (unsigned*)a.workspace;
    p.partial = (float*)((uint8_t*)a.workspace + linear_workspace_zeros());
    p.err_flag = a.err_flag;
    p.limit_ns = (unsigned long long)(a.wait_limit_s * 1e9);
    int pairs = 0;
    cudaError_t e = pairs_of<act8_wgrad_kernel>(kWgThreads, WgSmem::kTotal, &pairs);
    if (e != cudaSuccess) return (int)e;
    p.grid = plan_tiles((a.N + 2 * BM - 1) / (2 * BM), (a.K + kWgBN - 1) / kWgBN, (int)((a.tokens + BK - 1) / BK), pairs, 12);
    return (int)launch_pairs(act8_wgrad_kernel, kWgThreads, WgSmem::kTotal, p.grid.pairs, p, (cudaStream_t)stream);
}

}  // namespace psb
