// Weight gradient of a linear layer whose input was kept in 8 bits:
//
//   dw[n][k] = sum_t dy[t][n] * x[t][k],     x = q * 2^(e-127)                              (act8.cuh)
//   norm form: the layer's input was xhat * g + b, and xhat is what was kept:
//   dw[n][k] = g[k] * sum_t dy[t][n] * xhat[t][k] + b[k] * sum_t dy[t][n]
//
// q * 2^(e-127) is exact in bf16, so the products are those of the values that were kept. A layer of few outputs reads the
// checkpoint as it is (a byte and a 32nd per value) and turns it into bf16 in shared memory, on its way to the tensor cores; one
// of many outputs, which would do that again for every 256 of them, unpacks it once into scratch (act8_wgrad_scratch). The norm
// form is applied to the fp32 sums, where it needs no rounding of x. Layers with few tiles are unpacked as well and go to the
// clusters of linear_few.cuh (wgrad_few).
//
// CTA pairs on 256 x 256 tiles of dw as in linear_fused.cuh, both operands MN-major. Where x is converted, four more warps per
// CTA turn the pair's half of the checkpoint tile ([64 tokens][128 columns], 8 KB) into the swizzled bf16 tile that the MMA reads:
// per two values two byte permutes, a packed sum, a packed product and a conversion (sum and product in one: 450 of the 750 cycles of a k-step); dy, the
// checkpoint and the bf16 tiles have rings of their own, so that no part waits for another's space.
// The eight epilogue warps keep the tile's sums in registers: the tensor core adds to its fp32 accumulator with truncation, which
// loses 1e-9 of the sum per token (2e-5 at 16384, all towards zero), so a chain in TMEM ends after 512 tokens and the chains are
// added in round-to-nearest by the epilogue warps, one TMEM buffer behind the MMAs (1.5e-7 at 16384 tokens). Registers move
// from the producer and converter warps to them (setmaxnreg).
// 16384 tokens, 6144 x 2048: 300 us with a cold L2 (1375 TFLOP/s), 347 back to back at the power limit. Bound by the tensor cores and
// that limit.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "act8_wgrad.h"
#include "linear_few.cuh"

namespace psb {

namespace {

constexpr int kWgThreads = 512;          // warpgroups: 0 producer / MMA, 1 converters, 2 and 3 epilogue
constexpr int kWgChain = 8;              // k-steps (of 64 tokens) that are added inside TMEM
constexpr int kWgBN = 256;
constexpr int kRegsIssue = 40, kRegsConvert = 88, kRegsEpilogue = 192;   // 40 + 88 + 2 * 192 = 4 * 128, the launch's share
static_assert(kRegsIssue + kRegsConvert + 2 * kRegsEpilogue == 4 * (65536 / kWgThreads), "setmaxnreg would wait for registers that the launch does not have");

template <bool CONVERT>
struct WgSmem {
    static constexpr int kABytes = BM * BK * 2;       // dy: 2 blocks of [64 tokens][64 n]
    static constexpr int kBBytes = 128 * BK * 2;      // x in bf16: the same of the CTA's 128 columns
    static constexpr int kRawBytes = BK * 128;        // q: [64 tokens][128]
    static constexpr int kExpBytes = BK * 16;         // e: [64 tokens][16], four of them ours
    static constexpr int kRawStage = kRawBytes + kExpBytes;
    static constexpr int kA = 6, kB = CONVERT ? 4 : 6, kRaw = CONVERT ? 5 : 0;   // stages
    static constexpr int kBOff = kA * kABytes, kRawOff = kBOff + kB * kBBytes;
    static constexpr int kTileBytes = kRawOff + kRaw * kRawStage;
    static constexpr int kBarBytes = 512;
    static constexpr int kOutBytes = kLinEpilogueWarps * 2048;
    static constexpr int kTotal = kTileBytes + kBarBytes + kOutBytes + 1024;
};

constexpr int kWgUnpackN = 2048;   // from so many outputs on x is unpacked once (see act8_wgrad_scratch)

struct WgParams {
    CUtensorMap map_a, map_b, map_e;   // b: q, or x in bf16
    TileGrid grid;
    int N, K;             // rows and columns of dw
    int a_blocked, b_blocked;
    float* out;
    int64_t ldo;
    int accumulate;
    const __nv_bfloat16* weight;
    const __nv_bfloat16* bias;
    const float* dy_sum;
    float* partial;
    unsigned* arrived;
    unsigned* err_flag;
    unsigned long long limit_ns;
};

// Two of the bytes of `w` (unsigned, 128 more than the value; chosen by the selectors) as bf16 times the step: byte b in the
// second byte of 0x4700bb00 is the float 32768 + b, a packed sum takes off 32896 and a packed product scales, both exactly. (One
// multiply-add with -32896 steps would do, but that is infinite from a step of 2^113 on, and the format's largest is 2^122.)
__device__ __forceinline__ uint32_t convert2(uint32_t w, uint32_t s0, uint32_t s1, float step) {
    float a, b;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
        "add.rn.f32x2 x, x, z;\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(a), "=f"(b)
        : "r"(__byte_perm(w, 0x47000000u, s0)), "r"(__byte_perm(w, 0x47000000u, s1)), "f"(step), "f"(-32896.f));
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&v;
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// eight bytes (two words) as bf16 to 16 bytes of shared memory
__device__ __forceinline__ void sts_converted(uint32_t addr, uint32_t w0, uint32_t w1, float step) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(convert2(w0, 0x7404, 0x7414, step)),
                 "r"(convert2(w0, 0x7424, 0x7434, step)), "r"(convert2(w1, 0x7404, 0x7414, step)),
                 "r"(convert2(w1, 0x7424, 0x7434, step))
                 : "memory");
}

// WIDE: rows of dw start on 16-byte boundaries (a kernel of its own: the epilogue is long, and bound by instruction fetch)
template <bool CONVERT, bool WIDE>
__global__ void __launch_bounds__(kWgThreads, 1) act8_wgrad_kernel(const __grid_constant__ WgParams p) {
    using L = WgSmem<CONVERT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* afull_bar = (uint64_t*)(smem + L::kTileBytes);   // leader: dy of both CTAs has landed
    uint64_t* aempty_bar = afull_bar + L::kA;                  // both: the MMAs have read it
    uint64_t* rfull_bar = aempty_bar + L::kA;                  // own: q and e have landed
    uint64_t* rempty_bar = rfull_bar + L::kRaw;                // own: the converters have read them
    uint64_t* bfull_bar = rempty_bar + L::kRaw;                // leader: x in bf16 is there, in both CTAs
    uint64_t* bempty_bar = bfull_bar + L::kB;               // both: the MMAs have read it
    uint64_t* tfull_bar = bempty_bar + L::kB;
    uint64_t* tempty_bar = tfull_bar + 2;
    uint32_t* tmem_slot = (uint32_t*)(tempty_bar + 2);
    uint8_t* stage_out = smem + L::kTileBytes + L::kBarBytes;
    static_assert((2 * (L::kA + L::kRaw + L::kB) + 4) * 8 + 4 <= L::kBarBytes, "barriers");

    const int cr = (int)cluster_ctarank();
    const bool leader = cr == 0;
    const int pair = (int)blockIdx.x / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned long long limit_ns = p.limit_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kA; ++s) { mbar_init(&afull_bar[s], 1); mbar_init(&aempty_bar[s], 1); }
        for (int s = 0; s < L::kRaw; ++s) { mbar_init(&rfull_bar[s], 1); mbar_init(&rempty_bar[s], 4); }
        for (int s = 0; s < L::kB; ++s) { mbar_init(&bfull_bar[s], CONVERT ? 8 : 1); mbar_init(&bempty_bar[s], 1); }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull_bar[b], 1);
            mbar_init(&tempty_bar[b], 2 * kLinEpilogueWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_arrive_all();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)(2 * kWgBN))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    cluster_wait_all();   // the peer's barriers must exist before anything is signalled on them
    wait_predecessor();
    uint32_t tmem_base = 0;
    if (warp == 1 || warp >= 8) {   // (loads and converters need no TMEM and do not wait for it)
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        meet_named(2, 32 * (1 + kLinEpilogueWarps));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_base = tmem_address(tmem_slot);
        allow_successor();
    }

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        if (warp == 0 && lane == 0) {
            // ---- TMA producer of dy (and of x, where it is bf16) ----
            asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_a) : "memory");
            TileWalk walk(p.grid, pair);
            Tile t;
            uint32_t it = 0;
            bool ok = true;
            while (ok && walk.next(p.grid, t)) {
                const int m0 = t.m * 2 * BM + cr * BM, n0 = t.n * kWgBN + cr * 128;
                for (int k = 0; k < t.nk; ++k, ++it) {
                    const int s = it % L::kA;
                    // (one commit frees the stages of both operands, and they are as many: one wait covers both)
                    if (!mbar_wait(&aempty_bar[s], ((it / L::kA) & 1u) ^ 1u, limit_ns)) {
                        give_up_pair(p.err_flag, 31u, tmem_slot);
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + s * L::kABytes;
                    const int t0 = (t.k0 + k) * BK;   // first token
                    if (leader) mbar_expect_tx(&afull_bar[s], 2u * (uint32_t)(CONVERT ? L::kABytes : L::kABytes + L::kBBytes));
                    const uint32_t fb = mapa_cluster(smem_u32(&afull_bar[s]), 0);
                    if (p.a_blocked) {
                        tma_load_3d_pair(sa, &p.map_a, fb, 0, t0, m0 / 64);
                    } else {
                        tma_load_2d_pair(sa, &p.map_a, fb, m0, t0);
                        tma_load_2d_pair(sa + 64 * 128, &p.map_a, fb, m0 + 64, t0);
                    }
                    if constexpr (!CONVERT) {
                        uint8_t* sb = smem + L::kBOff + s * L::kBBytes;
                        if (p.b_blocked) {
                            tma_load_3d_pair(sb, &p.map_b, fb, 0, t0, n0 / 64);
                        } else {
                            tma_load_2d_pair(sb, &p.map_b, fb, n0, t0);
                            tma_load_2d_pair(sb + 64 * 128, &p.map_b, fb, n0 + 64, t0);
                        }
                    }
                }
            }
        } else if (CONVERT && warp == 2 && lane == 0) {
            // ---- TMA producer of the checkpoint ----
            asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_b) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&p.map_e) : "memory");
            TileWalk walk(p.grid, pair);
            Tile t;
            uint32_t it = 0;
            bool ok = true;
            while (ok && walk.next(p.grid, t)) {
                const int n0 = t.n * kWgBN + cr * 128;
                for (int k = 0; k < t.nk; ++k, ++it) {
                    const int s = it % L::kRaw;
                    if (!mbar_wait(&rempty_bar[s], ((it / L::kRaw) & 1u) ^ 1u, limit_ns)) {
                        give_up_pair(p.err_flag, 36u, tmem_slot);
                        ok = false;
                        break;
                    }
                    uint8_t* sq = smem + L::kRawOff + s * L::kRawStage;
                    const int t0 = (t.k0 + k) * BK;
                    mbar_expect_tx(&rfull_bar[s], (uint32_t)L::kRawStage);
                    tma_load_2d(sq, &p.map_b, &rfull_bar[s], n0, t0);
                    tma_load_2d(sq + L::kRawBytes, &p.map_e, &rfull_bar[s], (n0 / kAct8Block) & ~15, t0);   // x is a multiple of 16 bytes
                }
            }
        } else if (warp == 1 && lane == 0 && leader) {
            // ---- MMA issuer ----
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(kWgBN >> 3) << 17) |
                                   ((uint32_t)((2 * BM) >> 4) << 24);
            // The issue of an MMA blocks while the tensor core's queue is full, and the queue is short: what this thread does
            // between two k-steps is time in which it may run dry. So the next k-step's barriers are asked before the current
            // one's MMAs are issued, and descriptors and ring positions are kept as running values.
            const uint64_t desc_a = make_desc(smem_u32(smem), 8192, 1024), desc_b = make_desc(smem_u32(smem + L::kBOff), 8192, 1024);
            TileWalk walk(p.grid, pair);
            Tile t;
            uint32_t it = 0, tc = 0, ia = 0, ic = 0, pa = 0, pc = 0;
            bool ok = true, have = false;
            while (ok && walk.next(p.grid, t)) {
                for (int k = 0; ok && k < t.nk; ++tc) {
                    const uint32_t buf = tc & 1u;
                    if (!mbar_wait(&tempty_bar[buf], ((tc >> 1) & 1u) ^ 1u, limit_ns)) {
                        give_up_pair(p.err_flag, 34u, tmem_slot);
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t tmem_d = tmem_base + buf * (uint32_t)kWgBN;
                    const int lim = min(t.nk, k + kWgChain);
                    uint32_t add = 0;
                    for (; k < lim; ++k, ++it) {
                        if (!have && (!mbar_wait(&afull_bar[ia], pa, limit_ns * 2) || (CONVERT && !mbar_wait(&bfull_bar[ic], pc, limit_ns * 2)))) {
                            give_up_pair(p.err_flag, 32u, tmem_slot);
                            ok = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t na = ia + 1 == L::kA ? 0 : ia + 1, nc = ic + 1 == L::kB ? 0 : ic + 1;
                        const uint32_t npa = na == 0 ? pa ^ 1u : pa, npc = nc == 0 ? pc ^ 1u : pc;
                        const uint64_t da = desc_a + ia * (uint32_t)(L::kABytes >> 4), db = desc_b + ic * (uint32_t)(L::kBBytes >> 4);
                        umma_bf16_pair(tmem_d, da, db, idesc, add);
                        have = mbar_try_wait(&afull_bar[na], npa);
                        umma_bf16_pair(tmem_d, da + 128, db + 128, idesc, 1u);
                        if constexpr (CONVERT) have = have && mbar_try_wait(&bfull_bar[nc], npc);
                        umma_bf16_pair(tmem_d, da + 256, db + 256, idesc, 1u);
                        umma_bf16_pair(tmem_d, da + 384, db + 384, idesc, 1u);
                        umma_commit_pair(&aempty_bar[ia]);
                        if constexpr (CONVERT) umma_commit_pair(&bempty_bar[ic]);
                        add = 1;
                        ia = na; ic = nc; pa = npa; pc = npc;
                    }
                    umma_commit_pair(&tfull_bar[buf]);   // (also on error, so that the epilogue moves on)
                }
            }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        if constexpr (CONVERT) {
        // ---- converters ----
        // Eight lanes take 16 columns each of two neighbouring rows: columns 0-63 of the even row and 64-127 of the odd one,
        // then the other halves. Their loads cover 128 bytes of distinct banks, and so do their stores: the two 16-byte
        // chunks of a thread land at chunk ^ (row % 8) of the row's swizzled span, even positions for one row, odd for the
        // other. A thread does this for rows r0 and r0 + 32.
        const int ct = threadIdx.x - 128, gg = ct & 3, rr = (ct >> 2) & 1, r0 = 2 * (ct >> 3) + rr;
        const int c0 = ((2 * gg) ^ (r0 & 7)) << 4, c1 = ((2 * gg + 1) ^ (r0 & 7)) << 4;
        // One k-step ahead: the next k-step's bytes are requested before this one's are converted, and the barriers of the step
        // after are asked before they are needed.
        TileWalk walk(p.grid, pair);
        Tile t;
        const uint32_t q0 = smem_u32(smem + L::kRawOff) + r0 * 128 + gg * 16 + rr * 64;          // pass 0: row r0, columns of block rr
        const uint32_t x0 = smem_u32(smem + L::kRawOff + L::kRawBytes) + r0 * 16 + gg / 2 + rr * 2;
        const uint32_t d0 = smem_u32(smem + L::kBOff) + r0 * 128 + rr * 8192;
        const uint32_t bfull0 = mapa_cluster(smem_u32(&bfull_bar[0]), 0);
        const uint32_t other = rr != 0 ? 0u - 8192u : 8192u;   // from one column block of the converted tile to the other
        uint32_t ir = 0, pr = 0, ic = 0, pc = 1;
        uint32_t site = 0;   // of the wait that ran out
        uint4 raw[4], nraw[4];
        uint32_t e[4], ne[4];
        bool have = false;
        auto load = [&](uint32_t eb) -> bool {
            // (The warp's lanes decide together: one that left alone would be missed at the next __syncwarp. Asked once more after a
            // wait only: with one vote for both, 16384 tokens, 512 x 2048 take 61.1 us, so 59.8, and 58.9 if lanes could part.)
            if (!__all_sync(0xFFFFFFFFu, have) && !__all_sync(0xFFFFFFFFu, mbar_wait(&rfull_bar[ir], pr, limit_ns * 2))) {
                site = 35u;
                return false;
            }
            const uint32_t sq = q0 + ir * L::kRawStage, sx = x0 + ir * L::kRawStage + eb;
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // odd: the other column block of the row (neither eb nor gg / 2 touches that bit)
                nraw[i] = ld_smem_v4(((i & 1) ? (sq ^ 64u) : sq) + 32 * (i / 2) * 128);
                ne[i] = lds_u8(((i & 1) ? (sx ^ 2u) : sx) + 32 * (i / 2) * 16);
            }
            if (++ir == L::kRaw) { ir = 0; pr ^= 1u; }
            have = false;
            return true;
        };
        bool more = walk.next(p.grid, t);
        int left = t.nk;
        uint32_t eb = ((t.n * kWgBN + cr * 128) / kAct8Block) & 15;
        if (more) more = load(eb);
        while (more) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { raw[i] = nraw[i]; e[i] = ne[i]; }
            const uint32_t ir_now = ir == 0 ? L::kRaw - 1 : ir - 1;
            const bool room = mbar_try_wait(&bempty_bar[ic], pc);
            if (--left == 0) {
                more = walk.next(p.grid, t);
                left = t.nk;
                eb = ((t.n * kWgBN + cr * 128) / kAct8Block) & 15;
            }
            if (more) more = load(eb);
            if (!__all_sync(0xFFFFFFFFu, room) && !__all_sync(0xFFFFFFFFu, mbar_wait(&bempty_bar[ic], pc, limit_ns * 2))) {
                site = 37u;
                break;
            }
            const uint32_t sb = d0 + ic * L::kBBytes;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float step = act8_step(e[i]);
                const uint32_t w0 = raw[i].x ^ 0x80808080u, w1 = raw[i].y ^ 0x80808080u, w2 = raw[i].z ^ 0x80808080u, w3 = raw[i].w ^ 0x80808080u;
                const uint32_t dst = sb + ((i & 1) ? other : 0u) + 32 * (i / 2) * 128;
                sts_converted(dst + c0, w0, w1, step);
                sts_converted(dst + c1, w2, w3, step);
            }
            if (more) have = mbar_try_wait(&rfull_bar[ir], pr);
            fence_async_smem();   // the MMAs read through the async proxy
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_pair(bfull0 + ic * 8);
                // only now that the values have been used is it certain that they have been read: a load alone may be carried out
                // behind an arrival that follows it
                mbar_arrive(&rempty_bar[ir_now]);
            }
            if (++ic == L::kB) { ic = 0; pc ^= 1u; }
        }
        if (site != 0 && lane == 0) give_up_pair(p.err_flag, site, tmem_slot);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue));
        // ---- epilogue ----
        const int ew = warp - 8, quarter = warp & 3, half = ew >> 2;
        const uint32_t stage = smem_u32(stage_out) + (uint32_t)ew * 2048;
        TileWalk walk(p.grid, pair);
        Tile t;
        uint32_t tc = 0;
        bool ok = true;
        while (ok && walk.next(p.grid, t)) {
            const int row0 = t.m * 2 * BM + cr * BM + quarter * 32, colw = t.n * kWgBN + half * 128;
            // Chunk c of this lane's part of the gradient that is added to: four blocks of 16 bytes, or, where rows do not start on
            // 16-byte boundaries, sixteen values, so that the lanes cover two rows side by side. One chunk is always on its way.
            // (50 tokens, 4096 x 4096: 39 us, loaded when needed, between the stores: 57; 3336 x 2574, on no boundary: 32, 96.)
            float old[16];
            auto request_old = [&](int c) {
                const int col0 = colw + c * 16;
                if (!p.accumulate || c >= 8 || col0 >= p.K) return;   // warp-uniform
                if constexpr (WIDE) {
                    const int col = col0 + (lane & 3) * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = i * 8 + (lane >> 2);
                        const float* o = p.out + (int64_t)(row0 + r) * p.ldo + col;
                        if (row0 + r >= p.N) continue;
                        if (col + 4 <= p.K) {
                            const float4 x = *(const float4*)o;
                            old[4 * i] = x.x; old[4 * i + 1] = x.y; old[4 * i + 2] = x.z; old[4 * i + 3] = x.w;
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (col + k < p.K) old[4 * i + k] = o[k];
                        }
                    }
                } else {
                    const float* o = p.out + (int64_t)(row0 + (lane >> 4)) * p.ldo + col0 + (lane & 15);
                    const int left = col0 + (lane & 15) < p.K ? p.N - row0 - (lane >> 4) : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (2 * i < left) old[i] = o[2 * i * p.ldo];
                }
            };
#pragma unroll
            for (int i = 0; i < 16; ++i) old[i] = 0.f;
            if (t.runs == 1) request_old(0);
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.f;
            for (int k = 0; k < t.nk; k += kWgChain, ++tc) {
                const uint32_t buf = tc & 1u;
                // one warp asks for the chain's end, the others sleep (asking takes issue slots from the MMAs' thread)
                const bool waited = ew != 0 || mbar_wait(&tfull_bar[buf], (tc >> 1) & 1u, limit_ns * 4);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                if (!meet_all(1, 32 * kLinEpilogueWarps, waited)) {
                    if (!waited && lane == 0) give_up_pair(p.err_flag, 33u, tmem_slot);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * (uint32_t)kWgBN + (uint32_t)(half * 128);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t v[16];
                    tmem_ld16(taddr + (uint32_t)c * 16u, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[c * 16 + j] += __uint_as_float(v[j]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_cluster(smem_u32(&tempty_bar[buf]), 0));
            }
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
                request_old(0);
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] = 0.f;
#pragma unroll 1
                for (int r = 0; r < t.runs; ++r) {
                    const float* src = part_of(t.first + r, TileWalk::slot_of(p.grid, t, r));
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float4 x = __ldcg((const float4*)(src + j * 128));
                        acc[4 * j] += x.x; acc[4 * j + 1] += x.y; acc[4 * j + 2] += x.z; acc[4 * j + 3] += x.w;
                        if (j % 4 == 3) asm volatile("" ::: "memory");   // eight loads in flight: more would not fit the registers
                    }
                }
            }
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
                        st_smem_v4(stage + (uint32_t)(lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)),
                                   make_uint4(__float_as_uint(acc[c * 16 + 4 * j]), __float_as_uint(acc[c * 16 + 4 * j + 1]),
                                              __float_as_uint(acc[c * 16 + 4 * j + 2]), __float_as_uint(acc[c * 16 + 4 * j + 3])));
                    __syncwarp();
                    float now[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) now[i] = old[i];
                    request_old(c + 1);
                    const int col0 = colw + c * 16;
                    if constexpr (WIDE) {
                        const int cb = lane & 3, col = col0 + cb * 4;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = i * 8 + (lane >> 2);
                            if (row0 + r >= p.N) continue;
                            const uint4 w = ld_smem_v4(in_piece(stage, r, cb * 16));
                            const float x[4] = {__uint_as_float(w.x) + now[4 * i], __uint_as_float(w.y) + now[4 * i + 1],
                                                __uint_as_float(w.z) + now[4 * i + 2], __uint_as_float(w.w) + now[4 * i + 3]};
                            float* op = p.out + (int64_t)(row0 + r) * p.ldo + col;
                            if (col + 4 <= p.K) {
                                *(float4*)op = make_float4(x[0], x[1], x[2], x[3]);
                            } else {
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (col + k < p.K) op[k] = x[k];
                            }
                        }
                    } else {
                        float* o = p.out + (int64_t)(row0 + (lane >> 4)) * p.ldo + col0 + (lane & 15);
                        const int left = col0 + (lane & 15) < p.K ? p.N - row0 - (lane >> 4) : 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float x;
                            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(in_piece(stage, i * 2 + (lane >> 4), (lane & 15) * 4)) : "memory");
                            now[i] += x;
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (2 * i < left) o[2 * i * p.ldo] = now[i];
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    if (warp == 1) {
        if (gave_up(tmem_slot)) let_copies_land();
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

template <bool CONVERT, bool WIDE>
int plan_wgrad(WgParams& p, int64_t tokens) {
    int pairs = 0;
    cudaError_t e = pairs_of<act8_wgrad_kernel<CONVERT, WIDE>>(kWgThreads, WgSmem<CONVERT>::kTotal, &pairs);
    if (e != cudaSuccess) return (int)e;
    p.grid = plan_tiles((p.N + 2 * BM - 1) / (2 * BM), (p.K + kWgBN - 1) / kWgBN, (int)((tokens + BK - 1) / BK), pairs, 48, 8);
    return p.grid.shared > 0 && p.arrived == nullptr ? kNeedsWorkspace : 0;
}
template <bool CONVERT, bool WIDE>
int launch_wgrad(const WgParams& p, cudaStream_t s) {
    constexpr auto kern = act8_wgrad_kernel<CONVERT, WIDE>;
    return (int)launch_pairs(kern, kWgThreads, WgSmem<CONVERT>::kTotal, p.grid.pairs, p, s);
}

// Whether a layer has so few tiles that clusters on 128 x 128 of them are done first, from x in bf16. In k-steps (0.25 us), from
// sweeps: a pair's step takes 1.2, or 1.7 where it converts, its frame and epilogue 34 or 55 and a join of cut tiles 55; the small
// kernel's frame 24, with two CTAs on an SM 44, and the pass that unpacks x 10 and its bytes. us, without and with the small
// kernel: 1000 tokens, 512 x 512: 19.6, 10.1; 8192: 33.9, 20.2; 2048 tokens, 1024 x 1024: 26.5, 14.4; 300, 4096 x 1024: 13.0, 17.6.
bool wgrad_few(int64_t tokens, int N, int K) {
    const int64_t k_steps = (tokens + BK - 1) / BK, small = (int64_t)((N + BM - 1) / BM) * ((K + BM - 1) / BM);
    const int max_pairs = gemm_cta_limit() > 0 ? std::min(kMaxPairs, std::max(1, gemm_cta_limit() / 2)) : kMaxPairs;
    if (small > 4 * max_pairs) return false;
    const FewPlan plan = few_plan(N, K, tokens, true);
    if (plan.cluster == 0) return false;
    const TileGrid g = plan_tiles((N + 2 * BM - 1) / (2 * BM), (K + kWgBN - 1) / kWgBN, (int)k_steps, max_pairs, 48, 8);
    const int64_t tiles = (int64_t)g.m_tiles * g.n_tiles, whole = (tiles - g.shared + g.pairs - 1) / g.pairs;
    const float unpack = 10.f + (float)tokens * (float)K * 2.4e-6f;
    const bool converts = N < kWgUnpackN;
    const float pairs = (float)(whole * k_steps + (g.shared > 0 ? g.len : 0)) * (converts ? 1.7f : 1.2f) + (converts ? 55.f : 34.f + unpack) +
                        (g.shared > 0 ? 55.f : 0.f);
    return plan.steps + (small * plan.cluster > 2 * kMaxPairs ? 44.f : 24.f) + unpack < pairs;
}

int wgrad_on_few(const Act8WgradArgs& a, int64_t ldx, cudaStream_t s) {
    FewParams p = {};
    p.M = a.N;
    p.N = a.K;
    p.k_steps = (int)((a.tokens + BK - 1) / BK);
    p.columns = a.N <= 64 ? 64 : 128;
    p.n_tiles = (a.K + BM - 1) / BM;
    if (!make_map(&p.map_w, a.scratch, (uint64_t)a.tokens, (uint64_t)a.K, (uint64_t)ldx, 64) ||
        !make_map(&p.map_x, a.dy, (uint64_t)a.tokens, (uint64_t)a.N, (uint64_t)a.lddy, 64))
        return -3;
    p.dw = a.out;
    p.ldo = a.ldo;
    p.out_wide = ((uintptr_t)a.out % 16) == 0 && a.ldo % 4 == 0;
    p.accumulate = a.accumulate;
    p.gain = (const __nv_bfloat16*)a.weight;
    p.bias = (const __nv_bfloat16*)a.bias;
    p.dy_sum = a.bias != nullptr ? a.dy_sum : nullptr;
    p.err_flag = a.err_flag;
    p.limit_ns = (unsigned long long)(a.wait_limit_s * 1e9);
    const int rc = act8_unpack(0, a.x, a.scratch, ldx, a.tokens, a.K, s);
    return rc != 0 ? rc : launch_few<kFewWgrad, kActNone>(p, few_plan(a.N, a.K, a.tokens, true).cluster, s);
}

}  // namespace

int act8_wgrad(const Act8WgradArgs& a, void* stream) {
    if (a.N <= 0 || a.K <= 0) return 0;
    if (a.tokens <= 0 || a.tokens > 0x7FFFFFFFll - 64 || a.err_flag == nullptr || a.out == nullptr) return -2;
    if (a.bias != nullptr && a.dy_sum == nullptr) return -2;
    if (!rows16(a.dy, a.lddy) || ((uintptr_t)a.x.q % 16) || (a.x.ldq % 16) || ((uintptr_t)a.x.e % 16) || (a.x.lde % 16)) return -2;
    const uint64_t tokens = (uint64_t)a.tokens, blocks = (uint64_t)(a.K + kAct8Block - 1) / kAct8Block;
    const bool convert = a.scratch == nullptr;
    const int64_t ldx = ((int64_t)a.K + 7) / 8 * 8;
    if (!convert && wgrad_few(a.tokens, a.N, a.K)) return wgrad_on_few(a, ldx, (cudaStream_t)stream);
    WgParams p;
    p.N = a.N;
    p.K = a.K;
    p.arrived = (unsigned*)a.workspace;
    p.partial = a.workspace == nullptr ? nullptr : (float*)((uint8_t*)a.workspace + linear_workspace_zeros());
    const bool wide = ((uintptr_t)a.out % 16) == 0 && a.ldo % 4 == 0;
    int rc = convert ? (wide ? plan_wgrad<true, true>(p, a.tokens) : plan_wgrad<true, false>(p, a.tokens))
                     : (wide ? plan_wgrad<false, true>(p, a.tokens) : plan_wgrad<false, false>(p, a.tokens));
    if (rc == 0 && !convert) rc = act8_unpack(0, a.x, a.scratch, ldx, a.tokens, a.K, stream);
    if (rc != 0) return rc;
    p.a_blocked = a.N % 64 == 0 && a.N >= BM ? 1 : 0;
    p.b_blocked = a.K % 64 == 0 && a.K >= 128 ? 1 : 0;
    bool ok = p.a_blocked ? make_map_blocked(&p.map_a, a.dy, tokens, (uint64_t)a.N, (uint64_t)a.lddy, BM / 64)
                          : make_map(&p.map_a, a.dy, tokens, (uint64_t)a.N, (uint64_t)a.lddy, 64);
    if (convert) {
        ok = ok && make_byte_map(&p.map_b, a.x.q, tokens, (uint64_t)a.K, (uint64_t)a.x.ldq, 128) &&
             make_byte_map(&p.map_e, a.x.e, tokens, blocks, (uint64_t)a.x.lde, 16);
    } else {
        ok = ok && (p.b_blocked ? make_map_blocked(&p.map_b, a.scratch, tokens, (uint64_t)a.K, (uint64_t)ldx, 2)
                                : make_map(&p.map_b, a.scratch, tokens, (uint64_t)a.K, (uint64_t)ldx, 64));
        p.map_e = p.map_b;   // not used
    }
    if (!ok) return -3;
    p.out = a.out;
    p.ldo = a.ldo;
    p.accumulate = a.accumulate;
    p.weight = (const __nv_bfloat16*)a.weight;
    p.bias = (const __nv_bfloat16*)a.bias;
    p.dy_sum = a.dy_sum;
    p.err_flag = a.err_flag;
    p.limit_ns = (unsigned long long)(a.wait_limit_s * 1e9);
    cudaStream_t st = (cudaStream_t)stream;
    if (convert) return wide ? launch_wgrad<true, true>(p, st) : launch_wgrad<true, false>(p, st);
    return wide ? launch_wgrad<false, true>(p, st) : launch_wgrad<false, false>(p, st);
}

// Converting tile by tile repeats the work for every 256 rows of dw and costs the tensor cores a fifth of their time;
// unpacking once costs five bytes of traffic per value of x. Measured on 16384 tokens, tile by tile against unpacked, in us with
// a cold L2 and back to back: 6144 x 2048: 369, 300 and 416, 347; 2048 x 2048: 135, 120 and 137, 126; 1024 x 2048: 86, 89 and
// 79, 87; 512 x 2048: 61, 69 and 53, 63. On 1024 tokens 2048 x 2048: 27, 24.
int64_t act8_wgrad_scratch(int64_t tokens, int N, int K) {
    if (tokens <= 0 || N <= 0 || K <= 0) return 0;
    return N >= kWgUnpackN || wgrad_few(tokens, N, K) ? tokens * (((int64_t)K + 7) / 8 * 8) * 2 : 0;
}

}  // namespace psb
