// Products with few tiles, where the operands' way through the chip and the latency of one tile are the time:
//
//   forward   h = x w^T + b, y = act(h) + residual        dgrad   dh = (dy w) * act'(h), a = act(h)        (few tokens)
//   wgrad     dw = dy^T x, or (dy^T x) g + (sum dy) b^T    (few weights, x in bf16)
//
// The features of an output row take the tensor core's 128 rows, its rows (the tokens; outputs of the layer in wgrad) the columns,
// 16 to 128 of them, so that few tokens are not padded to a tile. A cluster of S CTAs has the same 128 features (and the same
// 128 rows, where there are more) and cuts the contraction in S parts; each CTA keeps its part's sums in TMEM. They meet in
// distributed shared memory: every CTA lays its sums down in its own, and CTA r reads the r-th share of the rows from all S,
// adds them in rank order (the same bits every time) and runs the epilogue for its share, with 32 neighbouring features in the
// lanes of a warp. Where more CTAs than SMs are needed, two fit an SM (16 tokens, 4096 -> 2048 in clusters of eight with one
// CTA to an SM: 17 us, two waves).
// The tensor core cuts its sums off towards zero, a billionth of them per token (act8_wgrad.cu): wgrad, whose contraction is long,
// starts a new chain in TMEM after 512 tokens, and the chains are added with rounding.
#pragma once
#include "linear_fused.cuh"

namespace psb {

namespace {

constexpr int kFewThreads = 512;
constexpr int kFewTokens = 128;    // of a tile
constexpr int kFewMaxStages = 12;
constexpr int kFewSmem = 220 * 1024, kFewSmemShared = 108 * 1024;   // one CTA on an SM, two
constexpr int kFewFwd = 0, kFewDgrad = 1, kFewWgrad = 2;
constexpr int kFewChain = 8;       // k-steps (of 64 tokens) of a wgrad chain
// CTAs that wait for one another (in a cluster, or a pair) must never share an SM with CTAs that hold the TMEM they still need.
// So each asks for shared memory in proportion to its TMEM: what fits one SM's shared memory fits its TMEM, whichever streams it is
// from. (The pair kernels have all the TMEM and 211 KB; 512 columns here take more than a 128-column CTA's share leaves.)
inline int few_smem_floor(int tmem_columns) { return (tmem_columns == 128 ? 58 : tmem_columns == 256 ? 114 : 172) * 1024; }

// tokens of a tile padded to what the tensor core takes here
inline int few_columns(int64_t M) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128; }

struct FewParams {
    CUtensorMap map_w, map_x;
    int M, N, k_steps;
    int n_tiles;
    int columns;          // rows of a tile padded to 16, 32, 64 or 128
    int tmem_columns;     // 128; wgrad: a power of two that has every chain's
    int stages, ring_bytes;
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
    int res_wide, out_wide, out2_wide, pre_wide;   // rows on 8-byte boundaries (wgrad's out: 16)
    // gated: the second factor's checkpoint, and whether its columns of pre and (dgrad) of out lie on 8-byte boundaries
    int8_t* q_up;
    int64_t ldq_up;
    uint8_t* e_up;
    int64_t lde_up;
    int pre_up_wide, out_up_wide;
    DropoutArgs drop;
    float* dw;            // wgrad: out, with the norm's weight (null: 1) and, with a bias, the sums of dy's rows
    const __nv_bfloat16* gain;
    const float* dy_sum;
    int accumulate;
    unsigned* err_flag;
    unsigned long long limit_ns;
};

__device__ __forceinline__ uint32_t cluster_nctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// Four neighbours of a bf16 row, `n` of them there; `wide`: the row's 8-byte blocks are aligned
__device__ __forceinline__ void load4(const __nv_bfloat16* p, int n, bool wide, float* f) {
    if (wide && n >= 4) {
        const uint2 r = *(const uint2*)p;
        f[0] = __uint_as_float(r.x << 16);
        f[1] = __uint_as_float(r.x & 0xFFFF0000u);
        f[2] = __uint_as_float(r.y << 16);
        f[3] = __uint_as_float(r.y & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = j < n ? __bfloat162float(p[j]) : 0.f;
    }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, int n, bool wide, const float* f) {
    if (wide && n >= 4) {
        uint2 r;
        __nv_bfloat162* h = (__nv_bfloat162*)&r;
        h[0] = __floats2bfloat162_rn(f[0], f[1]);
        h[1] = __floats2bfloat162_rn(f[2], f[3]);
        *(uint2*)p = r;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) p[j] = __float2bfloat16_rn(f[j]);
    }
}
// Four features' sums over the S CTAs, in rank order; all loads are on their way before the first is added (one round trip
// between SMs takes about 0.2 us).
template <int S>
__device__ __forceinline__ void add_parts(uint32_t at, float* v) {
    float4 part[S];
#pragma unroll
    for (int s = 0; s < S; ++s) part[s] = ld_cluster_v4(mapa_cluster(at, (uint32_t)s));
    v[0] = part[0].x; v[1] = part[0].y; v[2] = part[0].z; v[3] = part[0].w;
#pragma unroll
    for (int s = 1; s < S; ++s) { v[0] += part[s].x; v[1] += part[s].y; v[2] += part[s].z; v[3] += part[s].w; }
}

// The same for four features 32 apart
__device__ __forceinline__ void add_parts_apart(uint32_t at, int S, float* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0.f;
    for (int s = 0; s < S; ++s) {
        const uint32_t from = mapa_cluster(at, (uint32_t)s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(from + 128 * j) : "memory");
            v[j] = s == 0 ? x : v[j] + x;
        }
    }
}

template <int MODE, int ACT, int KIND = kLinPlain>
__global__ void __launch_bounds__(kFewThreads, KIND >= kLinDropout ? 2 : 1) linear_few_kernel(const __grid_constant__ FewParams p) {
    constexpr bool DGRAD = MODE == kFewDgrad, WGRAD = MODE == kFewWgrad, W_MN = MODE != kFewFwd;
    constexpr bool GATED_FWD = KIND == kLinGated && !DGRAD, GATED_DGRAD = KIND == kLinGated && DGRAD;
    constexpr int kWide = GATED_FWD ? BM / 2 : BM;   // outputs of a tile: of a gated one's features, half are the gate's
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = BM * BK * 2 + p.columns * BK * 2;
    const uint32_t parts = smem_u32(smem);   // float [tokens][128 features]: this CTA's sums, where the stages were
    uint64_t* full_bar = (uint64_t*)(smem + p.ring_bytes);
    uint64_t* empty_bar = full_bar + kFewMaxStages;
    uint64_t* done_bar = empty_bar + kFewMaxStages;
    uint32_t* tmem_slot = (uint32_t*)(done_bar + 1);

    const int S = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
    const int tile = (int)blockIdx.x / S, n0 = tile % p.n_tiles * kWide, m0 = tile / p.n_tiles * kFewTokens;
    const int tokens = min(p.M - m0, kFewTokens);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k_begin = (int)((int64_t)p.k_steps * rank / S), k_end = (int)((int64_t)p.k_steps * (rank + 1) / S), nk = k_end - k_begin;
    const int share = (p.columns + S - 1) / S;   // tokens that one CTA finishes
    auto load = [&](int k, int s) {
        const int k0 = (k_begin + k) * BK;
        uint8_t* sa = smem + s * stage_bytes;
        mbar_expect_tx(&full_bar[s], (uint32_t)stage_bytes);
        if constexpr (GATED_FWD) {
            tma_load_2d(sa, &p.map_w, &full_bar[s], k0, n0);   // [64 features][64 k] of the gate, and of the other factor
            tma_load_2d(sa + 64 * BK * 2, &p.map_w, &full_bar[s], k0, p.N + n0);
        } else if constexpr (!W_MN) {
            tma_load_2d(sa, &p.map_w, &full_bar[s], k0, n0);   // [128 features][64 k]
        } else {
            tma_load_2d(sa, &p.map_w, &full_bar[s], n0, k0);   // two blocks of [64 k][64 features]
            tma_load_2d(sa + 64 * 128, &p.map_w, &full_bar[s], n0 + 64, k0);
        }
        if constexpr (!WGRAD) {
            tma_load_2d(sa + BM * BK * 2, &p.map_x, &full_bar[s], k0, m0);   // [tokens][64 k]
        } else {
            for (int c = 0; c < p.columns; c += 64) tma_load_2d(sa + BM * BK * 2 + c * 128, &p.map_x, &full_bar[s], m0 + c, k0);   // [64 k][64 rows]
        }
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(done_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        wait_predecessor();
        for (int k = 0; k < min(nk, p.stages); ++k) load(k, k);   // the loads need no TMEM: they start before it is there
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)p.tmem_columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_address(tmem_slot);
    wait_predecessor();
    allow_successor();

    if (warp == 0) {
        if (lane == 0) {
            // ---- TMA producer ----
            uint32_t ph = 0;
            for (int k = p.stages, s = 0; k < nk; ++k) {
                if (!mbar_wait(&empty_bar[s], ph, p.limit_ns)) {
                    give_up(p.err_flag, 41u, tmem_slot);
                    break;
                }
                load(k, s);
                if (++s == p.stages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---- MMA issuer: D[feature][token] ----
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((W_MN ? 1u : 0u) << 15) | ((WGRAD ? 1u : 0u) << 16) | ((uint32_t)(p.columns >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            // running descriptors (in 16 bytes), and the next stage's barrier asked between this one's MMAs, as in linear_fused.cuh
            const uint64_t desc_w = make_desc(smem_u32(smem), W_MN ? 8192 : 16, 1024);
            const uint64_t desc_x = make_desc(smem_u32(smem) + BM * BK * 2, WGRAD ? 8192 : 16, 1024);
            constexpr uint32_t kNextW = W_MN ? 2048 >> 4 : 32 >> 4, kNextX = WGRAD ? 2048 >> 4 : 32 >> 4;
            uint32_t ph = 0, at = 0, tmem_d = tmem;
            bool have = false;
            for (int k = 0, s = 0; k < nk; ++k) {
                if (!have && !mbar_wait(&full_bar[s], ph, p.limit_ns * 2)) {
                    give_up(p.err_flag, 42u, tmem_slot);
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const bool wraps = s + 1 == p.stages;
                const uint64_t dw = desc_w + at, dx = desc_x + at;
                const bool opens = k == 0 || (WGRAD && k % kFewChain == 0);
                if (WGRAD && opens && k) tmem_d += (uint32_t)p.columns;
                umma_bf16(tmem_d, dw, dx, idesc, opens ? 0u : 1u);
#pragma unroll
                for (int u = 1; u < BK / UMMA_K; ++u) umma_bf16(tmem_d, dw + u * kNextW, dx + u * kNextX, idesc, 1u);
                const int next = wraps ? 0 : s + 1;
                have = mbar_try_wait(&full_bar[next], wraps ? ph ^ 1u : ph);   // (past the last step: not used)
                umma_commit(&empty_bar[s]);
                at = wraps ? 0u : at + ((uint32_t)stage_bytes >> 4);
                if (wraps) ph ^= 1u;
                s = next;
            }
            umma_commit(done_bar);   // (also on error, so that nobody waits for it)
        }
    }
    __syncwarp();
    // what the epilogue needs from memory, on its way meanwhile: a warp has a token, a lane four neighbouring features
    // (wgrad with rows that are not aligned: four features 32 apart, so that the lanes' single values lie side by side)
    const bool apart = WGRAD && p.out_wide == 0;
    // (gated: the lower sixteen lanes have the gate's features, the others those of the second factor at the same places)
    const bool up = GATED_FWD && lane >= 16;
    const int n = apart ? n0 + lane : n0 + (GATED_FWD ? lane & 15 : lane) * 4, have = p.N - n;   // features of this lane that exist (4 or more: all)
    const int bias_at = up ? p.N + n : n;
    const int stride = apart ? 32 : 1;                                 // between them
    const int t_end = min(tokens, (rank + 1) * share), t_first = rank * share + warp;
    float b[4] = {0.f, 0.f, 0.f, 0.f}, gain[4] = {1.f, 1.f, 1.f, 1.f}, aux[4], sum = 0.f;
    [[maybe_unused]] float aux_up[4];
    [[maybe_unused]] const DropKeys<KIND == kLinDropoutSeed> key(p.drop);
    if constexpr (WGRAD) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j * stride < have && p.gain != nullptr) gain[j] = __bfloat162float(p.gain[n + j * stride]);
    }
    if constexpr (!DGRAD) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j * stride < have)
                b[j] = p.bias32 != nullptr ? p.bias32[bias_at + j * stride] : p.bias != nullptr ? __bfloat162float(p.bias[bias_at + j * stride]) : 0.f;
    }
    auto fetch = [&](int t) {   // residual, or h
#pragma unroll
        for (int j = 0; j < 4; ++j) aux[j] = 0.f;
        if constexpr (GATED_DGRAD) {
#pragma unroll
            for (int j = 0; j < 4; ++j) aux_up[j] = 0.f;
        }
        if (have <= 0 || t >= t_end) return;
        const int64_t row = m0 + t;
        if constexpr (WGRAD) {
            if (p.dy_sum != nullptr) sum = p.dy_sum[row];
            if (!p.accumulate) return;
            const float* old = p.dw + row * p.ldo + n;
            if (p.out_wide != 0 && have >= 4) {
                const float4 o = *(const float4*)old;
                aux[0] = o.x; aux[1] = o.y; aux[2] = o.z; aux[3] = o.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j * stride < have) aux[j] = old[j * stride];
            }
        } else if constexpr (!DGRAD) {
            if (p.res != nullptr) load4(p.res + row * p.ldres + n, have, p.res_wide != 0, aux);
        } else if (p.q != nullptr) {
            const uint32_t w = *(const uint32_t*)(p.q + row * p.ldq + n) ^ 0x80808080u;   // (rows are padded to 16 bytes)
            const float step = act8_step(p.e[row * p.lde + n / kAct8Block]);
            aux[0] = s8_of_biased<0>(w) * step;
            aux[1] = s8_of_biased<1>(w) * step;
            aux[2] = s8_of_biased<2>(w) * step;
            aux[3] = s8_of_biased<3>(w) * step;
            if constexpr (GATED_DGRAD) {
                const uint32_t wu = *(const uint32_t*)(p.q_up + row * p.ldq_up + n) ^ 0x80808080u;
                const float step_up = act8_step(p.e_up[row * p.lde_up + n / kAct8Block]);
                aux_up[0] = s8_of_biased<0>(wu) * step_up;
                aux_up[1] = s8_of_biased<1>(wu) * step_up;
                aux_up[2] = s8_of_biased<2>(wu) * step_up;
                aux_up[3] = s8_of_biased<3>(wu) * step_up;
            }
        } else if (p.pre != nullptr) {
            load4(p.pre + row * p.ldpre + n, have, p.pre_wide != 0, aux);
            if constexpr (GATED_DGRAD) load4(p.pre + row * p.ldpre + p.N + n, have, p.pre_up_wide != 0, aux_up);
        }
    };
    fetch(t_first);
    // ---- this CTA's sums to its shared memory: the MMAs have read all stages, and no load is in flight ----
    // (One warp asks the barrier, the others sleep at the CTA's: with all sixteen asking, a k-step's four MMAs took 735 cycles to issue.)
    if (warp == 1 && !mbar_wait(done_bar, 0u, p.limit_ns * 4) && lane == 0) give_up(p.err_flag, 43u, tmem_slot);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    {
        // four warps share a quarter of TMEM's lanes (warp % 4) and take its columns in turn
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int quarter = warp & 3;
        for (int t0 = (warp >> 2) * 16; t0 < tokens; t0 += kFewThreads / 128 * 16) {
            uint32_t v[16];
            tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)t0, v);
            if constexpr (WGRAD) {
                for (int c = 1; c * kFewChain < nk; ++c) {
                    uint32_t w[16];
                    tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(c * p.columns + t0), w);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(w[j]));
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(parts + (uint32_t)((t0 + j) * BM + quarter * 32 + lane) * 4), "r"(v[j]) : "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    cluster_sync_all();
    if (warp == 1) {
        if (gave_up(tmem_slot)) let_copies_land();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)p.tmem_columns) : "memory");
    }
    // ---- epilogue of this CTA's tokens ----
    const uint32_t mine = parts + (uint32_t)lane * (apart ? 4 : 16);
    for (int t = t_first; t < t_end; t += kFewThreads / 32) {
        const int64_t row = m0 + t;
        float v[4];
        const uint32_t at = mine + (uint32_t)(t * BM) * 4;
        if (WGRAD && apart) add_parts_apart(at, S, v);
        else if (S == 8) add_parts<8>(at, v);
        else if (S == 4) add_parts<4>(at, v);
        else if (S == 2) add_parts<2>(at, v);
        else add_parts<1>(at, v);
        if constexpr (WGRAD) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = v[j] * gain[j] + sum * b[j] + aux[j];
            fetch(t + kFewThreads / 32);
            float* o = p.dw + row * p.ldo + n;
            if (p.out_wide != 0 && have >= 4) {
                *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j * stride < have) o[j * stride] = v[j];
            }
        } else if constexpr (!DGRAD) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += b[j];   // (0 past the last feature: its weights were read as zeros)
            if constexpr (GATED_FWD) {   // (behind the gate's last row of w, the tile has the other factor's first)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = j < have ? v[j] : 0.f;
            }
            if (p.pre != nullptr && have > 0) store4(p.pre + row * p.ldpre + bias_at, have, (up ? p.pre_up_wide : p.pre_wide) != 0, v);
            if (p.q != nullptr) {   // a block is eight lanes
                uint32_t m = abs_bits(abs_max(abs_max(v[0], v[1]), abs_max(v[2], v[3])));
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
                const uint32_t ex = act8_exponent(m);
                if (have > 0) {
                    int8_t* q = up ? p.q_up + row * p.ldq_up : p.q + row * p.ldq;
                    uint8_t* e = up ? p.e_up + row * p.lde_up : p.e + row * p.lde;
                    *(uint32_t*)(q + n) = ex == 255u ? 0u : act8_quantise4(v[0], v[1], v[2], v[3], act8_inverse_step(ex));
                    if ((lane & 7) == 0) e[n / kAct8Block] = (uint8_t)ex;
                }
            }
            if constexpr (GATED_FWD) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = act_of<ACT>(v[j]) * __shfl_xor_sync(0xFFFFFFFFu, v[j], 16);   // (meant in the lower lanes)
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = act_of<ACT>(v[j]);
                if constexpr (KIND >= kLinDropout) drop4(key, p.drop, (uint32_t)row, (uint32_t)n / 4, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += aux[j];
            }
            fetch(t + kFewThreads / 32);   // (before the stores: another lane's residual is never what this one writes)
            if (have > 0 && !up) store4(p.out + row * p.ldo + n, have, p.out_wide != 0, v);
        } else {
            float a[4];
            [[maybe_unused]] float du[4];
            if constexpr (GATED_DGRAD) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float slope = act_slope<ACT>(aux[j], &a[j]);
                    du[j] = v[j] * a[j];
                    a[j] *= aux_up[j];
                    v[j] *= aux_up[j] * slope;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= act_slope<ACT>(aux[j], &a[j]);
            }
            fetch(t + kFewThreads / 32);
            if (have > 0) {
                store4(p.out + row * p.ldo + n, have, p.out_wide != 0, v);
                if constexpr (GATED_DGRAD) store4(p.out + row * p.ldo + p.N + n, have, p.out_up_wide != 0, du);
                if (p.out2 != nullptr) store4(p.out2 + row * p.ldo2 + n, have, p.out2_wide != 0, a);
            }
        }
    }
    __syncwarp();
    cluster_sync_all();   // until here the others may read this CTA's shared memory
}

template <int MODE, int ACT, int KIND = kLinPlain>
int launch_few(FewParams& p, int cluster, cudaStream_t s) {
    constexpr auto kern = linear_few_kernel<MODE, ACT, KIND>;
    const int64_t ctas = (int64_t)p.n_tiles * ((p.M + kFewTokens - 1) / kFewTokens) * cluster;
    const int nk = (p.k_steps + cluster - 1) / cluster, chains = MODE == kFewWgrad ? (nk + kFewChain - 1) / kFewChain : 1;
    p.tmem_columns = 128;
    while (p.tmem_columns < chains * p.columns) p.tmem_columns *= 2;
    if (p.tmem_columns > 512) return -2;
    const int stage_bytes = (BM + p.columns) * BK * 2, extra = 1024 + 512;
    // (clusters of eight do not get SMs of their own: see few_plan)
    const int room = p.tmem_columns > 256 || (ctas <= 2 * kMaxPairs && cluster < 8) ? kFewSmem : kFewSmemShared;
    p.stages = std::min(std::min(kFewMaxStages, (room - extra) / stage_bytes), nk);
    p.ring_bytes = std::max(p.stages * stage_bytes, p.columns * BM * 4);
    const int smem = std::max(p.ring_bytes + extra, few_smem_floor(p.tmem_columns));
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.n_tiles * ((p.M + kFewTokens - 1) / kFewTokens) * cluster));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute a[2] = {in_clusters(cluster), start_early()};
    cfg.attrs = a;
    cfg.numAttrs = overlap_attrs(2);
    return (int)cudaLaunchKernelEx(&cfg, kern, p);
}

// How many CTAs share a tile's contraction, and the time of the whole in k-steps of a CTA that has its SM for itself (0.25 us).
// Fewer k-steps per CTA against the exchange of the sums: a 64th of a step per token for every doubling, and three steps more where
// two CTAs are on an SM. There a step of 128 tokens also takes half as long again (64 KB for both), one of fewer tokens less, since
// two CTAs wait for memory side by side. Measured, us (1, 2, 4, 8 CTAs): 16 x 8192 x 2048: 12.1, 9.7, 8.5; 128 x 2048 x 2048: 13.7, 9.2,
// 7.4, 8.8; 512 x 2048 x 2048: 13.9, 10.1, 11.3; 16 x 8192 x 512: 5.7, 4.7, 5.6. Within gemm_set_cta_limit() there are no more CTAs than
// that; a product with more tiles is the pairs' (cluster 0).
struct FewPlan {
    int cluster;
    float steps;
};
FewPlan few_plan(int64_t M, int64_t N, int64_t K, bool wgrad = false) {
    const int64_t tiles = (N + BM - 1) / BM * ((M + kFewTokens - 1) / kFewTokens), k_steps = (K + BK - 1) / BK;
    const bool limited = gemm_cta_limit() > 0;
    const int64_t sms = limited ? gemm_cta_limit() : 2 * kMaxPairs;
    const int columns = few_columns(M);
    FewPlan best = {0, 0.f};   // (wgrad: cluster 0 where the chains never fit TMEM, too)
    for (int cluster = 1, doublings = 0; cluster <= 8; cluster *= 2, ++doublings) {
        const int64_t ctas = tiles * cluster;
        // (chains past the first take TMEM that a second CTA would need)
        const int64_t fit = limited || (wgrad && k_steps > kFewChain * cluster) ? sms : 2 * sms;
        const bool crowded = ctas > sms && fit > sms;
        if (limited && ctas > sms) break;
        if (cluster > 1 && (ctas > fit || cluster > k_steps)) break;
        if (wgrad && (k_steps + cluster - 1) / cluster > (int64_t)kFewChain * 512 / BM) continue;
        // clusters of eight do not all fit the GPCs with an SM for each CTA: they share, with three stages for 128 tokens, or (wgrad with
        // more chains) come in two waves
        const bool eights = cluster == 8 && columns > 64 && 2 * ctas > sms;
        if (eights && fit > sms) break;
        const float step = !crowded ? 1.f : columns > 64 ? 1.5f : 0.6f;
        const float steps = (float)((k_steps + cluster - 1) / cluster) * step * (float)(eights ? 2 : (ctas + fit - 1) / fit) +
                            (float)doublings * ((float)columns / 64.f + (crowded ? 3.f : 0.f));
        if (best.cluster == 0 || steps < best.steps) best = {cluster, steps};
    }
    return best;
}

// Which kernel: up to 128 tokens this one wherever it can run; above, the one whose longest CTA is done first. A k-step of a pair's tile
// takes as long as one here; its launch, its prologue and its last tile's epilogue (half the warps for twice the values) cost 16 more.
// 512 x 8192 x 2048, in us: 20.5 here, 20.3; 1024 x 4096 x 4096: 31.9, 29.0; 1024 x 2048 x 8192: 31.6, 42.9.
bool few_tokens(const LinearArgs& a, int64_t features) {
    if (gemm_cta_limit() <= 0 && a.M <= kFewTokens) return true;
    const FewPlan plan = few_plan(a.M, features, a.K);
    if (plan.cluster == 0) return false;
    if (a.M <= kFewTokens) return true;
    const int64_t k_steps = (a.K + BK - 1) / BK, pairs = gemm_cta_limit() > 0 ? std::max(1, gemm_cta_limit() / 2) : kMaxPairs;
    const int64_t small = (int64_t)((features + BM - 1) / BM) * ((a.M + kFewTokens - 1) / kFewTokens), large = (int64_t)((features + 255) / 256) * ((a.M + 255) / 256);
    if (small > 4 * pairs) return false;
    return plan.steps < (float)((large + pairs - 1) / pairs * k_steps) + 16.f;
}

// Rows of products: of a gated layer's, each tile has 64 of the gate and the 64 that go with them
inline int64_t few_features(const LinearArgs& a) { return a.gated && !a.dgrad ? (a.N + 63) / 64 * (int64_t)BM : a.N; }

template <bool DGRAD, int KIND>
int linear_few(const LinearArgs& a, cudaStream_t s) {
    constexpr bool GATED_FWD = KIND == kLinGated && !DGRAD;
    FewParams p;
    p.M = a.M;
    p.N = a.N;
    p.k_steps = (a.K + BK - 1) / BK;
    p.columns = few_columns(a.M);
    if (!make_map(&p.map_x, a.a, (uint64_t)a.M, (uint64_t)a.K, (uint64_t)a.lda, p.columns)) return -3;
    if (!(DGRAD ? make_map(&p.map_w, a.w, (uint64_t)a.K, (uint64_t)a.N, (uint64_t)a.ldw, 64)
                : make_map(&p.map_w, a.w, (uint64_t)a.N * (GATED_FWD ? 2 : 1), (uint64_t)a.K, (uint64_t)a.ldw, GATED_FWD ? BM / 2 : BM)))
        return -3;
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
    auto wide = [](const void* r, int64_t ld) { return (uintptr_t)r % 8 == 0 && ld % 4 == 0 ? 1 : 0; };
    p.res_wide = wide(a.residual, a.ldres);
    p.out_wide = wide(a.out, a.ldo);
    p.out2_wide = wide(a.out2, a.ldo2);
    p.pre_wide = wide(a.pre, a.ldpre);
    p.drop = a.drop;
    if constexpr (KIND == kLinGated) {
        p.q_up = (int8_t*)a.q_up;
        p.ldq_up = a.ldq_up;
        p.e_up = (uint8_t*)a.e_up;
        p.lde_up = a.lde_up;
        p.pre_up_wide = p.pre != nullptr ? wide(p.pre + a.N, a.ldpre) : 0;
        p.out_up_wide = wide(p.out + a.N, a.ldo);
    }
    p.err_flag = a.err_flag;
    p.limit_ns = (unsigned long long)(a.wait_limit_s * 1e9);
    const int64_t features = few_features(a);
    p.n_tiles = (int)((features + BM - 1) / BM);
    const int cluster = few_plan(a.M, features, a.K).cluster;
    constexpr int MODE = DGRAD ? kFewDgrad : kFewFwd;
    switch (a.act) {
        case kActNone: return launch_few<MODE, kActNone, KIND>(p, cluster, s);
        case kActRelu: return launch_few<MODE, kActRelu, KIND>(p, cluster, s);
        case kActGelu: return launch_few<MODE, kActGelu, KIND>(p, cluster, s);
        case kActGeluTanh: return launch_few<MODE, kActGeluTanh, KIND>(p, cluster, s);
        case kActSilu: return launch_few<MODE, kActSilu, KIND>(p, cluster, s);
    }
    return -2;
}

// The kernel that takes such a product
template <bool DGRAD, int KIND>
int linear_by_size(const LinearArgs& a, cudaStream_t s) {
    return few_tokens(a, few_features(a)) ? linear_few<DGRAD, KIND>(a, s) : linear_typed<DGRAD, KIND>(a, s);
}

}  // namespace

}  // namespace psb
