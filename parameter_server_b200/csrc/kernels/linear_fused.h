// Host interface of the fused linear layers (linear_fused.cu): device pointers, leading dimensions in elements.
#pragma once
#include <cstdint>

#include "dropout.h"

namespace psb {

enum LinearActivation { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

struct LinearArgs {
    // forward:  h = a w^T + bias, out = act(h) + residual; a [M][K], w [N][K]; h kept in `pre` (bf16) or `q` / `e` (8 bits)
    // dgrad:    out = (a w) * act'(h), out2 = act(h);      a [M][K], w [K][N]; h read from `pre` or `q` / `e`
    // with `drop`:    out = dropout(act(h)) + residual
    // gated (N counts the outputs): forward  [g | u] = a w^T + bias, out = act(g) * u; w [2N][K], bias [2N]; g and u kept side by side in
    //                 `pre` [M][2N], or in `q` / `e` and `q_up` / `e_up`;  dgrad  a w = da, out [M][2N] = [da * u * act'(g) | da * act(g)],
    //                 out2 = act(g) * u, both with rows on 16-byte boundaries; w [K][N]
    int dgrad = 0;
    int gated = 0;
    int act = 0;
    const void* a = nullptr;
    int64_t lda = 0;
    const void* w = nullptr;
    int64_t ldw = 0;
    const void* bias = nullptr;      // [N], bf16, or fp32 with bias_f32
    int bias_f32 = 0;
    const void* residual = nullptr;  // bf16 [M][N]
    int64_t ldres = 0;
    void* out = nullptr;             // bf16 [M][N]
    int64_t ldo = 0;
    void* out2 = nullptr;            // bf16 [M][N] (dgrad), optional
    int64_t ldo2 = 0;
    void* pre = nullptr;             // bf16 [M][N]
    int64_t ldpre = 0;
    void* q = nullptr;               // int8 [M][N] and uint8 [M][N / 32], rows on 16-byte boundaries
    int64_t ldq = 0;
    void* e = nullptr;
    int64_t lde = 0;
    void* q_up = nullptr;            // gated: the second factor's, like q / e
    int64_t ldq_up = 0;
    void* e_up = nullptr;
    int64_t lde_up = 0;
    DropoutArgs drop;                // forward; threshold 0: none
    int M = 0, N = 0, K = 0;
    void* workspace = nullptr;       // linear_workspace_bytes() bytes; the first linear_workspace_zeros() are zero before the
                                     // first call and left zero by every call. Null: tried without (see kNeedsWorkspace)
    unsigned* err_flag = nullptr;    // device word, set non-zero when a bounded wait ran out
    double wait_limit_s = 2.0;
};

// Nothing was launched: tiles are cut along the contraction here and meet in a workspace, which is null.
constexpr int kNeedsWorkspace = -4;

// Returns 0, a cudaError_t, -2 (alignment or an argument that is not supported), -3 (tensor map) or kNeedsWorkspace.
int linear_fused(const LinearArgs& args, void* stream);
int64_t linear_workspace_bytes();
int64_t linear_workspace_zeros();

}  // namespace psb
