// Bindings of the decoder-block operators: layer norm, fused linear layers, 8-bit activation checkpoints.
#include <pybind11/pybind11.h>

#include "kernels/act8_wgrad.h"
#include "kernels/linear_fused.h"
#include "kernels/norm.h"

namespace py = pybind11;
using namespace psb;

namespace {
Act8View view(uintptr_t q, int64_t ldq, uintptr_t e, int64_t lde) { return Act8View{(void*)q, ldq, (void*)e, lde}; }
}  // namespace

void bind_block(py::module_& m) {
    m.def("layer_norm_fwd", [](int dtype, uintptr_t x, int64_t ldx, uintptr_t w, uintptr_t b, uintptr_t y, int64_t ldy, uintptr_t mean,
                               uintptr_t rstd, uintptr_t q, int64_t ldq, uintptr_t e, int64_t lde, int64_t rows, int64_t d, float eps,
                               uintptr_t s) {
        return layer_norm_fwd(dtype, (const void*)x, ldx, (const void*)w, (const void*)b, (void*)y, ldy, (float*)mean, (float*)rstd,
                              view(q, ldq, e, lde), rows, d, eps, (void*)s);
    });
    m.def("layer_norm_bwd", [](int dtype, uintptr_t dy, int64_t lddy, uintptr_t x, int64_t ldx, uintptr_t q, int64_t ldq, uintptr_t e,
                               int64_t lde, uintptr_t w, uintptr_t mean, uintptr_t rstd, uintptr_t join, int64_t ldjoin, uintptr_t dx,
                               int64_t lddx, uintptr_t dw, uintptr_t db, bool accumulate, uintptr_t partial, int64_t rows, int64_t d,
                               uintptr_t s) {
        return layer_norm_bwd(dtype, (const void*)dy, lddy, (const void*)x, ldx, view(q, ldq, e, lde), (const void*)w, (const float*)mean,
                              (const float*)rstd, (const void*)join, ldjoin, (void*)dx, lddx, (float*)dw, (float*)db, accumulate ? 1 : 0,
                              (float*)partial, rows, d, (void*)s);
    });
    m.def("layer_norm_bwd_scratch", &layer_norm_bwd_scratch);
    m.def("act8_pack", [](int dtype, uintptr_t x, int64_t ldx, uintptr_t q, int64_t ldq, uintptr_t e, int64_t lde, int64_t rows, int64_t cols,
                          uintptr_t s) { return act8_pack(dtype, (const void*)x, ldx, view(q, ldq, e, lde), rows, cols, (void*)s); });
    m.def("act8_unpack", [](int dtype, uintptr_t q, int64_t ldq, uintptr_t e, int64_t lde, uintptr_t x, int64_t ldx, int64_t rows, int64_t cols,
                            uintptr_t s) { return act8_unpack(dtype, view(q, ldq, e, lde), (void*)x, ldx, rows, cols, (void*)s); });
    m.def("column_sum", [](int dtype, uintptr_t x, int64_t ldx, int64_t rows, int64_t cols, uintptr_t out, bool accumulate, uintptr_t partial,
                           uintptr_t s) {
        return column_sum(dtype, (const void*)x, ldx, rows, cols, (float*)out, accumulate ? 1 : 0, (float*)partial, (void*)s);
    });
    m.def("column_sum_scratch", &column_sum_scratch);
    m.def("pad_rows", [](uintptr_t src, int64_t ld, uintptr_t dst, int64_t ldp, int64_t rows, int64_t cols, uintptr_t s) {
        return pad_rows((const void*)src, ld, (void*)dst, ldp, rows, cols, (void*)s);
    });
    m.def("linear_fused", [](bool dgrad, int act, int M, int N, int K, uintptr_t a, int64_t lda, uintptr_t w, int64_t ldw, uintptr_t bias,
                             bool bias_f32, uintptr_t residual, int64_t ldres, uintptr_t out, int64_t ldo, uintptr_t out2, int64_t ldo2,
                             uintptr_t pre, int64_t ldpre, uintptr_t q, int64_t ldq, uintptr_t e, int64_t lde, uintptr_t workspace,
                             uintptr_t err_flag, double wait_limit_s, uintptr_t s) {
        LinearArgs x;
        x.dgrad = dgrad ? 1 : 0;
        x.act = act;
        x.M = M;
        x.N = N;
        x.K = K;
        x.a = (const void*)a;
        x.lda = lda;
        x.w = (const void*)w;
        x.ldw = ldw;
        x.bias = (const void*)bias;
        x.bias_f32 = bias_f32 ? 1 : 0;
        x.residual = (const void*)residual;
        x.ldres = ldres;
        x.out = (void*)out;
        x.ldo = ldo;
        x.out2 = (void*)out2;
        x.ldo2 = ldo2;
        x.pre = (void*)pre;
        x.ldpre = ldpre;
        x.q = (void*)q;
        x.ldq = ldq;
        x.e = (void*)e;
        x.lde = lde;
        x.workspace = (void*)workspace;
        x.err_flag = (unsigned*)err_flag;
        x.wait_limit_s = wait_limit_s;
        return linear_fused(x, (void*)s);
    });
    m.def("act8_wgrad", [](uintptr_t dy, int64_t lddy, uintptr_t q, int64_t ldq, uintptr_t e, int64_t lde, uintptr_t out, int64_t ldo,
                           bool accumulate, uintptr_t weight, uintptr_t bias, uintptr_t dy_sum, int64_t tokens, int N, int K, uintptr_t scratch,
                           uintptr_t workspace, uintptr_t err_flag, double wait_limit_s, uintptr_t s) {
        Act8WgradArgs x;
        x.dy = (const void*)dy;
        x.lddy = lddy;
        x.x = view(q, ldq, e, lde);
        x.out = (float*)out;
        x.ldo = ldo;
        x.accumulate = accumulate ? 1 : 0;
        x.weight = (const void*)weight;
        x.bias = (const void*)bias;
        x.dy_sum = (const float*)dy_sum;
        x.tokens = tokens;
        x.scratch = (void*)scratch;
        x.N = N;
        x.K = K;
        x.workspace = (void*)workspace;
        x.err_flag = (unsigned*)err_flag;
        x.wait_limit_s = wait_limit_s;
        return act8_wgrad(x, (void*)s);
    });
    m.def("act8_wgrad_scratch", &act8_wgrad_scratch);
    m.def("linear_workspace_bytes", &linear_workspace_bytes);
    m.def("linear_workspace_zeros", &linear_workspace_zeros);
    m.attr("NEEDS_WORKSPACE") = kNeedsWorkspace;
}
