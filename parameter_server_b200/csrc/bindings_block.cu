// Bindings of the decoder-block operators: layer norm, fused linear layers, 8-bit activation checkpoints.
#include <pybind11/pybind11.h>

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
}
