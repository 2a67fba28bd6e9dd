// Host interface of layer norm, its gradients, the 8-bit checkpoints of rows, and reproducible column sums (norm.cu).
// Device pointers throughout; `dtype`: 0 = bf16, 1 = fp32. Leading dimensions are in elements. Returns 0, a cudaError_t,
// or -2 (a shape or dtype that is not supported).
#pragma once
#include <cstdint>

namespace psb {

struct Act8View {          // rows of int8 and of exponent bytes, one per 32 columns
    void* q = nullptr;
    int64_t ldq = 0;
    void* e = nullptr;
    int64_t lde = 0;
};

// y = (x - mean) * rstd * weight + bias; weight / bias (x's dtype) may be null. keep.q != null: the normalised rows go to
// an 8-bit checkpoint and `mean` may be null.
int layer_norm_fwd(int dtype, const void* x, int64_t ldx, const void* weight, const void* bias, void* y, int64_t ldy, float* mean,
                   float* rstd, const Act8View& keep, int64_t rows, int64_t d, float eps, void* stream);
// dx = rstd * (p - avg(p) - xhat * avg(p * xhat)) + join with p = dy * weight; dweight = sum dy * xhat; dbias = sum dy, both
// fp32 and optional. xhat from x, mean and rstd, or from kept.q. `partial`: layer_norm_bwd_scratch() floats.
int layer_norm_bwd(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, const Act8View& kept, const void* weight,
                   const float* mean, const float* rstd, const void* join, int64_t ldjoin, void* dx, int64_t lddx, float* dweight,
                   float* dbias, int accumulate, float* partial, int64_t rows, int64_t d, void* stream);
int64_t layer_norm_bwd_scratch(int64_t rows, int64_t d);

int act8_pack(int dtype, const void* x, int64_t ldx, const Act8View& out, int64_t rows, int64_t cols, void* stream);
int act8_unpack(int dtype, const Act8View& in, void* x, int64_t ldx, int64_t rows, int64_t cols, void* stream);

// out[n] (+)= sum_m x[m][n] in a fixed order. `partial`: column_sum_scratch() floats.
int column_sum(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, float* out, int accumulate, float* partial,
               void* stream);
int64_t column_sum_scratch(int64_t rows, int64_t cols);

// bf16 rows to rows on 16-byte boundaries (dst, ldp a multiple of 8 elements and at least cols rounded up to 8)
int pad_rows(const void* src, int64_t ld, void* dst, int64_t ldp, int64_t rows, int64_t cols, void* stream);

}  // namespace psb
