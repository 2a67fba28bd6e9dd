// Forward instances of the fused linear kernel.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_fused_fwd(const LinearArgs& a, cudaStream_t s) { return linear_by_size<false, kLinPlain>(a, s); }

int64_t linear_workspace_zeros() { return (kArrivedWords * 4 + 255) / 256 * 256; }
int64_t linear_workspace_bytes() { return linear_workspace_zeros() + kPartialFloats * 4; }

int linear_fused(const LinearArgs& a, void* stream) {
    if (a.M <= 0 || a.N <= 0) return 0;
    if (a.K <= 0 || a.err_flag == nullptr || a.out == nullptr) return -2;
    if (!rows16(a.a, a.lda) || !rows16(a.w, a.ldw)) return -2;
    if (a.q != nullptr && (((uintptr_t)a.q % 16) || (a.ldq % 16) || ((uintptr_t)a.e % 16) || (a.lde % 16))) return -2;
    if (a.gated) {
        if (a.residual != nullptr || a.drop.threshold != 0) return -2;
        if (a.dgrad && (!rows16(a.out, a.ldo) || (a.out2 != nullptr && !rows16(a.out2, a.ldo2)))) return -2;
        if (a.q != nullptr && (((uintptr_t)a.q_up % 16) || (a.ldq_up % 16) || ((uintptr_t)a.e_up % 16) || (a.lde_up % 16) || a.q_up == nullptr || a.e_up == nullptr)) return -2;
        return a.dgrad ? linear_gated_dgrad(a, (cudaStream_t)stream) : linear_gated_fwd(a, (cudaStream_t)stream);
    }
    if (a.drop.threshold != 0) {
        if (a.dgrad) return -2;
        return a.drop.seed_ptr == nullptr ? linear_dropout_fwd(a, (cudaStream_t)stream) : linear_dropout_seed_fwd(a, (cudaStream_t)stream);
    }
    return a.dgrad ? linear_fused_dgrad(a, (cudaStream_t)stream) : linear_fused_fwd(a, (cudaStream_t)stream);
}

}  // namespace psb
