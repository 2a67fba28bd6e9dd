// Input-gradient instances of the gated linear kernel.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_gated_dgrad(const LinearArgs& a, cudaStream_t s) {
    if (a.pre == nullptr && a.q == nullptr) return -2;
    return linear_by_size<true, kLinGated>(a, s);
}

}  // namespace psb
