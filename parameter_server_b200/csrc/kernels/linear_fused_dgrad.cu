// Input-gradient instances of the fused linear kernel.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_fused_dgrad(const LinearArgs& a, cudaStream_t s) {
    if (a.pre == nullptr && a.q == nullptr && a.act != kActNone) return -2;
    return linear_by_size<true, kLinPlain>(a, s);
}

}  // namespace psb
