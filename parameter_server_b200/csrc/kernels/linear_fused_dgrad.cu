// Input-gradient instances of the fused linear kernel.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_fused_dgrad(const LinearArgs& a, cudaStream_t s) {
    if (a.pre == nullptr && a.q == nullptr && a.act != kActNone) return -2;
    return few_tokens(a) ? linear_few<true>(a, s) : linear_typed<true>(a, s);
}

}  // namespace psb
