// Forward instances of the gated linear kernel.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_gated_fwd(const LinearArgs& a, cudaStream_t s) { return linear_by_size<false, kLinGated>(a, s); }

}  // namespace psb
