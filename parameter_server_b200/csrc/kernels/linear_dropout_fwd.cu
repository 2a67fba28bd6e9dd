// Instances of the fused linear kernel with dropout behind the activation.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_dropout_fwd(const LinearArgs& a, cudaStream_t s) { return linear_by_size<false, kLinDropout>(a, s); }

}  // namespace psb
