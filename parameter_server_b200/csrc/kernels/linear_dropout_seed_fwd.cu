// Instances of the fused linear kernel with dropout behind the activation, the seed in memory.
#include "linear_few.cuh"
#include "linear_fused.cuh"

namespace psb {

int linear_dropout_seed_fwd(const LinearArgs& a, cudaStream_t s) { return linear_by_size<false, kLinDropoutSeed>(a, s); }

}  // namespace psb
