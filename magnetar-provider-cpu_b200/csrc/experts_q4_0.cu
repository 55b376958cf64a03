// The expert products over Q4_0 weights.
#include "experts_launch.cuh"

namespace mgb {
template cudaError_t launch_moe_product<Q4_0>(const moe::Args *, int, int, int *, cudaStream_t);
}  // namespace mgb
