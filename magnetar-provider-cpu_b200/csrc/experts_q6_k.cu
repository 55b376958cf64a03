// The expert products over Q6_K weights.
#include "experts_launch.cuh"

namespace mgb {
template cudaError_t launch_moe_product<Q6_K>(const moe::Args *, int, int, int *, cudaStream_t);
}  // namespace mgb
