// The expert products over Q5_K weights.
#include "experts_launch.cuh"

namespace mgb {
template cudaError_t launch_moe_product<Q5_K>(const moe::Args *, int, int, int *, cudaStream_t);
}  // namespace mgb
