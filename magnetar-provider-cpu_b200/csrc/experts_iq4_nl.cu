// The expert products over IQ4_NL weights.
#include "experts_launch.cuh"

namespace mgb {
template cudaError_t launch_moe_product<IQ4_NL>(const moe::Args *, int, int, int *, cudaStream_t);
}  // namespace mgb
