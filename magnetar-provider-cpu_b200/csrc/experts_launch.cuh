// Launches of the packed expert products of one format.
#pragma once

#include <atomic>

#include "experts.cuh"

namespace mgb {

template <int FMT, int T>
static cudaError_t launch_moe_one(const moe::Args *args, int sms, int *ctas_per_sm,
                                  cudaStream_t stream) {
  using X = moe::Shape<FMT, T>;
  if (ctas_per_sm) *ctas_per_sm = X::CTAS;
  if (!args) return cudaSuccess;
  const moe::Args &a = *args;
  auto *kern = moe::mgb_moe_product_kernel<FMT, T>;
  // at least what keeps CTAs for which there is no TMEM off the SM
  uint32_t smem = X::FIXED + moe::plan_bytes(a.experts, a.slots);
  constexpr uint32_t least = 228 * 1024 / (512 / X::TMEM + 1);
  if (smem < least) smem = least;
  // the opt-in is an attribute of the function on a device: once each
  static std::atomic<uint64_t> opted{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!(opted.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return e;
    opted.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sms * X::CTAS));
  cfg.blockDim = dim3(moe::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int FMT>
cudaError_t launch_moe_product(const moe::Args *a, int tokens, int sms, int *ctas_per_sm,
                               cudaStream_t stream) {
  if (tokens == 8) return launch_moe_one<FMT, 8>(a, sms, ctas_per_sm, stream);
  return launch_moe_one<FMT, 16>(a, sms, ctas_per_sm, stream);
}

}  // namespace mgb
