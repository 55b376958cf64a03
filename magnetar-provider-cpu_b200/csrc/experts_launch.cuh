// Launches of the packed expert products of one format.
#pragma once

#include "experts.cuh"

namespace mgb {

template <int FMT, bool GATE_UP, int NT>
static cudaError_t launch_moe_one(const moe::Args &a, int sms, cudaStream_t stream) {
  const uint32_t smem = moe::WARPS * moe::warp_bytes<FMT>() + moe::plan_bytes(a.experts, a.slots);
  auto *kern = moe::mgb_moe_product_kernel<FMT, GATE_UP, NT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sms);
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
cudaError_t launch_moe_product(const moe::Args &a, bool gate_up, int nt, int sms,
                               cudaStream_t stream) {
  if (gate_up)
    return nt == 1   ? launch_moe_one<FMT, true, 1>(a, sms, stream)
           : nt == 2 ? launch_moe_one<FMT, true, 2>(a, sms, stream)
                     : launch_moe_one<FMT, true, 4>(a, sms, stream);
  return nt == 1   ? launch_moe_one<FMT, false, 1>(a, sms, stream)
         : nt == 2 ? launch_moe_one<FMT, false, 2>(a, sms, stream)
                   : launch_moe_one<FMT, false, 4>(a, sms, stream);
}

}  // namespace mgb
