// Low-rank adapters of many requests beside a shared projection:
//   y[r] = base[r] + s_a * (x[r] A_a^T) B_a^T,  a = ids[r],
// in two products: h[r] = s_a * A_a x[r] (rank values a row), y[r] = base[r] +
// B_a h[r].
#include "common.cuh"
#include "kernels.h"

namespace mgb {

// The adapter of a row: 0 .. count - 1, -1 for none, -2 for an invalid id.
__device__ __forceinline__ int adapter_of(float id, uint64_t count) {
  if (id < 0.0f) return -1;
  return floorf(id) == id && (double)id < (double)count ? (int)id : -2;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// One warp per (row, rank index).
template <typename T>
__global__ void mgb_adapter_shrink_kernel(const T *__restrict__ a, const float *__restrict__ scales,
                                          uint64_t count, uint64_t rank, uint64_t k,
                                          const float *__restrict__ ids, const float *__restrict__ x,
                                          uint64_t m, float *__restrict__ h, uint32_t *bad) {
  const int lane = threadIdx.x & 31;
  for (uint64_t i = (blockIdx.x * (uint64_t)blockDim.x + threadIdx.x) / 32; i < m * rank;
       i += (uint64_t)gridDim.x * blockDim.x / 32) {
    const uint64_t row = i / rank, r = i % rank;
    const int id = adapter_of(ids[row], count);
    if (id == -2 && r == 0 && lane == 0 && bad)
      atomicMin(bad, (uint32_t)(row < 0xFFFFFFFEull ? row : 0xFFFFFFFEull));
    if (id < 0) continue;
    float s = 0.f;
    for (uint64_t j = lane; j < k; j += 32)
      s = fmaf(to_f32(a[((uint64_t)id * rank + r) * k + j]), x[row * k + j], s);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) h[i] = scales ? s * scales[id] : s;
  }
}

// One thread per output.
template <typename T>
__global__ void mgb_adapter_expand_kernel(const T *__restrict__ b, uint64_t count, uint64_t rank,
                                          uint64_t n, const float *__restrict__ ids,
                                          const float *__restrict__ h, uint64_t m, const float *base,
                                          float *y) {
  for (uint64_t i = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; i < m * n;
       i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t row = i / n, c = i % n;
    const int id = adapter_of(ids[row], count);
    float v = base ? base[i] : 0.f;
    if (id >= 0) {
      float s = 0.f;
      for (uint64_t r = 0; r < rank; ++r)
        s = fmaf(to_f32(b[((uint64_t)id * n + c) * rank + r]), h[row * rank + r], s);
      v += s;
    }
    y[i] = v;
  }
}

uint64_t adapters_scratch_bytes(const mgb_adapters &ad, uint64_t m) {
  return ceil_div(m * ad.rank * 4, 16) * 16;
}

static unsigned capped(uint64_t blocks) { return (unsigned)(blocks > 65536 ? 65536 : blocks); }

template <typename T>
static cudaError_t launch_adapters_t(const mgb_adapters &ad, const float *ids, const float *x,
                                     uint64_t m, const float *base, float *y, uint32_t *bad,
                                     void *workspace, cudaStream_t stream) {
  float *h = static_cast<float *>(workspace);
  mgb_adapter_shrink_kernel<T><<<capped(ceil_div(m * ad.rank, 8)), 256, 0, stream>>>(
      static_cast<const T *>(ad.a), ad.scales, ad.count, ad.rank, ad.k, ids, x, m, h, bad);
  mgb_adapter_expand_kernel<T><<<capped(ceil_div(m * ad.n, 256)), 256, 0, stream>>>(
      static_cast<const T *>(ad.b), ad.count, ad.rank, ad.n, ids, h, m, base, y);
  return cudaGetLastError();
}

cudaError_t launch_adapters(const mgb_adapters &ad, const float *ids, const float *x, uint64_t m,
                            const float *base, float *y, uint32_t *bad, void *workspace,
                            cudaStream_t stream) {
  if (bad) {
    cudaError_t e = cudaMemsetAsync(bad, 0xFF, sizeof(uint32_t), stream);
    if (e != cudaSuccess) return e;
  }
  if (!m) return cudaSuccess;
  if (ad.dtype == MGB_DTYPE_F32)
    return launch_adapters_t<float>(ad, ids, x, m, base, y, bad, workspace, stream);
  if (ad.dtype == MGB_DTYPE_F16)
    return launch_adapters_t<__half>(ad, ids, x, m, base, y, bad, workspace, stream);
  return launch_adapters_t<__nv_bfloat16>(ad, ids, x, m, base, y, bad, workspace, stream);
}

}  // namespace mgb
