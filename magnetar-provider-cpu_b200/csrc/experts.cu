// A mixture-of-experts layer over packed experts, for a few tokens:
//   z = x R^T;  (e_j, w_j) = the top_k of z and their softmax weights;
//   y = addend + sum_j w_j D_ej (silu(G_ej x) * (U_ej x)).
#include "common.cuh"
#include "decode.cuh"
#include "kernels.h"

namespace mgb {

// The expert of a slot: 0 .. experts - 1, -1 for unused, -2 for an invalid id.
__device__ __forceinline__ int expert_of(float id, uint64_t experts) {
  if (id < 0.0f) return -1;
  return floorf(id) == id && (double)id < (double)experts ? (int)id : -2;
}

// One CTA per token: the logits by warps, then the choice by one thread.
__global__ void __launch_bounds__(256)
    mgb_moe_route_kernel(const float *__restrict__ router, int experts, int hidden,
                         const float *__restrict__ x, int top_k, int normalize, float scale,
                         float *__restrict__ ids, float *__restrict__ weights) {
  __shared__ double z[MGB_MOE_MAX_EXPERTS];
  const int token = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = warp; e < experts; e += 8) {
    double s = 0.0;
    for (int j = lane; j < hidden; j += 32)
      s += (double)(x[(size_t)token * hidden + j]) * (double)router[(size_t)e * hidden + j];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) z[e] = s;
  }
  __syncthreads();
  if (threadIdx.x) return;
  double total = 0.0, top = 0.0, sum = 0.0;
  unsigned long long taken[MGB_MOE_MAX_EXPERTS / 64] = {};
  for (int j = 0; j < top_k; ++j) {
    int best = -1;
    for (int e = 0; e < experts; ++e)
      if (!(taken[e >> 6] >> (e & 63) & 1) && (best < 0 || z[e] > z[best] || (z[best] != z[best] && z[e] == z[e])))
        best = e;
    taken[best >> 6] |= 1ull << (best & 63);
    if (j == 0) {
      top = z[best];
      for (int e = 0; e < experts; ++e) total += exp(z[e] - top);
    }
    sum += exp(z[best] - top);
    ids[(size_t)token * top_k + j] = (float)best;
  }
  for (int j = 0; j < top_k; ++j) {
    const int e = (int)ids[(size_t)token * top_k + j];
    weights[(size_t)token * top_k + j] = (float)(exp(z[e] - top) / (normalize ? sum : total) * scale);
  }
}

// h[slot, f] = silu(gate) * up: one warp per (slot, f).
__global__ void mgb_moe_gate_up_kernel(int fmt, const uint8_t *__restrict__ gate,
                                       const uint8_t *__restrict__ up, uint64_t experts,
                                       uint64_t hidden, uint64_t ffn, const float *__restrict__ x,
                                       const float *__restrict__ ids, uint64_t slots, uint64_t top_k,
                                       float *__restrict__ h, uint32_t *bad) {
  const Layout L(fmt, experts * ffn, hidden);
  const int lane = threadIdx.x & 31;
  for (uint64_t i = (blockIdx.x * (uint64_t)blockDim.x + threadIdx.x) / 32; i < slots * ffn;
       i += (uint64_t)gridDim.x * blockDim.x / 32) {
    const uint64_t slot = i / ffn, f = i % ffn;
    const int e = expert_of(ids[slot], experts);
    if (e == -2 && f == 0 && lane == 0 && bad) atomicMin(bad, (uint32_t)slot);
    if (e < 0) continue;
    float g = 0.f, u = 0.f;
    const float *xr = x + slot / top_k * hidden;
    for (uint64_t j = 0; j < hidden / RUN; ++j) {
      g = fmaf(decode_value(fmt, gate, L, e * ffn + f, j, lane), xr[j * RUN + lane], g);
      u = fmaf(decode_value(fmt, up, L, e * ffn + f, j, lane), xr[j * RUN + lane], u);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      g += __shfl_xor_sync(0xffffffffu, g, o);
      u += __shfl_xor_sync(0xffffffffu, u, o);
    }
    if (lane == 0) h[i] = g / (1.f + expf(-g)) * u;
  }
}

// y: one warp per (token, output).
__global__ void mgb_moe_down_kernel(int fmt, const uint8_t *__restrict__ down, uint64_t experts,
                                    uint64_t hidden, uint64_t ffn, const float *__restrict__ h,
                                    const float *__restrict__ ids, const float *__restrict__ weights,
                                    uint64_t m, uint64_t top_k, const float *addend, float *y) {
  const Layout L(fmt, experts * hidden, ffn);
  const int lane = threadIdx.x & 31;
  for (uint64_t i = (blockIdx.x * (uint64_t)blockDim.x + threadIdx.x) / 32; i < m * hidden;
       i += (uint64_t)gridDim.x * blockDim.x / 32) {
    const uint64_t token = i / hidden, c = i % hidden;
    float acc = 0.f;
    for (uint64_t j = 0; j < top_k; ++j) {
      const uint64_t slot = token * top_k + j;
      const int e = expert_of(ids[slot], experts);
      if (e < 0) continue;
      float s = 0.f;
      for (uint64_t u = 0; u < ffn / RUN; ++u)
        s = fmaf(decode_value(fmt, down, L, e * hidden + c, u, lane), h[slot * ffn + u * RUN + lane], s);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      acc = fmaf(weights[slot], s, acc);
    }
    if (lane == 0) y[i] = addend ? addend[i] + acc : acc;
  }
}

uint64_t moe_route_scratch_bytes(uint64_t, uint64_t, uint64_t) { return 0; }
uint64_t moe_experts_scratch_bytes(const mgb_experts &ex, uint64_t m, uint64_t top_k) {
  return m * top_k * ex.ffn * 4;
}

cudaError_t launch_moe_route(const float *router, uint64_t experts, uint64_t hidden,
                             const float *x, uint64_t m, uint64_t top_k, int normalize,
                             float scale, float *ids, float *weights, void *, cudaStream_t stream) {
  if (!m) return cudaSuccess;
  mgb_moe_route_kernel<<<(unsigned)m, 256, 0, stream>>>(router, (int)experts, (int)hidden, x,
                                                        (int)top_k, normalize, scale, ids, weights);
  return cudaGetLastError();
}

static unsigned capped(uint64_t blocks) { return (unsigned)(blocks > 65536 ? 65536 : blocks); }

cudaError_t launch_moe_experts(const mgb_experts &ex, const float *x, uint64_t m, const float *ids,
                               const float *weights, uint64_t top_k, const float *addend, float *y,
                               uint32_t *bad, void *workspace, cudaStream_t stream) {
  if (bad) {
    cudaError_t e = cudaMemsetAsync(bad, 0xFF, sizeof(uint32_t), stream);
    if (e != cudaSuccess) return e;
  }
  if (!m) return cudaSuccess;
  float *h = static_cast<float *>(workspace);
  mgb_moe_gate_up_kernel<<<capped(ceil_div(m * top_k * ex.ffn, 8)), 256, 0, stream>>>(
      ex.gate_up_format, static_cast<const uint8_t *>(ex.gate), static_cast<const uint8_t *>(ex.up),
      ex.experts, ex.hidden, ex.ffn, x, ids, m * top_k, top_k, h, bad);
  mgb_moe_down_kernel<<<capped(ceil_div(m * ex.hidden, 8)), 256, 0, stream>>>(
      ex.down_format, static_cast<const uint8_t *>(ex.down), ex.experts, ex.hidden, ex.ffn, h, ids,
      weights, m, top_k, addend, y);
  return cudaGetLastError();
}

}  // namespace mgb
