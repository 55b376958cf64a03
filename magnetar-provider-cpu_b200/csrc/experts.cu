// A mixture-of-experts layer over packed experts, for a few tokens:
//   z = x R^T;  (e_j, w_j) = the top_k of z and their softmax weights;
//   y = addend + sum_j w_j D_ej (silu(G_ej x) * (U_ej x)).
// Four launches, each a programmatic dependent of the one before: routing (a
// cluster per token, which also packs the token's activations), gate and up,
// down, and the weighted sum over a token's slots.  The two products are in
// experts.cuh.
#include <cooperative_groups.h>

#include "experts.cuh"

namespace mgb {

namespace cg = cooperative_groups;
using moe::expert_of;

constexpr int ROUTE_CTAS = 8;  // of a token's cluster
constexpr int ROUTE_THREADS = 256;

// The token's activations in packets for weights of format fmt: run by run over
// the warps `first`, first + step, ...
__device__ __forceinline__ void pack_token(int fmt, const float *x, int token,
                                           int hidden, int first, int step, uint8_t *packets,
                                           float2 *meta) {
  const int lane = threadIdx.x & 31, runs = hidden / RUN;
  for (int r = first; r < runs; r += step) {
    const size_t at = (size_t)token * runs + r;
    moe::write_packet(fmt, moe::ld_f32(x + (size_t)token * hidden + r * RUN + lane), lane,
                      packets + at * moe::PACKET, meta + at);
  }
}

__global__ void __launch_bounds__(256)
    mgb_moe_pack_kernel(int fmt, const float *x, int hidden, uint8_t *packets,
                        float2 *meta) {
  moe::grid_wait();
  moe::grid_dependents();
  pack_token(fmt, x, blockIdx.y, hidden, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8,
             packets, meta);
}

// One cluster per token: its warps take the experts' logits and, with
// `packets`, the token's runs; the first CTA's first warp then picks.  A logit
// is a sum of f32 products in chains of hidden / 128 a lane, joined in f64.
__global__ void __cluster_dims__(ROUTE_CTAS, 1, 1) __launch_bounds__(ROUTE_THREADS)
    mgb_moe_route_kernel(const float *__restrict__ router, int experts, int hidden,
                         const float *x, int top_k, int normalize, float scale, float *ids,
                         float *weights, int fmt,
                         uint8_t *packets, float2 *meta) {
  __shared__ double z[MGB_MOE_MAX_EXPERTS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int token = blockIdx.x / ROUTE_CTAS;
  const int warp = rank * (ROUTE_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  constexpr int WARPS = ROUTE_CTAS * ROUTE_THREADS / 32;
  moe::grid_wait();
  moe::grid_dependents();
  double *zs = cluster.map_shared_rank(z, 0);
  const float *xr = x + (size_t)token * hidden;
  const bool wide = hidden % 4 == 0 && ((uintptr_t)router & 15) == 0 && ((uintptr_t)x & 15) == 0;
  for (int e = warp; e < experts; e += WARPS) {
    const float *r = router + (size_t)e * hidden;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (wide) {
#pragma unroll 4
      for (int j = lane * 4; j < hidden; j += 128) {
        const uint4 a = moe::ld_v4(xr + j);
        const float4 b = __ldg(reinterpret_cast<const float4 *>(r + j));
        s[0] = fmaf(__uint_as_float(a.x), b.x, s[0]);
        s[1] = fmaf(__uint_as_float(a.y), b.y, s[1]);
        s[2] = fmaf(__uint_as_float(a.z), b.z, s[2]);
        s[3] = fmaf(__uint_as_float(a.w), b.w, s[3]);
      }
    } else {
      for (int j = lane; j < hidden; j += 128)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (j + 32 * c < hidden) s[c] = fmaf(moe::ld_f32(xr + j + 32 * c), r[j + 32 * c], s[c]);
    }
    double d = ((double)s[0] + (double)s[1]) + ((double)s[2] + (double)s[3]);
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) zs[e] = d;
  }
  if (packets) pack_token(fmt, x, token, hidden, warp, WARPS, packets, meta);
  cluster.sync();
  if (rank || threadIdx.x >= 32) return;

  // best-first: the largest logit left, the lowest id among equals, NaN last
  auto before = [](double a, int i, double b, int j) {  // (a, i) sorts before (b, j)
    if (i < 0 || j < 0) return i >= 0;
    const bool na = a != a, nb = b != b;
    if (na || nb) return na == nb ? i < j : nb;
    return a > b || (a == b && i < j);
  };
  uint32_t taken = 0;  // bit c: expert 32 c + lane
  double top = 0.0, total = 0.0, sum = 0.0, mine = 0.0;  // lane k keeps choice k's share
  for (int k = 0; k < top_k; ++k) {
    double v = 0.0;
    int best = -1;
    for (int c = 0; c * 32 + lane < experts; ++c)
      if (!(taken >> c & 1) && before(z[c * 32 + lane], c * 32 + lane, v, best))
        v = z[c * 32 + lane], best = c * 32 + lane;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, v, o);
      const int oi = __shfl_xor_sync(0xffffffffu, best, o);
      if (before(ov, oi, v, best)) v = ov, best = oi;
    }
    if ((best & 31) == lane) taken |= 1u << (best >> 5);
    if (k == 0) {
      top = v;
      if (!normalize) {
        for (int e = lane; e < experts; e += 32) total += exp(z[e] - top);
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      }
    }
    const double share = exp(v - top);
    sum += share;
    if (lane == k) mine = share, ids[(size_t)token * top_k + k] = (float)best;
  }
  if (lane < top_k)
    weights[(size_t)token * top_k + lane] = (float)(mine / (normalize ? sum : total) * (double)scale);
}

// y = addend + the weighted slots of a token, in slot order.
__global__ void __launch_bounds__(256)
    mgb_moe_combine_kernel(const float *out, const float *ids, const float *weights, int experts,
                           int hidden, int top_k, const float *addend, float *y) {
  moe::grid_wait();
  moe::grid_dependents();
  const int token = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= hidden) return;  // hidden is a multiple of 32
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < top_k; ++j) {
    const size_t slot = (size_t)token * top_k + j;
    if (expert_of(moe::ld_f32(ids + slot), experts) < 0) continue;
    const float w = moe::ld_f32(weights + slot);
    const uint4 v = moe::ld_v4(out + slot * hidden + c);
    a[0] = fmaf(w, __uint_as_float(v.x), a[0]);
    a[1] = fmaf(w, __uint_as_float(v.y), a[1]);
    a[2] = fmaf(w, __uint_as_float(v.z), a[2]);
    a[3] = fmaf(w, __uint_as_float(v.w), a[3]);
  }
  const size_t at = (size_t)token * hidden + c;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[at + i] = addend ? addend[at + i] + a[i] : a[i];
}

uint64_t moe_route_scratch_bytes(uint64_t, uint64_t, uint64_t) { return 0; }

// The products' scratch: x and h in packets with their run factors, the slots'
// outputs.
struct MoeScratch {
  uint64_t x, x_meta, h, h_meta, out, total;
  MoeScratch(const mgb_experts &ex, uint64_t m, uint64_t top_k) {
    const uint64_t slots = m * top_k;
    // in order, each 128-byte aligned
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
      const uint64_t r = at;
      at += (bytes + 127) / 128 * 128;
      return r;
    };
    x = take(m * ex.hidden * 4);
    x_meta = take(m * (ex.hidden / RUN) * 8);
    h = take(slots * ex.ffn * 4);
    h_meta = take(slots * (ex.ffn / RUN) * 8);
    out = take(slots * ex.hidden * 4);
    total = at;
  }
};

uint64_t moe_experts_scratch_bytes(const mgb_experts &ex, uint64_t m, uint64_t top_k) {
  return MoeScratch(ex, m, top_k).total;
}

template <typename... P, typename... A>
static cudaError_t launch_chained(void (*kern)(P...), dim3 grid, dim3 block, cudaStream_t stream,
                                  A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

cudaError_t launch_moe_route(const float *router, uint64_t experts, uint64_t hidden,
                             const float *x, uint64_t m, uint64_t top_k, int normalize,
                             float scale, float *ids, float *weights, const mgb_experts *pack_for,
                             void *workspace, cudaStream_t stream) {
  if (!m) return cudaSuccess;
  uint8_t *packets = nullptr;
  float2 *meta = nullptr;
  int fmt = 0;
  if (pack_for) {  // the products of mgb_moe_layer follow, with this workspace
    const MoeScratch s(*pack_for, m, top_k);
    packets = static_cast<uint8_t *>(workspace) + s.x;
    meta = reinterpret_cast<float2 *>(static_cast<uint8_t *>(workspace) + s.x_meta);
    fmt = pack_for->gate_up_format;
  }
  return launch_chained(mgb_moe_route_kernel, dim3((unsigned)m * ROUTE_CTAS), dim3(ROUTE_THREADS),
                        stream, router, (int)experts, (int)hidden, x, (int)top_k, normalize, scale,
                        ids, weights, fmt, packets, meta);
}

static cudaError_t moe_product(int fmt, const moe::Args &a, bool gate_up, int nt, int sms,
                               cudaStream_t stream) {
  switch (fmt) {
    case Q4_K: return launch_moe_product<Q4_K>(a, gate_up, nt, sms, stream);
    case Q5_K: return launch_moe_product<Q5_K>(a, gate_up, nt, sms, stream);
    case Q6_K: return launch_moe_product<Q6_K>(a, gate_up, nt, sms, stream);
    case Q8_0: return launch_moe_product<Q8_0>(a, gate_up, nt, sms, stream);
    case IQ4_NL: return launch_moe_product<IQ4_NL>(a, gate_up, nt, sms, stream);
    default: return launch_moe_product<Q4_0>(a, gate_up, nt, sms, stream);
  }
}

// Warps that share a tile's columns: as many as there are stages of a row (every
// warp then streams its own piece of it), and more, one of them idle, where the
// tiles would not cover the SMs.
static int column_slices(int fmt, int rows, int cols, int row_unit, int most, uint64_t slots,
                         int experts, int sms) {
  const int stage = fmt == Q4_K || fmt == Q4_0 || fmt == IQ4_NL ? 256 : 128;
  const int stages = (cols + stage - 1) / stage;
  const uint64_t used = slots < (uint64_t)experts ? slots : (uint64_t)experts;
  int ks = 1;
  while (ks < most) {
    const uint64_t tiles = used * ceil_div(rows, row_unit * (moe::WARPS / ks));
    if (ks * 2 <= stages || (ks < stages && tiles < (uint64_t)sms)) ks *= 2;
    else break;
  }
  return ks;
}

cudaError_t launch_moe_experts(const mgb_experts &ex, const float *x, uint64_t m, const float *ids,
                               const float *weights, uint64_t top_k, const float *addend, float *y,
                               uint32_t *bad, void *workspace, bool packed, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (bad) e = cudaMemsetAsync(bad, 0xFF, sizeof(uint32_t), stream);
  if (e != cudaSuccess || !m) return e;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = device_sms(dev);
  const MoeScratch s(ex, m, top_k);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  const int hidden = (int)ex.hidden, ffn = (int)ex.ffn, slots = (int)(m * top_k);
  // tokens of one expert in a pass over its rows: m is the most it can have
  const int nt = m <= 8 ? 1 : m <= 16 ? 2 : 4;
  if (!packed) {
    e = launch_chained(mgb_moe_pack_kernel, dim3((unsigned)ceil_div(hidden / RUN, 8), (unsigned)m),
                       dim3(256), stream, ex.gate_up_format, x, hidden, ws + s.x,
                       reinterpret_cast<float2 *>(ws + s.x_meta));
    if (e != cudaSuccess) return e;
  }
  moe::Args a = {};
  a.w0 = static_cast<const uint8_t *>(ex.gate);
  a.w1 = static_cast<const uint8_t *>(ex.up);
  a.packets = ws + s.x;
  a.meta = reinterpret_cast<const float2 *>(ws + s.x_meta);
  a.ids = ids;
  a.h_packets = ws + s.h;
  a.h_meta = reinterpret_cast<float2 *>(ws + s.h_meta);
  a.bad = bad;
  a.experts = (int)ex.experts;
  a.rows = ffn;
  a.cols = hidden;
  a.slots = slots;
  a.act_div = (int)top_k;
  a.ks = column_slices(ex.gate_up_format, ffn, hidden, 16, 8, slots, a.experts, sms);
  a.down_fmt = ex.down_format;
  e = moe_product(ex.gate_up_format, a, true, nt, sms, stream);
  if (e != cudaSuccess) return e;
  a.w0 = a.w1 = static_cast<const uint8_t *>(ex.down);
  a.packets = ws + s.h;
  a.meta = reinterpret_cast<const float2 *>(ws + s.h_meta);
  a.out = reinterpret_cast<float *>(ws + s.out);
  a.rows = hidden;
  a.cols = ffn;
  a.act_div = 1;
  a.ks = column_slices(ex.down_format, hidden, ffn, 32, 16, slots, a.experts, sms);
  e = moe_product(ex.down_format, a, false, nt, sms, stream);
  if (e != cudaSuccess) return e;
  return launch_chained(mgb_moe_combine_kernel, dim3((unsigned)ceil_div(hidden, 1024), (unsigned)m),
                        dim3(256), stream, static_cast<const float *>(a.out), ids, weights,
                        a.experts, hidden, (int)top_k, addend, y);
}

}  // namespace mgb
