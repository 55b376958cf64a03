// A mixture-of-experts layer over packed experts, for a few tokens:
//   z = x R^T;  (e_j, w_j) = the top_k of z and their softmax weights;
//   y = addend + sum_j w_j D_ej (silu(G_ej x) * (U_ej x)).
// Five launches, each a programmatic dependent of the one before: routing (a
// cluster per token, which also packs the token's activations), gate and up, h
// (a cluster per slot, packed again), down, and the weighted sum over a token's
// slots.  The two products are in experts.cuh.
#include <cooperative_groups.h>

#include <climits>

#include "experts.cuh"

namespace mgb {

namespace cg = cooperative_groups;
using moe::expert_of;

constexpr int ROUTE_CTAS = 8;  // of a token's cluster
constexpr int ROUTE_THREADS = 256;

// Packs row `row` of x for weights of format fmt: the runs first, first + step,
// ... by this CTA's warps (first, step count warps).  Every CTA finds the row's
// largest magnitude itself.
template <int CTA_THREADS>
__device__ __forceinline__ void pack_row(int fmt, const float *x, uint64_t row, int cols, int first,
                                         int step, const moe::Packed16 &o) {
  __shared__ float most[CTA_THREADS / 32];
  const int lane = threadIdx.x & 31;
  const float *xr = x + row * cols;
  float mx = 0.f;
#pragma unroll 8
  for (int j = threadIdx.x; j < cols; j += CTA_THREADS) mx = fmaxf(mx, fabsf(xr[j]));
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  if (lane == 0) most[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < CTA_THREADS / 32; ++w) mx = fmaxf(mx, most[w]);
  const int k = moe::scale_exponent(mx);
  for (int r = first; r < cols / RUN; r += step)
    moe::pack_run16(fmt, o, row, cols, r, k, lane, [&](int i) { return xr[r * RUN + i]; });
  if (first == 0 && lane == 0) o.scale[row] = moe::pow2(-k);
}

__global__ void __launch_bounds__(256)
    mgb_moe_pack_kernel(int fmt, const float *x, int cols, moe::Packed16 o) {
  moe::grid_wait();
  moe::grid_dependents();
  pack_row<256>(fmt, x, blockIdx.y, cols, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8, o);
}

// Doubles as integers in the same order, -0 as +0, NaN (0) below all, and back.
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return v != v ? 0 : b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double order_value(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k ^ 1ull << 63 : ~k));
}

// One cluster per token: its warps take the experts' logits and, with `pack`,
// the token's runs; the first CTA's first warp then picks.  A logit is summed in f32
// chains of at most CHAIN products, joined in f64, so that its error does not grow with
// the width: at most 2^-20 of its terms' magnitudes, far less in practice.  Eight steps'
// loads are under way at a time, and a chain is joined while they are: 64 experts of
// 4,096, one token 4.9 us, 64 tokens 8.2 us; 1,024 experts, 16 tokens 50 us; 64 of 2^18, 8
// tokens 259 us.  (As a nest of loops, whose loads wait for the joins: 6.4, 9.3, 61 and
// 489 us.  Four CTAs an SM are what the registers are kept to; unasked, the compiler takes
// fewer and 6.1, 9.3, 56 and 470 us.)
constexpr int CHAIN = 16;
__global__ void __cluster_dims__(ROUTE_CTAS, 1, 1) __launch_bounds__(ROUTE_THREADS, 4)
    mgb_moe_route_kernel(const float *__restrict__ router, int experts, int hidden,
                         const float *x, int top_k, int normalize, float scale, float *ids,
                         float *weights, bool pack, int fmt, moe::Packed16 packed) {
  __shared__ double z[MGB_MOE_MAX_EXPERTS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int token = blockIdx.x / ROUTE_CTAS;
  const int warp = rank * (ROUTE_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  constexpr int WARPS = ROUTE_CTAS * ROUTE_THREADS / 32;
  cluster.barrier_arrive();  // (the first CTA has started before its memory is written)
  moe::grid_wait();
  moe::grid_dependents();
  cluster.barrier_wait();
  double *zs = cluster.map_shared_rank(z, 0);
  const float *xr = x + (size_t)token * hidden;
  const bool wide = hidden % 4 == 0 && ((uintptr_t)router & 15) == 0 && ((uintptr_t)x & 15) == 0;
  // few experts: several warps each, a stretch of the columns a warp (rounded up, so
  // that the stretches cover every column; the last ones may be short or empty)
  int stretches = 1;
  while (experts * stretches * 2 <= WARPS && hidden >= 1024 * stretches) stretches *= 2;
  const int columns = ((hidden + stretches - 1) / stretches + 127) & ~127;
  for (int i = warp; i < experts * stretches; i += WARPS) {
    const int from = min(hidden, i % stretches * columns), to = min(hidden, from + columns);
    const float *r = router + (size_t)(i / stretches) * hidden;
    double d = 0.0;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    int n = 0;  // steps taken
    auto join = [&]() {
      d += ((double)s[0] + (double)s[1]) + ((double)s[2] + (double)s[3]);
      s[0] = s[1] = s[2] = s[3] = 0.f;
    };
    if (wide) {
      constexpr int AHEAD = 8;
      auto add = [&](const float4 &a, const float4 &b) {
        s[0] = fmaf(a.x, b.x, s[0]);
        s[1] = fmaf(a.y, b.y, s[1]);
        s[2] = fmaf(a.z, b.z, s[2]);
        s[3] = fmaf(a.w, b.w, s[3]);
      };
      int j = from + lane * 4;
      for (; j + 128 * (AHEAD - 1) < to; j += 128 * AHEAD, n += AHEAD) {
        float4 a[AHEAD], b[AHEAD];
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) {
          a[c] = *reinterpret_cast<const float4 *>(xr + j + 128 * c);
          b[c] = __ldg(reinterpret_cast<const float4 *>(r + j + 128 * c));
        }
        if (n % CHAIN == 0) join();  // (of the chain before, while the loads are under way)
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) add(a[c], b[c]);
      }
      for (; j < to; j += 128, ++n) {
        if (n % CHAIN == 0) join();
        add(*reinterpret_cast<const float4 *>(xr + j), __ldg(reinterpret_cast<const float4 *>(r + j)));
      }
    } else {
      for (int j = from + lane; j < to; j += 128, ++n) {
        if (n % CHAIN == 0) join();
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (j + 32 * c < to) s[c] = fmaf(xr[j + 32 * c], r[j + 32 * c], s[c]);
      }
    }
    join();
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) zs[i] = d;
  }
  if (pack) pack_row<ROUTE_THREADS>(fmt, x, token, hidden, warp, WARPS, packed);
  cluster.sync();
  if (rank || threadIdx.x >= 32) return;
  if (stretches > 1) {  // (at most 32 experts)
    double d = 0.0;
    if (lane < experts)
      for (int i = 0; i < stretches; ++i) d += z[lane * stretches + i];
    __syncwarp();
    if (lane < experts) z[lane] = d;
    __syncwarp();
  }

  // Best first: the largest logit left, the lowest id among equals, NaN last.  A lane
  // keeps the best of its experts lane, lane + 32, ..., and looks again when that is
  // taken; the warp's best by three reductions of words.
  uint32_t taken = 0;  // bit c: expert 32 c + lane
  uint64_t key = 0;
  int best = INT_MAX;
  auto look = [&]() {
    key = 0, best = INT_MAX;
    for (int c = 0; c * 32 + lane < experts; ++c) {
      if (taken >> c & 1) continue;
      const uint64_t k = order_key(z[c * 32 + lane]);
      if (best == INT_MAX || k > key) key = k, best = c * 32 + lane;
    }
  };
  look();
  uint64_t mine = 0;  // of the lane-th choice
  for (int k = 0; k < top_k; ++k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
    const bool a = (uint32_t)(key >> 32) == hi;
    const uint32_t lo = __reduce_max_sync(0xffffffffu, a ? (uint32_t)key : 0u);
    const int e = __reduce_min_sync(0xffffffffu, a && (uint32_t)key == lo ? best : INT_MAX);
    if (lane == k) mine = (uint64_t)hi << 32 | lo, ids[(size_t)token * top_k + k] = (float)e;
    if (e == best) {
      taken |= 1u << (e >> 5);
      look();
    }
  }
  const double v = order_value(mine), top = __shfl_sync(0xffffffffu, v, 0);
  const double share = lane < top_k ? exp(v - top) : 0.0;
  double total = share;
  if (!normalize) {
    total = 0.0;
    for (int e = lane; e < experts; e += 32) total += exp(z[e] - top);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane < top_k) weights[(size_t)token * top_k + lane] = (float)(share / total * (double)scale);
}

// How the parts of a product are found: what its kernel left and the shapes.
struct Parts {
  const float *out;
  const int32_t *place, *share;
  int tiles, nb, width;  // row tiles of a pass, stages of a row, values of a result row
};

// The parts of row tile `tile` of a slot's pass.
__device__ __forceinline__ int tile_parts(const Parts &p, int place, int share, int tile) {
  return moe::parts_of((place >> 16) * p.tiles + tile, p.nb, share);
}
// The sum of n parts of a slot's result, in order: four values (c and the rows' widths are multiples of 32).
__device__ __forceinline__ float4 part_sum4(const Parts &p, int place, int used, int n, int c) {
  const float *at = p.out + (uint64_t)(place & 0xFFFF) * p.width + c;
  const uint64_t step = (uint64_t)used * p.width;
  float4 s = *reinterpret_cast<const float4 *>(at);
  for (int i = 1; i < n; ++i) {
    const float4 v = *reinterpret_cast<const float4 *>(at + i * step);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  return s;
}

// h = silu(gate) * up of one slot, packed for the down projection: a cluster per
// slot, which finds the row's largest magnitude together.
constexpr int H_CTAS = 8;
constexpr int H_THREADS = 256;
// Runs of a CTA: whole row tiles.
__host__ __device__ inline int h_runs(int ffn) {
  const int per = (ffn / RUN + H_CTAS - 1) / H_CTAS;
  return (per + 3) & ~3;
}
__global__ void __cluster_dims__(H_CTAS, 1, 1) __launch_bounds__(H_THREADS)
    mgb_moe_h_kernel(const Parts p, int ffn, int fmt, moe::Packed16 o) {
  extern __shared__ float h[];  // this CTA's runs
  __shared__ float most[H_THREADS / 32];
  __shared__ float cta_most;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), slot = blockIdx.x / H_CTAS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  moe::grid_wait();
  moe::grid_dependents();
  const int place = p.place[slot];
  if (place < 0) return;  // the whole cluster
  const int share = p.share[0], used = p.share[1];
  const int runs = ffn / RUN, per = h_runs(ffn);
  const int r0 = min(runs, rank * per), r1 = min(runs, r0 + per);
  const int tiles1 = p.tiles / 2;
  float mx = 0.f;
  // a warp's four runs (r0 is a multiple of four) lie in one row tile
  for (int r = r0 + 4 * warp; r < r1; r += H_THREADS / 8) {
    const int tile = r * RUN / moe::TILE, f = r * RUN + 4 * lane;
    if (f >= r1 * RUN) continue;
    const int ng = tile_parts(p, place, share, tile), nu = tile_parts(p, place, share, tiles1 + tile);
    const float4 g = part_sum4(p, place, used, ng, f), u = part_sum4(p, place, used, nu, ffn + f);
    float4 v;
    v.x = g.x / (1.f + expf(-g.x)) * u.x;
    v.y = g.y / (1.f + expf(-g.y)) * u.y;
    v.z = g.z / (1.f + expf(-g.z)) * u.z;
    v.w = g.w / (1.f + expf(-g.w)) * u.w;
    *reinterpret_cast<float4 *>(h + f - r0 * RUN) = v;
    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  if (lane == 0) most[warp] = mx;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < H_THREADS / 32; ++w) mx = fmaxf(mx, most[w]);
    cta_most = mx;
  }
  cluster.sync();
  mx = 0.f;
  for (int r = 0; r < H_CTAS; ++r) mx = fmaxf(mx, *cluster.map_shared_rank(&cta_most, r));
  const int k = moe::scale_exponent(mx);
  for (int r = r0 + warp; r < r1; r += H_THREADS / 32)
    moe::pack_run16(fmt, o, slot, ffn, r, k, lane, [&](int i) { return h[(r - r0) * RUN + i]; });
  if (rank == 0 && threadIdx.x == 0) o.scale[slot] = moe::pow2(-k);
  cluster.sync();  // the others' reads of cta_most are done
}

// y = addend + the weighted slots of a token, in slot order.
__global__ void __launch_bounds__(256)
    mgb_moe_combine_kernel(const Parts p, const float *weights, int hidden, int top_k,
                           const float *addend, float *y) {
  moe::grid_wait();
  moe::grid_dependents();
  const int token = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
  if (c >= hidden) return;
  const int share = p.share[0], used = p.share[1];
  const uint64_t step = (uint64_t)used * p.width;
  float a = 0.f;
  for (int j0 = 0; j0 < top_k; j0 += 4) {  // four slots' loads at a time
    int n[4];
    float w[4], v[4], v1[4];
    const float *at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = token * top_k + min(j0 + i, top_k - 1);
      const int place = j0 + i < top_k ? p.place[j] : -1;
      w[i] = weights[j];
      n[i] = place < 0 ? 0 : tile_parts(p, place, share, c / moe::TILE);
      at[i] = p.out + (uint64_t)(place & 0xFFFF) * p.width + c;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = n[i] > 0 ? at[i][0] : 0.f;
      v1[i] = n[i] > 1 ? at[i][step] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!n[i]) continue;  // (not even a NaN weight of it counts)
      float s = v[i];
      if (n[i] > 1) s += v1[i];
      for (int q = 2; q < n[i]; ++q) s += at[i][q * step];
      a = fmaf(w[i], s, a);
    }
  }
  const size_t at = (size_t)token * hidden + c;
  y[at] = addend ? addend[at] + a : a;
}

static int current_sms() {
  int dev = 0;
  cudaGetDevice(&dev);
  return device_sms(dev);
}

// Tokens of one expert in a pass over its rows: 8 where no expert has more (m) or
// few will.  At 2, 4, 6 and 8 tokens an expert (64 or 16 experts, Q8_0) 8 a pass
// take 199, 263, 88 and 102 us and 16 take 245, 279, 98 and 103 us; in Q4_K 161, 194,
// 77 and 87 us, and 166, 196, 73 and 76 us.
static int pass_tokens(uint64_t m, uint64_t slots, uint64_t experts) {
  return m <= 8 || slots <= 4 * experts ? 8 : moe::MOST_TOKENS;
}

static cudaError_t moe_product(int fmt, const moe::Args *a, int tokens, int sms, int *ctas_per_sm,
                               cudaStream_t stream) {
  switch (fmt) {
    case Q4_K: return launch_moe_product<Q4_K>(a, tokens, sms, ctas_per_sm, stream);
    case Q5_K: return launch_moe_product<Q5_K>(a, tokens, sms, ctas_per_sm, stream);
    case Q6_K: return launch_moe_product<Q6_K>(a, tokens, sms, ctas_per_sm, stream);
    case Q8_0: return launch_moe_product<Q8_0>(a, tokens, sms, ctas_per_sm, stream);
    case IQ4_NL: return launch_moe_product<IQ4_NL>(a, tokens, sms, ctas_per_sm, stream);
    default: return launch_moe_product<Q4_0>(a, tokens, sms, ctas_per_sm, stream);
  }
}

// Result rows of a product: parts times used slots.  A tile is cut into more
// than two parts only where few passes share the CTAs: P parts need a share
// below nb / (P - 2) stages, so passes below ctas / (tiles (P - 2)).
static uint64_t part_rows(uint64_t slots, uint64_t tokens, uint64_t tiles, uint64_t ctas) {
  uint64_t most = 2 * slots;
  for (uint64_t P = 3; P <= moe::MAX_PARTS + 1; ++P) {
    const uint64_t rows = tokens * (ctas / (tiles * (P - 2)) + 1);
    const uint64_t need = P * (slots < rows ? slots : rows);
    most = most > need ? most : need;
  }
  return most;
}

// The products' scratch.
struct MoeScratch {
  uint64_t x_hi, x_lo, x_sums, x_scale, h_hi, h_lo, h_sums, h_scale, place[2], share[2], out, total;
  MoeScratch(const mgb_experts &ex, uint64_t m, uint64_t top_k, int sms) {
    const uint64_t slots = m * top_k;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {  // in order, each 128-byte aligned
      const uint64_t r = at;
      at += (bytes + 127) / 128 * 128;
      return r;
    };
    x_hi = take(m * ex.hidden * 2);
    x_lo = take(m * ex.hidden * 2);
    x_sums = take(m * (ex.hidden / 256) * 32);
    x_scale = take(m * 4);
    h_hi = take(slots * ex.ffn * 2);
    h_lo = take(slots * ex.ffn * 2);
    h_sums = take(slots * (ex.ffn / 256) * 32);
    h_scale = take(slots * 4);
    for (int i = 0; i < 2; ++i) place[i] = take(slots * 4), share[i] = take(8);
    // the second product's results take the first one's place
    auto rows = [&](int fmt, uint64_t tiles) {
      const int tokens = pass_tokens(m, slots, ex.experts);
      int per_sm = 0;
      moe_product(fmt, nullptr, tokens, sms, &per_sm, nullptr);
      return part_rows(slots, tokens, tiles, (uint64_t)sms * per_sm);
    };
    const uint64_t a = rows(ex.gate_up_format, 2 * ceil_div(ex.ffn, moe::TILE)) * 2 * ex.ffn;
    const uint64_t b = rows(ex.down_format, ceil_div(ex.hidden, moe::TILE)) * ex.hidden;
    out = take((a > b ? a : b) * 4);
    total = at;
  }
  moe::Packed16 x(uint8_t *ws) const {
    return {reinterpret_cast<__half *>(ws + x_hi), reinterpret_cast<__half *>(ws + x_lo),
            reinterpret_cast<__half *>(ws + x_sums), reinterpret_cast<float *>(ws + x_scale)};
  }
  moe::Packed16 h(uint8_t *ws) const {
    return {reinterpret_cast<__half *>(ws + h_hi), reinterpret_cast<__half *>(ws + h_lo),
            reinterpret_cast<__half *>(ws + h_sums), reinterpret_cast<float *>(ws + h_scale)};
  }
};

uint64_t moe_experts_scratch_bytes(const mgb_experts &ex, uint64_t m, uint64_t top_k) {
  return m ? MoeScratch(ex, m, top_k, current_sms()).total : 0;
}

template <typename... P, typename... A>
static cudaError_t launch_chained(void (*kern)(P...), dim3 grid, dim3 block, uint32_t smem,
                                  cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
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
  moe::Packed16 packed = {};
  if (pack_for)  // the products of mgb_moe_layer follow, with this workspace
    packed = MoeScratch(*pack_for, m, top_k, current_sms()).x(static_cast<uint8_t *>(workspace));
  return launch_chained(mgb_moe_route_kernel, dim3((unsigned)m * ROUTE_CTAS), dim3(ROUTE_THREADS), 0,
                        stream, router, (int)experts, (int)hidden, x, (int)top_k, normalize, scale,
                        ids, weights, pack_for != nullptr, pack_for ? pack_for->gate_up_format : 0,
                        packed);
}

cudaError_t launch_moe_experts(const mgb_experts &ex, const float *x, uint64_t m, const float *ids,
                               const float *weights, uint64_t top_k, const float *addend, float *y,
                               uint32_t *bad, void *workspace, bool packed, int *err,
                               cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (bad) e = cudaMemsetAsync(bad, 0xFF, sizeof(uint32_t), stream);
  if (e != cudaSuccess || !m) return e;
  const int sms = current_sms();
  const MoeScratch s(ex, m, top_k, sms);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  const int hidden = (int)ex.hidden, ffn = (int)ex.ffn, slots = (int)(m * top_k);
  const int tokens = pass_tokens(m, slots, ex.experts);
  if (!packed) {
    e = launch_chained(mgb_moe_pack_kernel, dim3((unsigned)ceil_div(hidden / RUN, 32), (unsigned)m),
                       dim3(256), 0, stream, ex.gate_up_format, x, hidden, s.x(ws));
    if (e != cudaSuccess) return e;
  }
  moe::Args a = {};
  a.w0 = static_cast<const uint8_t *>(ex.gate);
  a.w1 = static_cast<const uint8_t *>(ex.up);
  a.act = s.x(ws);
  a.ids = ids;
  a.out = reinterpret_cast<float *>(ws + s.out);
  a.place = reinterpret_cast<int32_t *>(ws + s.place[0]);
  a.share = reinterpret_cast<int32_t *>(ws + s.share[0]);
  a.bad = bad;
  a.err = err;
  a.experts = (int)ex.experts;
  a.matrices = 2;
  a.rows = ffn;
  a.cols = hidden;
  a.slots = slots;
  a.act_div = (int)top_k;
  e = moe_product(ex.gate_up_format, &a, tokens, sms, nullptr, stream);
  if (e != cudaSuccess) return e;
  const Parts gu{a.out, a.place, a.share, 2 * (int)ceil_div(ffn, moe::TILE),
                 (int)ceil_div(hidden, moe::stage_cols(ex.gate_up_format)), 2 * ffn};
  const uint32_t h_smem = (uint32_t)h_runs(ffn) * RUN * 4;
  if (h_smem > 40 * 1024) {  // (the widest rows' always: another thread's call may be between)
    e = cudaFuncSetAttribute(mgb_moe_h_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             h_runs(MGB_MOE_MAX_WIDTH) * RUN * 4);
    if (e != cudaSuccess) return e;
  }
  e = launch_chained(mgb_moe_h_kernel, dim3((unsigned)slots * H_CTAS), dim3(H_THREADS), h_smem, stream, gu,
                     ffn, ex.down_format, s.h(ws));
  if (e != cudaSuccess) return e;
  a.w0 = a.w1 = static_cast<const uint8_t *>(ex.down);
  a.act = s.h(ws);
  a.place = reinterpret_cast<int32_t *>(ws + s.place[1]);
  a.share = reinterpret_cast<int32_t *>(ws + s.share[1]);
  a.bad = nullptr;
  a.matrices = 1;
  a.rows = hidden;
  a.cols = ffn;
  a.act_div = 1;
  e = moe_product(ex.down_format, &a, tokens, sms, nullptr, stream);
  if (e != cudaSuccess) return e;
  const Parts dn{a.out, a.place, a.share, (int)ceil_div(hidden, moe::TILE),
                 (int)ceil_div(ffn, moe::stage_cols(ex.down_format)), hidden};
  return launch_chained(mgb_moe_combine_kernel, dim3((unsigned)ceil_div(hidden, 256), (unsigned)m),
                        dim3(256), 0, stream, dn, weights, hidden, (int)top_k, addend, y);
}

}  // namespace mgb
