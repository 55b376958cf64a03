// Low-rank adapters of many requests beside a shared projection:
//   y[r] = base[r] + s_a * (x[r] A_a^T) B_a^T,  a = ids[r],
// in two products: h[r] = s_a * A_a x[r] (rank values a row), y[r] = base[r] +
// B_a h[r], by one launch: a cluster of 8 CTAs takes one group of rows, each CTA
// an eighth of k for h, which they exchange through distributed shared memory,
// and then an eighth of the outputs (two chained launches cost one row 9.8 us
// against PLACEHOLDER).
//
// Rows are grouped by adapter into tiles of up to 16, the M of mma.sync
// m16n8k8 (tf32 operands, f32 accumulation), so that an adapter is read once
// for its rows whatever their order, and one row alone costs no more than its
// adapter's bytes.  The products are bound by those bytes or, with many rows,
// by base and y; arithmetic intensity never exceeds a few hundred operations a
// byte, far from what tcgen05 is for.
//
// f32 accuracy from tf32: x and h are held as hi + lo, two tf32 terms (22 bits);
// f16 and bf16 factors are tf32 numbers as they are, f32 factors are split too.
// The order of a product's K is free, so a lane takes runs of neighbouring
// values of its row: every load is 16 bytes where the buffers allow it.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace mgb {
namespace {

namespace cg = cooperative_groups;

constexpr int ROWS = 16;          // of a tile
constexpr int INLINE_ROWS = 128;  // up to here every CTA plans for itself
constexpr int BUCKETS = 4096;     // of the planning kernel's sort
constexpr int CTAS = 8;           // of a cluster
constexpr int WARPS = 8;          // of a CTA
constexpr int COLS = 32;          // outputs of a warp at a time

// The adapter of a row: 0 .. count - 1, -1 for none, -2 for an invalid id.
__device__ __forceinline__ int adapter_of(float id, uint64_t count) {
  if (id < 0.0f) return -1;
  return floorf(id) == id && (double)id < (double)count ? (int)id : -2;
}

struct Tile {
  int start, len, id;  // positions of the sorted order; the adapter or -1
};

struct Params {
  const void *a, *b;
  const float *scales, *ids, *x, *base;
  float *y;
  int32_t *order;    // [m]: the rows by adapter (m > INLINE_ROWS)
  Tile *tiles;       // and their tiles
  int32_t *ntiles;
  uint32_t *bad;
  uint64_t count;
  int m, k, n, rank;
  bool wide_a, wide_b, wide_x, wide_y;  // 16-byte loads are aligned
};

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- grouping ------------------------------------------------------------------------------

// Shared memory of a CTA that plans for itself.
struct SmallPlan {
  int id[INLINE_ROWS];
  int16_t order[INLINE_ROWS], head[INLINE_ROWS];
  Tile tiles[INLINE_ROWS];
  int ntiles;
};

// Rows sorted by (id, row), tiles of up to 16 rows of one id.
__device__ void plan_small(const Params &p, SmallPlan &s, bool report) {
  const int i = threadIdx.x;
  if (i == 0) s.ntiles = 0;
  int id = -1;
  if (i < p.m) {
    id = adapter_of(p.ids[i], p.count);
    if (id == -2) {
      if (report && p.bad) atomicMin(p.bad, (uint32_t)i);
      id = -1;
    }
    s.id[i] = id;
  }
  __syncthreads();
  int pos = 0, nth = 0, same = 0;
  if (i < p.m) {
    for (int j = 0; j < p.m; ++j) {
      const int o = s.id[j];
      pos += o < id || (o == id && j < i);
      nth += o == id && j < i;
      same += o == id;
    }
    s.order[pos] = (int16_t)i;
    s.head[pos] = nth % ROWS == 0;
  }
  __syncthreads();
  if (i < p.m && nth % ROWS == 0) {
    int t = 0;
    for (int j = 0; j < pos; ++j) t += s.head[j];
    s.tiles[t] = Tile{pos, min(ROWS, same - nth), id};
    if (pos + min(ROWS, same - nth) == p.m) s.ntiles = t + 1;
  }
  __syncthreads();
}

__device__ __forceinline__ int block_scan(int v, int *warp_sums, int &total) {  // exclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + s - v;
}

// One CTA: rows by bucket (the adapter, modulo 4,095; the last bucket holds the
// rows without one), then tiles of up to 16 neighbours of one adapter.  Which
// tile a row lands in does not affect its result.
__global__ void __launch_bounds__(1024) mgb_adapter_plan_kernel(const Params p) {
  __shared__ int at[BUCKETS];
  __shared__ int sums[32], s_carry[2];
  grid_wait();
  grid_dependents();
  for (int b = threadIdx.x; b < BUCKETS; b += 1024) at[b] = 0;
  __syncthreads();
  auto id_of = [&](int r) { return adapter_of(p.ids[r], p.count); };
  auto bucket = [&](int id) { return id < 0 ? BUCKETS - 1 : id % (BUCKETS - 1); };
  for (int r = threadIdx.x; r < p.m; r += 1024) {
    const int id = id_of(r);
    if (id == -2 && p.bad) atomicMin(p.bad, (uint32_t)r);
    atomicAdd(&at[bucket(id)], 1);
  }
  __syncthreads();
  {
    int c[4], v = 0, total;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = at[4 * threadIdx.x + i], v += c[i];
    int s = block_scan(v, sums, total);
#pragma unroll
    for (int i = 0; i < 4; ++i) at[4 * threadIdx.x + i] = s, s += c[i];
  }
  __syncthreads();
  for (int r = threadIdx.x; r < p.m; r += 1024) p.order[atomicAdd(&at[bucket(id_of(r))], 1)] = r;
  __syncthreads();
  // run heads, then tile heads (every 16th of a run)
  if (threadIdx.x == 0) s_carry[0] = 0, s_carry[1] = 0;
  __syncthreads();
  for (int p0 = 0; p0 < p.m; p0 += 1024) {
    const int i = p0 + threadIdx.x;
    int id = -3, prev = -3;
    if (i < p.m) {
      id = max(id_of(p.order[i]), -1);
      if (i) prev = max(id_of(p.order[i - 1]), -1);
    }
    const bool head = i < p.m && id != prev;
    // the run's start: an inclusive maximum of the head positions
    int start = head ? i : -1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, start, o);
      if (lane >= o) start = max(start, u);
    }
    __syncthreads();
    if (lane == 31) sums[warp] = start;
    __syncthreads();
    for (int w = 0; w < warp; ++w) start = max(start, sums[w]);
    start = max(start, s_carry[0]);
    const bool tile = i < p.m && (i - start) % ROWS == 0;
    int total;
    const int t = s_carry[1] + block_scan(tile, sums, total);
    __syncthreads();
    if (threadIdx.x == 1023) s_carry[0] = start;
    if (threadIdx.x == 0) s_carry[1] += total;
    if (tile) p.tiles[t] = Tile{i, 0, id};
    __syncthreads();
  }
  const int n = s_carry[1];
  if (threadIdx.x == 0) *p.ntiles = n;
  for (int t = threadIdx.x; t < n; t += 1024)
    p.tiles[t].len = (t + 1 < n ? p.tiles[t + 1].start : p.m) - p.tiles[t].start;
}

// The CTA's tile and its rows (row[i] of lanes' tokens, absent ones repeat the
// first); false: no such tile.
__device__ __forceinline__ bool find_tile(const Params &p, int t, SmallPlan &plan, int (&rows)[ROWS],
                                          bool report, Tile &tile) {
  const bool small = p.m <= INLINE_ROWS;
  if (small) plan_small(p, plan, report);
  if (t >= (small ? plan.ntiles : *p.ntiles)) return false;
  tile = small ? plan.tiles[t] : p.tiles[t];
  if (threadIdx.x < ROWS) {
    const int i = tile.start + (threadIdx.x < tile.len ? threadIdx.x : 0);
    rows[threadIdx.x] = small ? plan.order[i] : p.order[i];
  }
  __syncthreads();
  return true;
}

// ---- operands --------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t tf32(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
// v = hi + lo to 22 bits
__device__ __forceinline__ void split(float v, uint32_t &hi, uint32_t &lo) {
  hi = tf32(v);
  lo = tf32(v - __uint_as_float(hi));
}
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += (hi + lo) * (b0, b1) for factors of type T, to 22 bits of each
template <typename T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                         float b0, float b1) {
  if constexpr (sizeof(T) == 4) {
    uint32_t h0, h1, l0, l1;
    split(b0, h0, l0);
    split(b1, h1, l1);
    mma1688(c, lo, h0, h1);
    mma1688(c, hi, l0, l1);
    mma1688(c, hi, h0, h1);
  } else {
    mma1688(c, lo, __float_as_uint(b0), __float_as_uint(b1));
    mma1688(c, hi, __float_as_uint(b0), __float_as_uint(b1));
  }
}

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// N neighbouring values from `at`, `left` of which exist (the others are 0);
// wide: 16-byte aligned when all exist.
template <int N, typename T>
__device__ __forceinline__ void load_values(const T *at, int left, bool wide, float (&v)[N]) {
  constexpr int PER = 16 / sizeof(T);
  if (wide && left >= N) {
    if constexpr (N >= PER) {
#pragma unroll
      for (int i = 0; i < N / PER; ++i) {
        const uint4 w = *reinterpret_cast<const uint4 *>(at + i * PER);
        const T *t = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int j = 0; j < PER; ++j) v[i * PER + j] = as_f32(t[j]);
      }
    } else {  // half of 16 bytes
      const uint2 w = *reinterpret_cast<const uint2 *>(at);
      const T *t = reinterpret_cast<const T *>(&w);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = as_f32(t[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < left ? as_f32(at[j]) : 0.f;
  }
}

// ---- the kernel --------------------------------------------------------------------------------
//
// RC: ranks of a pass (a lane of the second product: RC / 4 neighbours, K of
// RC / 8 MMAs).  Shared memory: the warps' sums of a pass, then the whole h
// (`red`), and this CTA's part of h (`part`).
template <int RC>
__host__ __device__ constexpr uint32_t red_floats() {
  return WARPS * ROWS * (RC + 4);
}

template <typename T, int RC>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(32 * WARPS, 2)
    mgb_adapter_kernel(const Params p) {
  extern __shared__ __align__(16) float red[];
  __shared__ SmallPlan plan;
  __shared__ int rows[ROWS];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank();
  const int width = (p.rank + RC - 1) / RC * RC;  // ranks in whole passes
  float *part = red + max(red_floats<RC>(), (uint32_t)ROWS * (width + 4));  // [ROWS][width]
  grid_wait();
  grid_dependents();
  Tile tile;
  // (the whole cluster has one tile)
  if (!find_tile(p, blockIdx.x / CTAS, plan, rows, blockIdx.x == 0, tile)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // h = s A x: this CTA's eighth of k, in groups of 32 that its warps take in turn
  if (tile.id >= 0) {
    const T *a = static_cast<const T *>(p.a) + (uint64_t)tile.id * p.rank * p.k;
    const float *x0 = p.x + (uint64_t)rows[g] * p.k, *x1 = p.x + (uint64_t)rows[g + 8] * p.k;
    const int groups = (p.k + 31) / 32, per = (groups + CTAS - 1) / CTAS;
    const int g0 = min(groups, cta * per), g1 = min(groups, g0 + per);
    for (int r0 = 0; r0 < p.rank; r0 += RC) {
      float acc[RC / 8][4];
#pragma unroll
      for (int n = 0; n < RC / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
      for (int q = g0 + warp; q < g1; q += WARPS) {
        const int k0 = q * 32 + t * 8, left = p.k - k0;  // this lane's 8 values: K of four MMAs
        float v0[8], v1[8];
        load_values<8>(x0 + k0, left, p.wide_x, v0);
        load_values<8>(x1 + k0, left, p.wide_x, v1);
        uint32_t hi[4][4], lo[4][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          split(v0[2 * s], hi[s][0], lo[s][0]);
          split(v1[2 * s], hi[s][1], lo[s][1]);
          split(v0[2 * s + 1], hi[s][2], lo[s][2]);
          split(v1[2 * s + 1], hi[s][3], lo[s][3]);
        }
#pragma unroll
        for (int n = 0; n < RC / 8; ++n) {
          const int r = r0 + n * 8 + g;
          if (r0 + n * 8 >= p.rank) break;
          float w[8];
          load_values<8>(a + (uint64_t)min(r, p.rank - 1) * p.k + k0, r < p.rank ? left : 0, p.wide_a, w);
#pragma unroll
          for (int s = 0; s < 4; ++s) multiply<T>(acc[n], hi[s], lo[s], w[2 * s], w[2 * s + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < RC / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[(warp * ROWS + g + 8 * (i >> 1)) * (RC + 4) + n * 8 + 2 * t + (i & 1)] = acc[n][i];
      __syncthreads();
      for (int i = threadIdx.x; i < ROWS * RC; i += 32 * WARPS) {
        const int row = i / RC, c = i % RC;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += red[(w * ROWS + row) * (RC + 4) + c];
        part[row * width + r0 + c] = s;
      }
      __syncthreads();
    }
    cluster.sync();
    // the whole h, summed over the CTAs in order, in `red` ([ROWS][width + 4])
    const float scale = p.scales ? p.scales[tile.id] : 1.f;
    for (int i = threadIdx.x; i < ROWS * width; i += 32 * WARPS) {
      float v[CTAS], s = 0.f;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) v[c] = cluster.map_shared_rank(part, c)[i];
#pragma unroll
      for (int c = 0; c < CTAS; ++c) s += v[c];
      red[i / width * (width + 4) + i % width] = s * scale;
    }
    __syncthreads();
    cluster.barrier_arrive();  // (waited for before this CTA's part may go)
  }

  // y = base + B h: blocks of 32 outputs.  A warp's four MMA column blocks are
  // interleaved so that a lane ends up with 8 neighbouring outputs of a row.
  constexpr int PER = RC / 4, STEPS = RC / 8;
  const T *b = static_cast<const T *>(p.b) + (uint64_t)max(tile.id, 0) * p.n * p.rank;
  uint32_t hi[STEPS][4], lo[STEPS][4];
  auto load_h = [&](int r0) {
    const float *h0 = red + g * (width + 4) + r0 + t * PER, *h1 = h0 + 8 * (width + 4);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      split(h0[2 * s], hi[s][0], lo[s][0]);
      split(h1[2 * s], hi[s][1], lo[s][1]);
      split(h0[2 * s + 1], hi[s][2], lo[s][2]);
      split(h1[2 * s + 1], hi[s][3], lo[s][3]);
    }
  };
  if (tile.id >= 0 && p.rank <= RC) load_h(0);
  for (int c0 = (cta * WARPS + warp) * COLS; c0 < p.n; c0 += CTAS * WARPS * COLS) {
    // lane (g, t) ends with rows g and g + 8, outputs c0 + 8 t .. + 7
    const int c = c0 + 8 * t;
    const bool wide = p.wide_y && c + 8 <= p.n;
    float4 old[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (wide && p.base && g + 8 * h < tile.len)
          old[h][q] = *reinterpret_cast<const float4 *>(p.base + (uint64_t)rows[g + 8 * h] * p.n + c + 4 * q);
        else old[h][q] = make_float4(0.f, 0.f, 0.f, 0.f);
    float acc[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    if (tile.id >= 0)
      for (int r0 = 0; r0 < p.rank; r0 += RC) {
        if (p.rank > RC) load_h(r0);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          // MMA column g of block n: the outputs 8 (g / 2) + 2 n + g % 2
          const int col = c0 + 8 * (g >> 1) + 2 * n + (g & 1);
          float w[PER];
          load_values<PER>(b + (uint64_t)min(col, p.n - 1) * p.rank + r0 + t * PER,
                           col < p.n ? p.rank - r0 - t * PER : 0, p.wide_b, w);
#pragma unroll
          for (int s = 0; s < STEPS; ++s) multiply<T>(acc[n], hi[s], lo[s], w[2 * s], w[2 * s + 1]);
        }
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = g + 8 * h;
      if (row >= tile.len || c >= p.n) continue;
      const uint64_t at = (uint64_t)rows[row] * p.n + c;
      float v[8];
#pragma unroll
      for (int n = 0; n < 4; ++n) v[2 * n] = acc[n][2 * h], v[2 * n + 1] = acc[n][2 * h + 1];
      if (wide) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 s = old[h][q];
          *reinterpret_cast<float4 *>(p.y + at + 4 * q) =
              tile.id < 0 ? s
                          : make_float4(s.x + v[4 * q], s.y + v[4 * q + 1], s.z + v[4 * q + 2], s.w + v[4 * q + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.n) {
            const float s = p.base ? p.base[at + i] : 0.f;
            p.y[at + i] = tile.id < 0 ? s : s + v[i];
          }
      }
    }
  }
  if (tile.id >= 0) cluster.barrier_wait();
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The most tiles m rows can make.
uint64_t tile_bound(uint64_t m, uint64_t count) {
  // an adapter's last tile may be short; above the sort's buckets neighbours may
  // alternate
  const uint64_t most = count < BUCKETS - 1 || m <= INLINE_ROWS ? m / ROWS + count + 1 : m;
  return most < m ? most : m;
}

// The sort's scratch (rows up to INLINE_ROWS need none of it).
struct Scratch {
  uint64_t order, tiles, ntiles, total;
  Scratch(const mgb_adapters &ad, uint64_t m) {
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
      const uint64_t r = at;
      at += (bytes + 127) / 128 * 128;
      return r;
    };
    const uint64_t planned = m > INLINE_ROWS ? m : 0;
    order = take(planned * 4);
    tiles = take(planned ? tile_bound(m, ad.count) * sizeof(Tile) : 0);
    ntiles = take(4);
    total = at;
  }
};

cudaError_t launch_chained(void (*kern)(Params), unsigned grid, int threads, uint32_t smem,
                           cudaStream_t stream, const Params &p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, int RC>
cudaError_t launch_rc(const Params &p, unsigned tiles, cudaStream_t stream) {
  const uint32_t width = (uint32_t)ceil_div(p.rank, RC) * RC;
  const uint32_t whole = ROWS * (width + 4);
  const uint32_t smem = ((red_floats<RC>() > whole ? red_floats<RC>() : whole) + ROWS * width) * 4;
  auto *kern = mgb_adapter_kernel<T, RC>;
  if (RC == 64) {  // the others stay below what needs no opt-in
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(kern, tiles * CTAS, 32 * WARPS, smem, stream, p);
}

template <typename T>
cudaError_t launch_t(const Params &p, unsigned tiles, cudaStream_t stream) {
  return p.rank <= 16   ? launch_rc<T, 16>(p, tiles, stream)
         : p.rank <= 32 ? launch_rc<T, 32>(p, tiles, stream)
                        : launch_rc<T, 64>(p, tiles, stream);
}

}  // namespace

uint64_t adapters_scratch_bytes(const mgb_adapters &ad, uint64_t m) {
  return m ? Scratch(ad, m).total : 0;
}

cudaError_t launch_adapters(const mgb_adapters &ad, const float *ids, const float *x, uint64_t m,
                            const float *base, float *y, uint32_t *bad, void *workspace,
                            cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (bad) e = cudaMemsetAsync(bad, 0xFF, sizeof(uint32_t), stream);
  if (e != cudaSuccess || !m) return e;
  Params p = {};
  p.a = ad.a;
  p.b = ad.b;
  p.scales = ad.scales;
  p.ids = ids;
  p.x = x;
  p.base = base;
  p.y = y;
  p.bad = bad;
  p.count = ad.count;
  p.m = (int)m;
  p.k = (int)ad.k;
  p.n = (int)ad.n;
  p.rank = (int)ad.rank;
  const Scratch s(ad, m);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.order = reinterpret_cast<int32_t *>(ws + s.order);
  p.tiles = reinterpret_cast<Tile *>(ws + s.tiles);
  p.ntiles = reinterpret_cast<int32_t *>(ws + s.ntiles);
  const uint64_t per = ad.dtype == MGB_DTYPE_F32 ? 4 : 8;  // values in 16 bytes
  p.wide_a = aligned16(ad.a) && ad.k % per == 0;
  p.wide_b = aligned16(ad.b) && ad.rank % per == 0;
  p.wide_x = aligned16(x) && ad.k % 4 == 0;
  p.wide_y = aligned16(y) && aligned16(base) && ad.n % 4 == 0;
  if (m > INLINE_ROWS) {
    e = launch_chained(mgb_adapter_plan_kernel, 1, 1024, 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  const unsigned tiles = (unsigned)tile_bound(m, ad.count);
  if (ad.dtype == MGB_DTYPE_F32) return launch_t<float>(p, tiles, stream);
  if (ad.dtype == MGB_DTYPE_F16) return launch_t<__half>(p, tiles, stream);
  return launch_t<__nv_bfloat16>(p, tiles, stream);
}

}  // namespace mgb
