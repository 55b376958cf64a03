// Low-rank adapters of many requests beside a shared projection:
//   y[r] = base[r] + s_a * (x[r] A_a^T) B_a^T,  a = ids[r],
// in two products: h[r] = s_a * A_a x[r] (rank values a row), y[r] = base[r] +
// B_a h[r].  Up to 128 rows, where launches count, one launch does both: a
// cluster takes one group of rows, each of its CTAs a slice of k for h, which
// they exchange through distributed shared memory, and then a slice of the
// outputs.  More rows take three chained launches (grouping, h, y) and hand h over
// through global memory: at 64 rows a group the exchange of 8 CTAs' parts by
// remote reads of shared memory alone took 47 us of 187 (2,048 rows, rank 64).
//
// Rows are grouped by adapter into tiles of up to 64, so that an adapter is read
// once for its rows whatever their order, and one row alone costs no more than
// its adapter's bytes.  16 rows are the M of mma.sync m16n8k8 (tf32 operands, f32
// accumulation); tiles of up to four rows take plain f32 multiply-adds.  The
// products are bound by the adapters' bytes or, with many rows, by base and y: rank
// operations a value, far from what tcgen05 is for.
//
// Measured on the device (floors at the copy's rate): one row, k = n = 4,096, rank 16,
// 5.8 us, a chain of the plan, A, the exchange and B; 64 rows of some 40 adapters, n =
// 14,336, 18.6 us (4.7), of which B takes 5 to 7 us at nine warps an SM (with the tensor
// cores' tiles 29.1 us, at 300 instructions a block of 32 outputs); 2,048 rows of rank
// 64, bf16 94 us (42), f16 160, f32 187: in bf16 grouping 6, h 22, y 66, which waits for
// base a block ahead and for the tensor cores (two blocks ahead: the same time).
//
// f32 accuracy from tf32: x and h are held as hi + lo, two tf32 terms (22 bits);
// f16 factors are tf32 numbers as they are, f32 factors are split too.  Beside bf16
// factors x and h are three bf16 terms, of m16n8k16: a quarter fewer MMAs, and no
// factor is converted (2,048 rows 102 us instead of 107 when that came).
// The order of a product's K is free, so a lane takes runs of neighbouring
// values of its row: every load is 16 bytes where the buffers allow it.
#include <cooperative_groups.h>

#include <atomic>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace mgb {
namespace {

namespace cg = cooperative_groups;

constexpr int M = 16;             // rows of an MMA
constexpr int MOST_ROWS = 64;     // of a tile
constexpr int INLINE_ROWS = 128;  // up to here every CTA plans for itself
constexpr int BUCKETS = 4096;     // of the planning kernel's sort
constexpr int MOST_CTAS = 8;      // of a cluster
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
  float *y, *h;      // h: [splits][m, sorted][h_width] (m > INLINE_ROWS)
  int32_t *order;    // [m]: the rows by adapter (m > INLINE_ROWS)
  Tile *tiles;       // and their tiles
  int32_t *ntiles;
  uint32_t *bad;
  uint64_t count;
  int m, k, n, rank;
  int tile_rows;     // rows of a tile: 16, 32 or 64
  int splits;        // slices of k (the CTAs of a cluster, or of the grid)
  bool wide_a, wide_b, wide_x, wide_y;  // 16-byte loads are aligned
  bool early;        // B's ring and the parts of h do not share their place
};

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- grouping ------------------------------------------------------------------------------

// Shared memory of a CTA that plans for itself.
struct SmallPlan {
  alignas(16) int id[INLINE_ROWS];
  int16_t order[INLINE_ROWS];
  Tile tiles[INLINE_ROWS];
  uint32_t heads[INLINE_ROWS / 32];  // the positions at which tiles start
};

// Rows sorted by (id, row), tiles of up to tile_rows rows of one id; returns their
// number.
__device__ __forceinline__ int plan_small(const Params &p, SmallPlan &s, bool report) {
  if (threadIdx.x < INLINE_ROWS) {
    const int i = threadIdx.x;
    int id = INT_MAX;
    if (i < p.m) {
      id = adapter_of(p.ids[i], p.count);
      if (id == -2) {
        if (report && p.bad) atomicMin(p.bad, (uint32_t)i);
        id = -1;
      }
    }
    s.id[i] = id;
    if (i < INLINE_ROWS / 32) s.heads[i] = 0;
  }
  __syncthreads();
  // two threads a row, four where that is all of them
  const int several = p.m <= 64 ? 4 : 2, i = threadIdx.x / several, sub = threadIdx.x % several;
  static_assert(32 * WARPS == 2 * INLINE_ROWS, "two threads a row");
  const int id = s.id[i];
  int pos = 0, nth = 0, same = 0;
  if (i < p.m)
    for (int j0 = 4 * sub; j0 < p.m; j0 += 4 * several) {
      const int4 four = *reinterpret_cast<const int4 *>(s.id + j0);
      const int o[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool before = o[c] == id && j0 + c < i;
        pos += o[c] < id || before;
        nth += before;
        same += o[c] == id;
      }
    }
  for (int d = 1; d < several; d <<= 1) {
    pos += __shfl_xor_sync(0xffffffffu, pos, d);
    nth += __shfl_xor_sync(0xffffffffu, nth, d);
    same += __shfl_xor_sync(0xffffffffu, same, d);
  }
  const bool row = i < p.m && sub == 0, head = row && nth % p.tile_rows == 0;
  if (row) s.order[pos] = (int16_t)i;
  if (head) atomicOr(&s.heads[pos >> 5], 1u << (pos & 31));
  __syncthreads();
  int before = 0, all = 0;  // tiles that start earlier; tiles
#pragma unroll
  for (int w = 0; w < INLINE_ROWS / 32; ++w) {
    const uint32_t h = s.heads[w];
    all += __popc(h);
    before += __popc(w < pos >> 5 ? h : w == pos >> 5 ? h & ((1u << (pos & 31)) - 1) : 0u);
  }
  if (head) s.tiles[before] = Tile{pos, min(p.tile_rows, same - nth), id};
  __syncthreads();
  return all;
}

__device__ __forceinline__ int warp_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Exclusive sum over 1,024 threads; warp_sums [32].
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = warp_scan(v);
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  const int sums = warp_scan(warp_sums[lane]);
  total = __shfl_sync(0xffffffffu, sums, 31);
  const int before = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
  return (warp ? before : 0) + s - v;
}

// One CTA: rows by bucket (the adapter, modulo 4,095; the last bucket holds the
// rows without one), in row order within a bucket (where a row lands decides in which
// order its sums are taken), then tiles of up to tile_rows neighbours of one adapter.
// Up to CACHED rows in shared memory, by two stable passes of 6 bits: every warp
// counts its stretch of the rows and then places it, its digits' places known from a
// scan over (digit, warp).  (2,048 rows took 12 us, now 6, with the warps placing their
// rows one after the other, which more than CACHED rows still do.)
constexpr int CACHED = 24576;
// Dynamic shared memory: the ids by row and the rows after each pass; not cached: the
// buckets.
inline uint32_t plan_bytes(uint64_t m) { return m <= CACHED ? (uint32_t)(m + 1) / 2 * 16 : BUCKETS * 4; }
__global__ void __launch_bounds__(1024) mgb_adapter_plan_kernel(const Params p) {
  extern __shared__ __align__(16) int ids[];
  const int even = (p.m + 1) & ~1;
  uint16_t *half = reinterpret_cast<uint16_t *>(ids + even), *sorted = half + even;
  __shared__ int counts[64 * 32];                  // [digit][warp]
  __shared__ int sums[32], s_carry[2];
  static_assert(BUCKETS == 64 * 64 && CACHED < 65536, "two digits; rows in 16 bits");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_wait();
  grid_dependents();
  const bool cached = p.m <= CACHED;
  auto bucket = [&](int id) { return id < 0 ? BUCKETS - 1 : id % (BUCKETS - 1); };
  if (cached) {
    for (int r = threadIdx.x; r < p.m; r += 1024) {
      int id = adapter_of(p.ids[r], p.count);
      if (id == -2) {
        if (p.bad) atomicMin(p.bad, (uint32_t)r);
        id = -1;
      }
      ids[r] = id;
    }
    const int per = ((p.m + 31) / 32 + 31) & ~31, i0 = warp * per, i1 = min(p.m, i0 + per);
    for (int shift = 0; shift < 12; shift += 6) {
      const uint16_t *from = shift ? half : nullptr;  // (first: the rows as they are)
      uint16_t *to = shift ? sorted : half;
      counts[threadIdx.x] = counts[threadIdx.x + 1024] = 0;
      __syncthreads();
      for (int place = 0; place < 2; ++place) {
        for (int i = i0 + lane; i - lane < i1; i += 32) {
          const int r = i < i1 ? from ? from[i] : i : -1;
          const int d = r < 0 ? 64 : bucket(ids[r]) >> shift & 63;
          const uint32_t same = __match_any_sync(0xffffffffu, d);
          int *at = counts + d * 32 + warp;  // this warp's own
          if (place && r >= 0) to[*at + __popc(same & ((1u << lane) - 1))] = (uint16_t)r;
          __syncwarp();
          if (r >= 0 && (same >> lane) == 1u) *at += __popc(same);  // the last of its digit
          __syncwarp();
        }
        __syncthreads();
        if (place) break;
        const int c0 = counts[2 * threadIdx.x], c1 = counts[2 * threadIdx.x + 1];
        int total;
        const int s = block_scan(c0 + c1, sums, total);
        counts[2 * threadIdx.x] = s;
        counts[2 * threadIdx.x + 1] = s + c0;
        __syncthreads();
      }
    }
  } else {
    int *at = ids;
    for (int b = threadIdx.x; b < BUCKETS; b += 1024) at[b] = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < p.m; r += 1024) {
      const int id = adapter_of(p.ids[r], p.count);
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
    for (int r0 = 0; r0 < p.m; r0 += 1024) {
      const int r = r0 + threadIdx.x;
      const int b = r < p.m ? bucket(adapter_of(p.ids[r], p.count)) : BUCKETS;
      const uint32_t same = __match_any_sync(0xffffffffu, b);
      for (int w = 0; w < 32 && r0 + 32 * w < p.m; ++w) {
        if (warp == w) {  // (the whole warp)
          const int i = r < p.m ? at[b] + __popc(same & ((1u << lane) - 1)) : 0;
          __syncwarp();
          if (r < p.m) {
            p.order[i] = r;
            if ((same >> lane) == 1u) at[b] = i + 1;  // the last of its bucket
          }
        }
        __syncthreads();
      }
    }
  }
  auto id_at = [&](int i) {
    return cached ? ids[sorted[i]] : max(adapter_of(p.ids[p.order[i]], p.count), -1);
  };
  // run heads, then tile heads (every tile_rows-th row of a run)
  if (threadIdx.x == 0) s_carry[0] = 0, s_carry[1] = 0;
  __syncthreads();
  for (int p0 = 0; p0 < p.m; p0 += 1024) {
    const int i = p0 + threadIdx.x;
    int id = -3, prev = -3;
    if (i < p.m) {
      id = id_at(i);
      if (i) prev = id_at(i - 1);
      if (cached) p.order[i] = sorted[i];
    }
    const bool head = i < p.m && id != prev;
    // the run's start: an inclusive maximum of the head positions
    int start = head ? i : -1;
    auto warp_max = [&](int v) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, u);
      }
      return v;
    };
    start = warp_max(start);
    __syncthreads();
    if (lane == 31) sums[warp] = start;
    __syncthreads();
    const int warps = warp_max(sums[lane]), before = __shfl_sync(0xffffffffu, warps, max(warp - 1, 0));
    start = max(max(start, warp ? before : -1), s_carry[0]);
    const bool tile = i < p.m && (i - start) % p.tile_rows == 0;
    int total;
    const int t = s_carry[1] + block_scan(tile, sums, total);
    __syncthreads();
    if (threadIdx.x == 1023) s_carry[0] = start;
    if (threadIdx.x == 0) s_carry[1] += total;
    if (tile) {
      p.tiles[t] = Tile{i, 0, id};
      if (cached) half[t] = (uint16_t)i;
    }
    __syncthreads();
  }
  const int n = s_carry[1];
  if (threadIdx.x == 0) *p.ntiles = n;
  for (int t = threadIdx.x; t < n; t += 1024) {
    if (cached) p.tiles[t].len = (t + 1 < n ? (int)half[t + 1] : p.m) - half[t];
    else p.tiles[t].len = (t + 1 < n ? p.tiles[t + 1].start : p.m) - p.tiles[t].start;
  }
}

// The CTA's tile and its rows (absent ones repeat the first); false: no such tile.  Up
// to INLINE_ROWS rows, by a plan of its own, and from the grouped rows.
__device__ __forceinline__ bool plan_tile(const Params &p, int t, SmallPlan &plan, int (&rows)[MOST_ROWS],
                                          bool report, Tile &tile) {
  if (t >= plan_small(p, plan, report)) return false;
  tile = plan.tiles[t];
  if (threadIdx.x < MOST_ROWS) rows[threadIdx.x] = plan.order[tile.start + (threadIdx.x < tile.len ? threadIdx.x : 0)];
  __syncthreads();
  return true;
}
__device__ __forceinline__ bool grouped_tile(const Params &p, int t, int (&rows)[MOST_ROWS], Tile &tile) {
  if (t >= *p.ntiles) return false;
  tile = p.tiles[t];
  if (threadIdx.x < MOST_ROWS) rows[threadIdx.x] = p.order[tile.start + (threadIdx.x < tile.len ? threadIdx.x : 0)];
  __syncthreads();
  return true;
}

// ---- operands --------------------------------------------------------------------------------

// Rounded to a term of an operand, infinities and what would round to one to the largest
// finite term of their sign: what is left of them is for the next term.  (An infinity
// here would leave NaN or one of the other sign.)  The conversion does it at no cost; a
// minimum and a maximum a term took 0.5 us of 100 (2,048 rows of rank 64).
__device__ __forceinline__ uint32_t tf32(float v) {
  uint32_t r;
  asm("cvt.rna.satfinite.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
  uint32_t r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
// v = hi + lo to 22 bits.  lo is cut where it could be rounded to half of that error: the
// largest value's rest would be rounded up, and the sum overflow.
__device__ __forceinline__ void split(float v, uint32_t &hi, uint32_t &lo) {
  hi = tf32(v);
  lo = __float_as_uint(v - __uint_as_float(hi)) & 0xFFFFE000u;
}
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += (hi + lo) * (b0, b1) for factors of type T, to 22 bits of each, in two parts.
// (lo times lo is up to 2^-22: without it 2,048 rows of f32 factors take 173 us, not 187,
// and a product is off by half more.)
template <typename T>
__device__ __forceinline__ void multiply_small(float (&c)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                               float b0, float b1) {
  if constexpr (sizeof(T) == 4) {
    uint32_t h0, h1, l0, l1;
    split(b0, h0, l0);
    split(b1, h1, l1);
    uint32_t finite[4];  // (an infinity, which lo carries, times a lower term may be NaN)
#pragma unroll
    for (int i = 0; i < 4; ++i) finite[i] = fabsf(__uint_as_float(lo[i])) <= FLT_MAX ? lo[i] : 0u;
    mma1688(c, finite, l0, l1);
    mma1688(c, lo, h0, h1);
    mma1688(c, hi, l0, l1);
  } else {
    mma1688(c, lo, __float_as_uint(b0), __float_as_uint(b1));
  }
}
template <typename T>
__device__ __forceinline__ void multiply_large(float (&c)[4], const uint32_t (&hi)[4], float b0, float b1) {
  if constexpr (sizeof(T) == 4) mma1688(c, hi, tf32(b0), tf32(b1));
  else mma1688(c, hi, __float_as_uint(b0), __float_as_uint(b1));
}
template <typename T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                         float b0, float b1) {
  multiply_small<T>(c, hi, lo, b0, b1);
  multiply_large<T>(c, hi, b0, b1);
}

// bf16 factors: K is 16, and the other operand's f32 values are three bf16 terms
// (24 bits).
template <typename T>
constexpr bool THREE = std::is_same<T, __nv_bfloat16>::value;
__device__ __forceinline__ void split3(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
  auto take = [&]() {
    const uint32_t r = bf16_pair(x, y);
    x -= __uint_as_float(r << 16);
    y -= __uint_as_float(r & 0xFFFF0000u);
    return r;
  };
  hi = take();
  mid = take();
  const __nv_bfloat162 rest = __floats2bfloat162_rn(x, y);
  lo = *reinterpret_cast<const uint32_t *>(&rest);
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// N neighbouring values in pairs as they are stored (16-bit types), or one by one.
template <typename T, int N>
struct Pairs {
  static constexpr int REGS = sizeof(T) == 4 ? N : N / 2;
  uint32_t r[REGS];
  __device__ __forceinline__ void load(const T *at, int left, bool wide) {
    if (wide && left >= N) {
      if constexpr (REGS >= 4) {
#pragma unroll
        for (int i = 0; i < REGS / 4; ++i) {
          const uint4 v = reinterpret_cast<const uint4 *>(at)[i];
          r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w;
        }
      } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(at);
        r[0] = v.x, r[1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < REGS; ++i) r[i] = 0;
      T *d = reinterpret_cast<T *>(r);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) d[i] = at[i];
    }
  }
  // values 2 s and 2 s + 1
  __device__ __forceinline__ float2 pair(int s) const {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(r[2 * s]), __uint_as_float(r[2 * s + 1]));
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return make_float2(__uint_as_float(r[s] << 16), __uint_as_float(r[s] & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&r[s]));
  }
};

// ---- the kernel --------------------------------------------------------------------------------

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// RC: ranks of a pass (a lane of the second product: RC / 4 neighbours, K of
// RC / 8 MMAs).  Shared memory: h as MMA operands (hi and lo, [rows / 16][ranks /
// 8][lane][4], or three terms of 16 ranks), then in turn this CTA's part of h ([rows][ranks + 4]) and, where
// the buffers allow 16-byte copies (WIDE), a ring of B's rows for every warp.
template <typename T, int RC>
struct Shared {
  static constexpr uint32_t ROW = RC * sizeof(T) + 16;  // neighbouring rows in different banks
  static constexpr uint32_t STAGE = COLS * ROW;
  // as many stages as two CTAs an SM leave room for (f32 factors: one)
  static constexpr int DEPTH = sizeof(T) == 4 || RC == 64 ? 2 : 96 / RC;
  static constexpr uint32_t RING = WARPS * DEPTH * STAGE;
};
__host__ __device__ inline int h_width(int rank, int rc) { return (rank + rc - 1) / rc * rc; }
template <typename T>
__host__ __device__ inline uint32_t h_bytes(int tile_rows, int width) {
  return tile_rows * width * (THREE<T> ? 6 : 8);
}
__host__ __device__ inline uint32_t part_bytes(int tile_rows, int width) {
  return tile_rows * (width + 4) * 4;
}

// part = A x over groups g0 .. g1 of 32 of k, by the whole CTA.  A warp takes one
// block of rows (of 1, 2 or 4) and every kparts-th group.
template <typename T, int RC>
__device__ __forceinline__ void shrink(const Params &p, const Tile &tile, const int (&rows)[MOST_ROWS],
                                       int g0, int g1, int width, float *part) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int mts = (tile.len + M - 1) / M, stride = width + 4;
  const int split_m = mts > 2 ? 4 : mts, kparts = WARPS / split_m;
  const int mt = warp % split_m, kp = warp / split_m;
  const T *a = static_cast<const T *>(p.a) + (uint64_t)tile.id * p.rank * p.k;
  const float *x0 = p.x + (uint64_t)rows[mt * M + g] * p.k, *x1 = p.x + (uint64_t)rows[mt * M + g + 8] * p.k;
  for (int r0 = 0; r0 < p.rank; r0 += RC) {
    float acc[RC / 8][4];
#pragma unroll
    for (int n = 0; n < RC / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    if (mt < mts)
      for (int q = g0 + kp; q < g1; q += kparts) {
        const int k0 = q * 32 + t * 8, left = p.k - k0;  // this lane's 8 values: K of four MMAs
        float v0[8], v1[8];
        Pairs<T, 8> w[RC / 8];
        load_values<8>(x0 + k0, left, p.wide_x, v0);
        load_values<8>(x1 + k0, left, p.wide_x, v1);
#pragma unroll
        for (int n = 0; n < RC / 8; ++n) {
          const int r = r0 + n * 8 + g;
          w[n].load(a + (uint64_t)min(r, p.rank - 1) * p.k + k0, r < p.rank ? left : 0, p.wide_a);
        }
        // A group's products in the tensor core, the small terms first, and its sum to the
        // others by f32 additions: the tensor core cuts its sums instead of rounding them
        // (a chain over all of k: 20,000 rows of k = 4,096 off by 7e-6 to 1.4e-5 of y, now 3e-7).
        if constexpr (THREE<T>) {
          uint32_t hi[2][4], mid[2][4], lo[2][4];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            split3(v0[4 * s], v0[4 * s + 1], hi[s][0], mid[s][0], lo[s][0]);
            split3(v1[4 * s], v1[4 * s + 1], hi[s][1], mid[s][1], lo[s][1]);
            split3(v0[4 * s + 2], v0[4 * s + 3], hi[s][2], mid[s][2], lo[s][2]);
            split3(v1[4 * s + 2], v1[4 * s + 3], hi[s][3], mid[s][3], lo[s][3]);
          }
#pragma unroll
          for (int n = 0; n < RC / 8; ++n) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 2; ++s) mma16816(c, lo[s], w[n].r[2 * s], w[n].r[2 * s + 1]);
#pragma unroll
            for (int s = 0; s < 2; ++s) mma16816(c, mid[s], w[n].r[2 * s], w[n].r[2 * s + 1]);
#pragma unroll
            for (int s = 0; s < 2; ++s) mma16816(c, hi[s], w[n].r[2 * s], w[n].r[2 * s + 1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] += c[i];
          }
        } else {
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
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const float2 v = w[n].pair(s);
              multiply_small<T>(c, hi[s], lo[s], v.x, v.y);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const float2 v = w[n].pair(s);
              multiply_large<T>(c, hi[s], v.x, v.y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] += c[i];
          }
        }
      }
    // the warps' sums, in order
    for (int k = 0; k < kparts; ++k) {
      if (kp == k && mt < mts)
#pragma unroll
        for (int n = 0; n < RC / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = r0 + n * 8 + 2 * t + (i & 1);
            float *at = part + (mt * M + g + 8 * (i >> 1)) * stride + r;
            // (behind the last rank 0, whatever x: infinities times zeros are none)
            *at = r >= p.rank ? 0.f : k ? *at + acc[n][i] : acc[n][i];
          }
      __syncthreads();
    }
  }
}

// Few rows (of an adapter of up to 64 ranks): plain f32 arithmetic, of which a tensor
// core's tile would leave most unused.  48 rows in tiles of 1, 2, 3 and 4 (k = 4,096, n =
// 8,192): rank 16 bf16 10.5, 8.6, 10.3 and 8.5 us, as MMAs 17.8, 12.6, 12.4 and 10.8;
// rank 64 f32 41.5, 25.9, 30.8 and 16.7, as MMAs 83, 50, 50 and 26.5.  More rows' partial
// sums would not fit a tile's shared memory.
constexpr int FEW = 4;
__device__ __forceinline__ bool few_rows(const Params &p, const Tile &tile) {
  return tile.len <= FEW && p.tile_rows == MOST_ROWS;
}

// shrink for few rows, two of them at a time.  A thread takes 4 neighbouring k of 16
// ranks; a warp's lanes hand one another halves of their sums until each has one.
template <typename T>
__device__ __forceinline__ void shrink_few(const Params &p, const Tile &tile, const int (&rows)[MOST_ROWS],
                                           int g0, int g1, int width, float *part) {
  constexpr int RB = 16, PAIR = 2;
  static_assert(FEW * (1 + WARPS) <= MOST_ROWS, "a part a warp");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stride = width + 4;
  const T *a = static_cast<const T *>(p.a) + (uint64_t)tile.id * p.rank * p.k;
  float *mine = part + (FEW + warp * FEW) * stride;
  const int end = min(p.k, g1 * 32);
  const bool wide = p.wide_a && p.wide_x;  // (k is a multiple of 4 then)
  for (int i0 = 0; i0 < tile.len; i0 += PAIR) {
    const float *x0 = p.x + (uint64_t)rows[i0] * p.k, *x1 = p.x + (uint64_t)rows[min(i0 + 1, tile.len - 1)] * p.k;
    for (int r0 = 0; r0 < width; r0 += RB) {
      float acc[PAIR][RB];
#pragma unroll
      for (int i = 0; i < PAIR; ++i)
#pragma unroll
        for (int r = 0; r < RB; ++r) acc[i][r] = 0.f;
      for (int k = g0 * 32 + threadIdx.x * 4; k < end; k += WARPS * 128) {
        Pairs<T, 4> w[RB];
        Pairs<float, 4> v[PAIR];
        if (wide) {  // (all loads before the first use)
#pragma unroll
          for (int r = 0; r < RB; ++r) w[r].load(a + (uint64_t)min(r0 + r, p.rank - 1) * p.k + k, 4, true);
          v[0].load(x0 + k, 4, true);
          v[1].load(x1 + k, 4, true);
        } else {
#pragma unroll
          for (int r = 0; r < RB; ++r)
            w[r].load(a + (uint64_t)min(r0 + r, p.rank - 1) * p.k + k, end - k, false);
          v[0].load(x0 + k, end - k, false);
          v[1].load(x1 + k, end - k, false);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float2 f = w[r].pair(s);
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
              const float2 u = v[i].pair(s);
              acc[i][r] = fmaf(f.y, u.y, fmaf(f.x, u.x, acc[i][r]));
            }
          }
      }
#pragma unroll
      for (int i = 0; i < PAIR; ++i) {
#pragma unroll
        for (int o = 16, half = RB / 2; half; o >>= 1, half >>= 1)
#pragma unroll
          for (int r = 0; r < half; ++r) {
            const float keep = lane & o ? acc[i][r + half] : acc[i][r];
            const float give = lane & o ? acc[i][r] : acc[i][r + half];
            acc[i][r] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
        const float s = acc[i][0] + __shfl_xor_sync(0xffffffffu, acc[i][0], 1);
        const int r = r0 + (lane >> 1);
        if ((lane & 1) == 0 && i0 + i < tile.len) mine[(i0 + i) * stride + r] = r < p.rank ? s : 0.f;
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < tile.len * width; e += 32 * WARPS) {
    const int at = e / width * stride + e % width;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += part[(FEW + w * FEW) * stride + at];
    part[at] = s;
  }
  __syncthreads();
}

// h of few rows, [rows][width].
template <typename F>
__device__ __forceinline__ void h_values(float *h, int len, int width, const F &sum) {
  for (int e = threadIdx.x; e < len * width / 2; e += 32 * WARPS) {
    const int row = e / (width / 2), r = e % (width / 2) * 2;
    *reinterpret_cast<float2 *>(h + row * width + r) = sum(row, r);
  }
}

// h as operands: lane (g, t) of step q RC / 8 + s multiplies ranks q RC + t RC / 4 +
// 2 s and the next (THREE: of step q RC / 16 + s, 4 s and the next three).
// sum(row, r): h of the tile's row at ranks r and r + 1.
template <typename T, int RC, typename F>
__device__ __forceinline__ void h_operands(uint4 *hs, int mts, int width, const F &sum) {
  constexpr int K = THREE<T> ? 16 : 8;
  const int steps = width / K;
  for (int i = threadIdx.x; i < mts * steps * 32; i += 32 * WARPS) {
    const int l = i & 31, step = (i >> 5) % steps, b = (i >> 5) / steps, row = b * M + (l >> 2);
    const int r = step / (RC / K) * RC + (l & 3) * (RC / 4) + K / 4 * (step % (RC / K));
    const float2 v0 = sum(row, r), v1 = sum(row + 8, r);
    if constexpr (THREE<T>) {
      const float2 v2 = sum(row, r + 2), v3 = sum(row + 8, r + 2);
      uint4 hi, mid, lo;
      split3(v0.x, v0.y, hi.x, mid.x, lo.x);
      split3(v1.x, v1.y, hi.y, mid.y, lo.y);
      split3(v2.x, v2.y, hi.z, mid.z, lo.z);
      split3(v3.x, v3.y, hi.w, mid.w, lo.w);
      uint4 *at = hs + (b * steps + step) * 96 + l;
      at[0] = hi, at[32] = mid, at[64] = lo;
    } else {
      uint4 hi, lo;
      split(v0.x, hi.x, lo.x);
      split(v1.x, hi.y, lo.y);
      split(v0.y, hi.z, lo.z);
      split(v1.y, hi.w, lo.w);
      uint4 *at = hs + (b * steps + step) * 64 + l;
      at[0] = hi, at[32] = lo;
    }
  }
}

// A warp's copies of B where 16-byte copies are aligned (WIDE): its blocks of 32
// outputs first, first + step, ..., a pass of RC ranks of a block a stage, DEPTH
// ahead.
template <typename T, int RC, bool WIDE>
struct Copies {
  using SM = Shared<T, RC>;
  static constexpr int CHUNKS = RC * sizeof(T) / 16;
  static constexpr int ROWS = 32 / CHUNKS;  // of B at a time: a lane copies chunk lane % CHUNKS of one
  const T *b;
  uint8_t *ring;
  int n, last, next, passes;
  int fc, fp = 0, fslot = 0;
  const uint8_t *src;                         // this lane's first chunk of the stage to be fetched
  uint32_t dst, rows_step, block_step, have;  // bytes; have: of a row from the lane's chunk on
  __device__ __forceinline__ Copies(const Params &p, const Tile &tile, int width, uint8_t *rings, int first,
                                    int end, int step)
      : b(static_cast<const T *>(p.b) + (uint64_t)max(tile.id, 0) * p.n * p.rank),
        ring(rings + (threadIdx.x >> 5) * SM::DEPTH * SM::STAGE), n(p.n), last(min(p.n, end * COLS)),
        next(step * COLS), passes(tile.id >= 0 ? width / RC : 0), fc(first * COLS) {
    const int lane = threadIdx.x & 31, row = lane / CHUNKS, c = lane % CHUNKS;
    const uint32_t row_bytes = (uint32_t)p.rank * sizeof(T);
    src = reinterpret_cast<const uint8_t *>(b) + (uint64_t)(fc + row) * row_bytes + c * 16;
    dst = smem_u32(ring) + row * SM::ROW + c * 16;
    rows_step = ROWS * row_bytes;
    block_step = (uint32_t)next * row_bytes;
    have = max((int)row_bytes - c * 16, 0);
  }
  __device__ __forceinline__ void fetch() {
    if (fc < last && passes) {
      const int left = n - fc - (threadIdx.x & 31) / CHUNKS;
      const bool in = fp * RC * (int)sizeof(T) < (int)have;  // (zeros behind the last rank)
      const uint8_t *from = in ? src : reinterpret_cast<const uint8_t *>(b);
      const uint32_t step = in ? rows_step : 0;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i)
        if (i * ROWS < left)
          cp_async16(dst + fslot * SM::STAGE + i * ROWS * SM::ROW, from + (uint64_t)(uint32_t)i * step, in ? 16 : 0);
      fslot = fslot + 1 == SM::DEPTH ? 0 : fslot + 1;
      src += RC * sizeof(T);
      if (++fp == passes) {
        src += (uint64_t)block_step - (uint32_t)(passes * RC * (int)sizeof(T));
        fp = 0;
        fc += next;
      }
    }
    cp_async_commit();
  }
  __device__ __forceinline__ void start() {
    if (WIDE)
#pragma unroll
      for (int i = 0; i < SM::DEPTH; ++i) fetch();
  }
};

// y = base + B h for few rows of up to RC ranks: a lane an output, two blocks of 32 of
// the warp together, whose part of base is loaded two blocks ahead.  h: [rows][width].
template <typename T, int RC, bool WIDE>
__device__ __forceinline__ void expand_few(const Params &p, const Tile &tile, const int (&rows)[MOST_ROWS],
                                           const float *h, int width, int first, Copies<T, RC, WIDE> &copies) {
  using SM = Shared<T, RC>;
  constexpr int TWO = 2, RB = 16;
  const int lane = threadIdx.x & 31, last = copies.last;
  const bool adapted = copies.passes != 0;
  uint64_t at[FEW];  // this lane's first output of a row
#pragma unroll
  for (int i = 0; i < FEW; ++i) at[i] = (uint64_t)rows[i] * p.n + lane;
  struct Old {
    float v[TWO][FEW];
  };
  auto load_old = [&](Old &o, int c0) {
    const bool in[TWO] = {p.base && c0 < last && c0 + lane < p.n,
                          p.base && c0 + copies.next < last && c0 + copies.next + lane < p.n};
#pragma unroll
    for (int i = 0; i < FEW; ++i) {
      if (i >= tile.len) break;
#pragma unroll
      for (int u = 0; u < TWO; ++u) o.v[u][i] = in[u] ? p.base[at[i] + c0 + u * copies.next] : 0.f;
    }
  };
  Old next;
  load_old(next, first);
  int slot = 0;
  for (int c0 = first; c0 < last; c0 += TWO * copies.next) {
    const Old old = next;
    load_old(next, c0 + TWO * copies.next);
    float acc[TWO][FEW];
#pragma unroll
    for (int u = 0; u < TWO; ++u)
#pragma unroll
      for (int i = 0; i < FEW; ++i) acc[u][i] = 0.f;
    if (adapted) {
      if (WIDE) {
        cp_async_wait<SM::DEPTH - TWO>();
        __syncwarp();
      }
#pragma unroll
      for (int r0 = 0; r0 < RC; r0 += RB) {
        if (r0 >= p.rank) break;
        Pairs<T, RB> w[TWO];
#pragma unroll
        for (int u = 0; u < TWO; ++u) {
          if (WIDE) {
            const int at = slot + u >= SM::DEPTH ? slot + u - SM::DEPTH : slot + u;
            w[u].load(reinterpret_cast<const T *>(copies.ring + at * SM::STAGE + lane * SM::ROW) + r0, RB, true);
          } else {
            w[u].load(copies.b + (uint64_t)min(c0 + u * copies.next + lane, p.n - 1) * p.rank + r0, p.rank - r0,
                      false);
          }
        }
#pragma unroll
        for (int i = 0; i < FEW; ++i) {
          if (i >= tile.len) break;
#pragma unroll
          for (int s = 0; s < RB / 2; ++s) {
            const float2 v = *reinterpret_cast<const float2 *>(h + i * width + r0 + 2 * s);
#pragma unroll
            for (int u = 0; u < TWO; ++u) {
              const float2 f = w[u].pair(s);
              acc[u][i] = fmaf(f.y, v.y, fmaf(f.x, v.x, acc[u][i]));
            }
          }
        }
      }
      if (WIDE) {
        __syncwarp();
        slot = slot + TWO >= SM::DEPTH ? slot + TWO - SM::DEPTH : slot + TWO;
        copies.fetch();
        copies.fetch();
      }
    }
    const bool in[TWO] = {c0 + lane < p.n, c0 + copies.next < last && c0 + copies.next + lane < p.n};
#pragma unroll
    for (int i = 0; i < FEW; ++i) {
      if (i >= tile.len) break;
#pragma unroll
      for (int u = 0; u < TWO; ++u)
        if (in[u])
          p.y[at[i] + c0 + u * copies.next] =
              !adapted ? old.v[u][i] : p.base ? old.v[u][i] + acc[u][i] : acc[u][i];
    }
  }
  if (WIDE) cp_async_wait<0>();
}

// y = base + B h for the copies' blocks of 32 outputs, which have been started.  An
// MMA's four column blocks are interleaved so that a lane ends up with 8
// neighbouring outputs of a row: column g of block n is output 8 (g / 2) + 2 n +
// g % 2.
template <typename T, int RC, bool WIDE>
__device__ __forceinline__ void expand(const Params &p, const Tile &tile, const int (&rows)[MOST_ROWS],
                                       const uint4 *hs, int width, int first, Copies<T, RC, WIDE> &copies) {
  using SM = Shared<T, RC>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int mts = (tile.len + M - 1) / M;
  constexpr int PER = RC / 4, STEPS = RC / (THREE<T> ? 16 : 8);
  const int NEXT = copies.next, last = copies.last;
  const T *b = copies.b;
  const uint8_t *ring = copies.ring;
  const int passes = copies.passes, steps = width / (THREE<T> ? 16 : 8);
  int slot = 0;
  // base (after the first pass: y) of lane (g, t)'s outputs c .. c + 7, c = c0 + 8 t,
  // of rows g and g + 8 of a block of rows; loaded one block ahead
  struct Old {
    float v[2][8];
  };
  auto load_old = [&](Old &o, int c0, int q, int mt) {
    const float *from = q ? p.y : p.base;
    const int c = c0 + 8 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = mt * M + g + 8 * h;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[h][i] = 0.f;
      if (!from || row >= tile.len) continue;
      const float *at = from + (uint64_t)rows[row] * p.n + c;
      if (p.wide_y && c + 8 <= p.n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 v = *reinterpret_cast<const float4 *>(at + 4 * i);
          o.v[h][4 * i] = v.x, o.v[h][4 * i + 1] = v.y, o.v[h][4 * i + 2] = v.z, o.v[h][4 * i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.n) o.v[h][i] = at[i];
      }
    }
  };
  Old next;
  int c0 = first;
  if (c0 < last) load_old(next, c0, 0, 0);
  for (; c0 < last; c0 += NEXT) {
    const int c = c0 + 8 * t;
    const bool wide = p.wide_y && c + 8 <= p.n;
    for (int q = 0; q < max(passes, 1); ++q) {
      Pairs<T, PER> w[4];
      if (passes) {
        if (WIDE) {
          cp_async_wait<SM::DEPTH - 1>();
          __syncwarp();
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int col = 8 * (g >> 1) + 2 * n + (g & 1);
          if (WIDE)
            w[n].load(reinterpret_cast<const T *>(ring + slot * SM::STAGE + col * SM::ROW) + t * PER, PER, true);
          else
            w[n].load(b + (uint64_t)min(c0 + col, p.n - 1) * p.rank + q * RC + t * PER,
                      c0 + col < p.n ? p.rank - q * RC - t * PER : 0, p.wide_b);
        }
        if (WIDE) {
          __syncwarp();
          slot = slot + 1 == SM::DEPTH ? 0 : slot + 1;
          copies.fetch();
        }
      }
      const bool add = q || p.base;  // (more than one pass: the sums so far are in y)
      for (int mt = 0; mt < mts; ++mt) {
        const Old old = next;
        if (mt + 1 < mts) load_old(next, c0, q, mt + 1);
        else if (q + 1 < passes && mts > 1) load_old(next, c0, q + 1, 0);  // (one block: not written yet)
        else if (q + 1 >= passes && c0 + NEXT < last) load_old(next, c0 + NEXT, 0, 0);
        float acc[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
        if (passes)
#pragma unroll
          for (int s = 0; s < STEPS; ++s) {
            if constexpr (THREE<T>) {
              const uint4 *f = hs + (mt * steps + q * STEPS + s) * 96 + lane;
#pragma unroll
              for (int term = 2; term >= 0; --term) {
                const uint4 a = f[32 * term];
                const uint32_t v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) mma16816(acc[n], v, w[n].r[2 * s], w[n].r[2 * s + 1]);
              }
            } else {
              const uint4 *f = hs + (mt * steps + q * STEPS + s) * 64 + lane;
              const uint4 h0 = f[0], l0 = f[32];
              const uint32_t hi[4] = {h0.x, h0.y, h0.z, h0.w}, lo[4] = {l0.x, l0.y, l0.z, l0.w};
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                const float2 v = w[n].pair(s);
                multiply<T>(acc[n], hi, lo, v.x, v.y);
              }
            }
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (mt * M + g + 8 * h >= tile.len) continue;
          float v[8];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              v[2 * n + e] = !passes ? old.v[h][2 * n + e]
                             : add   ? old.v[h][2 * n + e] + acc[n][2 * h + e]
                                     : acc[n][2 * h + e];
          float *y = p.y + (uint64_t)rows[mt * M + g + 8 * h] * p.n + c;
          if (wide) {
            *reinterpret_cast<float4 *>(y) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(y + 4) = make_float4(v[4], v[5], v[6], v[7]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c + i < p.n) y[i] = v[i];
          }
        }
        if (mts == 1 && q + 1 < passes) load_old(next, c0, q + 1, 0);
      }
    }
  }
  if (WIDE) cp_async_wait<0>();
}

// Both products of one tile by a cluster of `splits` CTAs.
template <typename T, int RC, bool WIDE>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 4 ? 1 : 2) mgb_adapter_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ SmallPlan plan;
  __shared__ int rows[MOST_ROWS];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), ctas = p.splits, warp = threadIdx.x >> 5;
  const int width = h_width(p.rank, RC);
  uint4 *hs = reinterpret_cast<uint4 *>(smem);
  float *part = reinterpret_cast<float *>(smem + h_bytes<T>(p.tile_rows, width));
  grid_wait();
  grid_dependents();
  Tile tile;
  // (the whole cluster has one tile)
  if (!plan_tile(p, blockIdx.x / ctas, plan, rows, blockIdx.x == 0, tile)) return;
  const bool few = few_rows(p, tile);
  // B's first copies are under way while h is taken, where shared memory holds both
  const int first = cta * WARPS + warp;
  Copies<T, RC, WIDE> copies(p, tile, width,
                             smem + h_bytes<T>(p.tile_rows, width) + (p.early ? part_bytes(p.tile_rows, width) : 0),
                             first, (p.n + COLS - 1) / COLS, ctas * WARPS);
  if (p.early) copies.start();
  if (tile.id >= 0) {
    const int groups = (p.k + 31) / 32, per = (groups + ctas - 1) / ctas;
    const int g0 = min(groups, cta * per), g1 = min(groups, g0 + per);
    if (few) shrink_few<T>(p, tile, rows, g0, g1, width, part);
    else shrink<T, RC>(p, tile, rows, g0, g1, width, part);
    cluster.sync();
    const float scale = p.scales ? p.scales[tile.id] : 1.f;
    auto sum = [&](int row, int r) {
      float2 s = make_float2(0.f, 0.f);
      if (row >= tile.len) return s;
#pragma unroll 4
      for (int c = 0; c < ctas; ++c) {  // in order
        const float2 u = *reinterpret_cast<const float2 *>(
            cluster.map_shared_rank(part + row * (width + 4) + r, c));
        s.x += u.x, s.y += u.y;
      }
      return make_float2(s.x * scale, s.y * scale);
    };
    if (few) h_values(reinterpret_cast<float *>(hs), tile.len, width, sum);
    else h_operands<T, RC>(hs, (tile.len + M - 1) / M, width, sum);
    cluster.sync();  // h is complete, and no CTA reads another's part any more
  }
  if (!p.early) copies.start();
  if (few) expand_few<T, RC, WIDE>(p, tile, rows, reinterpret_cast<float *>(hs), width, first * COLS, copies);
  else expand<T, RC, WIDE>(p, tile, rows, hs, width, first * COLS, copies);
}

// The two products apart, for grouped rows: CTA (slice of k, tile), and CTA
// (slice of the outputs, tile).
template <typename T, int RC>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 4 ? 1 : 2) mgb_adapter_h_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int rows[MOST_ROWS];
  const int width = h_width(p.rank, RC);
  float *part = reinterpret_cast<float *>(smem);
  grid_wait();
  grid_dependents();
  Tile tile;
  const int split = blockIdx.x % p.splits;
  if (!grouped_tile(p, blockIdx.x / p.splits, rows, tile) || tile.id < 0) return;
  const int groups = (p.k + 31) / 32, per = (groups + p.splits - 1) / p.splits;
  const int g0 = min(groups, split * per), g1 = min(groups, g0 + per);
  if (few_rows(p, tile)) shrink_few<T>(p, tile, rows, g0, g1, width, part);
  else shrink<T, RC>(p, tile, rows, g0, g1, width, part);
  const float scale = p.scales ? p.scales[tile.id] : 1.f;
  float *h = p.h + ((uint64_t)split * p.m + tile.start) * width;
  for (int i = threadIdx.x; i < tile.len * width; i += 32 * WARPS)
    h[i] = part[i / width * (width + 4) + i % width] * scale;
}
template <typename T, int RC, bool WIDE>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 4 ? 1 : 2)
    mgb_adapter_y_kernel(const Params p, int slices) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int rows[MOST_ROWS];
  const int width = h_width(p.rank, RC), warp = threadIdx.x >> 5;
  uint4 *hs = reinterpret_cast<uint4 *>(smem);
  grid_wait();
  grid_dependents();
  Tile tile;
  const int slice = blockIdx.x % slices;
  if (!grouped_tile(p, blockIdx.x / slices, rows, tile)) return;
  const bool few = few_rows(p, tile);
  if (tile.id >= 0) {
    auto sum = [&](int row, int r) {
      float2 s = make_float2(0.f, 0.f);
      if (row >= tile.len) return s;
      const float *at = p.h + (uint64_t)(tile.start + row) * width + r;
      for (int c = 0; c < p.splits; ++c) {  // in order
        const float2 u = *reinterpret_cast<const float2 *>(at + (uint64_t)c * p.m * width);
        s.x += u.x, s.y += u.y;
      }
      return s;
    };
    if (few) h_values(reinterpret_cast<float *>(hs), tile.len, width, sum);
    else h_operands<T, RC>(hs, (tile.len + M - 1) / M, width, sum);
    __syncthreads();
  }
  const int blocks = (p.n + COLS - 1) / COLS, per = (blocks + slices - 1) / slices;
  const int first = slice * per + warp;
  Copies<T, RC, WIDE> copies(p, tile, width, smem + h_bytes<T>(p.tile_rows, width), first,
                             min(blocks, (slice + 1) * per), WARPS);
  copies.start();
  if (few) expand_few<T, RC, WIDE>(p, tile, rows, reinterpret_cast<float *>(hs), width, first * COLS, copies);
  else expand<T, RC, WIDE>(p, tile, rows, hs, width, first * COLS, copies);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The most tiles m rows can make.
uint64_t tile_bound(uint64_t m, uint64_t count, uint64_t tile_rows) {
  // an adapter's last tile may be short; above the sort's buckets neighbours may
  // alternate
  const uint64_t most = count < BUCKETS - 1 || m <= INLINE_ROWS ? m / tile_rows + count + 1 : m;
  return most < m ? most : m;
}

// Rows of a tile: h of 64 rows as operands takes 512 bytes a rank of shared
// memory, which two CTAs an SM allow up to rank 64.
int tile_rows_of(uint64_t rank) { return rank <= 64 ? 64 : rank <= 128 ? 32 : 16; }

int pass_ranks(uint64_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

// The most slices of k of a grid.
constexpr uint64_t MOST_SPLITS = 16;
uint64_t most_splits(const mgb_adapters &ad) {
  const uint64_t groups = ceil_div(ceil_div(ad.k, 32), WARPS);
  return groups < MOST_SPLITS ? groups : MOST_SPLITS;
}

// Slices of k.  A cluster: as many CTAs as keep all clusters on the SMs at once
// (two CTAs each), so that 64 rows of 64 adapters do not run in two waves.  The
// grid: enough for two CTAs an SM, at least a group of 32 a warp.
int k_splits(const mgb_adapters &ad, uint64_t m, int sms) {
  const uint64_t tiles = tile_bound(m, ad.count, tile_rows_of(ad.rank));
  if (m <= INLINE_ROWS) {
    int s = MOST_CTAS;
    while (s > 1 && tiles * s > 2 * (uint64_t)sms) s /= 2;
    return s;
  }
  const uint64_t want = ceil_div(2 * (uint64_t)sms, tiles), most = most_splits(ad);
  return (int)(want < most ? want : most);
}

// The most rows of h that any batch of up to m rows has, over its slices of k.  More
// rows can have fewer slices and so fewer rows of h; a workspace of the largest batch
// serves every smaller one all the same.
uint64_t most_h_rows(const mgb_adapters &ad, uint64_t m, int sms) {
  const uint64_t tile_rows = tile_rows_of(ad.rank);
  uint64_t most = m;
  for (uint64_t s = 2; s <= MOST_SPLITS; ++s) {
    // s slices or more: ceil(2 sms / tiles) >= s, so up to `tiles` tiles
    const uint64_t tiles = (2 * (uint64_t)sms - 1) / (s - 1);
    uint64_t rows = tiles;  // the most that stay within them (tile_bound's inverse)
    if (ad.count < BUCKETS - 1 && tiles > ad.count && (tiles - ad.count) * tile_rows - 1 > rows)
      rows = (tiles - ad.count) * tile_rows - 1;
    if (rows > m) rows = m;
    if (s <= most_splits(ad) && s * rows > most) most = s * rows;
  }
  return most;
}

// Grouped rows' scratch (up to INLINE_ROWS rows need none of it).
struct Scratch {
  uint64_t order, tiles, ntiles, h, total;
  Scratch(const mgb_adapters &ad, uint64_t m, int sms) {
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
      const uint64_t r = at;
      at += (bytes + 127) / 128 * 128;
      return r;
    };
    const uint64_t planned = m > INLINE_ROWS ? m : 0;
    order = take(planned * 4);
    tiles = take(planned ? tile_bound(m, ad.count, tile_rows_of(ad.rank)) * sizeof(Tile) : 0);
    ntiles = take(4);
    h = take((planned ? most_h_rows(ad, m, sms) : 0) * h_width((int)ad.rank, pass_ranks(ad.rank)) * 4);
    total = at;
  }
};

int current_sms() {
  int dev = 0;
  cudaGetDevice(&dev);
  return device_sms(dev);
}

// A programmatic dependent launch, in clusters of `cluster` CTAs.
template <typename... A>
cudaError_t launch_chained(void (*kern)(A...), unsigned grid, int threads, uint32_t smem, int cluster,
                           cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Lets a kernel use its dynamic shared memory: an attribute of the function on a
// device, set once each.
template <typename K>
cudaError_t opt_in(K kern, std::atomic<uint64_t> &opted) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || opted.load(std::memory_order_relaxed) >> (dev & 63) & 1) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024);
  if (e == cudaSuccess) opted.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  return e;
}

template <typename T, int RC, bool WIDE>
cudaError_t launch_rc(const Params &p, unsigned tiles, int sms, cudaStream_t stream) {
  static std::atomic<uint64_t> opted[3];
  const int width = h_width(p.rank, RC);
  const uint32_t h = h_bytes<T>(p.tile_rows, width), part = part_bytes(p.tile_rows, width);
  const uint32_t ring = WIDE ? Shared<T, RC>::RING : 0;
  cudaError_t e;
  if (p.m <= INLINE_ROWS) {
    if ((e = opt_in(mgb_adapter_kernel<T, RC, WIDE>, opted[0])) != cudaSuccess) return e;
    Params q = p;
    const uint32_t most = (sizeof(T) == 4 ? 216 : 108) * 1024;  // of one CTA an SM, of two
    q.early = h + part + ring <= most;
    return launch_chained(mgb_adapter_kernel<T, RC, WIDE>, tiles * p.splits, 32 * WARPS,
                          h + (q.early ? part + ring : part > ring ? part : ring), p.splits, stream, q);
  }
  if ((e = opt_in(mgb_adapter_h_kernel<T, RC>, opted[1])) != cudaSuccess) return e;
  if ((e = opt_in(mgb_adapter_y_kernel<T, RC, WIDE>, opted[2])) != cudaSuccess) return e;
  e = launch_chained(mgb_adapter_h_kernel<T, RC>, tiles * p.splits, 32 * WARPS, part, 1, stream, p);
  if (e != cudaSuccess) return e;
  // Slices of the outputs: those with the fewest waves of CTAs (two an SM) times the
  // blocks of a warp and one more, about what a CTA takes before its first block (the
  // rows, h as operands); summed for the fewest tiles that the rows can make and for the
  // middle of that and the most.  2,048 rows, 32 to 41 tiles, 14,336 outputs, y alone when
  // the rule was set: 8 slices, a wave, 76 us (now 66); 14 slices 91 us, 28 slices 100 us.
  const uint64_t blocks = ceil_div(p.n, COLS), full = ceil_div(p.m, p.tile_rows);
  uint64_t slices = 1, least = ~0ull;
  for (uint64_t s = 1; s <= 64 && s <= ceil_div(blocks, WARPS); ++s) {
    const uint64_t waves =
        ceil_div((tiles + full) / 2 * s, 2 * (uint64_t)sms) + ceil_div(full * s, 2 * (uint64_t)sms);
    const uint64_t cost = waves * (ceil_div(ceil_div(blocks, s), WARPS) + 1);
    if (cost <= least) least = cost, slices = s;
  }
  const uint64_t fit = 0x7FFFFFFFull / tiles;  // CTAs of a grid
  if (slices > fit) slices = fit;
  return launch_chained(mgb_adapter_y_kernel<T, RC, WIDE>, (unsigned)(tiles * slices), 32 * WARPS, h + ring,
                        1, stream, p, (int)slices);
}

template <typename T>
cudaError_t launch_t(const Params &p, unsigned tiles, int sms, cudaStream_t stream) {
  const int rc = pass_ranks(p.rank);
  if (p.wide_b && p.wide_y)
    return rc == 16   ? launch_rc<T, 16, true>(p, tiles, sms, stream)
           : rc == 32 ? launch_rc<T, 32, true>(p, tiles, sms, stream)
                      : launch_rc<T, 64, true>(p, tiles, sms, stream);
  return rc == 16   ? launch_rc<T, 16, false>(p, tiles, sms, stream)
         : rc == 32 ? launch_rc<T, 32, false>(p, tiles, sms, stream)
                    : launch_rc<T, 64, false>(p, tiles, sms, stream);
}

}  // namespace

uint64_t adapters_scratch_bytes(const mgb_adapters &ad, uint64_t m) {
  return m ? Scratch(ad, m, current_sms()).total : 0;
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
  p.tile_rows = tile_rows_of(ad.rank);
  const int sms = current_sms();
  p.splits = k_splits(ad, m, sms);
  const Scratch s(ad, m, sms);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.order = reinterpret_cast<int32_t *>(ws + s.order);
  p.tiles = reinterpret_cast<Tile *>(ws + s.tiles);
  p.ntiles = reinterpret_cast<int32_t *>(ws + s.ntiles);
  p.h = reinterpret_cast<float *>(ws + s.h);
  const uint64_t per = ad.dtype == MGB_DTYPE_F32 ? 4 : 8;  // values in 16 bytes
  p.wide_a = aligned16(ad.a) && ad.k % per == 0;
  p.wide_b = aligned16(ad.b) && ad.rank % per == 0;
  p.wide_x = aligned16(x) && ad.k % 4 == 0;
  p.wide_y = aligned16(y) && aligned16(base) && ad.n % 4 == 0;
  if (m > INLINE_ROWS) {
    static std::atomic<uint64_t> opted{0};
    if ((e = opt_in(mgb_adapter_plan_kernel, opted)) != cudaSuccess) return e;
    e = launch_chained(mgb_adapter_plan_kernel, 1, 1024, plan_bytes(m), 1, stream, p);
    if (e != cudaSuccess) return e;
  }
  const unsigned tiles = (unsigned)tile_bound(m, ad.count, p.tile_rows);
  if (ad.dtype == MGB_DTYPE_F32) return launch_t<float>(p, tiles, sms, stream);
  if (ad.dtype == MGB_DTYPE_F16) return launch_t<__half>(p, tiles, sms, stream);
  return launch_t<__nv_bfloat16>(p, tiles, sms, stream);
}

}  // namespace mgb
