// One token per row of logits from given random numbers: temperature, top-k,
// top-p and min-p, then a draw in index order.
//
// Order.  Logits are compared as 32-bit keys (the float's bits made
// monotonic, -0 as +0; 0 for -inf and NaN, which are masked).  Every cut keeps
// a prefix of the tokens sorted by (key descending, index ascending), so what
// is kept is described by a key tau and how many tokens of key tau (the lowest
// indices) stay: no sort of the vocabulary is needed, only the search for tau.
//
// A row is held by a cluster, whose CTAs agree on one number after another through
// distributed shared memory.  Few rows: up to eight CTAs of 256 threads a row, each
// its part in shared memory.  Rows that fill the SMs by themselves: two CTAs of 512
// threads a row, which read it again from L2; what a batch costs then is the
// instructions a token takes, and one CTA a row would leave the SMs of greedy rows
// idle beside those of broad ones (256 rows of 128,256, every row its own settings:
// 320 us with one, 204 us with two; all rows top-k 50: 52 us and 74 us).
//  - Small top_k: the top_k-th largest of the threads' own largest logits is a bound
//    that at least top_k of a CTA's tokens reach and few others do.  One from the
//    first quarter of the CTA's part bounds the rest as it is read; the first CTA
//    sorts the tokens that reach all bounds and does what is left.
//  - Otherwise the border is searched by histograms of counts (top-k) or of mass
//    (top-p) over the distance to the largest logit, where tokens spread evenly over
//    the bins: of 1/16, and if that holds too many tokens of 1/16384; the first CTA
//    sorts the border bin's.  Where even that is too much (equal or nearly equal
//    logits), by ever smaller ranges of keys.
// Measured on the device, 256 rows of 128,256 (131 MB; 20 us at the copy's rate): greedy
// 31 us, no cuts 133 us (a weight costs some 45 instructions), min-p 76 us, top-k 50 72 us,
// top-k 1,000 150 us, top-p 0.95 360 us (two histograms, two lists, the sum).  One row of
// 32,000, top-k 50 and top-p: 15 us, a chain of dependent steps.
//
// Mass.  A token's weight is 2^((logit - max) log2(e) / T) as a 64-bit integer
// in units of 2^-43: integer sums are the same in every order, so atomics and
// any split of a row give the same token, and a border is only missed where
// weights round (2^-31 relative, and half a unit).  2^20 tokens of weight 1 stay below
// 2^63.  A log-probability takes the kept total from them, and the token's own part from
// its logit: a weight of few units has few bits.
#include <cooperative_groups.h>

#include <atomic>
#include <cfloat>

#include "common.cuh"
#include "kernels.h"

namespace mgb {

namespace cg = cooperative_groups;

constexpr int ONE_BITS = 43;  // weight 1

// 2^(j / 64) in units of 2^-31.
__constant__ uint32_t g_pow2[64] = {
    2147483648u, 2170868212u, 2194507417u, 2218404036u, 2242560872u, 2266980759u, 2291666561u, 2316621173u,
    2341847524u, 2367348571u, 2393127307u, 2419186755u, 2445529972u, 2472160047u, 2499080105u, 2526293303u,
    2553802834u, 2581611923u, 2609723834u, 2638141863u, 2666869345u, 2695909648u, 2725266179u, 2754942382u,
    2784941738u, 2815267765u, 2845924021u, 2876914102u, 2908241642u, 2939910317u, 2971923842u, 3004285971u,
    3037000500u, 3070071267u, 3103502151u, 3137297074u, 3171459999u, 3205994934u, 3240905930u, 3276197082u,
    3311872529u, 3347936457u, 3384393094u, 3421246719u, 3458501653u, 3496162267u, 3534232978u, 3572718252u,
    3611622603u, 3650950594u, 3690706840u, 3730896002u, 3771522796u, 3812591987u, 3854108391u, 3896076880u,
    3938502376u, 3981389855u, 4024744348u, 4068570940u, 4112874773u, 4157661043u, 4202935003u, 4248701965u};

__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 -> +0
  if (!(v > __int_as_float(0xff800000))) return 0;  // -inf, NaN
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The weight function of a row.
struct Weigh {
  float top, chi, clo;  // the largest logit; log2(e) / T as the sum of two floats
  const uint32_t *pow2;  // g_pow2 in shared memory: lanes look different entries up,
                         // which constant memory serves one after the other, and two
                         // words in each bank keep few of them waiting for one another
  // the distance to the largest logit in octaves: monotonic
  __device__ __forceinline__ float octaves(float v) const { return (top - v) * chi; }
  __device__ __forceinline__ uint64_t operator()(float v) const {
    if (__isinff(top)) return v == top ? 1ull << ONE_BITS : 0;  // +inf
    // v - top = d + e exactly; times (chi + clo): p + r
    const float d = v - top, b = d - v;
    const float e = (v - (d - b)) + (-top - b);
    const float p = d * chi;
    if (!(p > -44.f)) return 0;  // below half a unit (also v = -inf, NaN)
    float r = fmaf(d, chi, -p);
    r = fmaf(d, clo, r);
    r = fmaf(e, chi, r);
    // 2^(p + r) = 2^N 2^(j / 64) 2^s, |s| <= 1/128; the last factor by its Taylor
    // polynomial (next term 2^-44).  (Rounding by adding 1.5 2^23 leaves the integer
    // in the float's bits: the conversion units are far slower than the arithmetic.)
    const float big = fmaf(p, 64.f, 12582912.f), n = big - 12582912.f;
    const float s = fmaf(n, -0.015625f, p) + r;
    float q = fmaf(s, 0.009618129107628f, 0.055504108664822f);
    q = fmaf(s, q, 0.240226506959101f);
    q = fmaf(s, q, 0.693147180559945f);
    q *= s;
    const int ni = __float_as_int(big) - 0x4B400000, N = ni >> 6;
    const uint32_t lead = pow2[ni & 63];
    // the last two factors in units of 2^-31 (below 2): lead (1 + q), q in 2^-38
    const uint32_t one = lead + ((__mulhi((int)(lead >> 1), __float2int_rn(q * 0x1p38f)) + 16) >> 5);
    const int down = 31 - ONE_BITS - N;
    if (down > 0) return ((one >> (down - 1)) + 1) >> 1;  // (down <= 32)
    return (uint64_t)one << -down;
  }
};

constexpr int BINS = 1024;
constexpr int MOST_CTAS = 8;      // of a cluster
constexpr int LIST = 1024;        // tokens the first CTA sorts at most
constexpr uint32_t LOWEST = 0x00800000u;  // the key of the lowest finite value
// A token's distance to the largest logit (in octaves of the weight where masses
// are summed) as a number of 20 bits, monotonic: 1,024 bins of 1/16, of 1,024 parts.
constexpr float CODE_SCALE = 16384.f;
constexpr int CODE_MOST = (1 << 20) - 1;
constexpr uint32_t MOST_TOKENS = 1 << 17;  // of a CTA

typedef unsigned long long u64;  // what atomicAdd and shuffles take

// A token in the order: larger is earlier.
__device__ __forceinline__ u64 place_of(uint32_t key, uint32_t index) {
  return ((u64)key << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint32_t index_of(u64 place) { return 0xFFFFFFFFu - (uint32_t)place; }

template <bool MASS>
__device__ __forceinline__ int code_of(const Weigh &weigh, float v) {
  const int c = (int)((MASS ? weigh.octaves(v) : weigh.top - v) * CODE_SCALE);  // (saturates)
  return c < CODE_MOST ? c : CODE_MOST;
}

template <int THREADS>
struct Shared {
  static constexpr int WARPS = THREADS / 32;
  u64 list[LIST];                       // the first CTA: its cluster's tokens; a histogram
  alignas(8) uint32_t part[3][BINS];    // a histogram as it is filled (32-bit atomics are native:
                                        // masses in three digits); the sort's buffer
  u64 scan[WARPS];
  // what the CTAs tell each other, by rank
  u64 top[MOST_CTAS];                   // the place of the largest logit
  u64 mass[MOST_CTAS];
  float bound[MOST_CTAS];
  uint32_t live[MOST_CTAS], found[MOST_CTAS], count[MOST_CTAS], ties[MOST_CTAS], kept[MOST_CTAS];
  // the first CTA's answers
  u64 found_above, cut, target;
  uint32_t lo, hi;
  int border, many;
  // of the CTA
  u64 above, warp_mass[WARPS];
  uint32_t warp_ties[WARPS], warp_count[WARPS], taken, bin;
};

template <int THREADS>
__device__ __forceinline__ u64 block_max(u64 v, Shared<THREADS> &s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 u = __shfl_xor_sync(0xffffffffu, v, o);
    v = v > u ? v : u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v = v > s.scan[w] ? v : s.scan[w];
  return v;
}

// Inclusive sum over the CTA's threads.
template <int THREADS>
__device__ __forceinline__ u64 block_scan(u64 v, Shared<THREADS> &s, u64 &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) s.scan[warp] = v;
  __syncthreads();
  total = 0;
  u64 before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s.scan[w];
    total += s.scan[w];
  }
  return before + v;
}

// The first of n entries (n a multiple of THREADS) at which the running sum
// reaches target, and the sum before it; all threads.
template <int PER, int THREADS>
__device__ __forceinline__ void find_entry(const u64 *e, u64 target, Shared<THREADS> &s, int &at, u64 &before) {
  u64 c[PER], v = 0, total;
#pragma unroll
  for (int i = 0; i < PER; ++i) c[i] = e[threadIdx.x * PER + i], v += c[i];
  u64 run = block_scan(v, s, total) - v;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (run < target && run + c[i] >= target) s.bin = threadIdx.x * PER + i, s.above = run;
    run += c[i];
  }
  __syncthreads();
  at = (int)s.bin;
  before = s.above;
  __syncthreads();
}

// n different places (n <= LIST) into descending order, in place.
template <int THREADS>
__device__ __forceinline__ void sort_places(u64 *e, uint32_t n) {
  if (n <= 256 && n <= THREADS) {  // each counts those before it (a barrier a step costs more)
    const u64 mine = threadIdx.x < n ? e[threadIdx.x] : 0;
    uint32_t at = 0;
    if (threadIdx.x < n)
#pragma unroll 4
      for (uint32_t i = 0; i < n; ++i) at += e[i] > mine;
    __syncthreads();
    if (threadIdx.x < n) e[at] = mine;
    __syncthreads();
    return;
  }
  uint32_t size = 2;
  while (size < n) size <<= 1;
  for (uint32_t i = n + threadIdx.x; i < size; i += THREADS) e[i] = 0;
  __syncthreads();
  for (uint32_t k = 2; k <= size; k <<= 1)
    for (uint32_t j = k >> 1; j; j >>= 1) {
      for (uint32_t i = threadIdx.x; i < size / 2; i += THREADS) {
        const uint32_t a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = e[a], y = e[b];
        if ((x < y) == ((a & k) == 0)) e[a] = y, e[b] = x;
      }
      __syncthreads();
    }
}

// Whether a token's place is above a given one, without building its key.
struct Over {
  float v;
  uint32_t limit;
  __device__ __forceinline__ explicit Over(u64 place) {
    v = place >> 32 ? value_of((uint32_t)(place >> 32)) : __int_as_float(0xff800000);
    limit = place >> 32 ? 0xFFFFFFFFu - (uint32_t)place : 0;
  }
  __device__ __forceinline__ bool operator()(float x, uint32_t index) const {
    return x > v || (x == v && index < limit);
  }
};

struct Row {
  const float *v;      // this CTA's part of the row
  uint32_t first, n;   // index of its first token, tokens
  float top;           // the row's largest logit
  uint32_t top_key;
};

// Calls f(logit, position) for the tokens [from, to) of the CTA's part (from a
// multiple of 4), spread over THREADS threads, 16 bytes at a time where it can, and copies them; a thread's
// positions rise.  (AHEAD loads are issued before the first f, whose atomics and
// stores no load is moved over: the candidates of 256 rows of 128,256 took 34 us of
// a row's time without that.)
template <int THREADS, int AHEAD = 4, bool COPY = false, typename F>
__device__ __forceinline__ void for_each(const float *v, uint32_t from, uint32_t to, const F &f,
                                         float *copy = nullptr, uint32_t thread = threadIdx.x) {
  uint32_t i = from;
  if ((reinterpret_cast<uintptr_t>(v) & 15) == 0) {
    const float4 *v4 = reinterpret_cast<const float4 *>(v);
    const uint32_t n4 = to / 4;
    auto four = [&](const float4 &x, uint32_t at) {
      if (COPY) reinterpret_cast<float4 *>(copy)[at] = x;
      f(x.x, 4 * at);
      f(x.y, 4 * at + 1);
      f(x.z, 4 * at + 2);
      f(x.w, 4 * at + 3);
    };
    uint32_t j = from / 4 + thread;
    for (; j + (AHEAD - 1) * THREADS < n4; j += AHEAD * THREADS) {
      float4 x[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) x[a] = v4[j + a * THREADS];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) four(x[a], j + a * THREADS);
    }
    for (; j < n4; j += THREADS) four(v4[j], j);
    i = max(from, 4 * n4);
  }
  i += thread;
  auto one = [&](float x, uint32_t at) {
    if (COPY) copy[at] = x;
    f(x, at);
  };
  for (; i + 3 * THREADS < to; i += 4 * THREADS) {
    float x[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) x[a] = v[i + a * THREADS];
#pragma unroll
    for (int a = 0; a < 4; ++a) one(x[a], i + a * THREADS);
  }
  for (; i < to; i += THREADS) one(v[i], i);
}

// A value that at least k of the threads' keys reach and few more (the lowest
// finite value where fewer than k are live).
template <int THREADS>
__device__ __forceinline__ float kth_largest(uint32_t own, uint32_t k) {
  uint32_t lo = LOWEST, hi = 0xFF800000u;  // (+inf)
  while (lo < hi) {
    const uint32_t m = lo + (hi - lo + 1) / 2;
    const uint32_t n = __syncthreads_count(own >= m);
    if (n >= k) lo = m;
    else hi = m - 1;
    if (n >= k && n <= k + k / 8) break;
  }
  return value_of(lo);
}

// The tokens' counts (MASS: masses) by bin, summed over the cluster in the first
// CTA's part[0..1], as u64.  bin(v, position): a token's bin, or -1.  A mass is
// added in digits, whose sums over a CTA's tokens stay below 2^32: 15 bits, three of
// them, for MOST_TOKENS; with NARROW and about half of those, two of 16 bits.
// NARROW: bin b's weights are multiples of 2^low(b) and at most 2^32 of that (a
// thousandth more where they round up).
template <bool MASS, bool NARROW, int THREADS, typename B, typename L>
__device__ __forceinline__ u64 *histogram(const Row &row, const B &bin, const L &low, const Weigh &weigh,
                                          Shared<THREADS> &s, cg::cluster_group &cluster) {
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const bool two = NARROW && row.n <= 65000;
  const int D = two ? 16 : 15;
  const uint32_t mask = (1u << D) - 1;
  for (int i = threadIdx.x; i < BINS; i += THREADS)
#pragma unroll
    for (int d = 0; d < (MASS ? 3 : 1); ++d) s.part[d][i] = 0;
  __syncthreads();
  for_each<THREADS>(row.v, 0, row.n, [&](float v, uint32_t i) {
    const int b = bin(v, i);
    if (b < 0) return;
    if (MASS) {
      const uint64_t w = weigh(v) >> low(b);
      if (!w) return;
      atomicAdd(&s.part[0][b], (uint32_t)w & mask);
      if (two) {
        atomicAdd(&s.part[1][b], (uint32_t)(w >> 16));
      } else {
        const uint32_t d1 = (uint32_t)(w >> 15) & mask, d2 = (uint32_t)(w >> 30);
        atomicAdd(&s.part[1][b], d1);
        if (d2) atomicAdd(&s.part[2][b], d2);
      }
    } else {
      atomicAdd(&s.part[0][b], 1u);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS)
    s.list[i] = MASS ? (s.part[0][i] + ((u64)s.part[1][i] << D) + ((u64)s.part[2][i] << 30)) << low(i)
                     : s.part[0][i];
  cluster.sync();
  u64 *all = reinterpret_cast<u64 *>(s.part[0]);  // [BINS]: two of the three
  if (rank == 0) {
    u64 c[BINS / THREADS];
#pragma unroll
    for (int j = 0; j < BINS / THREADS; ++j) c[j] = 0;
    for (int o = 0; o < ctas; ++o) {
      const u64 *h = cluster.map_shared_rank(s.list, o);
#pragma unroll
      for (int j = 0; j < BINS / THREADS; ++j) c[j] += h[j * THREADS + threadIdx.x];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < BINS / THREADS; ++j) all[j * THREADS + threadIdx.x] = c[j];
    __syncthreads();
  }
  return all;
}

// The largest key in [lo, hi] at which the count (MASS: the mass) of the keys from
// hi down to it, of places above `over`, reaches `target` (>= 1, at most what
// there is); above: the count or mass of the keys over it.  The whole cluster.
template <bool MASS, int THREADS>
__device__ __noinline__ uint32_t find_key(const Row &row, uint32_t lo, uint32_t hi, u64 over, u64 target,
                                          const Weigh &weigh, Shared<THREADS> &s, cg::cluster_group cluster,
                                          u64 &above) {
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  above = 0;
  while (lo < hi) {
    int shift = 0;
    while (((hi - lo) >> shift) >= BINS) ++shift;
    const u64 *all = histogram<MASS, false, THREADS>(
        row,
        [&](float v, uint32_t i) {
          const uint32_t key = key_of(v);
          return key >= lo && key <= hi && place_of(key, row.first + i) > over ? (int)((hi - key) >> shift) : -1;
        },
        [](int) { return 0; }, weigh, s, cluster);
    if (rank == 0) {
      int bin;
      u64 before;
      find_entry<BINS / THREADS>(all, target - above, s, bin, before);
      if (threadIdx.x < (unsigned)ctas) {
        const uint32_t nhi = hi - ((uint32_t)bin << shift), width = (1u << shift) - 1;
        Shared<THREADS> *o = cluster.map_shared_rank(&s, threadIdx.x);
        o->lo = nhi - lo > width ? nhi - width : lo;
        o->hi = nhi;
        o->found_above = above + before;
      }
    }
    cluster.sync();
    lo = s.lo;
    hi = s.hi;
    above = s.found_above;
  }
  __syncthreads();
  return hi;
}

// What is kept: the places above `over`, and `ties` tokens of key tau besides (the
// lowest indices).
struct Cut {
  u64 over;
  uint32_t tau;
  u64 ties;
};

// The first CTA: what its cluster's list holds from `bound` on, best first, in
// part[0..1]; returns its number.
template <int THREADS>
__device__ __forceinline__ uint32_t sort_list(int ctas, uint32_t room, const uint32_t *count, float bound,
                                              Shared<THREADS> &s) {
  u64 *sorted = reinterpret_cast<u64 *>(s.part[0]);
  __syncthreads();
  if (threadIdx.x == 0) s.taken = 0;
  __syncthreads();
  for (int c = 0; c < ctas; ++c)
    for (uint32_t i = threadIdx.x; i < count[c]; i += THREADS) {
      const u64 place = s.list[c * room + i];
      if (value_of((uint32_t)(place >> 32)) >= bound) sorted[atomicAdd(&s.taken, 1u)] = place;
    }
  __syncthreads();
  const uint32_t n = s.taken;
  sort_places<THREADS>(sorted, n);
  return n;
}

// Where a border cannot be listed: the key at which the count (MASS: the mass) of
// what is kept so far reaches target, and how many of its tokens stay.
template <bool MASS, int THREADS>
__device__ __noinline__ void cut_by_key(const Row &row, u64 target, const Weigh &weigh, Shared<THREADS> &s,
                                        cg::cluster_group cluster, Cut &cut) {
  u64 above;
  const uint32_t lo = cut.ties ? cut.tau : LOWEST;
  const uint32_t key = find_key<MASS, THREADS>(row, lo, row.top_key, cut.ties ? 0 : cut.over, target, weigh, s,
                                               cluster, above);
  const u64 w = MASS ? weigh(value_of(key)) : 1;
  u64 need = w ? (target - above + w - 1) / w : 1;
  if (cut.ties && key == cut.tau && cut.ties < need) need = cut.ties;
  cut.tau = key;
  cut.ties = need;
  cut.over = place_of(key, 0);  // every place of a larger key
}

// Cuts behind the token at which the count (MASS: the mass) of what is kept so
// far, in order, reaches its target: target_of(all of it), at least 1.  Histograms
// of the distance to the largest logit find the border's bin, and part of the bin
// where that holds too many tokens; the first CTA sorts those.  The whole cluster.
template <bool MASS, int THREADS, typename F>
__device__ void cut_at(const Row &row, const F &target_of, const Weigh &weigh, Shared<THREADS> &s,
                       cg::cluster_group cluster, Cut &cut) {
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const uint32_t room = LIST / ctas;
  const Over over(cut.over);
  // the first CTA finds the entry of its histogram and tells all; the total counts
  // where it is the first level's
  auto tell = [&](const u64 *all, bool first_level) {
    if (rank == 0) {
      u64 c[BINS / THREADS], v = 0, total;
#pragma unroll
      for (int i = 0; i < BINS / THREADS; ++i) c[i] = all[threadIdx.x * (BINS / THREADS) + i], v += c[i];
      block_scan(v, s, total);
      if (cut.ties) total += cut.ties * (MASS ? weigh(value_of(cut.tau)) : 1);
      const u64 target = first_level ? target_of(total) : s.target;
      const u64 above = first_level ? 0 : s.found_above;
      __syncthreads();
      int bin;
      u64 before;
      find_entry<BINS / THREADS>(all, target - above, s, bin, before);
      if (threadIdx.x < (unsigned)ctas) {
        Shared<THREADS> *o = cluster.map_shared_rank(&s, threadIdx.x);
        o->border = bin;
        // more tokens than can be listed (of masses: even if each had its bin's most)
        o->many = (MASS ? exp2f(bin * 0.0625f - (float)ONE_BITS) : 1.f) * (float)all[bin] > (float)LIST;
        o->found_above = above + before;
        o->target = target;
      }
    }
    if (threadIdx.x == 0) s.taken = 0;
    cluster.sync();
  };
  if (cut.ties == 0 && !__isinff(row.top)) {
    // a bin's weights lie within 1/16 octave, and have 32 bits
    tell(histogram<MASS, true, THREADS>(
             row,
             [&](float v, uint32_t i) { return over(v, row.first + i) ? code_of<MASS>(weigh, v) >> 10 : -1; },
             [](int b) { return b < 11 * 16 ? 11 - (b >> 4) : 0; }, weigh, s, cluster),
         true);
    const int border = s.border;
    int part = -1;
    for (int level = s.many; level < 2; ++level) {
      if (level == 1) {
        tell(histogram<MASS, true, THREADS>(
                 row,
                 [&](float v, uint32_t i) {
                   if (!over(v, row.first + i)) return -1;
                   const int c = code_of<MASS>(weigh, v);
                   return c >> 10 == border ? c & 1023 : -1;
                 },
                 [=](int) { return border < 11 * 16 ? 11 - (border >> 4) : 0; }, weigh, s, cluster),
             false);
        part = (border << 10) | s.border;
      }
      auto inside = [&](float v, uint32_t i) {
        if (!over(v, row.first + i)) return false;
        const int c = code_of<MASS>(weigh, v);
        return part < 0 ? c >> 10 == border : c == part;
      };
      u64 *list = cluster.map_shared_rank(s.list, 0) + rank * room;
      for_each<THREADS>(row.v, 0, row.n, [&](float v, uint32_t i) {
        if (!inside(v, i)) return;
        const uint32_t at = atomicAdd(&s.taken, 1u);
        if (at < room) list[at] = place_of(key_of(v), row.first + i);
      });
      __syncthreads();
      if (threadIdx.x < (unsigned)ctas) cluster.map_shared_rank(&s, threadIdx.x)->count[rank] = s.taken;
      cluster.sync();
      bool listed = true;
      for (int c = 0; c < ctas; ++c) listed = listed && s.count[c] <= room;
      if (listed) {
        if (rank == 0) {
          const u64 *sorted = reinterpret_cast<const u64 *>(s.part[0]);
          const uint32_t n = sort_list<THREADS>(ctas, room, s.count, -FLT_MAX, s);
          for (uint32_t i = threadIdx.x; i < LIST; i += THREADS)
            s.list[i] = i >= n ? 0 : MASS ? weigh(value_of((uint32_t)(sorted[i] >> 32))) : 1;
          __syncthreads();
          int at;
          u64 unused;
          find_entry<LIST / THREADS>(s.list, s.target - s.found_above, s, at, unused);
          if (threadIdx.x < (unsigned)ctas) cluster.map_shared_rank(&s, threadIdx.x)->cut = sorted[at] - 1;
        }
        cluster.sync();
        cut.over = s.cut;
        __syncthreads();
        return;
      }
    }
  } else {
    tell(histogram<MASS, false, THREADS>(
             row, [&](float v, uint32_t i) { return over(v, row.first + i) ? 0 : -1; }, [](int) { return 0; },
             weigh, s, cluster),
         true);
  }
  cut_by_key<MASS, THREADS>(row, s.target, weigh, s, cluster, cut);  // too many tokens in one place
}

__device__ __forceinline__ void answer(const SampleArgs &p, uint64_t r, float id, float logprob,
                                       uint32_t kept) {
  if (p.ids) p.ids[r] = id;
  if (p.logprob) p.logprob[r] = logprob;
  if (p.kept) p.kept[r] = kept;
}

// One row a cluster.  STAGED: each CTA's part of the row is in its shared memory;
// otherwise it is read again (from L2, mostly).
template <int THREADS, bool STAGED>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 2)
    mgb_sample_kernel(const SampleArgs p, uint32_t chunk) {
  constexpr int WARPS = THREADS / 32;
  __shared__ Shared<THREADS> s;
  __shared__ uint32_t pow2[64];
  extern __shared__ __align__(16) float data[];
  if (threadIdx.x < 64) pow2[threadIdx.x] = g_pow2[threadIdx.x];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t r = blockIdx.x / ctas;
  const uint32_t vocab = (uint32_t)p.vocab;
  cluster.barrier_arrive();  // (waited for before another CTA's memory is touched: it has started)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  Row row;
  row.first = min(vocab, rank * chunk);
  row.n = min(chunk, vocab - row.first);
  const float *src = p.logits + r * p.ld + row.first;
  const float temp = p.temperature ? p.temperature[r] : 1.f;
  const bool greedy = !(temp > 0.f) || !p.uniform;
  const float kf = p.top_k ? p.top_k[r] : 0.f;

  // the thread's largest key and its position, and the live tokens
  uint32_t own = 0, own_at = 0, live = 0;
  auto see = [&](float v, uint32_t i) {
    const uint32_t key = key_of(v);
    live += key != 0;
    if (key > own) own = key, own_at = i;  // (positions rise: the first of equals stays)
  };
  // small top_k: this CTA's candidates, to the first CTA's list
  static_assert(LIST <= BINS && BINS * 8 <= sizeof(s.part), "the sort's buffer");
  const uint32_t room = LIST / ctas;
  const bool few = !greedy && kf >= 1.f && kf < 257.f && kf < (float)room + 1.f;
  u64 *list = cluster.map_shared_rank(s.list, 0) + rank * room;
  float bound;
  auto take = [&](float v, uint32_t i) {
    if (!(v >= bound)) return;
    const uint32_t at = atomicAdd(&s.taken, 1u);
    if (at < room) list[at] = place_of(key_of(v), row.first + i);
  };
  // From the threads' largest of a first part comes a bound for the rest, whose
  // candidates are so listed as they are read.
  const uint32_t head = few && row.n >= 32 * THREADS ? row.n / 4 & ~3u : row.n;
  if (threadIdx.x == 0) s.taken = 0;
  for_each<THREADS, 8, STAGED>(src, 0, head, see, data);
  cluster.barrier_wait();
  if (head < row.n) {
    bound = kth_largest<THREADS>(own, (uint32_t)kf);
    for_each<THREADS, 8, STAGED>(
        src, head, row.n,
        [&](float v, uint32_t i) {
          see(v, i);
          take(v, i);
        },
        data);
  }
  row.v = STAGED ? data : src;
  u64 best = block_max(own ? place_of(own, row.first + own_at) : 0ull, s);
  {
    u64 total;
    block_scan(live, s, total);
    live = (uint32_t)total;
  }
  uint32_t found = 0xFFFFFFFFu;  // none sent
  if (few) {
    // what is listed is a superset: the first CTA leaves out what is below all bounds
    bound = live > room ? kth_largest<THREADS>(own, (uint32_t)kf) : -FLT_MAX;
    const bool kept = s.taken <= room;
    __syncthreads();
    if (!kept && threadIdx.x == 0) s.taken = 0;
    __syncthreads();
    for_each<THREADS>(row.v, 0, kept ? head : row.n, take);
    __syncthreads();
    found = s.taken;  // (above room: too many tokens reach the bound)
  }
  if (threadIdx.x < (unsigned)ctas) {
    Shared<THREADS> *o = cluster.map_shared_rank(&s, threadIdx.x);
    o->top[rank] = best;
    o->live[rank] = live;
    o->found[rank] = found;
    o->bound[rank] = bound;
  }
  cluster.sync();
  bool listed = few;
  best = 0, live = 0;
  for (int c = 0; c < ctas; ++c) {
    best = best > s.top[c] ? best : s.top[c];
    live += s.live[c];
    listed = listed && s.found[c] <= room;
  }
  row.top_key = (uint32_t)(best >> 32);
  if (!row.top_key || greedy) {
    if (rank == 0 && threadIdx.x == 0) {
      if (!row.top_key) answer(p, r, -1.f, __int_as_float(0xff800000), 0);
      else answer(p, r, (float)index_of(best), 0.f, 1);
    }
    return;
  }
  row.top = value_of(row.top_key);
  Weigh weigh;
  weigh.top = row.top;
  weigh.pow2 = pow2;
  const double log2e_t = 1.4426950408889634 / (double)temp;
  {
    const double c = fmin(log2e_t, (double)FLT_MAX);  // (finite for every T that is not subnormal)
    weigh.chi = (float)c;
    weigh.clo = (float)(c - (double)weigh.chi);
  }
  const float pf = p.top_p ? p.top_p[r] : 1.f, mf = p.min_p ? p.min_p[r] : 0.f;
  const float uf = p.uniform[r];
  const double u = uf > 0.f ? (double)fminf(uf, 0.99999994f) : 0.0;
  // min-p compares probabilities by their logits: their weights are rounded, and small
  // ones have few bits or none
  const bool min_p = mf > 0.f;
  const double deepest = min_p ? -log2((double)fminf(mf, 1.f)) : 0.0;  // octaves below the largest
  auto likely = [&](float v) { return v == row.top || ((double)row.top - (double)v) * log2e_t <= deepest; };
  auto logprob_of = [&](float v, u64 total) {
    const double own = v == row.top ? 0.0 : ((double)v - (double)row.top) / (double)temp;
    return (float)(own - log((double)total * (1.0 / (double)(1ull << ONE_BITS))));
  };
  auto mass_target = [&](u64 total) {  // of top-p, in [1, total]
    const double want = ceil((double)fmaxf(pf, 0.f) * (double)total);
    const u64 t = want < 1.0 ? 1ull : (u64)want;
    return t < total ? t : total;
  };

  if (listed) {
    // ---- the first CTA sorts the candidates, best first, and does the rest
    if (rank) return;
    const u64 *sorted = reinterpret_cast<const u64 *>(s.part[0]);
    float least_bound = s.bound[0];
    for (int c = 1; c < ctas; ++c) least_bound = fmaxf(least_bound, s.bound[c]);
    uint32_t n = sort_list<THREADS>(ctas, room, s.found, least_bound, s);
    const uint32_t i = threadIdx.x;
    n = min(n, (uint32_t)kf);  // <= THREADS
    const u64 mine = i < n ? sorted[i] : 0;
    const uint32_t key = (uint32_t)(mine >> 32);
    const u64 w = i < n ? weigh(value_of(key)) : 0;
    u64 total;
    const u64 sum = block_scan(w, s, total);
    if (pf < 1.f) n = __syncthreads_count(i < n && sum - w < mass_target(total));
    if (min_p) n = __syncthreads_count(i < n && likely(value_of(key)));
    s.list[i] = w;
    if (i + 1 == n) s.above = sum;  // the kept total
    __syncthreads();
    total = s.above;
    u64 target = (u64)(u * (double)total);
    if (target >= total) target = total - 1;
    if (i < n) {
      u64 upto = 0;  // the kept mass of the tokens up to this one
      for (uint32_t j = 0; j < n; ++j)
        if ((uint32_t)sorted[j] >= (uint32_t)mine) upto += s.list[j];
      if (upto > target && upto - w <= target)
        answer(p, r, (float)index_of(mine), logprob_of(value_of(key), total), n);
    }
    return;
  }

  // ---- the cuts
  Cut cut{0, 0, 0};  // every live token (their places are above 0)
  if (kf >= 1.f && floorf(kf) < (float)live)
    cut_at<false, THREADS>(row, [&](u64) { return (u64)kf; }, weigh, s, cluster, cut);
  if (pf < 1.f) cut_at<true, THREADS>(row, mass_target, weigh, s, cluster, cut);
  if (min_p) {  // probabilities fall with the key: the smallest that is likely enough
    uint32_t l = LOWEST, h = row.top_key;
    while (l < h) {
      const uint32_t m = l + (h - l) / 2;
      if (likely(value_of(m))) h = m;
      else l = m + 1;
    }
    const u64 light = ((u64)l << 32) - 1;
    cut.over = cut.over > light ? cut.over : light;
    if (cut.tau < l) cut.ties = 0;
  }
  const u64 wt = cut.ties ? weigh(value_of(cut.tau)) : 0;
  const Over over(cut.over);

  // ---- kept mass and ties of every warp's stretch of the CTA's part
  const uint32_t stretch = ((row.n + WARPS - 1) / WARPS + 3) & ~3u;
  const uint32_t s0 = min(row.n, warp * stretch), s1 = min(row.n, s0 + stretch);
  const uint32_t tie_key = cut.ties ? cut.tau : 0;
  {
    u64 mass = 0;
    uint32_t tied = 0, count = 0;
    auto add = [&](float v, uint32_t i) {
      if (over(v, row.first + i)) {
        mass += weigh(v);
        ++count;
      } else if (tie_key && key_of(v) == tie_key) {
        ++tied;
      }
    };
    for_each<32>(row.v, s0, s1, add, nullptr, lane);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
      tied += __shfl_xor_sync(0xffffffffu, tied, o);
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    __syncthreads();
    if (lane == 0) s.warp_mass[warp] = mass, s.warp_ties[warp] = tied, s.warp_count[warp] = count;
    __syncthreads();
    if (threadIdx.x < (unsigned)ctas) {
      Shared<THREADS> *o = cluster.map_shared_rank(&s, threadIdx.x);
      u64 m = 0;
      uint32_t t = 0, c = 0;
      for (int w = 0; w < WARPS; ++w) m += s.warp_mass[w], t += s.warp_ties[w], c += s.warp_count[w];
      o->mass[rank] = m;
      o->ties[rank] = t;
      o->kept[rank] = c;
    }
  }
  cluster.sync();  // (the last one: nothing remote is touched after it)
  // the order's running sums: over the CTAs, then over the warps' stretches of the
  // CTA that holds the token
  u64 total = 0, left = cut.ties;
  uint32_t count = 0;
  for (int c = 0; c < ctas; ++c) {
    const u64 take = left < s.ties[c] ? left : s.ties[c];
    total += s.mass[c] + take * wt;
    count += s.kept[c] + (uint32_t)take;
    left -= take;
  }
  u64 target = (u64)(u * (double)total);  // the first sum above it
  if (target >= total) target = total - 1;
  u64 run = 0;
  left = cut.ties;
  int owner = 0;
  for (;; ++owner) {
    const u64 take = left < s.ties[owner] ? left : s.ties[owner], m = s.mass[owner] + take * wt;
    if (target < run + m) break;
    run += m;
    left -= take;
  }
  if (rank != owner) return;
  int w = 0;
  u64 quota = 0;  // ties that stay in the stretch
  for (;; ++w) {
    quota = left < s.warp_ties[w] ? left : s.warp_ties[w];
    const u64 m = s.warp_mass[w] + quota * wt;
    if (target < run + m) break;
    run += m;
    left -= quota;
  }
  // a few neighbouring tokens of the stretch a thread
  const uint32_t b0 = min(row.n, w * stretch), b1 = min(row.n, b0 + stretch);
  const uint32_t each = (b1 - b0 + THREADS - 1) / THREADS;
  const uint32_t t0 = min(b1, b0 + threadIdx.x * each), t1 = min(b1, t0 + each);
  u64 mass = 0, tied = 0, unused;
#pragma unroll 4
  for (uint32_t i = t0; i < t1; ++i) {
    const float v = row.v[i];
    if (over(v, row.first + i)) mass += weigh(v);
    else if (tie_key && key_of(v) == tie_key) ++tied;
  }
  u64 ties_before = tie_key ? block_scan(tied, s, unused) - tied : 0;
  const u64 mine = ties_before >= quota ? 0 : tied < quota - ties_before ? tied : quota - ties_before;
  mass += mine * wt;
  u64 sum = run + block_scan(mass, s, unused) - mass;
  if (target < sum || target >= sum + mass) return;
  for (uint32_t i = t0; i < t1; ++i) {
    const float v = row.v[i];
    u64 weight = 0;
    if (over(v, row.first + i)) weight = weigh(v);
    else if (tie_key && key_of(v) == tie_key && ties_before++ < quota) weight = wt;
    sum += weight;
    if (sum > target) {
      answer(p, r, (float)(row.first + i), logprob_of(v, total), count);
      return;
    }
  }
}

template <int THREADS, bool STAGED>
static cudaError_t launch_sample_kernel(const SampleArgs &a, uint32_t ctas, uint32_t chunk, int dev,
                                        cudaStream_t stream) {
  auto *kern = mgb_sample_kernel<THREADS, STAGED>;
  if (STAGED) {  // the opt-in is an attribute of the function on a device: once each
    static std::atomic<uint64_t> opted{0};
    if (!(opted.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024);
      if (e != cudaSuccess) return e;
      opted.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = STAGED ? chunk * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  // a grid holds 2^31 - 1 CTAs
  const uint64_t most = 0x7FFFFFFFull / ctas;
  for (uint64_t r = 0; r < a.rows; r += most) {
    SampleArgs part = a;
    part.rows = a.rows - r < most ? a.rows - r : most;
    part.logits += r * a.ld;
    for (const float **q : {&part.temperature, &part.top_k, &part.top_p, &part.min_p, &part.uniform})
      if (*q) *q += r;
    if (part.ids) part.ids += r;
    if (part.logprob) part.logprob += r;
    if (part.kept) part.kept += r;
    cfg.gridDim = dim3((unsigned)(part.rows * ctas));
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, part, chunk);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t stream) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t sms = (uint64_t)device_sms(dev);
  // Rows that fill the SMs by themselves: CTAs of 512 threads, two an SM.  Two of
  // them a row, so that rows with little to do leave their SMs to the others.
  if (a.rows > sms / 2 && a.vocab >= 4096) {
    uint32_t ctas = 2;
    while (ceil_div(a.vocab, ctas) > MOST_TOKENS) ctas *= 2;
    const uint32_t chunk = (uint32_t)(ceil_div(ceil_div(a.vocab, ctas), 4) * 4);
    return launch_sample_kernel<512, false>(a, ctas, chunk, dev, stream);
  }
  // Fewer: a cluster each, parts of up to 16,384 tokens (64 KB), and as many CTAs
  // as leave each 2,048.
  uint32_t ctas = 1;
  while (ctas < MOST_CTAS && (ceil_div(a.vocab, ctas) > 16384 ||
                              (a.rows * ctas * 2 <= sms && ceil_div(a.vocab, 2 * ctas) >= 2048)))
    ctas *= 2;
  const uint32_t chunk = (uint32_t)(ceil_div(ceil_div(a.vocab, ctas), 4) * 4);
  if (chunk <= 48 * 1024) return launch_sample_kernel<256, true>(a, ctas, chunk, dev, stream);
  return launch_sample_kernel<256, false>(a, ctas, chunk, dev, stream);
}

}  // namespace mgb
