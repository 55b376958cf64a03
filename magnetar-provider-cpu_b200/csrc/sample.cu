// One token per row of logits from given random numbers: temperature, top-k,
// top-p and min-p, then a draw in index order.
//
// Order.  Logits are compared as 32-bit keys (the float's bits made
// monotonic, -0 as +0; 0 for -inf and NaN, which are masked).  Every cut keeps
// a prefix of the tokens sorted by (key descending, index ascending), so what
// is kept is described by a key tau and how many tokens of key tau (the lowest
// indices) stay: no sort of the vocabulary is needed, only the search for tau.
//
// A row is read once: a cluster of CTAs holds it in shared memory (a few CTAs an
// SM, so that one row's loads overlap another's arithmetic), and the CTAs agree
// on one number after another through distributed shared memory.
//  - Small top_k: the top_k-th largest of a CTA's 256 threads' own largest logits
//    is a bound that at least top_k of its tokens reach and few others do; the
//    first CTA sorts the tokens that reach their CTA's and does the rest: one
//    cluster barrier a row.
//  - Otherwise tau is searched by histograms of counts (top-k) or of mass (top-p)
//    over ever smaller key ranges: first by distance to the largest logit, where
//    tokens spread evenly over the bins, then by key.
//
// Mass.  A token's weight is 2^((logit - max) log2(e) / T) as a 64-bit integer
// in units of 2^-43: integer sums are the same in every order, so atomics and
// any split of a row give the same token, and a border is only missed where
// weights round (2^-31 relative).  2^20 tokens of weight 1 stay below 2^63.
#include <cooperative_groups.h>

#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace mgb {

namespace cg = cooperative_groups;

constexpr int ONE_BITS = 43;  // weight 1

// 2^(j / 64): the nearest multiple of 2^-23 (in those units) and the rest.
struct Pow2Table {
  uint32_t hi[64];
  float lo[64];
};
__constant__ Pow2Table g_pow2 = {
    {
     8388608u, 8479954u, 8572295u, 8665641u, 8760003u, 8855394u, 8951823u, 9049301u,
     9147842u, 9247455u, 9348154u, 9449948u, 9552851u, 9656875u, 9762032u, 9868333u,
     9975792u, 10084422u, 10194234u, 10305242u, 10417458u, 10530897u, 10645571u, 10761494u,
     10878679u, 10997140u, 11116891u, 11237946u, 11360319u, 11484025u, 11609078u, 11735492u,
     11863283u, 11992466u, 12123055u, 12255067u, 12388516u, 12523418u, 12659789u, 12797645u,
     12937002u, 13077877u, 13220286u, 13364245u, 13509772u, 13656884u, 13805598u, 13955931u,
     14107901u, 14261526u, 14416824u, 14573813u, 14732511u, 14892937u, 15055111u, 15219050u,
     15384775u, 15552304u, 15721658u, 15892855u, 16065917u, 16240863u, 16417715u, 16596492u},
    {
     0.00000000e+00f, -5.71160541e-09f, -4.81155986e-08f, -2.80908932e-08f, 4.83347016e-08f,
     -4.90716943e-08f, -5.93375198e-08f, 5.46159455e-08f, -1.30775399e-08f, 4.26050200e-08f,
     -5.43554002e-08f, 3.12364143e-08f, 5.38622231e-08f, 2.19222827e-08f, -4.05144149e-08f,
     2.56697508e-08f, 3.79763527e-08f, -5.06975653e-08f, -3.26739489e-08f, -4.13620036e-08f,
     4.49683810e-08f, 7.32223748e-09f, 1.41933332e-09f, -3.81662169e-08f, -4.01899953e-08f,
     -3.49657157e-08f, -3.49637332e-08f, -3.46167397e-08f, -1.01233493e-08f, -3.84588184e-08f,
     -5.87557736e-08f, 8.68943406e-09f, 2.42032350e-08f, -1.34299292e-08f, 3.32419994e-08f,
     -3.62865755e-08f, -4.50089885e-08f, -3.42362014e-08f, -2.49593732e-08f, -1.76285688e-08f,
     8.07090483e-09f, -2.57646651e-08f, -5.66102543e-08f, -4.90313679e-10f, 9.83621717e-09f,
     -1.72600831e-08f, -5.12497209e-08f, -3.92029875e-08f, -2.47553267e-08f, -2.86514723e-08f,
     -4.84961760e-08f, -5.85022342e-08f, -9.23577037e-09f, 5.34319788e-08f, -1.14150449e-08f,
     3.73625824e-08f, -1.12392780e-08f, 1.43656118e-08f, -4.66300563e-08f, 2.81033845e-08f,
     9.84532811e-09f, 5.35707230e-08f, -1.70218044e-08f, 6.03272632e-09f}};

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
  const uint2 *pow2;    // g_pow2 in shared memory (lanes look different entries up,
                        // which constant memory serves one after the other: 562
                        // against PLACEHOLDER us for 256 rows of 128,256)
  __device__ __forceinline__ uint64_t operator()(float v) const {
    if (__isinff(top)) return v == top ? 1ull << ONE_BITS : 0;  // +inf
    // v - top = d + e exactly; times (chi + clo): p + r
    const float d = v - top, b = d - v;
    const float e = (v - (d - b)) + (-top - b);
    const float p = d * chi;
    if (!(p > -60.f)) return 0;  // below half a unit (also v = -inf, NaN)
    float r = fmaf(d, chi, -p);
    r = fmaf(d, clo, r);
    r = fmaf(e, chi, r);
    // 2^(p + r) = 2^N 2^(j / 64) 2^s, |s| <= 1/128; the last factor by its
    // Taylor polynomial (next term 2^-44)
    const float n = rintf(p * 64.f);
    const float s = fmaf(n, -0.015625f, p) + r;
    float q = fmaf(s, 0.009618129107628f, 0.055504108664822f);
    q = fmaf(s, q, 0.240226506959101f);
    q = fmaf(s, q, 0.693147180559945f);
    q *= s;
    const int ni = (int)n, j = ni & 63, N = ni >> 6;
    const uint2 power = pow2[j];
    const float hi = (float)power.x * 1.1920929e-7f;  // exact
    const int32_t tail = __float2int_rn(fmaf(hi, q, __uint_as_float(power.y)) * 68719476736.f);  // 2^36
    const uint64_t one = ((uint64_t)power.x << (ONE_BITS - 23)) +
                         (uint64_t)((int64_t)tail << (ONE_BITS - 36));
    if (N >= 0) return one << N;  // s may round p up to 0
    return (one + (1ull << (-N - 1))) >> -N;
  }
};

constexpr int BINS = 1024;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MOST_CTAS = 8;      // of a cluster
constexpr int LIST = 1024;        // candidates the first CTA sorts
constexpr int MOST_TOP_K = THREADS;  // of the candidate path
constexpr uint32_t LOWEST = 0x00800000u;  // the key of the lowest finite value
constexpr float BIN_SCALE = 16.f;    // bins of the distance to the largest logit

// The bin of a live logit by its distance to the largest one: monotonic.
__device__ __forceinline__ int distance_bin(float top, float v) {
  const int b = (int)((top - v) * BIN_SCALE);  // (saturates)
  return b < BINS - 1 ? b : BINS - 1;
}

struct Shared {
  unsigned long long list[LIST];        // the first CTA: its cluster's candidates; a histogram
  alignas(8) uint32_t part[3][BINS];    // a histogram as it is filled (32-bit atomics are native:
                                        // masses in three digits); the sort's buffer
  unsigned long long scan[WARPS];
  // what the CTAs tell each other, by rank
  unsigned long long top[MOST_CTAS];    // (key, ~index) of the largest logit
  unsigned long long mass[MOST_CTAS], cut_mass[MOST_CTAS];
  uint32_t live[MOST_CTAS], found[MOST_CTAS], ties[MOST_CTAS], count[MOST_CTAS];
  // the first CTA's answers
  unsigned long long found_above;
  uint32_t lo, hi;
  // of the CTA
  unsigned long long warp_mass[WARPS];
  unsigned long long above;
  uint32_t warp_ties[WARPS], warp_count[WARPS], own[THREADS], taken, bin;
};

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, Shared &s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = v > u ? v : u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v = v > s.scan[w] ? v : s.scan[w];
  return v;
}

// Inclusive sum over the CTA's threads.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, Shared &s,
                                                         unsigned long long &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) s.scan[warp] = v;
  __syncthreads();
  total = 0;
  unsigned long long before = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s.scan[w];
    total += s.scan[w];
  }
  return before + v;
}

// The first bin at which the running sum of hist reaches target, and the sum
// before it; all threads (sums of `hist`, which 4 bins a thread).
__device__ __forceinline__ void find_bin(const unsigned long long *hist, unsigned long long target,
                                         Shared &s, int &bin, unsigned long long &before) {
  unsigned long long c[BINS / THREADS], v = 0, total;
#pragma unroll
  for (int i = 0; i < BINS / THREADS; ++i) c[i] = hist[threadIdx.x * (BINS / THREADS) + i], v += c[i];
  unsigned long long run = block_scan(v, s, total) - v;
#pragma unroll
  for (int i = 0; i < BINS / THREADS; ++i) {
    if (run < target && run + c[i] >= target)
      s.bin = threadIdx.x * (BINS / THREADS) + i, s.above = run;
    run += c[i];
  }
  __syncthreads();
  bin = (int)s.bin;
  before = s.above;
}

struct Row {
  const float *v;      // this CTA's part of the row
  uint32_t first, n;   // index of its first token, tokens
  float top;           // the row's largest logit
  uint32_t top_key;
};

// A mass in three digits of a histogram: a CTA's part of at most 2^17 tokens (a
// row of 2^20 in 8 CTAs) keeps the sums of 15-bit digits below 2^32; a mass is
// below 2^45.
constexpr int DIGIT = 15;

// The largest key in [lo, hi] at which the count (MASS: the mass) of the keys from
// hi down to it reaches `target` (>= 1, at most what [lo, hi] holds); above: the
// count or mass of the keys over it.  The whole cluster.
template <bool MASS>
__device__ uint32_t find_key(const Row &row, uint32_t lo, uint32_t hi, unsigned long long target,
                             const Weigh &weigh, Shared &s, cg::cluster_group &cluster,
                             unsigned long long &above) {
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  bool linear = !__isinff(row.top);
  above = 0;
  while (lo < hi) {
    int shift = 0;
    while (((hi - lo) >> shift) >= BINS) ++shift;
    for (int i = threadIdx.x; i < BINS; i += THREADS)
#pragma unroll
      for (int d = 0; d < (MASS ? 3 : 1); ++d) s.part[d][i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < row.n; i += THREADS) {
      const float v = row.v[i];
      const uint32_t key = key_of(v);
      if (key < lo || key > hi) continue;
      const int b = linear ? distance_bin(row.top, v) : (int)((hi - key) >> shift);
      if (MASS) {
        const uint64_t w = weigh(v);
        const uint32_t d0 = (uint32_t)w & ((1u << DIGIT) - 1), d1 = (uint32_t)(w >> DIGIT) & ((1u << DIGIT) - 1),
                       d2 = (uint32_t)(w >> (2 * DIGIT));
        if (d0) atomicAdd(&s.part[0][b], d0);
        if (d1) atomicAdd(&s.part[1][b], d1);
        if (d2) atomicAdd(&s.part[2][b], d2);
      } else {
        atomicAdd(&s.part[0][b], 1u);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += THREADS)
      s.list[i] = MASS ? s.part[0][i] + ((unsigned long long)s.part[1][i] << DIGIT) +
                             ((unsigned long long)s.part[2][i] << (2 * DIGIT))
                       : s.part[0][i];
    cluster.sync();
    if (rank == 0) {
      unsigned long long c[BINS / THREADS];
#pragma unroll
      for (int j = 0; j < BINS / THREADS; ++j) c[j] = 0;
      for (int o = 0; o < ctas; ++o) {
        const unsigned long long *h = cluster.map_shared_rank(s.list, o);
#pragma unroll
        for (int j = 0; j < BINS / THREADS; ++j) c[j] += h[j * THREADS + threadIdx.x];
      }
      unsigned long long *all = reinterpret_cast<unsigned long long *>(s.part[0]);  // [BINS]: two of three
#pragma unroll
      for (int j = 0; j < BINS / THREADS; ++j) all[j * THREADS + threadIdx.x] = c[j];
      __syncthreads();
      int bin;
      unsigned long long before;
      find_bin(all, target - above, s, bin, before);
      if (threadIdx.x < (unsigned)ctas) {
        uint32_t nlo = lo, nhi = hi;
        if (linear) {
          // bins fall as keys grow: the keys of the bin, by bisection
          auto edge = [&](int b) {  // the smallest key in [lo, hi] whose bin is at most b
            uint32_t l = lo, h = hi;
            while (l < h) {
              const uint32_t m = l + (h - l) / 2;
              if (distance_bin(row.top, value_of(m)) <= b) h = m;
              else l = m + 1;
            }
            return l;
          };
          nlo = edge(bin);
          nhi = bin ? edge(bin - 1) - 1 : hi;
        } else {
          nhi = hi - ((uint32_t)bin << shift);
          const uint32_t width = (1u << shift) - 1;
          nlo = nhi - lo > width ? nhi - width : lo;
        }
        Shared *o = cluster.map_shared_rank(&s, threadIdx.x);
        o->lo = nlo;
        o->hi = nhi;
        o->found_above = above + before;
      }
    }
    cluster.sync();
    lo = s.lo;
    hi = s.hi;
    above = s.found_above;
    linear = false;
  }
  __syncthreads();
  return hi;
}

__device__ __forceinline__ void answer(const SampleArgs &p, uint64_t r, float id, float logprob,
                                       uint32_t kept) {
  if (p.ids) p.ids[r] = id;
  if (p.logprob) p.logprob[r] = logprob;
  if (p.kept) p.kept[r] = kept;
}

// One row a cluster.  STAGED: each CTA's part of the row is in its shared memory;
// otherwise (vocabularies that do not fit) it is read from global memory again.
template <bool STAGED>
__global__ void __launch_bounds__(THREADS, 3) mgb_sample_kernel(const SampleArgs p, uint32_t chunk) {
  __shared__ Shared s;
  __shared__ uint2 pow2[64];
  extern __shared__ __align__(16) float data[];
  if (threadIdx.x < 64) pow2[threadIdx.x] = make_uint2(g_pow2.hi[threadIdx.x], __float_as_uint(g_pow2.lo[threadIdx.x]));
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

  // the CTA's largest (key, ~index) and live tokens; the row comes in once
  unsigned long long best = 0;
  uint32_t live = 0;
  auto see = [&](float v, uint32_t i) {
    const uint32_t key = key_of(v);
    live += key != 0;
    const unsigned long long c = ((unsigned long long)key << 32) | (0xFFFFFFFFu - (row.first + i));
    if (key && c > best) best = c;
  };
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const uint32_t n4 = row.n / 4;
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < n4; i += THREADS) {
      const float4 v = reinterpret_cast<const float4 *>(src)[i];
      if (STAGED) reinterpret_cast<float4 *>(data)[i] = v;
      see(v.x, 4 * i);
      see(v.y, 4 * i + 1);
      see(v.z, 4 * i + 2);
      see(v.w, 4 * i + 3);
    }
    for (uint32_t i = 4 * n4 + threadIdx.x; i < row.n; i += THREADS) {
      const float v = src[i];
      if (STAGED) data[i] = v;
      see(v, i);
    }
  } else {
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < row.n; i += THREADS) {
      const float v = src[i];
      if (STAGED) data[i] = v;
      see(v, i);
    }
  }
  row.v = STAGED ? data : src;
  const uint32_t own = (uint32_t)(best >> 32);  // this thread's largest key
  best = block_max(best, s);
  {
    unsigned long long total;
    block_scan(live, s, total);
    live = (uint32_t)total;
  }

  cluster.barrier_wait();

  // small top_k: this CTA's candidates, to the first CTA's list
  static_assert(LIST <= BINS && BINS * 8 <= sizeof(s.part), "the sort's buffer");
  const uint32_t room = LIST / ctas;
  const bool few = !greedy && kf >= 1.f && kf < (float)MOST_TOP_K + 1.f && kf < (float)room + 1.f;
  uint32_t found = 0xFFFFFFFFu;  // none sent
  if (few) {
    const uint32_t k = (uint32_t)kf;
    uint32_t bound = 1;  // every live token
    if (threadIdx.x == 0) s.taken = 0;
    if (live > room) {
      s.own[threadIdx.x] = own;
      __syncthreads();
      // the k-th largest of the threads' largest keys (k <= THREADS): the one with
      // fewer than k above it and k at least as large
      uint32_t over = 0, level = 0;
#pragma unroll 8
      for (int j = 0; j < THREADS; ++j) over += s.own[j] > own, level += s.own[j] == own;
      if (over < k && over + level >= k) s.bin = own;  // (equal keys agree)
      __syncthreads();
      bound = max(s.bin, 1u);
    } else {
      __syncthreads();
    }
    unsigned long long *list = cluster.map_shared_rank(s.list, 0) + rank * room;
    for (uint32_t i = threadIdx.x; i < row.n; i += THREADS) {
      const uint32_t key = key_of(row.v[i]);
      if (key >= bound) {
        const uint32_t at = atomicAdd(&s.taken, 1u);
        if (at < room) list[at] = ((unsigned long long)key << 32) | (0xFFFFFFFFu - (row.first + i));
      }
    }
    __syncthreads();
    found = s.taken;  // (above room: too many tokens reach the bound)
  }
  if (threadIdx.x < (unsigned)ctas) {
    Shared *o = cluster.map_shared_rank(&s, threadIdx.x);
    o->top[rank] = best;
    o->live[rank] = live;
    o->found[rank] = found;
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
      else answer(p, r, (float)(0xFFFFFFFFu - (uint32_t)best), 0.f, 1);
    }
    return;
  }
  row.top = value_of(row.top_key);
  Weigh weigh;
  weigh.top = row.top;
  weigh.pow2 = pow2;
  {
    const double c = fmin(1.4426950408889634 / (double)temp, 1e30);  // 1 / T stays finite
    weigh.chi = (float)c;
    weigh.clo = (float)(c - (double)weigh.chi);
  }
  const float pf = p.top_p ? p.top_p[r] : 1.f, mf = p.min_p ? p.min_p[r] : 0.f;
  const float uf = p.uniform[r];
  const double u = uf > 0.f ? (double)fminf(uf, 0.99999994f) : 0.0;
  const unsigned long long least =
      mf > 0.f ? (unsigned long long)ceil((double)fminf(mf, 1.f) * (double)(1ull << ONE_BITS)) : 0;
  auto mass_target = [&](unsigned long long total) {  // of top-p, in [1, total]
    const double want = ceil((double)fmaxf(pf, 0.f) * (double)total);
    const unsigned long long t = want < 1.0 ? 1ull : (unsigned long long)want;
    return t < total ? t : total;
  };

  if (listed) {
    // ---- the first CTA sorts the candidates, best first, and does the rest
    if (rank) return;
    unsigned long long *sorted = reinterpret_cast<unsigned long long *>(s.part[0]);  // [LIST]: two of three
    uint32_t n = 0;
    for (int c = 0; c < ctas; ++c) {
      for (uint32_t i = threadIdx.x; i < s.found[c]; i += THREADS) sorted[n + i] = s.list[c * room + i];
      n += s.found[c];
    }
    uint32_t size = 2;
    while (size < n) size <<= 1;
    for (uint32_t i = n + threadIdx.x; i < size; i += THREADS) sorted[i] = 0;
    __syncthreads();
    for (uint32_t k = 2; k <= size; k <<= 1)
      for (uint32_t j = k >> 1; j; j >>= 1) {
        for (uint32_t i = threadIdx.x; i < size / 2; i += THREADS) {
          const uint32_t a = 2 * i - (i & (j - 1)), b = a + j;
          const unsigned long long x = sorted[a], y = sorted[b];
          if ((x < y) == ((a & k) == 0)) sorted[a] = y, sorted[b] = x;
        }
        __syncthreads();
      }
    const uint32_t i = threadIdx.x;
    n = min(n, (uint32_t)kf);  // <= THREADS
    const unsigned long long mine = i < n ? sorted[i] : 0;
    const uint32_t key = (uint32_t)(mine >> 32), token = 0xFFFFFFFFu - (uint32_t)mine;
    const unsigned long long w = i < n ? weigh(value_of(key)) : 0;
    unsigned long long total;
    const unsigned long long sum = block_scan(w, s, total);
    if (pf < 1.f) n = __syncthreads_count(i < n && sum - w < mass_target(total));
    n = __syncthreads_count(i < n && (w >= least || key == row.top_key));
    s.list[i] = w;
    if (i + 1 == n) s.above = sum;  // the kept total
    __syncthreads();
    total = s.above;
    unsigned long long target = (unsigned long long)(u * (double)total);
    if (target >= total) target = total - 1;
    if (i < n) {
      unsigned long long upto = 0;  // the kept mass of the tokens up to this one
      for (uint32_t j = 0; j < n; ++j)
        if ((uint32_t)sorted[j] >= (uint32_t)mine) upto += s.list[j];
      if (upto > target && upto - w <= target)
        answer(p, r, (float)token, (float)(log((double)w) - log((double)total)), n);
    }
    return;
  }

  // ---- the cuts: everything above tau, and `ties` tokens of key tau
  uint32_t tau = 0;
  unsigned long long ties = 0, above;
  if (kf >= 1.f && floorf(kf) < (float)live) {
    const unsigned long long k = (unsigned long long)kf;
    tau = find_key<false>(row, LOWEST, row.top_key, k, weigh, s, cluster, above);
    ties = k - above;
  }
  if (pf < 1.f) {
    unsigned long long gt = 0, total;
    for (uint32_t i = threadIdx.x; i < row.n; i += THREADS) {
      const float v = row.v[i];
      if (key_of(v) > tau) gt += weigh(v);
    }
    block_scan(gt, s, total);
    if (threadIdx.x < (unsigned)ctas) cluster.map_shared_rank(&s, threadIdx.x)->cut_mass[rank] = total;
    cluster.sync();
    total = ties * (tau ? weigh(value_of(tau)) : 0);
    for (int c = 0; c < ctas; ++c) total += s.cut_mass[c];
    const unsigned long long target = mass_target(total);
    const uint32_t key = find_key<true>(row, tau ? tau : LOWEST, row.top_key, target, weigh, s, cluster, above);
    const unsigned long long w = weigh(value_of(key));
    const unsigned long long need = w ? (target - above + w - 1) / w : 1;
    ties = key == tau && ties < need ? ties : need;
    tau = key;
  }
  const unsigned long long wt = tau ? weigh(value_of(tau)) : 0;
  if (tau && tau != row.top_key && wt < least) ties = 0;

  // ---- kept mass and ties of every warp's stretch of the CTA's part
  const uint32_t stretch = (row.n + WARPS - 1) / WARPS;
  const uint32_t s0 = min(row.n, warp * stretch), s1 = min(row.n, s0 + stretch);
  auto kept = [&](float v, uint32_t key) {  // the weight of a token above tau, if it stays
    const unsigned long long w = weigh(v);
    return w >= least || key == row.top_key ? w : 0;
  };
  {
    unsigned long long mass = 0;
    uint32_t tied = 0, count = 0;
    for (uint32_t i = s0 + lane; i < s1; i += 32) {
      const float v = row.v[i];
      const uint32_t key = key_of(v);
      if (key > tau) {
        const unsigned long long w = weigh(v);
        const bool in = w >= least || key == row.top_key;
        mass += in ? w : 0;
        count += in;
      } else if (key && key == tau) {
        ++tied;
      }
    }
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
      Shared *o = cluster.map_shared_rank(&s, threadIdx.x);
      unsigned long long m = 0;
      uint32_t t = 0, c = 0;
      for (int w = 0; w < WARPS; ++w) m += s.warp_mass[w], t += s.warp_ties[w], c += s.warp_count[w];
      o->mass[rank] = m;
      o->ties[rank] = t;
      o->count[rank] = c;
    }
  }
  cluster.sync();  // (the last one: nothing remote is touched after it)
  unsigned long long total = 0, before = 0, left = ties;
  uint32_t count = 0, mine_ties = 0;
  for (int c = 0; c < ctas; ++c) {
    if (c == rank) {  // this warp's place in the order
      unsigned long long l = left;
      before = total;
      for (int w = 0; w < WARPS; ++w) {
        const unsigned long long take = l < s.warp_ties[w] ? l : s.warp_ties[w];
        if (w == warp) {
          mine_ties = (uint32_t)take;
          break;
        }
        before += s.warp_mass[w] + take * wt;
        l -= take;
      }
    }
    const unsigned long long take = left < s.ties[c] ? left : s.ties[c];
    total += s.mass[c] + take * wt;
    count += s.count[c] + (uint32_t)take;
    left -= take;
  }
  unsigned long long target = (unsigned long long)(u * (double)total);  // the first sum above it
  if (target >= total) target = total - 1;
  if (before > target || target >= before + s.warp_mass[warp] + mine_ties * wt) return;
  unsigned long long run = before;
  uint32_t tie_run = 0;
  for (uint32_t i0 = s0; i0 < s1; i0 += 32) {
    const uint32_t i = i0 + lane;
    const float v = i < s1 ? row.v[i] : 0.f;
    const uint32_t key = i < s1 ? key_of(v) : 0;
    const bool tie = key && key == tau;
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    unsigned long long w = 0;
    if (tie) w = tie_run + __popc(tie_mask & ((1u << lane) - 1)) < mine_ties ? wt : 0;
    else if (key > tau) w = kept(v, key);
    tie_run += __popc(tie_mask);
    unsigned long long sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, w && run + sum > target);
    if (hit) {
      if (lane == __ffs(hit) - 1)
        answer(p, r, (float)(row.first + i), (float)(log((double)w) - log((double)total)), count);
      return;
    }
    run += __shfl_sync(0xffffffffu, sum, 31);
  }
}

uint64_t sample_scratch_bytes(uint64_t, uint64_t) { return 0; }

cudaError_t launch_sample(const SampleArgs &a, void *, cudaStream_t stream) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int sms = device_sms(dev);
  // CTAs of a row: parts of up to 16,384 tokens (64 KB: three CTAs an SM), and,
  // with few rows, as many as leave each 2,048
  uint32_t ctas = 1;
  while (ctas < MOST_CTAS && (ceil_div(a.vocab, ctas) > 16384 ||
                              (a.rows * ctas * 2 <= (uint64_t)sms && ceil_div(a.vocab, 2 * ctas) >= 2048)))
    ctas *= 2;
  const uint32_t chunk = (uint32_t)(ceil_div(ceil_div(a.vocab, ctas), 4) * 4);
  const bool staged = chunk <= 48 * 1024;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = staged ? chunk * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  auto *kern = staged ? mgb_sample_kernel<true> : mgb_sample_kernel<false>;
  if (staged) {  // the opt-in is an attribute of the function on a device: once each
    static std::atomic<uint64_t> opted{0};
    if (!(opted.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 196608);
      if (e != cudaSuccess) return e;
      opted.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    }
  }
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
    e = cudaLaunchKernelEx(&cfg, kern, part, chunk);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mgb
