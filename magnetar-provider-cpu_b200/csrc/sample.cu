// One token per row of logits from given random numbers: temperature, top-k,
// top-p and min-p, then a draw in index order.
//
// Order.  Logits are compared as 32-bit keys (the float's bits made
// monotonic, -0 as +0; 0 for -inf and NaN, which are masked).  Every cut keeps
// a prefix of the tokens sorted by (key descending, index ascending), so what
// is kept is described by a key tau and how many tokens of key tau (the lowest
// indices) stay: no sort is needed, only the search for tau.  It is searched
// by histograms over key ranges, 2,048 bins a level, of counts (top-k) or of
// probability mass (top-p).
//
// Mass.  A token's weight is 2^((logit - max) log2(e) / T) as a 64-bit integer
// in units of 2^-43: integer sums are the same in every order, so atomics and
// any split of a row give the same token, and a border is only missed where
// weights round (2^-31 relative).  2^20 tokens of weight 1 stay below 2^63.
#include "common.cuh"
#include "kernels.h"

namespace mgb {

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
    const float hi = (float)g_pow2.hi[j] * 1.1920929e-7f;  // exact
    const int32_t tail = __float2int_rn(fmaf(hi, q, g_pow2.lo[j]) * 68719476736.f);  // 2^36
    const uint64_t one = ((uint64_t)g_pow2.hi[j] << (ONE_BITS - 23)) +
                         (uint64_t)((int64_t)tail << (ONE_BITS - 36));
    if (N >= 0) return one << N;  // s may round p up to 0
    return (one + (1ull << (-N - 1))) >> -N;
  }
};

constexpr int BINS = 2048;
constexpr int THREADS = 1024;

struct Found {
  uint32_t key;
  uint64_t above;  // count or mass of the keys above it
};

// The largest key in [lo, hi] at which the count (MASS: the mass) of the keys
// from hi down to it reaches `target` (>= 1, at most what [lo, hi] holds).
template <bool MASS>
__device__ Found find_key(const float *__restrict__ row, uint32_t vocab, uint32_t lo, uint32_t hi,
                          uint64_t target, const Weigh &weigh, uint64_t *hist) {
  __shared__ uint64_t s_above, s_warp[THREADS / 32];
  __shared__ uint32_t s_bin;
  uint64_t above = 0;
  while (lo < hi) {
    int shift = 0;
    while (((hi - lo) >> shift) >= BINS) ++shift;
    for (int i = threadIdx.x; i < BINS; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < vocab; t += THREADS) {
      const float v = row[t];
      const uint32_t key = key_of(v);
      if (key < lo || key > hi || !key) continue;
      atomicAdd((unsigned long long *)&hist[(hi - key) >> shift], MASS ? weigh(v) : 1ull);
    }
    __syncthreads();
    // inclusive sums from the highest bin; two bins a thread
    const uint64_t a = hist[2 * threadIdx.x], b = hist[2 * threadIdx.x + 1];
    uint64_t s = a + b;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    if (lane == 31) s_warp[warp] = s;
    __syncthreads();
    uint64_t before = above;
    for (int w = 0; w < warp; ++w) before += s_warp[w];
    const uint64_t end = before + s, start = end - a - b;
    if (start < target && end >= target) {
      const bool second = start + a < target;
      s_bin = 2 * threadIdx.x + second;
      s_above = second ? start + a : start;
    }
    __syncthreads();
    above = s_above;
    const uint32_t bin = s_bin;
    hi = hi - (bin << shift);
    const uint32_t width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    __syncthreads();
  }
  return {hi, above};
}

template <typename T>
__device__ T block_sum(T v, T *scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  T s = 0;
  for (int w = 0; w < THREADS / 32; ++w) s += scratch[w];
  return s;
}

__global__ void __launch_bounds__(THREADS) mgb_sample_kernel(const SampleArgs p) {
  __shared__ uint64_t hist[BINS];
  __shared__ uint64_t scratch[THREADS / 32], seg_mass[THREADS / 32];
  __shared__ uint32_t seg_ties[THREADS / 32], s_low;
  __shared__ uint32_t s_max;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t vocab = (uint32_t)p.vocab;
  for (uint64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const float *row = p.logits + r * p.ld;
    __syncthreads();
    if (threadIdx.x == 0) s_max = 0, s_low = 0xFFFFFFFFu;
    __syncthreads();
    uint32_t mx = 0;
    uint64_t live = 0;
    for (uint32_t t = threadIdx.x; t < vocab; t += THREADS) {
      const uint32_t key = key_of(row[t]);
      mx = max(mx, key);
      live += key != 0;
    }
    atomicMax(&s_max, mx);
    live = block_sum(live, scratch);
    const uint32_t top = s_max;
    if (!top) {
      if (threadIdx.x == 0) {
        if (p.ids) p.ids[r] = -1.f;
        if (p.logprob) p.logprob[r] = __int_as_float(0xff800000);
        if (p.kept) p.kept[r] = 0;
      }
      continue;
    }
    const float temp = p.temperature ? p.temperature[r] : 1.f;
    if (!(temp > 0.f) || !p.uniform) {
      for (uint32_t t = threadIdx.x; t < vocab; t += THREADS)
        if (key_of(row[t]) == top) {
          atomicMin(&s_low, t);
          break;
        }
      __syncthreads();
      if (threadIdx.x == 0) {
        if (p.ids) p.ids[r] = (float)s_low;
        if (p.logprob) p.logprob[r] = 0.f;
        if (p.kept) p.kept[r] = 1;
      }
      continue;
    }
    Weigh weigh;
    weigh.top = value_of(top);
    // 1 / T stays finite
    const double c = fmin(1.4426950408889634 / (double)temp, 1e30);
    weigh.chi = (float)c;
    weigh.clo = (float)(c - (double)weigh.chi);

    // top-k
    uint32_t tau = 1;  // every live key
    uint64_t ties = vocab;
    const float kf = p.top_k ? p.top_k[r] : 0.f;
    if (kf >= 1.f && floorf(kf) < (float)live) {
      const uint64_t k = (uint64_t)kf;
      const Found f = find_key<false>(row, vocab, 1, top, k, weigh, hist);
      tau = f.key;
      ties = k - f.above;
    }
    // top-p
    const float pf = p.top_p ? p.top_p[r] : 1.f;
    if (pf < 1.f) {
      uint64_t gt = 0;
      for (uint32_t t = threadIdx.x; t < vocab; t += THREADS) {
        const float v = row[t];
        const uint32_t key = key_of(v);
        if (key > tau || (key == tau && tau == 1)) gt += weigh(v);
      }
      uint64_t total = block_sum(gt, scratch);
      if (tau > 1) total += ties * weigh(value_of(tau));
      const double want = ceil((double)fmaxf(pf, 0.f) * (double)total);
      uint64_t target = want < 1.0 ? 1 : (uint64_t)want;
      if (target > total) target = total;
      const Found f = find_key<true>(row, vocab, tau, top, target, weigh, hist);
      const uint64_t w = weigh(value_of(f.key));
      const uint64_t need = w ? (target - f.above + w - 1) / w : 1;
      ties = f.key == tau ? min(ties, need) : need;
      tau = f.key;
    }
    const float mf = p.min_p ? p.min_p[r] : 0.f;
    const uint64_t least =
        mf > 0.f ? (uint64_t)ceil((double)fminf(mf, 1.f) * (double)(1ull << ONE_BITS)) : 0;
    if (tau == 1) ties = 0, tau = 0;  // no cut: every live key is above tau
    if (tau && tau != top && weigh(value_of(tau)) < least) ties = 0;
    const uint64_t wt = tau ? weigh(value_of(tau)) : 0;

    // one contiguous segment a warp: kept mass and ties
    const uint32_t seg = (vocab + THREADS / 32 - 1) / (THREADS / 32);
    const uint32_t s0 = min(vocab, warp * seg), s1 = min(vocab, s0 + seg);
    uint64_t mass = 0, count = 0;
    uint32_t tied = 0;
    for (uint32_t t = s0 + lane; t < s1; t += 32) {
      const float v = row[t];
      const uint32_t key = key_of(v);
      if (!key || key < tau) continue;
      if (key == tau) {
        ++tied;
        continue;
      }
      const uint64_t w = weigh(v);
      if (w < least && key != top) continue;
      mass += w;
      ++count;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
      tied += __shfl_xor_sync(0xffffffffu, tied, o);
    }
    if (lane == 0) seg_mass[warp] = mass, seg_ties[warp] = tied;
    count = block_sum(count, scratch);
    uint64_t total = 0, before = 0, mine = 0, mine_ties = 0, left = ties;
    for (int w = 0; w < THREADS / 32; ++w) {
      const uint64_t take = min(left, (uint64_t)seg_ties[w]);
      if (w == warp) before = total, mine = seg_mass[w] + take * wt, mine_ties = take;
      left -= take;
      total += seg_mass[w] + take * wt;
    }
    const float uf = p.uniform[r];
    const double u = uf > 0.f ? (double)fminf(uf, 0.99999994f) : 0.0;
    uint64_t target = (uint64_t)(u * (double)total);  // the first running sum above it
    if (target >= total) target = total - 1;
    if (before <= target && target < before + mine) {
      uint64_t run = before;
      uint32_t tie_run = 0;
      for (uint32_t t0 = s0; t0 < s1; t0 += 32) {
        const uint32_t t = t0 + lane;
        const float v = t < s1 ? row[t] : 0.f;
        const uint32_t key = t < s1 ? key_of(v) : 0;
        const bool tie = key && key == tau;
        const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
        uint64_t w = 0;
        if (tie) w = tie_run + __popc(tie_mask & ((1u << lane) - 1)) < mine_ties ? wt : 0;
        else if (key > tau) {
          w = weigh(v);
          if (w < least && key != top) w = 0;
        }
        tie_run += __popc(tie_mask);
        uint64_t s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t up = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += up;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, w && run + s > target);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            if (p.ids) p.ids[r] = (float)t;
            if (p.logprob) p.logprob[r] = (float)(log((double)w) - log((double)total));
          }
          break;
        }
        run += __shfl_sync(0xffffffffu, s, 31);
      }
    }
    if (threadIdx.x == 0 && p.kept) p.kept[r] = (uint32_t)(count + (ties - left));
  }
}

uint64_t sample_scratch_bytes(uint64_t, uint64_t) { return 0; }

cudaError_t launch_sample(const SampleArgs &a, void *, cudaStream_t stream) {
  mgb_sample_kernel<<<(unsigned)(a.rows < 65535 ? a.rows : 65535), THREADS, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace mgb
