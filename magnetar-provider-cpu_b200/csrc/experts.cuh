// The packed products of a mixture-of-experts layer for a few tokens, on the
// 5th-generation tensor cores.
//
// Every expert that a token chose has its packed rows streamed once for up to T
// of its tokens: 128 weight rows are the MMA's M, the tokens its N.  With so few
// tokens the weight stream is the work, so what counts is how few instructions
// a weight costs and that nothing stands between the stream and the tensor core.
//
// Weights.  A thread owns a weight row.  Its codes become f16 integers without
// rounding: a code masked out of its quant word is an f16 subnormal (q 2^-24, or
// 16 times that for the next nibble), one f16 multiply by the run's integer
// scale (Q4_K, Q5_K: sc q <= 1953 < 2048) or one multiply-add with the code's
// offset gives an exact number.  Two codes a register, written to TMEM
// (tcgen05.st) as the A operand: nothing goes back through shared memory.  What
// is left of a weight's scale is one f32 factor per row and 256 values (K
// formats) or per row and 32 values (the others), which multiplies the MMA's
// result as it is read from TMEM into the row's f32 sums.  Q6_K's products
// sc (q - 32) need 13 bits: they enter as two operands, sc n of the low nibble
// and 16 sc (h - 2) of the two high bits, which so need no joining (one token of
// two wide experts: 132 us with joined codes split by their lowest bit, 112 us so).
// Q4_K's and Q5_K's mins multiply the runs' activation sums, by one more MMA a
// block (8 runs, two terms each).
//
// Activations.  A row is held as 2^-k (hi + lo), two f16 terms with k such that
// the row's largest value lies in [2^13, 2^14): 22 bits of every value down to
// 2^-27 of the largest.  hi and lo are separate columns of N, added in f32.
//
// Work is split by stages of 256 columns (128 for the wider formats): the stages
// of all row tiles form one sequence, of which every CTA takes an equal part.  A
// tile whose stages fall to several CTAs gets a partial result from each; the
// kernel that reads the product adds them in order.
//
// Measured on the device: 64 tokens, 8 experts of 4,096 x 14,336, Q4_K and Q5_K 475 to
// 480 us the layer (132 at the copy's rate of the packed bytes); 16 tokens on 64 experts
// of 4,096 x 1,536, Q8_0, 270 us (175); one token on two wide experts 111 us (36).  Bound by
// instruction issue (2.4 to 2.6 a cycle and SM, 3.6 lane instructions a Q4_K weight,
// 6.8 a Q6_K one) and, for one token, by what every launch takes before its first
// weight.  Smaller steps with two A operands in TMEM: 143 us and 644 us instead of
// 130 and 540 at the time; a run unpacked before the wait: no gain.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace mgb {
namespace moe {

constexpr int TILE = 128;      // weight rows of a tile
constexpr int THREADS = 160;   // four warps of rows, one that feeds the tensor core
constexpr int MAX_PARTS = 8;   // a tile is cut into at most one more

__host__ __device__ constexpr bool k_format(int f) { return f == Q4_K || f == Q5_K || f == Q6_K; }
__host__ __device__ constexpr bool has_min(int f) { return f == Q4_K || f == Q5_K; }

// ---- activations ---------------------------------------------------------------------------

// The order in which a run's values come out of the quant words: the value at
// f16 position p of the run.  Bytes in value order come out as 0 2 1 3 of every
// four, nibble pairs as 0 4 1 5 2 6 3 7 of every eight.
__host__ __device__ __forceinline__ int value_at(int fmt, int p) {
  if (fmt == Q8_0 || fmt == IQ4_NL) return (p & ~3) | ((p & 1) << 1) | ((p >> 1) & 1);
  return (p & ~7) | ((p & 1) << 2) | ((p >> 1) & 3);
}

// Packed activations of `rows` rows of `cols` values.
struct Packed16 {
  __half *hi, *lo;  // [rows][cols]
  __half *sums;     // [rows][blocks][16]: 2^-5 times the 8 runs' sums, high terms, low terms
  float *scale;     // [rows]: 2^-k
};
constexpr float SUM_UNIT = 32.f;

// k with the largest magnitude mx (as float bits; 0 <= mx) in [2^13, 2^14).
// Infinities and NaN keep k in range and reach hi as they are.
__device__ __forceinline__ int scale_exponent(float mx) {
  const int k = 13 + 127 - (int)((__float_as_uint(mx) >> 23) & 255);
  return k > 126 ? 126 : k;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// One run by one warp, lane p writing position p; v(i) is value i of the run.
template <typename V>
__device__ __forceinline__ void pack_run16(int fmt, const Packed16 &o, uint64_t row, int cols,
                                           int run, int k, int lane, const V &v) {
  const float x = v(value_at(fmt, lane)) * pow2(k);
  const __half hi = __float2half_rn(x);
  const __half lo = __float2half_rn(x - __half2float(hi));
  const uint64_t at = row * cols + run * RUN + lane;
  o.hi[at] = hi;
  o.lo[at] = lo;
  if (has_min(fmt)) {
    float s = x;
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= 1.f / SUM_UNIT;
    const __half sh = __float2half_rn(s);
    if (lane == 0) {
      __half *q = o.sums + (row * (cols / 256) + run / 8) * 16 + run % 8;
      q[0] = sh;
      q[8] = __float2half_rn(s - __half2float(sh));
    }
  }
}

// ---- PTX -------------------------------------------------------------------------------------

__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// A bounded wait for phase `parity` that leaves the issue slots to the warps with
// work: each try suspends the warp for up to half a millisecond (the default
// limit is so short that the polls of waiting warps took a third of the issue
// slots).  Gives up, and records it, after about two seconds.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, int *err) {
  for (int i = 0; i < 4096; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(500000u)
        : "memory");
    if (ok) return true;
    if (err && *(volatile int *)err != 0) return false;
  }
  record_error(err, ERR_WAIT_TIMEOUT);
  return false;
}

// D[tmem] (+)= A[tmem] (f16, 128 rows x 16) * B[smem] (f16, K-major)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_done(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t at, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(at));
}
// The loads above have arrived (their registers pass through, so that no use
// of them is scheduled before the wait).
__device__ __forceinline__ void tmem_ld_wait(float (&a)[8], float (&b)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(a[0]), "+f"(a[1]), "+f"(a[2]), "+f"(a[3]), "+f"(a[4]), "+f"(a[5]), "+f"(a[6]), "+f"(a[7]),
                 "+f"(b[0]), "+f"(b[1]), "+f"(b[2]), "+f"(b[3]), "+f"(b[4]), "+f"(b[5]), "+f"(b[6]), "+f"(b[7])::"memory");
}

// K-major, SWIZZLE_128B: 8-row groups 1,024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// K-major without a swizzle: cores of 8 rows and 16 bytes, two along K side by side,
// 8-row groups 256 bytes apart.
__device__ __forceinline__ uint64_t desc_cores(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(256 >> 4) << 32) |
         ((uint64_t)1 << 46);
}
// D f32, A and B f16, M = 128
__device__ __forceinline__ uint32_t idesc_f16(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
}

// ---- codes -----------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b),
                            *reinterpret_cast<__half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ constexpr uint32_t both(uint32_t h) { return h | (h << 16); }
constexpr uint32_t H_2P14 = 0x7400u, H_2P10 = 0x6400u, H_2P6 = 0x5400u;  // f16 2^14, 2^10, 2^6

// What a warp stages of its 32 rows at a time: RUNS runs of each row.
template <int FMT>
struct Stage {
  static constexpr int RUNS = FMT == Q4_K || FMT == Q4_0 || FMT == IQ4_NL ? 8 : 4;
  static constexpr int QS = (FMT == Q8_0 ? 32 : FMT == Q6_K ? 24 : 16) * RUNS;
  // 8 rows of one run fall into different banks: by a gap, or 128-byte rows by an
  // exclusive or of the chunk with the row
  static constexpr bool SWIZZLED = QS == 128;
  static constexpr int STRIDE = SWIZZLED ? 128 : QS + 16;
  // the super-block's header (Q5_K: and these runs' fifth bits), or an f16 a run
  static constexpr int HEAD = FMT == Q4_K ? 16 : FMT == Q5_K || FMT == Q6_K ? 32 : 2 * RUNS;
  static constexpr uint32_t WARP_BYTES = 32 * (STRIDE + HEAD);
  // f32 factor that undoes the codes' scaling
  static constexpr float UNIT = FMT == Q4_K || FMT == Q5_K ? 16384.f : FMT == Q6_K ? 1048576.f : FMT == Q4_0 ? 1024.f : 1.f;
};
__host__ __device__ constexpr int stage_cols(int f) {
  return f == Q4_K || f == Q4_0 || f == IQ4_NL ? 256 : 128;
}

// Run j of a row's stage, run jb of its super-block, as A operand registers: 16
// (Q6_K: o and then the low part in o2).  sw: what the row's chunks are permuted with.
template <int FMT>
__device__ __forceinline__ void unpack(const uint8_t *row, int sw, const uint8_t *head, const uint4 &h, int j,
                                       int jb, const uint32_t (&lut)[4], uint32_t (&o)[16],
                                       uint32_t (&o2)[16]) {
  if (FMT == Q4_K || FMT == Q5_K) {
    uint32_t sc, mn;
    q4k_scale_min(jb, h.y, h.z, h.w, sc, mn);
    const uint32_t s = sub2(sc * 0x10001u + both(0x6400u), both(0x6400u));  // (1024 + sc) - 1024
    const uint32_t f = mul2(s, both(H_2P10)), f16th = FMT == Q4_K ? mul2(s, both(H_2P6)) : f;
    const uint4 q = *reinterpret_cast<const uint4 *>(row + ((j ^ sw) << 4));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const uint32_t hb = FMT == Q5_K ? *reinterpret_cast<const uint32_t *>(head + 16 + 4 * j) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (FMT == Q4_K) {
        const uint32_t u = w[i] >> 8;
        o[4 * i] = mul2(w[i] & 0x000F000Fu, f);
        o[4 * i + 1] = mul2(w[i] & 0x00F000F0u, f16th);
        o[4 * i + 2] = mul2(u & 0x000F000Fu, f);
        o[4 * i + 3] = mul2(u & 0x00F000F0u, f16th);
      } else {
        uint32_t ev, od;
        q5k_codes(w[i], hb, i, ev, od);
        o[4 * i] = mul2(ev & 0x00FF00FFu, f);
        o[4 * i + 1] = mul2(od & 0x00FF00FFu, f);
        o[4 * i + 2] = mul2((ev >> 8) & 0x00FF00FFu, f);
        o[4 * i + 3] = mul2((od >> 8) & 0x00FF00FFu, f);
      }
    }
  } else if (FMT == Q6_K) {
    const uint8_t *p = row + (j >> 1) * 48;
    const uint4 q = *reinterpret_cast<const uint4 *>(p + (j & 1) * 16);
    const uint2 hw = *reinterpret_cast<const uint2 *>(p + 32 + (j & 1) * 8);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const uint32_t sp = *reinterpret_cast<const uint16_t *>(head + 2 * jb) ^ 0x8080u;  // + 128 each
#pragma unroll
    for (int a = 0; a < 2; ++a) {  // 16 values of one scale
      const uint32_t sc = (a ? sp >> 8 : sp) & 0xFFu;
      const uint32_t s = sub2(sc * 0x10001u + both(0x6400u), both(0x6480u));  // - 1152
      const uint32_t s2 = mul2(s, both(0x4400u)), s4 = mul2(s, both(0x4C00u));  // s 2^2, s 2^4
      const uint32_t s6 = mul2(s, both(H_2P6)), s8 = mul2(s, both(0x5C00u));
      const uint32_t off = mul2(s, both(0x8200u));  // -s 2^-15
      const uint32_t hs = a ? hw.y : hw.x, ht = hs >> 8;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t n = w[2 * a + b], u = n >> 8;
        const int at = 8 * a + 4 * b;
        o[at] = mul2(n & 0x000F000Fu, s4);
        o[at + 1] = mul2(n & 0x00F000F0u, s);
        o[at + 2] = mul2(u & 0x000F000Fu, s4);
        o[at + 3] = mul2(u & 0x00F000F0u, s);
        const uint32_t even = b ? 0x00300030u : 0x00030003u, odd = even << 2;
        o2[at] = fma2(hs & even, b ? s4 : s8, off);
        o2[at + 1] = fma2(hs & odd, b ? s2 : s6, off);
        o2[at + 2] = fma2(ht & even, b ? s4 : s8, off);
        o2[at + 3] = fma2(ht & odd, b ? s2 : s6, off);
      }
    }
  } else if (FMT == Q4_0) {
    const uint4 q = *reinterpret_cast<const uint4 *>(row + ((j ^ sw) << 4));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i] >> 8;  // (q - 8) 2^-10
      o[4 * i] = fma2(w[i] & 0x000F000Fu, both(H_2P14), both(0xA000u));
      o[4 * i + 1] = fma2(w[i] & 0x00F000F0u, both(H_2P10), both(0xA000u));
      o[4 * i + 2] = fma2(u & 0x000F000Fu, both(H_2P14), both(0xA000u));
      o[4 * i + 3] = fma2(u & 0x00F000F0u, both(H_2P10), both(0xA000u));
    }
  } else {
    uint32_t c[8];  // value + 128, bytes in value order
    if (FMT == Q8_0) {
      const uint4 a = *reinterpret_cast<const uint4 *>(row + (((2 * j) ^ sw) << 4));
      const uint4 b = *reinterpret_cast<const uint4 *>(row + (((2 * j + 1) ^ sw) << 4));
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = w[i] ^ 0x80808080u;
    } else {
      const uint4 q = *reinterpret_cast<const uint4 *>(row + ((j ^ sw) << 4));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t s = w[i / 2] >> (16 * (i & 1)), sel = s & 0x7777u;
        const uint32_t low = __byte_perm(lut[0], lut[1], sel), high = __byte_perm(lut[2], lut[3], sel);
        c[i] = __byte_perm(low, high, 0x3210u | ((s & 0x8888u) >> 1));
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // the bytes under 0x64: (1024 + c) - 1152
      o[2 * i] = sub2(__byte_perm(c[i], 0x64646464u, 0x4240u), both(0x6480u));
      o[2 * i + 1] = sub2(__byte_perm(c[i], 0x64646464u, 0x4341u), both(0x6480u));
    }
  }
}

// ---- the product --------------------------------------------------------------------------------

struct Args {
  const uint8_t *w0, *w1;  // one matrix, or two of the same shape (their tiles follow one another)
  Packed16 act;
  const float *ids;        // [slots]
  float *out;              // [parts][used slots][matrices * rows]
  int32_t *place;          // [slots]: pass << 16 | position among the used slots; -1 unused
  int32_t *share;          // blocks a CTA takes; then the number of used slots
  uint32_t *bad;
  int *err;
  int experts, matrices, rows, cols;
  int slots, act_div;      // activation row of a slot: slot / act_div
};

__device__ __forceinline__ int expert_of(float id, int experts) {
  if (id < 0.0f) return -1;
  return floorf(id) == id && id < (float)experts ? (int)id : -2;
}

// Parts of a tile (see the top): the CTAs that its blocks [u nb, (u + 1) nb)
// fall to.
__host__ __device__ __forceinline__ int first_cta(int u, int nb, int share) {
  return (int)((uint32_t)(u * nb) / (uint32_t)share);  // (all stages: below 2^31)
}
__host__ __device__ __forceinline__ int parts_of(int u, int nb, int share) {
  return (int)((uint32_t)((u + 1) * nb - 1) / (uint32_t)share) - first_cta(u, nb, share) + 1;
}

// Tokens a pass takes at most.  32 would take 256 TMEM columns, two CTAs an SM: 64
// tokens of eight experts (Q4_K, Q5_K) took 567 us with them and 472 us without, and
// of a smaller layer 256 tokens, 64 an expert, 345 us and 324 us.
constexpr int MOST_TOKENS = 16;

// The shape of a kernel for up to T tokens a pass.  TMEM: the A operand of a
// step (16 columns a run, Q6_K 32), the mins as an operand (8), the results (N a
// step, or N a run), the min products.  They fit 128 columns, so that four CTAs
// share an SM: their waits for the tensor core, TMEM and memory cover one another.
template <int FMT, int T>
struct Shape {
  using S = Stage<FMT>;
  static constexpr int N = 2 * T;
  static constexpr int STEP = FMT == Q6_K || (!k_format(FMT) && T > 8) ? 2 : 4;  // runs
  static constexpr int STEPS = S::RUNS / STEP;
  static constexpr int A_COLS = STEP * (FMT == Q6_K ? 32 : 16);
  static constexpr int SUM_ROWS = 16;  // N of the min product
  static constexpr int MIN_A = A_COLS;
  static constexpr int D = MIN_A + (has_min(FMT) ? 8 : 0);
  static constexpr int MIN_D = D + (k_format(FMT) ? N : STEP * N);
  static constexpr int USED = MIN_D + (has_min(FMT) ? SUM_ROWS : 0);
  static constexpr int TMEM = 128;
  static_assert(USED <= TMEM && T <= SUM_ROWS, "TMEM columns");
  // shared memory: the activation ring (a step: T rows of high and T of low
  // terms, 64 bytes a run), the sums of two stages, the warps' weight rings,
  // barriers; the plan follows
  static constexpr int B_DEPTH = T > 8 || has_min(FMT) ? 2 : 3;
  static constexpr uint32_t B_ATOM = N * 128;  // two runs of every row
  static constexpr uint32_t B_STEP = B_ATOM * (STEP / 2);
  static constexpr uint32_t SUMS = has_min(FMT) ? SUM_ROWS * 32 : 0;
  static constexpr uint32_t BEFORE = 1024 + B_DEPTH * B_STEP + 2 * SUMS + 64;
  static constexpr uint32_t ROOM = 55 * 1024;  // of a CTA
  static constexpr int W_FIT = (int)((ROOM - BEFORE) / (4 * S::WARP_BYTES));
  static constexpr int W_DEPTH = W_FIT < 2 ? 2 : W_FIT > 4 ? 4 : W_FIT;
  static constexpr uint32_t W_RING = 4 * W_DEPTH * S::WARP_BYTES;
  static constexpr uint32_t FIXED = BEFORE + W_RING;
  static constexpr int CTAS = FIXED <= 56 * 1024 ? 4 : 3;
};
__host__ __device__ inline uint32_t plan_bytes(int experts, int slots) {
  return (uint32_t)(2 * (experts + 1) * 4 + slots * 2 + 15) / 16 * 16;
}

template <int FMT, int T>
__global__ void __launch_bounds__(THREADS, Shape<FMT, T>::CTAS) mgb_moe_product_kernel(const Args p) {
  using S = Stage<FMT>;
  using X = Shape<FMT, T>;
  constexpr bool KF = k_format(FMT);
  constexpr int N = X::N, STEP = X::STEP, STEPS = X::STEPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *b_ring = smem;                              // 1,024-byte aligned
  uint8_t *sum_ring = b_ring + X::B_DEPTH * X::B_STEP; // also
  uint8_t *w_ring = sum_ring + 2 * X::SUMS;
  uint64_t *full = reinterpret_cast<uint64_t *>(w_ring + X::W_RING);
  uint64_t *done = full + 1;
  uint32_t *tmem_at = reinterpret_cast<uint32_t *>(done + 1);
  uint32_t *first = tmem_at + 12;                                       // [experts + 1]
  uint32_t *pass0 = first + p.experts + 1;                              // [experts + 1]
  uint16_t *list = reinterpret_cast<uint16_t *>(pass0 + p.experts + 1); // [slots]: activation rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(full, 4);
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)),
                 "r"((uint32_t)X::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_at;
  grid_wait();
  grid_dependents();

  // ---- the plan: the used slots by expert in slot order (every CTA has to come
  // to the same passes), and passes of up to T slots of one expert
  uint16_t *chosen = reinterpret_cast<uint16_t *>(b_ring);  // [slots], before the rings are used
  uint32_t *next = reinterpret_cast<uint32_t *>(b_ring + ((p.slots * 2 + 15) & ~15));  // [experts]
  for (int e = threadIdx.x; e < p.experts; e += THREADS) next[e] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < p.slots; s += THREADS) {
    const int e = expert_of(p.ids[s], p.experts);
    chosen[s] = (uint16_t)(e < 0 ? 0xFFFF : e);
    if (e >= 0) atomicAdd(&next[e], 1u);
    else if (e == -2 && p.bad && blockIdx.x == 0) atomicMin(p.bad, (uint32_t)s);
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t run_f = 0, run_p = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const uint32_t n = e < p.experts ? next[e] : 0, q = (n + T - 1) / T;
      uint32_t a = n, b = q;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += ua, b += ub;
      }
      if (e < p.experts) first[e] = next[e] = run_f + a - n, pass0[e] = run_p + b - q;
      run_f += __shfl_sync(0xffffffffu, a, 31);
      run_p += __shfl_sync(0xffffffffu, b, 31);
    }
    if (lane == 0) first[p.experts] = run_f, pass0[p.experts] = run_p;
    __syncwarp();
    for (int s0 = 0; s0 < p.slots; s0 += 32) {
      const int s = s0 + lane, e = s < p.slots ? chosen[s] : 0xFFFF;
      const uint32_t same = __match_any_sync(0xffffffffu, e);
      const uint32_t at = e != 0xFFFF ? next[e] + __popc(same & ((1u << lane) - 1)) : 0;
      if (e != 0xFFFF) list[at] = (uint16_t)(s / p.act_div);
      if (blockIdx.x == 0 && s < p.slots)
        p.place[s] = e != 0xFFFF ? (int32_t)(((pass0[e] + (at - first[e]) / T) << 16) | at) : -1;
      __syncwarp();
      if (e != 0xFFFF && (same >> lane) == 1u) next[e] = at + 1;  // the last of its expert
      __syncwarp();
    }
  }
  __syncthreads();  // `chosen` and `next` are done with: the rings may be filled
  const int used = (int)first[p.experts], passes = (int)pass0[p.experts];
  const int runs = p.cols / RUN, nb = (runs + S::RUNS - 1) / S::RUNS;
  const int tiles1 = (p.rows + TILE - 1) / TILE, tiles = tiles1 * p.matrices;
  const int total = passes * tiles * nb;
  int share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
  share = max(share, (nb + MAX_PARTS - 1) / MAX_PARTS);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.share[0] = share, p.share[1] = used;

  const Layout L(FMT, (uint64_t)p.experts * p.rows, (uint64_t)p.cols);
  const int i0 = min(total, (int)blockIdx.x * share), i1 = min(total, i0 + share);
  // A position in the sequence of stages: stage b of unit u (a row tile of a
  // pass), with the unit's expert and slots.
  struct Cursor {
    int left, u, b;  // stages still to come (this one included)
    int expert, begin, n, tile;
  };
  auto load_unit = [&](Cursor &c) {
    const int pass = c.u / tiles;
    c.tile = c.u - pass * tiles;
    int lo = 0, hi = p.experts - 1;  // the last expert whose first pass is at most this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if ((int)pass0[mid] <= pass) lo = mid;
      else hi = mid - 1;
    }
    c.expert = lo;
    c.begin = (int)first[lo] + (pass - (int)pass0[lo]) * T;
    c.n = min(T, (int)first[lo + 1] - c.begin);
  };
  auto start = [&]() {
    Cursor c = {};
    c.left = i1 - i0;
    if (c.left > 0) {
      c.u = i0 / nb;
      c.b = i0 - c.u * nb;
      load_unit(c);
    }
    return c;
  };
  // returns whether the unit changed
  auto advance = [&](Cursor &c) {
    --c.left;
    if (++c.b < nb) return false;
    c.b = 0;
    ++c.u;
    if (c.left > 0) load_unit(c);
    return true;
  };
  // steps of stage b: all, or what the last stage's runs need
  // (the K formats' rows are whole stages)
  auto steps_of = [&](int b) {
    return KF ? STEPS : min(STEPS, (runs - b * S::RUNS + STEP - 1) / STEP);
  };

  if (warp == 4) {
    // ---------------- activations and MMAs ----------------
    bool ok = true;
    // the copies run B_DEPTH - 1 steps ahead.  A lane copies chunk `ch` of every
    // second (CH 8: fourth) row; the pass's tokens take rows 0 .. n - 1 of the
    // operand with their high terms and rows T8 .. T8 + n - 1, T8 = n rounded up
    // to 8, with their low ones.
    constexpr int CH = STEP * 4;       // 16-byte chunks of a row
    constexpr int LANES = 32 / CH;     // rows a copy round
    const int ch = lane % CH, r0 = lane / CH;
    Cursor f = start();
    int fs = 0, fslot = 0, fsum = 0;
    auto fetch = [&]() {
      if (f.left > 0) {
        const int run0 = f.b * S::RUNS + fs * STEP;
        const bool mine = KF || ch < (runs - run0) * 4;
        const uint32_t dst = smem_u32(b_ring + fslot * X::B_STEP) + (ch >> 3) * X::B_ATOM;
        const __half *hi = p.act.hi + run0 * RUN + ch * 8, *lo = p.act.lo + run0 * RUN + ch * 8;
        const int t8 = (f.n + 7) & ~7;
        if (mine)
          for (int t = r0; t < f.n; t += LANES) {
            const uint64_t at = (uint64_t)list[f.begin + t] * (uint32_t)p.cols;
            const uint32_t d = dst + t * 128 + (((ch ^ t) & 7) << 4);
            cp_async16_at(d, hi + at);
            cp_async16_at(d + t8 * 128, lo + at);
          }
        if (has_min(FMT) && fs == 0) {
          const uint32_t sd = smem_u32(sum_ring + fsum * X::SUMS);
          const int blocks = runs / 8, block = f.b * S::RUNS / 8;
          for (int q = lane; q < 2 * f.n; q += 32) {
            const int t = q >> 1, c = q & 1;
            cp_async16_at(sd + (t >> 3) * 256 + c * 128 + (t & 7) * 16,
                          p.act.sums + ((uint64_t)list[f.begin + t] * blocks + block) * 16 + c * 8);
          }
          fsum ^= 1;
        }
        fslot = fslot + 1 == X::B_DEPTH ? 0 : fslot + 1;
        if (++fs == steps_of(f.b)) fs = 0, advance(f);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < X::B_DEPTH - 1; ++i) fetch();
    const uint64_t b0 = desc_sw128(smem_u32(b_ring)), s0 = desc_cores(smem_u32(sum_ring));
    Cursor c = start();
    int slot = 0, sum_slot = 0;
    uint32_t q = 0;
    while (c.left > 0 && ok) {
      const int b = c.b, steps = steps_of(b);
      const uint32_t idesc = idesc_f16(2 * ((c.n + 7) & ~7));
      for (int s = 0; s < steps; ++s, ++q) {
        cp_async_wait<X::B_DEPTH - 2>();
        fence_proxy_async_smem();  // this lane's copies, for the tensor core's reads
        __syncwarp();
        ok = __all_sync(0xffffffffu, wait_phase(full, q & 1, p.err));
        if (!ok) break;
        if (lane == 0) {
          fence_after();
          const uint64_t bd = b0 + (((uint64_t)slot * X::B_STEP) >> 4);
          const uint32_t a = tmem;
          const int r = min(STEP, runs - b * S::RUNS - s * STEP);
#pragma unroll
          for (int j = 0; j < STEP; ++j) {
            if (!KF && j >= r) break;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
              const int k = 2 * j + kk;  // 16 values: 32 bytes of the step's atoms
              const uint64_t bk = bd + (uint64_t)(((k >> 2) * X::B_ATOM + (k & 3) * 32) >> 4);
              if (FMT == Q6_K) {
                mma_ts(tmem + X::D, a + k * 8, bk, idesc, s > 0 || k > 0);
                mma_ts(tmem + X::D, a + X::A_COLS / 2 + k * 8, bk, idesc, true);
              } else if (KF) {
                mma_ts(tmem + X::D, a + k * 8, bk, idesc, s > 0 || k > 0);
              } else {
                mma_ts(tmem + X::D + j * N, a + k * 8, bk, idesc, kk > 0);
              }
            }
          }
          if (has_min(FMT) && s == 0)
            mma_ts(tmem + X::MIN_D, tmem + X::MIN_A, s0 + (((uint64_t)sum_slot * X::SUMS) >> 4),
                   idesc_f16(X::SUM_ROWS), false);
          mma_done(done);
        }
        __syncwarp();
        if (has_min(FMT) && s == 0) sum_slot ^= 1;
        slot = slot + 1 == X::B_DEPTH ? 0 : slot + 1;
        // `full` of this step came after the rows' warps saw the step before it
        // done, so that step's slot is free
        fetch();
      }
      advance(c);
    }
    cp_async_wait<0>();
    // the last MMAs have been performed before TMEM goes back
    if (q > 0) wait_phase(done, (q - 1) & 1, p.err);
    __syncwarp();
  } else {
    // ---------------- weights ----------------
    uint8_t *ring = w_ring + warp * X::W_DEPTH * S::WARP_BYTES;
    const bool aligned = KF || L.sc_row % 16 == 0;
    constexpr int PER_ROW = S::QS / 16, AT_ONCE = 32 / PER_ROW;  // chunks of a row; rows a copy round
    Cursor f = start();
    int fslot = 0, frow0 = 0;
    const uint8_t *fq = nullptr, *fh = nullptr;  // this lane's quants and header of stage 0
    auto point = [&]() {
      const bool second = f.tile >= tiles1;
      const uint8_t *w = second ? p.w1 : p.w0;
      frow0 = (second ? f.tile - tiles1 : f.tile) * TILE + warp * 32;
      const uint64_t row = (uint64_t)f.expert * p.rows + frow0;
      fq = w + (row + lane / PER_ROW) * L.qs_row + (lane % PER_ROW) * 16;
      fh = w + L.qs_bytes + (row + lane) * L.sc_row;
    };
    if (f.left > 0) point();
    auto fetch = [&]() {
      if (f.left > 0) {
        uint8_t *st = ring + fslot * S::WARP_BYTES;
        const int left = runs - f.b * S::RUNS;
        const int chunks = left >= S::RUNS ? PER_ROW : FMT == Q8_0 ? 2 * left : FMT == Q6_K ? left * 3 / 2 : left;
        const uint32_t at = (uint32_t)f.b * S::QS;
        const int r = lane / PER_ROW, ch = lane % PER_ROW;
        const bool mine = r < AT_ONCE && ch < chunks;
        // (SWIZZLED: rows r + 4 c, of which every second has the same low bits)
        const uint32_t d = smem_u32(st + r * S::STRIDE) + ((S::SWIZZLED ? ch ^ r : ch) << 4);
        const int rows = min(32, p.rows - frow0) - r;  // this lane's rows are below it
#pragma unroll
        for (int c = 0; c < (31 + AT_ONCE) / AT_ONCE; ++c)
          if (mine && c * AT_ONCE < rows)
            cp_async16_at((S::SWIZZLED && (c & 1) ? d ^ 64u : d) + c * AT_ONCE * S::STRIDE,
                          fq + at + (uint64_t)(c * AT_ONCE) * L.qs_row);
        if (frow0 + lane < p.rows && aligned) {
          uint8_t *d = st + 32 * S::STRIDE + lane * S::HEAD;
          if (FMT == Q5_K) {
            cp_async16(d, fh + (f.b >> 1) * 48);
            cp_async16(d + 16, fh + (f.b >> 1) * 48 + 16 + (f.b & 1) * 16);
          } else if (FMT == Q6_K) {
            cp_async16(d, fh + (f.b >> 1) * 32);
            cp_async16(d + 16, fh + (f.b >> 1) * 32 + 16);
          } else if (S::HEAD == 16) {
            cp_async16(d, fh + f.b * 16);
          } else {
            cp_async8(d, fh + f.b * 8);
          }
        }
        fslot = fslot + 1 == X::W_DEPTH ? 0 : fslot + 1;
        if (advance(f) && f.left > 0) point();
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < X::W_DEPTH; ++i) fetch();
    uint32_t lut[4] = {0, 0, 0, 0};
    if (FMT == IQ4_NL)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) lut[i] |= (uint32_t)((iq4nl_value(4 * i + c) + 128) & 0xFF) << (8 * c);

    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const int sw = S::SWIZZLED ? lane & 7 : 0;
    float acc[T];
#pragma unroll
    for (int t = 0; t < T; ++t) acc[t] = 0.f;
    // what the step before left in TMEM: its factors, and whether it ends a stage
    // (the K formats' results are complete then) and a segment of a unit
    float fac[4] = {0.f, 0.f, 0.f, 0.f};
    bool stage_end = false, segment_end = false;
    int prev_runs = 0;
    Cursor prev = {};
    uint32_t q = 0;
    bool ok = true;

    // waits for step q - 1 and adds its results
    auto collect = [&]() {
      ok = __all_sync(0xffffffffu, wait_phase(done, (q - 1) & 1, p.err));
      if (!ok) return;
      fence_after();
      if (KF && !stage_end) return;
      const int t8 = (prev.n + 7) & ~7;
#pragma unroll
      for (int t0 = 0; t0 < T; t0 += 8) {
        if (t0 >= prev.n) break;
        if (KF) {
          float hi[8], lo[8];
          tmem_ld8(lanes + X::D + t0, hi);
          tmem_ld8(lanes + X::D + t8 + t0, lo);
          if (has_min(FMT)) {
            float mn[8];
            tmem_ld8(lanes + X::MIN_D + t0, mn);
            tmem_ld_wait(hi, lo);
            tmem_ld_wait(mn, hi);
#pragma unroll
            for (int t = 0; t < 8; ++t) acc[t0 + t] = fmaf(-fac[1], mn[t], acc[t0 + t]);
          } else {
            tmem_ld_wait(hi, lo);
          }
#pragma unroll
          for (int t = 0; t < 8; ++t) acc[t0 + t] = fmaf(fac[0], hi[t] + lo[t], acc[t0 + t]);
        } else {
#pragma unroll
          for (int j = 0; j < STEP; ++j) {
            if (j >= prev_runs) break;
            float hi[8], lo[8];
            tmem_ld8(lanes + X::D + j * N + t0, hi);
            tmem_ld8(lanes + X::D + j * N + t8 + t0, lo);
            tmem_ld_wait(hi, lo);
#pragma unroll
            for (int t = 0; t < 8; ++t) acc[t0 + t] = fmaf(fac[j], hi[t] + lo[t], acc[t0 + t]);
          }
        }
      }
      if (segment_end) {  // the segment's result: this thread's row, one value per token
        const int m = prev.tile >= tiles1;
        const int row = (m ? prev.tile - tiles1 : prev.tile) * TILE + warp * 32 + lane;
        const int part = (int)blockIdx.x - first_cta(prev.u, nb, share);
        float *o = p.out + ((uint64_t)part * used + prev.begin) * ((uint64_t)p.matrices * p.rows) +
                   (uint64_t)m * p.rows + row;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          if (t < prev.n && row < p.rows)
            o[(uint64_t)t * ((uint64_t)p.matrices * p.rows)] =
                acc[t] * p.act.scale[list[prev.begin + t]];
          acc[t] = 0.f;
        }
      }
    };

    Cursor c = start();
    int slot = 0;
    while (c.left > 0 && ok) {
      cp_async_wait<X::W_DEPTH - 1>();
      __syncwarp();
      const uint8_t *st = ring + slot * S::WARP_BYTES;
      const uint8_t *row = st + lane * S::STRIDE;
      const uint8_t *head = st + 32 * S::STRIDE + lane * S::HEAD;
      const uint4 h = has_min(FMT) ? *reinterpret_cast<const uint4 *>(head) : make_uint4(0, 0, 0, 0);
      const int left = runs - c.b * S::RUNS, steps = steps_of(c.b);
      const int jb0 = S::RUNS == 4 ? (c.b & 1) * 4 : 0;  // the stage's first run in its super-block
      const uint16_t *direct = nullptr;  // the row's scales where rows are not 16-byte aligned
      if (!aligned) {
        const int m = c.tile >= tiles1;
        const int r = min(p.rows - 1, (m ? c.tile - tiles1 : c.tile) * TILE + warp * 32 + lane);
        direct = reinterpret_cast<const uint16_t *>(
                     (m ? p.w1 : p.w0) + L.qs_bytes + ((uint64_t)c.expert * p.rows + r) * L.sc_row) +
                 c.b * S::RUNS;
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (!KF && s >= steps) break;
        const int r = KF ? STEP : min(STEP, left - s * STEP);
        if (q > 0) {  // the step before has read the A operand
          collect();
          if (!ok) break;
        }
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
          if (!KF && j >= r) break;
          uint32_t o[16], o2[16];
          unpack<FMT>(row, sw, head, h, s * STEP + j, jb0 + s * STEP + j, lut, o, o2);
          tmem_st16(lanes + j * 16, o);
          if (FMT == Q6_K) tmem_st16(lanes + X::A_COLS / 2 + j * 16, o2);
        }
        if (has_min(FMT) && s == 0) {
          // the stage's mins as f16 integers (zero for the runs of the super-block's
          // other stage), twice: for the high and the low terms of the sums
          uint32_t m[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t sc, m0, m1;
            q4k_scale_min(2 * j, h.y, h.z, h.w, sc, m0);
            q4k_scale_min(2 * j + 1, h.y, h.z, h.w, sc, m1);
            m[j] = sub2((m0 | (m1 << 16)) + both(0x6400u), both(0x6400u));
            if (S::RUNS == 4 && (j >> 1) != (jb0 >> 2)) m[j] = 0;
            m[j + 4] = m[j];
          }
          tmem_st8(lanes + X::MIN_A, m);
        }
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
        // for `collect` after the next step
        if (has_min(FMT)) {
          fac[0] = f16_bits_to_f32(h.x) * S::UNIT;
          fac[1] = f16_bits_to_f32(h.x >> 16) * SUM_UNIT;
        } else if (FMT == Q6_K) {
          fac[0] = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(head + 16)) * S::UNIT;
        } else {
#pragma unroll
          for (int j = 0; j < STEP; ++j)
            if (j < r)
              fac[j] = f16_bits_to_f32(direct ? direct[s * STEP + j]
                                              : *reinterpret_cast<const uint16_t *>(
                                                    head + 2 * (s * STEP + j))) * S::UNIT;
        }
        prev_runs = r;
        stage_end = s == steps - 1;
        segment_end = stage_end && (c.b == nb - 1 || c.left == 1);
        if (segment_end || q == 0) prev = c;
        prev.n = c.n;
        ++q;
      }
      __syncwarp();
      slot = slot + 1 == X::W_DEPTH ? 0 : slot + 1;
      fetch();
      advance(c);
    }
    if (q > 0 && ok) collect();
    cp_async_wait<0>();
    fence_before();
  }
  __syncthreads();
  fence_after();
  if (warp == 4)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"((uint32_t)X::TMEM)
                 : "memory");
}

}  // namespace moe

// One launch of a product (instantiated per format in experts_*.cu): `tokens`
// is what a pass takes, `sms` the device's; returns the CTAs of an SM instead of
// launching when a is null.
template <int FMT>
cudaError_t launch_moe_product(const moe::Args *a, int tokens, int sms, int *ctas_per_sm,
                               cudaStream_t stream);

}  // namespace mgb
