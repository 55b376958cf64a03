// The packed products of a mixture-of-experts layer for a few tokens.
//
// Every expert that a token chose has its packed rows streamed once and
// multiplied with all of its tokens by mma.sync m16n8k16 (f16 operands, f32
// accumulation): 16 weight rows are the MMA's rows, 8 tokens its columns, and
// the work is bound by the weight stream, so what counts is how few
// instructions a weight costs.
//
// Weights.  The codes of a 32-value run enter the MMA as they are: a 4-bit code
// masked in place (w & 0x000F000F) is a pair of f16 subnormals q 2^-24, the next
// nibble (w & 0x00F000F0) q 2^-20, byte codes likewise, so unpacking 8 weights
// takes a shift and four ANDs and is exact.  The run's scale multiplies the
// MMA's result in f32, and its min (and a code's offset) multiplies the run's
// activation sum: both factors are exact in f32.
//
// Activations.  A run of 32 values is held as x = 2^-k (hi + lo) with k chosen
// so that the largest |2^k x| lies in [2^13, 2^14): two f16 terms keep 22 bits
// of every value down to 2^-27 of the run's largest.  They are stored in the
// order in which a lane's codes come out of the quant words (`packet_slot`), so
// that a lane's B operands of a run are one 16-byte load a term.
#pragma once

#include "common.cuh"
#include "decode.cuh"
#include "kernels.h"

namespace mgb {
namespace moe {

constexpr int WARPS = 16;
constexpr int THREADS = 32 * WARPS;
constexpr int ROWS = 32;       // weight rows of a warp's tile (two MMA row blocks)
constexpr int RED_STRIDE = 36; // floats of a token's row in the reduction buffer
constexpr uint32_t SIDE_BYTES = 8 * RED_STRIDE * 4;  // a warp's factors, then its partial sums

// ---- activations in packets ------------------------------------------------------------
//
// One (row, run): 64 bytes of high terms, 64 of low terms; quarter t of each is
// what lane t of a quad multiplies with.  Beside it a float2: 2^-k and the sum
// of the run.

constexpr uint32_t PACKET = 128;

// Value i of a run sits in quarter t at f16 position `pos`, divided by 16 when
// its code comes out of the quant word times 16.
struct PacketSlot {
  int t, pos;
  bool sixteenth;
};
__host__ __device__ __forceinline__ PacketSlot packet_slot(int fmt, int i) {
  const int v = i & 7;
  if (fmt == Q6_K) {  // a half-run per MMA: values 4 t .. 4 t + 3 of each half
    const int r = i & 3;
    return {(i & 15) >> 2, (i >> 4) * 4 + (r == 1 ? 2 : r == 2 ? 1 : r), false};
  }
  if (fmt == Q8_0 || fmt == IQ4_NL)  // bytes in value order: 0 2 1 3 4 6 5 7
    return {i >> 3, (v & 4) | ((v & 1) << 1) | ((v >> 1) & 1), false};
  // nibble pairs: 0 4 1 5 2 6 3 7
  return {i >> 3, ((v & 3) << 1) | (v >> 2), fmt != Q5_K && (v & 1)};
}

// Writes value i (lane i of a full warp holds it) of one run: its packet and
// its (2^-k, sum).
__device__ __forceinline__ void write_packet(int fmt, float v, int lane, uint8_t *packet,
                                             float2 *meta) {
  float mx = fabsf(v), sum = v;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  // exponent of the largest value (NaN and infinities keep theirs: they reach
  // hi as they are), k within what 2^k and 2^-k hold
  int k = 13 + 127 - (int)((__float_as_uint(mx) >> 23) & 255);
  k = k > 126 ? 126 : k;
  const float up = __uint_as_float((uint32_t)(k + 127) << 23);
  const float down = __uint_as_float((uint32_t)(127 - k) << 23);
  const PacketSlot s = packet_slot(fmt, lane);
  float x = v * up;
  if (s.sixteenth) x *= 0.0625f;
  const __half hi = __float2half_rn(x);
  const __half lo = __float2half_rn(x - __half2float(hi));
  *reinterpret_cast<__half *>(packet + s.t * 16 + s.pos * 2) = hi;
  *reinterpret_cast<__half *>(packet + 64 + s.t * 16 + s.pos * 2) = lo;
  if (lane == 0) *meta = make_float2(down, sum);
}

// ---- the device layout by stages -----------------------------------------------------------
//
// A warp's stage holds RUNS runs of its 32 rows: their quant bytes at a padded
// row stride (8 rows of one run fall into different banks), then their scale
// headers.

template <int FMT>
struct Stage {
  static constexpr int RUNS = FMT == Q8_0 || FMT == Q6_K || FMT == Q5_K ? 4 : 8;
  static constexpr int QS = FMT == Q8_0 ? 32 * RUNS : FMT == Q6_K ? 24 * RUNS : 16 * RUNS;
  static constexpr int STRIDE = QS + (FMT == Q8_0 ? 32 : 16);
  static constexpr bool BLOCK256 = FMT == Q4_K || FMT == Q5_K || FMT == Q6_K;
  // header bytes of a row: the super-block's (Q5_K: its 16 bytes and the runs'
  // fifth bits), or an f16 per run
  static constexpr int HEAD = FMT == Q4_K ? 16 : FMT == Q5_K || FMT == Q6_K ? 32 : 2 * RUNS;
  static constexpr uint32_t BYTES = (STRIDE + HEAD) * ROWS;
  static constexpr int DEPTH = 2;
};

__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// What an earlier kernel of the chain wrote: ordinary loads through pointers
// that are not restrict-qualified (the read-only path is not ordered by the
// grid dependency, and inline assembly that the compiler takes for arithmetic
// may be moved in front of the branch that makes its address valid).
__device__ __forceinline__ uint4 ld_v4(const void *p) { return *static_cast<const uint4 *>(p); }
__device__ __forceinline__ float2 ld_v2(const void *p) { return *static_cast<const float2 *>(p); }
__device__ __forceinline__ float ld_f32(const float *p) { return *p; }

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The codes of run j of one staged row, quarter t, as the f16 pairs of two MMAs:
// a[0], a[2] of the first and of the second.
template <int FMT>
__device__ __forceinline__ void unpack(const uint8_t *row, const uint8_t *head, int j, int t,
                                       const uint32_t (&lut)[4], uint32_t (&o)[4]) {
  if (FMT == Q4_K || FMT == Q4_0) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(row + j * 16 + t * 4), s = w >> 8;
    o[0] = w & 0x000F000Fu, o[1] = w & 0x00F000F0u;
    o[2] = s & 0x000F000Fu, o[3] = s & 0x00F000F0u;
  } else if (FMT == Q5_K) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(row + j * 16 + t * 4);
    const uint32_t hb = *reinterpret_cast<const uint32_t *>(head + 16 + j * 4);
    uint32_t ev, od;
    q5k_codes(w, hb, t, ev, od);
    o[0] = ev & 0x00FF00FFu, o[1] = od & 0x00FF00FFu;
    o[2] = (ev >> 8) & 0x00FF00FFu, o[3] = (od >> 8) & 0x00FF00FFu;
  } else if (FMT == Q8_0) {
    const uint2 w = *reinterpret_cast<const uint2 *>(row + j * 32 + t * 8);
    const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;  // q + 128
    o[0] = x & 0x00FF00FFu, o[1] = (x >> 8) & 0x00FF00FFu;
    o[2] = y & 0x00FF00FFu, o[3] = (y >> 8) & 0x00FF00FFu;
  } else if (FMT == IQ4_NL) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(row + j * 16 + t * 4);
    uint32_t c[2];  // codebook bytes + 128 of values 0..3 and 4..7
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t s = w >> (16 * h), sel = s & 0x7777u;
      const uint32_t low = __byte_perm(lut[0], lut[1], sel), high = __byte_perm(lut[2], lut[3], sel);
      c[h] = __byte_perm(low, high, 0x3210u | ((s & 0x8888u) >> 1));
    }
    o[0] = c[0] & 0x00FF00FFu, o[1] = (c[0] >> 8) & 0x00FF00FFu;
    o[2] = c[1] & 0x00FF00FFu, o[3] = (c[1] >> 8) & 0x00FF00FFu;
  } else {  // Q6_K: 48 bytes per two runs; a half-run per MMA
    const uint8_t *p = row + (j >> 1) * 48;
    const uint2 hw = *reinterpret_cast<const uint2 *>(p + 32 + (j & 1) * 8);
    const __half2 offset = __halves2half2(__ushort_as_half(32), __ushort_as_half(32));
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint32_t n = *reinterpret_cast<const uint16_t *>(p + (j & 1) * 16 + a * 8 + t * 2);
      const uint32_t low = __byte_perm(n, 0, 0x4140u);
      const uint32_t high = __byte_perm(a ? hw.y : hw.x, 0, t & 1 ? 0x4342u : 0x4140u) >> (4 * (t >> 1));
      const uint32_t e = (low & 0x000F000Fu) | ((high & 0x00030003u) << 4);
      const uint32_t d = ((low >> 4) & 0x000F000Fu) | ((high << 2) & 0x00300030u);
      // code - 32, exact in subnormals
      const __half2 eh = __hsub2(*reinterpret_cast<const __half2 *>(&e), offset);
      const __half2 dh = __hsub2(*reinterpret_cast<const __half2 *>(&d), offset);
      o[2 * a] = *reinterpret_cast<const uint32_t *>(&eh);
      o[2 * a + 1] = *reinterpret_cast<const uint32_t *>(&dh);
    }
  }
}

// Codes come out in units of 2^-24.
constexpr float UNIT = 16777216.f;

// The two f32 factors of a run: Q6_K the scales of its halves, otherwise the
// scale and minus what multiplies the activation sum (min and code offset).
// `head`: the staged header; `direct`: the row's scales in global memory (f16
// formats whose rows are not 16-byte aligned), else null.
template <int FMT>
__device__ __forceinline__ float2 factors(const uint8_t *head, const uint8_t *direct, int run,
                                          int j) {
  if (FMT == Q4_K || FMT == Q5_K) {
    const uint4 h = *reinterpret_cast<const uint4 *>(head);
    const float d = f16_bits_to_f32(h.x), dmin = f16_bits_to_f32(h.x >> 16);
    uint32_t s, m;
    q4k_scale_min(run & 7, h.y, h.z, h.w, s, m);
    return make_float2(d * UNIT * (float)s, -dmin * (float)m);
  }
  if (FMT == Q6_K) {
    const float d = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(head + 16)) * UNIT;
    const uint32_t s = *reinterpret_cast<const uint16_t *>(head + 2 * (run & 7));
    return make_float2(d * (float)(int8_t)(s & 0xFF), d * (float)(int8_t)(s >> 8));
  }
  const uint16_t bits = direct ? __ldg(reinterpret_cast<const uint16_t *>(direct) + run)
                               : *reinterpret_cast<const uint16_t *>(head + 2 * j);
  const float d = f16_bits_to_f32(bits);
  return make_float2(d * UNIT, d * (FMT == Q4_0 ? -8.f : -128.f));
}

struct Args {
  const uint8_t *w0, *w1;   // gate and up, or down twice
  const uint8_t *packets;   // activations [rows][runs][PACKET]
  const float2 *meta;       // [rows][runs]
  const float *ids;         // [slots]
  uint8_t *h_packets;       // gate/up: h as packets of the down format
  float2 *h_meta;
  float *out;               // down: [slots][rows]
  uint32_t *bad;
  int experts, rows, cols;  // an expert's stored rows; values a row
  int slots, top_k;
  int act_div;              // activation row of a slot: slot / act_div
  int ks;                   // warps that share a tile's columns; 16 / ks tiles side by side
  int down_fmt;
};

__device__ __forceinline__ int expert_of(float id, int experts) {
  if (id < 0.0f) return -1;
  return floorf(id) == id && id < (float)experts ? (int)id : -2;
}

// Shared memory behind the warps' stages: the slots of every expert.
__host__ __device__ inline uint32_t plan_bytes(int experts, int slots) {
  return (uint32_t)(2 * (experts + 1) * 4 + slots * 2 + 15) / 16 * 16;
}
template <int FMT>
__host__ __device__ constexpr uint32_t warp_bytes() {
  return Stage<FMT>::BYTES * Stage<FMT>::DEPTH + SIDE_BYTES;
}

// One product.  GATE_UP: h = silu(gate x) * (up x), a warp's 32 rows are 16 of
// gate and the same 16 of up.  Otherwise out[slot] = down h[slot], 32 rows of
// down.  A CTA's 16 warps are `ks` slices of the columns times 16 / ks row
// tiles; the slices are summed in shared memory in order.  NT: groups of 8
// tokens that one pass over the rows multiplies.
template <int FMT, bool GATE_UP, int NT>
__global__ void __launch_bounds__(THREADS, 1) mgb_moe_product_kernel(const Args p) {
  using S = Stage<FMT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t *stages = smem + warp * warp_bytes<FMT>();
  float2 *fac = reinterpret_cast<float2 *>(stages + S::BYTES * S::DEPTH);  // [4 runs][ROWS]
  uint32_t *first = reinterpret_cast<uint32_t *>(smem + WARPS * warp_bytes<FMT>());  // [experts + 1]
  uint32_t *pass0 = first + p.experts + 1;                                           // [experts + 1]
  uint16_t *list = reinterpret_cast<uint16_t *>(pass0 + p.experts + 1);              // [slots]

  grid_wait();
  grid_dependents();

  // the plan: slots by expert in slot order (every CTA has to come to the same
  // passes), and passes (up to 8 NT slots of one expert each)
  uint16_t *chosen = reinterpret_cast<uint16_t *>(smem);  // [slots], before the stages are used
  for (int e = threadIdx.x; e <= p.experts; e += THREADS) pass0[e] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < p.slots; s += THREADS) {
    const int e = expert_of(ld_f32(p.ids + s), p.experts);
    chosen[s] = (uint16_t)(e < 0 ? 0xFFFF : e);
    if (e >= 0) atomicAdd(&pass0[e], 1u);
    else if (e == -2 && GATE_UP && p.bad && blockIdx.x == 0) atomicMin(p.bad, (uint32_t)s);
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t run_f = 0, run_p = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const uint32_t n = e < p.experts ? pass0[e] : 0, q = (n + 8 * NT - 1) / (8 * NT);
      uint32_t a = n, b = q;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += ua, b += ub;
      }
      if (e < p.experts) first[e] = run_f + a - n, pass0[e] = run_p + b - q;
      run_f += __shfl_sync(0xffffffffu, a, 31);
      run_p += __shfl_sync(0xffffffffu, b, 31);
    }
    if (lane == 0) first[p.experts] = run_f, pass0[p.experts] = run_p;
  }
  __syncthreads();
  // place them; first[e] becomes the end of e's slots
  if (warp == 0)
    for (int s0 = 0; s0 < p.slots; s0 += 32) {
      const int s = s0 + lane, e = s < p.slots ? chosen[s] : 0xFFFF;
      const uint32_t same = __match_any_sync(0xffffffffu, e);
      const uint32_t at = e != 0xFFFF ? first[e] + __popc(same & ((1u << lane) - 1)) : 0;
      if (e != 0xFFFF) list[at] = (uint16_t)s;
      __syncwarp();
      if (e != 0xFFFF && (same >> lane) == 1u) first[e] = at + 1;  // the last of its expert
      __syncwarp();
    }
  __syncthreads();

  const int ks = p.ks, mg = WARPS / ks;
  const int slice = warp % ks, group = warp / ks;
  const int tile_rows = (GATE_UP ? 16 : 32) * mg;
  const int tiles = (p.rows + tile_rows - 1) / tile_rows;
  const int passes = (int)pass0[p.experts];
  const int runs = p.cols / RUN;
  const int nstages = (runs + S::RUNS - 1) / S::RUNS;  // of a row
  const int mine = (nstages - slice + ks - 1) / ks;    // of this warp's slice
  const Layout L(FMT, (uint64_t)p.experts * p.rows, (uint64_t)p.cols);
  const bool aligned = S::BLOCK256 || L.sc_row % 16 == 0;
  uint32_t lut[4] = {0, 0, 0, 0};
  if (FMT == IQ4_NL)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b) lut[i] |= (uint32_t)((iq4nl_value(4 * i + b) + 128) & 0xFF) << (8 * b);

  // work item w: pass w / tiles, row tile w % tiles
  auto expert_at = [&](int pass) {
    int lo = 0, hi = p.experts - 1;  // the last expert whose first pass is <= pass and that has one
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if ((int)pass0[mid] <= pass) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  const int total = passes * tiles;
  // the warp's copies: stage i of its slice of work item w
  auto fetch = [&](int w, int e, int i, int slot) {
    uint8_t *st = stages + slot * S::BYTES;
    const int base = (w % tiles) * tile_rows + group * (GATE_UP ? 16 : 32);
    const int b = slice + i * ks;  // stage of the row
    const int left = min(S::RUNS, runs - b * S::RUNS);
    const int chunks = FMT == Q8_0 ? 2 * left : FMT == Q6_K ? left * 3 / 2 : left;
    constexpr int PER_ROW = S::QS / 16;
#pragma unroll
    for (int c0 = 0; c0 < PER_ROW * ROWS; c0 += 32) {
      const int r = (c0 + lane) / PER_ROW, c = (c0 + lane) % PER_ROW;
      const int row = GATE_UP ? base + (r & 15) : base + r;
      if (row < p.rows && c < chunks)
        cp_async16(st + r * S::STRIDE + c * 16,
                   (GATE_UP && r >= 16 ? p.w1 : p.w0) + ((uint64_t)e * p.rows + row) * L.qs_row +
                       (uint64_t)b * S::QS + c * 16);
    }
    const int row = GATE_UP ? base + (lane & 15) : base + lane;
    if (row < p.rows) {
      const uint8_t *src = (GATE_UP && lane >= 16 ? p.w1 : p.w0) + L.qs_bytes +
                           ((uint64_t)e * p.rows + row) * L.sc_row;
      uint8_t *dst = st + ROWS * S::STRIDE + lane * S::HEAD;
      if (FMT == Q4_K) {
        cp_async16(dst, src + (uint64_t)b * 16);
      } else if (FMT == Q5_K) {
        cp_async16(dst, src + (uint64_t)(b >> 1) * 48);
        cp_async16(dst + 16, src + (uint64_t)(b >> 1) * 48 + 16 + (b & 1) * 16);
      } else if (FMT == Q6_K) {
        cp_async16(dst, src + (uint64_t)(b >> 1) * 32);
        cp_async16(dst + 16, src + (uint64_t)(b >> 1) * 32 + 16);
      } else if (aligned) {
        if (S::HEAD == 16) cp_async16(dst, src + (uint64_t)b * 16);
        else cp_async8(dst, src + (uint64_t)b * 8);
      }
    }
  };

  // a warp's sequence of (work item, stage): the fetches run DEPTH ahead
  int fw = blockIdx.x, fi = 0, fe = fw < total ? expert_at(fw / tiles) : 0, fslot = 0;
  auto fetch_next = [&]() {
    if (fw < total && mine > 0) {
      fetch(fw, fe, fi, fslot);
      fslot = fslot + 1 == S::DEPTH ? 0 : fslot + 1;
      if (++fi == mine) {
        fi = 0;
        fw += gridDim.x;
        if (fw < total) fe = expert_at(fw / tiles);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S::DEPTH; ++i) fetch_next();
  int slot = 0;

  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    const int pass = w / tiles, e = expert_at(pass);
    const int end = (int)first[e];
    const int begin = (e ? (int)first[e - 1] : 0) + (pass - (int)pass0[e]) * 8 * NT;
    const int n = min(8 * NT, end - begin);
    const int row0 = (w % tiles) * tile_rows + group * (GATE_UP ? 16 : 32);
    // this lane's activation rows: token g of every group (operand), tokens 2 t
    // and 2 t + 1 (results); absent ones repeat the last and are not written
    // (offsets in packets: the host keeps packet bytes below 2^32)
    uint32_t act[NT], me[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      auto act_row = [&](int i) { return (uint32_t)(list[begin + min(i, n - 1)] / p.act_div) * runs; };
      act[nt] = act_row(nt * 8 + g) * PACKET + t * 16;
      me[nt][0] = act_row(nt * 8 + 2 * t);
      me[nt][1] = act_row(nt * 8 + 2 * t + 1);
    }
    float acc[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][mt][i] = 0.f;

    for (int i = 0; i < mine; ++i) {
      cp_async_wait<S::DEPTH - 1>();
      __syncwarp();
      const uint8_t *st = stages + slot * S::BYTES;
      const uint8_t *heads = st + ROWS * S::STRIDE;
      const int b = slice + i * ks;
      const int left = min(S::RUNS, runs - b * S::RUNS);
#pragma unroll
      for (int j0 = 0; j0 < S::RUNS; j0 += 4) {
        if (j0 >= left) break;
        {  // factors of four runs, lane = row
          const int row = GATE_UP ? row0 + (lane & 15) : row0 + lane;
          const uint8_t *direct = nullptr;
          if (!aligned && row < p.rows)
            direct = (GATE_UP && lane >= 16 ? p.w1 : p.w0) + L.qs_bytes +
                     ((uint64_t)e * p.rows + row) * L.sc_row;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j0 + j < left && (aligned || direct))
              fac[j * ROWS + lane] = factors<FMT>(heads + lane * S::HEAD, direct,
                                                  b * S::RUNS + j0 + j, j0 + j);
        }
        __syncwarp();
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const int j = j0 + jj;
          if (j >= left) break;
          const int run = b * S::RUNS + j;
          uint32_t o[2][2][4];
          float2 f[2][2];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = mt * 16 + h * 8 + g;
              unpack<FMT>(st + r * S::STRIDE, heads + r * S::HEAD, j, t, lut, o[mt][h]);
              f[mt][h] = fac[jj * ROWS + r];
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (NT > 1 && nt * 8 >= n) break;
            const uint8_t *at = p.packets + (act[nt] + (uint32_t)run * PACKET);
            const uint4 hi = ld_v4(at), lo = ld_v4(at + 64);
            const float2 m0 = ld_v2(p.meta + (me[nt][0] + run)), m1 = ld_v2(p.meta + (me[nt][1] + run));
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const uint32_t(&x)[4] = o[mt][0], (&y)[4] = o[mt][1];
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816(c, x[0], y[0], x[1], y[1], hi.x, hi.y);
              mma16816(c, x[0], y[0], x[1], y[1], lo.x, lo.y);
              float *a = acc[nt][mt];
              if (FMT == Q6_K) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(d, x[2], y[2], x[3], y[3], hi.z, hi.w);
                mma16816(d, x[2], y[2], x[3], y[3], lo.z, lo.w);
                a[0] = fmaf(fmaf(f[mt][0].y, d[0], f[mt][0].x * c[0]), m0.x, a[0]);
                a[1] = fmaf(fmaf(f[mt][0].y, d[1], f[mt][0].x * c[1]), m1.x, a[1]);
                a[2] = fmaf(fmaf(f[mt][1].y, d[2], f[mt][1].x * c[2]), m0.x, a[2]);
                a[3] = fmaf(fmaf(f[mt][1].y, d[3], f[mt][1].x * c[3]), m1.x, a[3]);
              } else {
                mma16816(c, x[2], y[2], x[3], y[3], hi.z, hi.w);
                mma16816(c, x[2], y[2], x[3], y[3], lo.z, lo.w);
                a[0] = fmaf(f[mt][0].x, c[0] * m0.x, fmaf(f[mt][0].y, m0.y, a[0]));
                a[1] = fmaf(f[mt][0].x, c[1] * m1.x, fmaf(f[mt][0].y, m1.y, a[1]));
                a[2] = fmaf(f[mt][1].x, c[2] * m0.x, fmaf(f[mt][1].y, m0.y, a[2]));
                a[3] = fmaf(f[mt][1].x, c[3] * m1.x, fmaf(f[mt][1].y, m1.y, a[3]));
              }
            }
          }
        }
        __syncwarp();
      }
      slot = slot + 1 == S::DEPTH ? 0 : slot + 1;
      fetch_next();
    }

    // the slices' sums, one group of 8 tokens at a time: [warp][token][row]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 8 >= n) break;
      float *red = reinterpret_cast<float *>(fac);
      __syncwarp();
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[(2 * t + (i & 1)) * RED_STRIDE + mt * 16 + (i >> 1) * 8 + g] = acc[nt][mt][i];
      __syncthreads();
      auto sum = [&](int grp, int tok, int r) {
        const uint8_t *at = smem + (size_t)grp * ks * warp_bytes<FMT>() + S::BYTES * S::DEPTH;
        float s = 0.f;
        for (int k = 0; k < ks; ++k)
          s += reinterpret_cast<const float *>(at + (size_t)k * warp_bytes<FMT>())[tok * RED_STRIDE + r];
        return s;
      };
      const int toks = min(8, n - nt * 8);
      if (GATE_UP) {
        // a warp per (token, run of 32 rows of h): two 16-row groups
        for (int q = warp; q < toks * (mg / 2); q += WARPS) {
          const int tok = q % toks, pair = q / toks;
          const int run0 = (w % tiles) * tile_rows + pair * 32;
          if (run0 >= p.rows) continue;
          const float gate = sum(2 * pair + (lane >> 4), tok, lane & 15);
          const float up = sum(2 * pair + (lane >> 4), tok, 16 + (lane & 15));
          const float h = gate / (1.f + expf(-gate)) * up;
          const uint64_t at = (uint64_t)list[begin + nt * 8 + tok] * (p.rows / RUN) + run0 / RUN;
          write_packet(p.down_fmt, h, lane, p.h_packets + at * PACKET, p.h_meta + at);
        }
      } else {
        for (int q = warp; q < toks * mg; q += WARPS) {
          const int tok = q % toks, grp = q / toks;
          const int row = (w % tiles) * tile_rows + grp * 32 + lane;
          if (row >= p.rows) continue;
          p.out[(uint64_t)list[begin + nt * 8 + tok] * p.rows + row] = sum(grp, tok, lane);
        }
      }
      __syncthreads();
    }
  }
}

}  // namespace moe

// One launch of a product (instantiated per format in experts_*.cu).
template <int FMT>
cudaError_t launch_moe_product(const moe::Args &a, bool gate_up, int nt, int sms,
                               cudaStream_t stream);

}  // namespace mgb
