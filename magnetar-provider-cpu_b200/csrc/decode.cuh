// Element access to the device layout: a run's codes and factors, and single
// values, with the reference's roundings (bit-exact to `decode`,
// src/native/quant.rs:100-195).
#pragma once

#include "common.cuh"

namespace mgb {

// The 32 quant values of run `u` of `row` (as ints) and the run's scale and
// min of each 16-value half (the same for both halves except Q6_K's scales).
__device__ __forceinline__ void decode_run(int fmt, const uint8_t *__restrict__ w, const Layout &L,
                                           uint64_t row, uint64_t u, int q[32], float scale[2],
                                           float min[2]) {
  const uint8_t *sc = w + L.qs_bytes + row * L.sc_row;
  if (fmt == Q6_K) {
    const uint8_t *qrow = w + row * L.qs_row;
    const uint4 v = *reinterpret_cast<const uint4 *>(qrow + q6k_nib_offset(u));
    const uint2 hh = *reinterpret_cast<const uint2 *>(qrow + q6k_high_offset(u));
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
    for (int wd = 0; wd < 4; ++wd) {
      uint32_t ev, od;
      q6k_codes(words[wd], wd < 2 ? hh.x : hh.y, wd, ev, od);
      for (int j = 0; j < 4; ++j) {
        q[8 * wd + 2 * j] = (int)((ev >> (8 * j)) & 0xFF) - 32;
        q[8 * wd + 2 * j + 1] = (int)((od >> (8 * j)) & 0xFF) - 32;
      }
    }
    const uint8_t *hd = sc + (u / 8) * 32;
    const float d = f16_bits_to_f32(hd[16] | (hd[17] << 8));
    const int r = (int)(u % 8);
    for (int p = 0; p < 2; ++p) {
      scale[p] = __fmul_rn(d, (float)(int8_t)hd[2 * r + p]);
      min[p] = 0.0f;
    }
    return;
  }
  if (fmt == Q8_0) {
    const uint4 a = *reinterpret_cast<const uint4 *>(w + row * L.qs_row + u * 32);
    const uint4 b = *reinterpret_cast<const uint4 *>(w + row * L.qs_row + u * 32 + 16);
    const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    for (int i = 0; i < 32; ++i) q[i] = (int)(int8_t)((words[i / 4] >> (8 * (i % 4))) & 0xff);
    scale[0] = scale[1] = f16_bits_to_f32(sc[u * 2] | (sc[u * 2 + 1] << 8));
    min[0] = min[1] = 0.0f;
    return;
  }
  const uint4 v = *reinterpret_cast<const uint4 *>(w + row * L.qs_row + u * 16);
  const uint32_t words[4] = {v.x, v.y, v.z, v.w};
  if (fmt == Q5_K) {
    const uint8_t *hd = sc + (u / 8) * 48;
    const uint32_t hb = *reinterpret_cast<const uint32_t *>(hd + 16 + 4 * (u % 8));
    for (int wd = 0; wd < 4; ++wd) {
      uint32_t ev, od;
      q5k_codes(words[wd], hb, wd, ev, od);
      for (int j = 0; j < 4; ++j) {
        q[8 * wd + 2 * j] = (int)((ev >> (8 * j)) & 0xFF);
        q[8 * wd + 2 * j + 1] = (int)((od >> (8 * j)) & 0xFF);
      }
    }
    const uint4 h = *reinterpret_cast<const uint4 *>(hd);
    const float d = f16_bits_to_f32(h.x), dmin = f16_bits_to_f32(h.x >> 16);
    uint32_t s, m;
    q4k_scale_min((int)(u % 8), h.y, h.z, h.w, s, m);
    scale[0] = scale[1] = __fmul_rn(d, (float)s);
    min[0] = min[1] = __fmul_rn(dmin, (float)m);
    return;
  }
  for (int i = 0; i < 32; ++i) {
    const uint32_t nib = (words[i / 8] >> (4 * (i % 8))) & 0xF;
    q[i] = fmt == Q4_K ? (int)nib : (fmt == Q4_0 ? (int)nib - 8 : iq4nl_value((int)nib));
  }
  if (fmt == Q4_K) {
    const uint4 h = *reinterpret_cast<const uint4 *>(sc + (u / 8) * 16);
    const float d = f16_bits_to_f32(h.x), dmin = f16_bits_to_f32(h.x >> 16);
    uint32_t s, m;
    q4k_scale_min((int)(u % 8), h.y, h.z, h.w, s, m);
    scale[0] = scale[1] = __fmul_rn(d, (float)s);
    min[0] = min[1] = __fmul_rn(dmin, (float)m);
  } else {
    scale[0] = scale[1] = f16_bits_to_f32(sc[u * 2] | (sc[u * 2 + 1] << 8));
    min[0] = min[1] = 0.0f;
  }
}

// One element of decode_run: value i of run u of stored row `row`, as
// scale[i / 16] * q[i] - min[i / 16] with the same roundings, decoding only
// that element's code and its run's factors (the input-major product and the
// embedding lookup use one value of a run at a time).
__device__ __forceinline__ float decode_value(int fmt, const uint8_t *__restrict__ w,
                                              const Layout &L, uint64_t row, uint64_t u, int i) {
  const uint8_t *sc = w + L.qs_bytes + row * L.sc_row;
  const uint8_t *qrow = w + row * L.qs_row;
  int q;
  float scale, mn = 0.0f;
  if (fmt == Q6_K) {
    const int wd = i / 8;
    const uint32_t word = *reinterpret_cast<const uint32_t *>(qrow + q6k_nib_offset(u) + 4 * wd);
    const uint32_t hw = *reinterpret_cast<const uint32_t *>(qrow + q6k_high_offset(u) + 4 * (wd >> 1));
    uint32_t ev, od;
    q6k_codes(word, hw, wd, ev, od);
    q = (int)((((i & 1) ? od : ev) >> (8 * ((i % 8) / 2))) & 0xFF) - 32;
    const uint8_t *hd = sc + (u / 8) * 32;
    const float d = f16_bits_to_f32(hd[16] | (hd[17] << 8));
    scale = __fmul_rn(d, (float)(int8_t)hd[2 * (int)(u % 8) + i / 16]);
  } else if (fmt == Q8_0) {
    q = (int)(int8_t)qrow[u * 32 + i];
    scale = f16_bits_to_f32(sc[u * 2] | (sc[u * 2 + 1] << 8));
  } else {
    const uint32_t word = *reinterpret_cast<const uint32_t *>(qrow + u * 16 + 4 * (i / 8));
    if (fmt == Q5_K || fmt == Q4_K) {
      const uint8_t *hd = sc + (u / 8) * (fmt == Q5_K ? 48 : 16);
      if (fmt == Q5_K) {
        const uint32_t hb = *reinterpret_cast<const uint32_t *>(hd + 16 + 4 * (u % 8));
        uint32_t ev, od;
        q5k_codes(word, hb, i / 8, ev, od);
        q = (int)((((i & 1) ? od : ev) >> (8 * ((i % 8) / 2))) & 0xFF);
      } else {
        q = (int)((word >> (4 * (i % 8))) & 0xF);
      }
      const uint4 h = *reinterpret_cast<const uint4 *>(hd);
      const float d = f16_bits_to_f32(h.x), dmin = f16_bits_to_f32(h.x >> 16);
      uint32_t s, m;
      q4k_scale_min((int)(u % 8), h.y, h.z, h.w, s, m);
      scale = __fmul_rn(d, (float)s);
      mn = __fmul_rn(dmin, (float)m);
    } else {
      const int nib = (int)((word >> (4 * (i % 8))) & 0xF);
      q = fmt == Q4_0 ? nib - 8 : iq4nl_value(nib);
      scale = f16_bits_to_f32(sc[u * 2] | (sc[u * 2 + 1] << 8));
    }
  }
  return __fsub_rn(__fmul_rn(scale, (float)q), mn);
}

}  // namespace mgb
