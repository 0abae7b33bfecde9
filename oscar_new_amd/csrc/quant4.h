// Clip + 4-bit quantize of one 256-element vector by one wavefront (lane l: elements 4 l .. 4 l + 3):
//   zero = fp16(min x), scale = fp16(max((max - min) / 15, 2^-14)) of the clipped values,
//   code = clamp(trunc((x - zero) / scale + 0.5), 0, 15)        (IEEE fp32, no contraction),
// clipped as quant.h clips (a quantile of |x|, a factor of its maximum, or the factor of eight with the
// least squared error). Floors and ties follow quant.h's 2-bit rule, with 15 steps instead of 3.
#pragma once

#include <type_traits>

#include "quant.h"
#include "record4.h"

namespace oscar {

struct Quantized4 {
  uint32_t codes;        // this lane's four codes, 16 bits
  uint32_t scale, zero;  // fp16 bits
};

// The quotient is taken through the scale's reciprocal (within one ulp), as in quant.h: for y in
// [0.5, 15.5], fma(d, r, 0.5) differs from fl(fl(d / scale) + 0.5) by at most
// 15 (2^-23 + 2^-24) + 2 x 2^-21 < 4e-6, so a value further than 2^-16 from every integer truncates to
// the same code; a wavefront with a nearer one takes the IEEE quotient. `code`: the codes as floats.
__device__ __forceinline__ Quantized4 quantize4(const float x[4], float thr, float mn, float mx,
                                                float (&code)[4], float& sf, float& zf) {
#pragma clang fp contract(off)
  const bool whole = mn == mn && mx == mx;  // no NaN (wave_min_max has one as an extreme)
  float xc[4];
  if (thr == INFINITY) {
#pragma unroll
    for (int i = 0; i < 4; ++i) xc[i] = x[i];
  } else {
    clamp4(x, thr, xc);
    mn = clamp1(mn, thr);
    mx = clamp1(mx, thr);
  }
  float spread = (mx - mn) / 15.0f;
  spread = spread < 6.103515625e-05f ? 6.103515625e-05f : spread;
  if (!whole) spread = mn = __uint_as_float(0x7fc00000u);  // so are the record's values
  Quantized4 q;
  q.zero = float_to_f16_bits(mn);
  q.scale = float_to_f16_bits(spread);
  zf = f16_bits_to_float(q.zero);
  sf = f16_bits_to_float(q.scale);
  const float r = scale_rcp(sf);
  float y[4];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = __builtin_fmaf(xc[i] - zf, r, 0.5f);
    near |= fabsf(y[i] - rintf(y[i])) < 1.52587890625e-05f;
  }
  if (__any(near)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (xc[i] - zf) / sf + 0.5f;
  }
  q.codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int c = static_cast<int>(y[i]);
    c = c < 0 ? 0 : (c > 15 ? 15 : c);
    code[i] = static_cast<float>(c);
    q.codes |= static_cast<uint32_t>(c) << (4 * i);
  }
  return q;
}

// Codes to `codes` (128 bytes), scale and zero to `side` (4 bytes); nothing is written when codes is
// null.
__device__ __forceinline__ void quantize_store4(const float x[4], int mode, float ratio, float factor,
                                                uint8_t* codes, uint8_t* side) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63;
  float mn, mx, code[4], sf, zf;
  wave_min_max(x, mn, mx);
  const float maxabs = fmaxf(fabsf(mn), fabsf(mx));
  float thr = INFINITY;
  if (mode == OSCAR_CLIP_FACTOR) {
    thr = maxabs * factor;
  } else if (mode == OSCAR_CLIP_SEARCH) {
    // Every candidate's codes and their squared error, in order; the first least one stays.
    float least = INFINITY;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const float t = maxabs * search_factor(i);
      quantize4(x, t, mn, mx, code, sf, zf);
      float sq[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float err = x[e] - (code[e] * sf + zf);
        sq[e] = err * err;
      }
      const float sum = wave_tree_sum_dpp((sq[0] + sq[1]) + (sq[2] + sq[3]));
      if (i == 0 || sum < least) {
        least = sum;
        thr = t;
      }
    }
  } else if (ratio != 0.0f) {
    thr = percentile_threshold(x, ratio);
  }
  const Quantized4 q = quantize4(x, thr, mn, mx, code, sf, zf);
  if (codes) {
    reinterpret_cast<uint16_t*>(codes)[lane] = static_cast<uint16_t>(q.codes);
    if (lane == 0) *reinterpret_cast<uint32_t*>(side) = q.scale | (q.zero << 16);
  }
}

}  // namespace oscar
