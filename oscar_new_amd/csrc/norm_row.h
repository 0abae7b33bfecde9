// Loads, scaling and the root of a row's norm, shared by norm_rope.hip and append.hip so that both give
// the same bits.
#pragma once

#include "common.h"

namespace oscar {
namespace {

__device__ __forceinline__ float load_value(const void* p, int64_t i, int fp32) {
  return fp32 ? static_cast<const float*>(p)[i]
              : bf16_to_float(static_cast<const uint16_t*>(p)[i]);
}
// Eight consecutive values (16-byte aligned bf16, or fp32).
__device__ __forceinline__ void load_eight(const void* p, int64_t i, int fp32, float (&v)[8]) {
  if (fp32) {
    const f32x4* s = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    const f32x4 lo = s[0], hi = s[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = lo[e];
      v[4 + e] = hi[e];
    }
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = bf16_to_float(w[e] & 0xffffu);
      v[2 * e + 1] = bf16_to_float(w[e] >> 16);
    }
  }
}
__device__ __forceinline__ void unpack_eight(u32x4 w, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = bf16_to_float(w[e] & 0xffffu);
    v[2 * e + 1] = bf16_to_float(w[e] >> 16);
  }
}

// Eight packed values times a power of two (rounded where that leaves bf16's range).
__device__ __forceinline__ u32x4 scale_eight(u32x4 w, float by) {
  float v[8];
  unpack_eight(w, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(v[2 * e] * by, v[2 * e + 1] * by);
  return w;
}

// What a row is multiplied by ahead of its norm: a power of two where fp32 does not hold its squares or
// their mean with eps (magnitudes above 1e18, which would give zeros; below 4e-15 with as small an eps,
// infinities), else 1. The scaled mean lies in [2^-114, 2^120], whatever the finite bf16 row.
__device__ __forceinline__ float range_scale(float mean) {
  return mean == INFINITY ? 0x1p-72f : mean < 0x1p-96f ? 0x1p80f : 1.f;
}

// 1 / sqrt(mean), NaN for a bad row: the hardware's reciprocal root (within one unit of the last
// place), whose argument may not be subnormal.
__device__ __forceinline__ float inverse_root(float mean, bool bad) {
  const float inv = __builtin_amdgcn_rsqf(mean);
  return bad ? __uint_as_float(0x7fc00000u) : inv;
}

}  // namespace
}  // namespace oscar
