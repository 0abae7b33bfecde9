// Loads, scaling and the root of a row's norm, shared by norm_rope.hip and append.hip so that both give
// the same bits.
#pragma once

#include "common.h"

namespace oscar {

// Angles of tokens with several positions: pair j turns by the table's row at the position of its axis.
struct AxisTable {
  const void* table;  // [rows][rotary]: cos of every pair, then sin
  int64_t rows, stride;
  const int64_t* positions;  // axis a of token t at a * position_stride + t
  int64_t position_stride;
  const int32_t* axes;  // of every pair, 16-byte aligned
  int32_t count, rotary;
};

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

// Axes of the kN pairs from pair0 on (a multiple of 4), and whether they are one of the positions' alone:
// sections are mostly longer than a lane's pairs, and then one row and one load serve all of them.
template <int kN>
struct PairAxes {
  int axis[kN];
  bool one;
};
template <int kN>
__device__ __forceinline__ PairAxes<kN> pair_axes(const AxisTable& t, int pair0) {
  PairAxes<kN> r;
#pragma unroll
  for (int i = 0; i < kN / 4; ++i) {
    const u32x4 v = reinterpret_cast<const u32x4*>(t.axes + pair0)[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) r.axis[4 * i + e] = static_cast<int>(v[e]);
  }
  r.one = r.axis[0] >= 0 && r.axis[0] < t.count;
#pragma unroll
  for (int e = 1; e < kN; ++e) r.one &= r.axis[e] == r.axis[0];
  return r;
}

// Packed cosines and sines (bf16 pairs, or fp32 words) of those pairs of a live token. Where some lane's
// pairs are mixed, each axis' row is loaded in turn by the lanes that have a pair of it, and its values
// selected (loads of single values instead held up the address units: 16384 tokens of 7 heads 54 us). A
// pair of no axis gets NaN; so does, with its whole row, one whose position is outside the table.
// `position`: the token's on an axis.
template <int kN, bool kFp32, int kWords, class Position>
__device__ __forceinline__ void axis_words(const AxisTable& t, Position position, int pair0,
                                           const PairAxes<kN>& pairs, uint32_t (&c)[kWords],
                                           uint32_t (&s)[kWords]) {
  static_assert(kWords * (kFp32 ? 1 : 2) == kN, "kN angles");
  const int half = t.rotary >> 1;
  constexpr int kBytes = kFp32 ? 4 : 2;
  auto load = [](const char* from, uint32_t (&w)[kWords]) {
    if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(from);
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 v = reinterpret_cast<const u32x4*>(from)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
      }
    }
  };
  auto row_of = [&](int axis) {
    const int64_t p = position(axis);
    const int64_t row = p >= 0 && p < t.rows ? p : 0;  // the token's rows are NaN where it is not
    return static_cast<const char*>(t.table) + (row * t.stride + pair0) * kBytes;
  };
  if (__all(pairs.one)) {
    const char* at = row_of(pairs.axis[0]);
    load(at, c);
    load(at + half * kBytes, s);
    return;
  }
#pragma unroll
  for (int w = 0; w < kWords; ++w) c[w] = s[w] = kFp32 ? 0x7fc00000u : 0x7fc07fc0u;
  for (int k = 0; k < t.count; ++k) {
    uint32_t take[kWords], any = 0;  // the words' bits that are of axis k
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      if (kFp32)
        take[w] = pairs.axis[w % kN] == k ? 0xffffffffu : 0u;
      else
        take[w] = (pairs.axis[2 * w % kN] == k ? 0xffffu : 0u) |
                  (pairs.axis[(2 * w + 1) % kN] == k ? 0xffff0000u : 0u);
      any |= take[w];
    }
    const char* at = row_of(k);  // by all lanes: `position` may read another's
    if (!any) continue;
    uint32_t cv[kWords], sv[kWords];
    load(at, cv);
    load(at + half * kBytes, sv);
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      c[w] = (cv[w] & take[w]) | (c[w] & ~take[w]);
      s[w] = (sv[w] & take[w]) | (s[w] & ~take[w]);
    }
  }
}

// Whether a live token's position on `axis` lies outside the table.
__device__ __forceinline__ bool bad_position(const AxisTable& t, int64_t token, int axis) {
  const int64_t p = t.positions[axis * t.position_stride + token];
  return p < 0 || p >= t.rows;
}

}  // namespace
}  // namespace oscar
