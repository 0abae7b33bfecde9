// Unpacking and paging of 4-bit records, shared by the history kernels that read them (history4.hip).
#pragma once

#include "attention.h"
#include "record4.h"

namespace oscar {

typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2_ptr_t;

constexpr uint32_t kNoBlock4 = 0xffffffffu;

// Eight codes of a dword as bf16 or fp16 values, in the order 0, 2, 4, 6, 1, 3, 5, 7: a nibble in a byte
// of its own is the e4m3 value c 2^-9 (a subnormal, or the first power above), which the conversion
// with scale 2^9 turns into c exactly. Seven instructions for eight codes.
__device__ __forceinline__ u32x4 codes_bf16(uint32_t w) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;
  auto pair = [](uint32_t b, auto high) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                                            b, 512.0f, decltype(high)::value));
  };
  return u32x4{pair(even, std::false_type()), pair(even, std::true_type()),
               pair(odd, std::false_type()), pair(odd, std::true_type())};
}
__device__ __forceinline__ u32x4 codes_f16(uint32_t w) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;
  auto pair = [](uint32_t b, auto high) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(
                                            b, 512.0f, decltype(high)::value));
  };
  return u32x4{pair(even, std::false_type()), pair(even, std::true_type()),
               pair(odd, std::false_type()), pair(odd, std::true_type())};
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Round to nearest even, as static_cast does.
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const f16x2_t v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ f32x4 mfma16x16x32_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Eight bf16 values, packed in pairs, in that order.
__device__ __forceinline__ u32x4 code_order(u32x4 w) {
  return u32x4{__builtin_amdgcn_perm(w[1], w[0], 0x05040100u),
               __builtin_amdgcn_perm(w[3], w[2], 0x05040100u),
               __builtin_amdgcn_perm(w[1], w[0], 0x07060302u),
               __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
}

// Offset (16-byte units) of kernel block kb of this request and head, or kNoBlock4: an unmapped block,
// or one that does not lie inside the history buffer.
__device__ __forceinline__ uint32_t block_offset4(const AttnArgs& a, const Task& t, int head, int kb) {
  if (kb < 0 || kb >= a.table_columns) return kNoBlock4;
  const int blk = a.table[static_cast<int64_t>(t.req) * a.table_stride + kb];
  if (blk < 0) return kNoBlock4;
  const uint32_t page = fastdiv(static_cast<uint32_t>(blk), a.L.bpp_div);
  const uint32_t inpage = static_cast<uint32_t>(blk) - page * a.L.bpp;
  const int64_t off = static_cast<int64_t>(page) * a.L.page_bytes +
                      (static_cast<int64_t>(inpage) * a.L.bk * a.L.kv_heads + head) * kSlot4;
  if (off + static_cast<int64_t>(a.L.bk) * a.L.kv_heads * kSlot4 > a.history_bytes + head * kSlot4)
    return kNoBlock4;
  return static_cast<uint32_t>(off >> 4);
}

}  // namespace oscar
