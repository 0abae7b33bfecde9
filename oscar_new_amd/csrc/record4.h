// Records of 4-bit codes: 272 bytes per (token, KV head),
//   [0, 128) K codes, [128, 256) V codes: dim d in bits 4 (d % 2) of byte d / 2,
//   [256, 264) K scale, K zero, V scale, V zero (fp16), [264, 272) never written.
// The value of code c is zero + scale c. Both vectors' codes start 16-byte aligned and the scales lie
// together, so that a record is 17 pieces of 16 bytes, and a stride of 68 dwords spreads the records
// of 16 tokens over all LDS banks.
#pragma once

#include "common.h"

namespace oscar {

constexpr int kSlot4 = 272, kVector4 = 132, kCodes4 = 128, kSide4 = 256;

}  // namespace oscar
