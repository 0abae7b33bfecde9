// Norms of the queries and keys of each head with the position rotation in the same pass, and
// optionally the rotation of the queries by R_k that the INT2 history wants.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (w, or 1 + w with a unit offset)
//   (a, b) -> (a cos - b sin, b cos + a sin)     for the pairs of the first `rotary` dims: dims
//                                                i and i + rotary / 2, or 2 i and 2 i + 1
//   q_rot = bf16(y) R_k                          (fp32 accumulation, the bits of oscar_rotate)
//
// No reference counterpart: the reference's layer gets its queries and keys after this
// (oscar_ascend/backend.py:125-140). Sums, norms and angles are fp32; a row is rounded to bf16 once,
// and the rotation by R_k reads the rounded row, as the attention's BF16 branch does.
//
// Half a wavefront holds a row: 32 lanes of 8 dims, one 16-byte load each, the sum of squares
// through DPP moves and one lane swap. A pair's other half is read again from memory (the row is
// in the cache by then) rather than moved between lanes: one 16-byte load, in flight with the
// lane's own, against four cross-lane moves behind it.
#include "rotate.h"

namespace oscar {
namespace {

enum PairMode { kPairHalves = 0, kPairAdjacent = 1, kPairGeneric = 2 };

struct NormArgs {
  const uint16_t* x;
  int64_t s0, s1;  // token and head strides, elements
  const void* weight;
  uint16_t* out;  // [tokens][heads][256]
  int64_t rows;
  int32_t heads;
  FastDiv h_div;
};

struct NormRopeArgs {
  NormArgs q, k;
  const void* table;  // [table_rows][rotary]: cos of every pair, then sin
  int64_t table_rows, table_stride;
  const int64_t* positions;
  const int32_t* counts;  // null: every token is live
  int64_t n;
  int32_t rotary, weight_fp32, table_fp32, adjacent;
  float offset, eps;
  const uint16_t* rk_t;  // R_k^T [256][256]
  uint16_t* q_rot;
  int32_t q_groups;  // workgroups of the query rows (kRotate)
};

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

// The lane's dims 8 l .. 8 l + 7 within a row: weights of its own dims and of their partners.
struct LaneWeights {
  float own[8], pair[8];
};

// Partner of dim d, the index of its angle and the sign of the partner's term.
__device__ __forceinline__ void pair_of(const NormRopeArgs& a, int d, int& pair, int& angle,
                                        float& sign) {
  const int half = a.rotary >> 1;
  if (a.adjacent) {
    pair = d ^ 1;
    angle = d >> 1;
    sign = d & 1 ? 1.f : -1.f;
  } else {
    pair = d < half ? d + half : d - half;
    angle = d < half ? d : d - half;
    sign = d < half ? -1.f : 1.f;
  }
}

template <int kMode>
__device__ __forceinline__ void load_weights(const NormRopeArgs& a, const void* weight, int l,
                                             LaneWeights& w) {
  load_eight(weight, 8 * l, a.weight_fp32, w.own);
#pragma unroll
  for (int e = 0; e < 8; ++e) w.own[e] += a.offset;
  const int half = a.rotary >> 1;
  if (kMode == kPairHalves) {
    const int d = 8 * l < half ? 8 * l + half : 8 * l - half;
    load_eight(weight, 8 * l < a.rotary ? d : 0, a.weight_fp32, w.pair);
#pragma unroll
    for (int e = 0; e < 8; ++e) w.pair[e] += a.offset;
  } else if (kMode == kPairAdjacent) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w.pair[e] = w.own[e ^ 1];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int p = 0, j;
      float s;
      if (8 * l + e < a.rotary) pair_of(a, 8 * l + e, p, j, s);
      w.pair[e] = load_value(weight, p, a.weight_fp32) + a.offset;
    }
  }
}

// What a row needs from memory: its lane's values, their partners and the angles.
struct RowLoads {
  u32x4 x;
  float pair[8], c[8], s[8];
  bool live, bad;  // a live token; its position is outside the table
};

template <int kMode>
__device__ __forceinline__ void load_row(const NormRopeArgs& a, const NormArgs& t, int64_t row,
                                         int64_t active, int l, RowLoads& r) {
  const int64_t safe = row < t.rows ? row : 0;
  const int64_t token = fastdiv(static_cast<uint32_t>(safe), t.h_div);
  const uint16_t* x = t.x + token * t.s0 + (safe - token * t.heads) * t.s1;
  r.live = row < t.rows && token < active;
  r.x = *reinterpret_cast<const u32x4*>(x + 8 * l);
  const int64_t pos = r.live ? a.positions[token] : 0;
  r.bad = a.rotary > 0 && (pos < 0 || pos >= a.table_rows);
  const int64_t at = (r.bad ? 0 : pos) * a.table_stride;
  const int half = a.rotary >> 1;
  if (8 * l >= a.rotary) return;  // nothing else is read
  if (kMode == kPairHalves) {
    const bool low = 8 * l < half;
    const int d = low ? 8 * l : 8 * l - half;
    unpack_eight(*reinterpret_cast<const u32x4*>(x + (low ? 8 * l + half : 8 * l - half)), r.pair);
    load_eight(a.table, at + d, a.table_fp32, r.c);
    load_eight(a.table, at + half + d, a.table_fp32, r.s);
#pragma unroll
    for (int e = 0; e < 8; ++e) r.s[e] = low ? -r.s[e] : r.s[e];
  } else if (kMode == kPairAdjacent) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float c = load_value(a.table, at + 4 * l + e, a.table_fp32);
      const float s = load_value(a.table, at + half + 4 * l + e, a.table_fp32);
      r.c[2 * e] = r.c[2 * e + 1] = c;
      r.s[2 * e] = -s;
      r.s[2 * e + 1] = s;
    }
    float v[8];
    unpack_eight(r.x, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) r.pair[e] = v[e ^ 1];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (8 * l + e >= a.rotary) break;
      int p, j;
      float sign;
      pair_of(a, 8 * l + e, p, j, sign);
      r.pair[e] = bf16_to_float(x[p]);
      r.c[e] = load_value(a.table, at + j, a.table_fp32);
      r.s[e] = sign * load_value(a.table, at + half + j, a.table_fp32);
    }
  }
}

// The row's 8 dims of this lane as bf16: zeros past the live tokens, NaN at a position outside the
// table (never a row of wrong angles).
__device__ __forceinline__ u32x4 finish_row(const NormRopeArgs& a, const LaneWeights& w,
                                            const RowLoads& r, int l) {
  float v[8], sum = 0.f;
  unpack_eight(r.x, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
  sum += dpp<kDppQuadXor1>(sum);
  sum += dpp<kDppQuadXor2>(sum);
  sum += dpp<kDppRowHalfMirror>(sum);
  sum += dpp<kDppRowMirror>(sum);
  sum = sum_xor16(sum);
  const float inv = r.bad ? __uint_as_float(0x7fc00000u)
                          : 1.0f / sqrtf(fmaf(sum, 1.0f / kHeadDim, a.eps));
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = v[e] * inv * w.own[e], p = r.pair[e] * inv * w.pair[e];
    o[e] = 8 * l + e < a.rotary ? fmaf(y, r.c[e], p * r.s[e]) : y;
  }
  u32x4 bits;
#pragma unroll
  for (int e = 0; e < 4; ++e) bits[e] = r.live ? pack_bf16x2(o[2 * e], o[2 * e + 1]) : 0u;
  return bits;
}

__device__ __forceinline__ int64_t live_tokens(const NormRopeArgs& a) {
  return a.counts ? min(static_cast<int64_t>(max(a.counts[1], 0)), a.n) : a.n;
}

// ---- no rotation by R_k: 8 rows per workgroup, query rows first.
template <int kMode>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeArgs a,
                                                             int64_t q_blocks) {
  const int l = threadIdx.x & 31;
  const bool is_q = blockIdx.x < q_blocks;
  const NormArgs& t = is_q ? a.q : a.k;
  const int64_t row = (blockIdx.x - (is_q ? 0 : q_blocks)) * 8 + (threadIdx.x >> 5);
  RowLoads r;
  LaneWeights w;
  load_row<kMode>(a, t, row, live_tokens(a), l, r);
  load_weights<kMode>(a, t.weight, l, w);
  const u32x4 bits = finish_row(a, w, r, l);
  if (row < t.rows) *reinterpret_cast<u32x4*>(t.out + row * kHeadDim + 8 * l) = bits;
}

// ---- with the rotation: workgroups of 8 wavefronts walk 16-row blocks of the queries. A wavefront
// keeps its 16 kTiles columns of R_k in registers for the whole walk (kTiles 2: the workgroup holds
// R_k once, 64 registers a lane; kTiles 1: two workgroups share the columns of a block, for the few
// rows of a decode step). The block's rows go through LDS (16-byte piece p of row r at p ^ r) as the
// B operand; the columns are the A operand, so that a lane ends with 4 kTiles consecutive columns
// of one row and stores them at once. Key rows are workgroups of their own behind the queries'.
constexpr int kRopeWaves = 8;

template <int kMode, int kTiles>
__global__ __launch_bounds__(kRopeWaves * kWave, kTiles == 2 || kMode == kPairGeneric ? 2 : 4) void norm_rope_rotate_kernel(
    const NormRopeArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t s_rows[2][16 * kHeadDim * 2];
  const int tid = threadIdx.x, l = tid & 31, r16 = tid >> 5;
  const int64_t active = live_tokens(a);
  const bool is_q = static_cast<int>(blockIdx.x) < a.q_groups;
  LaneWeights w;
  if (!is_q) {
    if (blockIdx.y) return;
    const int64_t row = static_cast<int64_t>(blockIdx.x - a.q_groups) * 16 + r16;
    RowLoads r;
    load_row<kMode>(a, a.k, row, active, l, r);
    load_weights<kMode>(a, a.k.weight, l, w);
    const u32x4 bits = finish_row(a, w, r, l);
    if (row < a.k.rows) *reinterpret_cast<u32x4*>(a.k.out + row * kHeadDim + 8 * l) = bits;
    return;
  }
  const int lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  // A row n of tile t is column base + 4 kTiles (n / 4) + 4 t + n % 4.
  const int base = 16 * kTiles * (kRopeWaves * blockIdx.y + wave);
  const int64_t blocks = (a.q.rows + 15) / 16;
  RowLoads r;
  load_row<kMode>(a, a.q, static_cast<int64_t>(blockIdx.x) * 16 + r16, active, l, r);
  load_weights<kMode>(a, a.q.weight, l, w);
  u32x4 rk[kTiles][8];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const uint16_t* col =
        a.rk_t + static_cast<int64_t>(base + 4 * kTiles * (n >> 2) + 4 * t + (n & 3)) * kHeadDim;
#pragma unroll
    for (int m = 0; m < 8; ++m) rk[t][m] = *reinterpret_cast<const u32x4*>(col + 32 * m + 8 * g);
  }
  int buf = 0;
  for (int64_t b = blockIdx.x; b < blocks; b += a.q_groups, buf ^= 1) {
    const int64_t row = b * 16 + r16;
    const u32x4 bits = finish_row(a, w, r, l);
    *reinterpret_cast<u32x4*>(&s_rows[buf][r16 * 512 + 16 * (l ^ r16)]) = bits;
    if (blockIdx.y == 0 && row < a.q.rows)
      *reinterpret_cast<u32x4*>(a.q.out + row * kHeadDim + 8 * l) = bits;
    // The next block's rows are in flight while this one's are multiplied.
    if (b + a.q_groups < blocks) load_row<kMode>(a, a.q, row + 16ll * a.q_groups, active, l, r);
    __syncthreads();  // one barrier per block: the other buffer's readers are a block behind it
    f32x4 acc[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(&s_rows[buf][n * 512 + 16 * ((4 * m + g) ^ n)]);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) acc[t] = mfma16x16x32(rk[t][m], x, acc[t]);
    }
    const int64_t orow = b * 16 + n;
    if (orow < a.q.rows) {
      uint16_t* out = a.q_rot + orow * kHeadDim + base + 4 * kTiles * g;
      if constexpr (kTiles == 2) {
        *reinterpret_cast<u32x4*>(out) =
            u32x4{pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3]),
                  pack_bf16x2(acc[1][0], acc[1][1]), pack_bf16x2(acc[1][2], acc[1][3])};
      } else {
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3]));
      }
    }
  }
}

// Query blocks up to which two workgroups share a block's columns: with fewer blocks than CUs the
// second workgroup halves what each reads of R_k.
constexpr int64_t kSharedColumnBlocks = 128;
constexpr int64_t kRotateGroups = 256;  // one workgroup per CU walks the blocks

template <int kMode>
void launch_norm_rope(NormRopeArgs& a, hipStream_t s) {
  if (!a.rk_t) {
    const int64_t q_blocks = (a.q.rows + 7) / 8, k_blocks = (a.k.rows + 7) / 8;
    hipLaunchKernelGGL((norm_rope_kernel<kMode>), dim3(static_cast<unsigned>(q_blocks + k_blocks)),
                       dim3(kThreads), 0, s, a, q_blocks);
    return;
  }
  const int64_t blocks = (a.q.rows + 15) / 16;
  a.q_groups = static_cast<int32_t>(blocks < kRotateGroups ? blocks : kRotateGroups);
  const unsigned x = static_cast<unsigned>(a.q_groups + (a.k.rows + 15) / 16);
  if (blocks <= kSharedColumnBlocks)
    hipLaunchKernelGGL((norm_rope_rotate_kernel<kMode, 1>), dim3(x, 2), dim3(kRopeWaves * kWave), 0,
                       s, a);
  else
    hipLaunchKernelGGL((norm_rope_rotate_kernel<kMode, 2>), dim3(x, 1), dim3(kRopeWaves * kWave), 0,
                       s, a);
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace oscar

extern "C" int oscar_qk_norm_rope(const void* query, int64_t q_s0, int64_t q_s1, const void* key,
                                  int64_t k_s0, int64_t k_s1, int64_t n, int64_t hq, int64_t hk,
                                  const void* q_weight, const void* k_weight, int32_t weight_fp32,
                                  int32_t unit_offset, float eps, const void* cos_sin,
                                  int64_t table_rows, int64_t table_stride, int32_t table_fp32,
                                  int32_t rotary_dim, int32_t interleaved,
                                  const int64_t* positions, const int32_t* counts, void* q_out,
                                  void* k_out, const void* rk_t, void* q_rot, void* stream) {
  using namespace oscar;
  if (n < 0 || hq <= 0 || hk <= 0 || (rotary_dim && table_rows < 1)) return OSCAR_E_SHAPE;
  if (rotary_dim < 0 || rotary_dim > kHeadDim || rotary_dim % 2 || table_stride < rotary_dim)
    return OSCAR_E_SHAPE;
  if (!(eps >= 0.f) || !(eps < INFINITY)) return OSCAR_E_UNSUPPORTED;
  if (n == 0) return OSCAR_OK;
  if (!query || !key || !q_weight || !k_weight || !positions || !q_out || !k_out ||
      (rotary_dim && !cos_sin) || !rk_t != !q_rot)
    return OSCAR_E_NULL;
  if (hq > 0x7fffffffll / n || hk > 0x7fffffffll / n) return OSCAR_E_SHAPE;
  if (q_s0 % 8 || q_s1 % 8 || k_s0 % 8 || k_s1 % 8 || !aligned16(query) || !aligned16(key) ||
      !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(q_out) || !aligned16(k_out) ||
      (rk_t && (!aligned16(rk_t) || !aligned16(q_rot))))
    return OSCAR_E_ALIGN;
  NormRopeArgs a;
  a.q = {static_cast<const uint16_t*>(query), q_s0, q_s1, q_weight, static_cast<uint16_t*>(q_out),
         n * hq, static_cast<int32_t>(hq), make_fastdiv(static_cast<uint32_t>(hq))};
  a.k = {static_cast<const uint16_t*>(key), k_s0, k_s1, k_weight, static_cast<uint16_t*>(k_out),
         n * hk, static_cast<int32_t>(hk), make_fastdiv(static_cast<uint32_t>(hk))};
  a.table = cos_sin;
  a.table_rows = table_rows;
  a.table_stride = table_stride;
  a.positions = positions;
  a.counts = counts;
  a.n = n;
  a.rotary = rotary_dim;
  a.weight_fp32 = weight_fp32 ? 1 : 0;
  a.table_fp32 = table_fp32 ? 1 : 0;
  a.adjacent = interleaved ? 1 : 0;
  a.offset = unit_offset ? 1.f : 0.f;
  a.eps = eps;
  a.rk_t = static_cast<const uint16_t*>(rk_t);
  a.q_rot = static_cast<uint16_t*>(q_rot);
  a.q_groups = 0;
  hipStream_t s = as_stream(stream);
  const bool rows16 = aligned16(cos_sin) && table_stride % 8 == 0;
  if (interleaved && rotary_dim % 8 == 0)
    launch_norm_rope<kPairAdjacent>(a, s);
  else if (!interleaved && rotary_dim % 16 == 0 && rows16)
    launch_norm_rope<kPairHalves>(a, s);
  else
    launch_norm_rope<kPairGeneric>(a, s);
  return static_cast<int>(hipGetLastError());
}
