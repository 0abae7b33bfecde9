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
//
// What bounds it (us, calls back to back in a graph): without R_k the memory (16384 tokens of 7 heads,
// 120 MB: 26.5, 4.5 TB/s; 31.6 where three inputs alternate and none is in the last-level cache); with
// R_k the memory too for many rows (the same with R_k, 170 MB: 35.2), the loads of rows and R_k and then
// R_k's reads from LDS for a chunk (2048 tokens of 14 heads, 42 MB: 14.1); a decode step its chain of
// loads (32 tokens of 7 heads: 5.2, 4.3 without R_k).
#include <type_traits>

#include "dma.h"
#include "norm_row.h"
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
  int32_t rotary, weight_fp32, adjacent;
  float offset, eps;
  const uint16_t* rk_t;  // R_k^T [256][256]
  uint16_t* q_rot;
  AxisTable axes;  // tokens with several positions (norm_rope_axes_kernel)
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

// The weight of every dim (with the offset), in LDS: sixteen values a lane would cost the walking
// kernel registers that it needs. Threads from .. from + 31 of the workgroup write it.
__device__ __forceinline__ void stage_weights(const NormRopeArgs& a, const void* weight,
                                              float* s_weight, int from) {
  const int i = static_cast<int>(threadIdx.x) - from;
  if (i < 0 || i >= 32) return;
  float w[8];
  load_eight(weight, 8 * i, a.weight_fp32, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) s_weight[8 * i + e] = w[e] + a.offset;
  if (i == 0)
#pragma unroll
    for (int e = 0; e < 8; ++e) s_weight[kHeadDim + e] = 0.f;
}

// A token's angles for the lane's dims, as they lie in the table: bf16 or fp32 words of the
// cosines and sines, or (generic) the fp32 values themselves. They stay packed while a load is in
// flight, as do the rows: a conversion waits for it.
template <int kMode, bool kFp32>
struct Angles {
  static constexpr int kWords = kMode == kPairGeneric || (kMode == kPairHalves && kFp32) ? 2 : 1;
  u32x4 c[kWords], s[kWords];
  bool live, bad;  // a live token; its position is outside the table
};
struct RowLoads {
  u32x4 x, pair;  // the lane's values and, where halves are paired, their partners
};

template <int kMode, bool kFp32>
__device__ __forceinline__ void load_angles(const NormRopeArgs& a, int64_t token, int64_t position,
                                            int64_t active, int l, Angles<kMode, kFp32>& r) {
  r.live = token < active;
  const int64_t pos = r.live ? position : 0;
  r.bad = a.rotary > 0 && (pos < 0 || pos >= a.table_rows);
  if (8 * l >= a.rotary) return;  // keeps its identity turn (start_row)
  const int64_t at = (r.bad ? 0 : pos) * a.table_stride;
  const int half = a.rotary >> 1;
  if constexpr (kMode == kPairHalves) {
    const int64_t c = at + (8 * l < half ? 8 * l : 8 * l - half);
#pragma unroll
    for (int w = 0; w < r.kWords; ++w) {
      const char* p = static_cast<const char*>(a.table) + 16 * w;
      r.c[w] = *reinterpret_cast<const u32x4*>(p + c * (kFp32 ? 4 : 2));
      r.s[w] = *reinterpret_cast<const u32x4*>(p + (c + half) * (kFp32 ? 4 : 2));
    }
  } else if constexpr (kMode == kPairAdjacent) {  // four pairs a lane
    if constexpr (kFp32) {
      r.c[0] = *reinterpret_cast<const u32x4*>(static_cast<const float*>(a.table) + at + 4 * l);
      r.s[0] = *reinterpret_cast<const u32x4*>(static_cast<const float*>(a.table) + at + half + 4 * l);
    } else {
      const uint16_t* t = static_cast<const uint16_t*>(a.table) + at + 4 * l;
      const uint2 c = *reinterpret_cast<const uint2*>(t);
      const uint2 s = *reinterpret_cast<const uint2*>(t + half);
      r.c[0] = u32x4{c.x, c.y, 0u, 0u};
      r.s[0] = u32x4{s.x, s.y, 0u, 0u};
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (8 * l + e >= a.rotary) break;
      int p, j;
      float sign;
      pair_of(a, 8 * l + e, p, j, sign);
      r.c[e >> 2][e & 3] = __float_as_uint(load_value(a.table, at + j, kFp32));
      r.s[e >> 2][e & 3] = __float_as_uint(load_value(a.table, at + half + j, kFp32));
    }
  }
}

// A lane past the rotary dims turns by cosine 1, sine 0 and a partner of 0 times 0: set once, since
// the loads leave such lanes alone. (A lane that ends inside them, as generic dims may, is selected
// per element.)
template <int kMode, bool kFp32>
__device__ __forceinline__ void start_row(Angles<kMode, kFp32>& t, RowLoads& r) {
  const bool fp32 = kFp32 || kMode == kPairGeneric;
#pragma unroll
  for (int w = 0; w < t.kWords; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t.c[w][e] = fp32 ? 0x3f800000u : 0x3f803f80u;
      t.s[w][e] = 0u;
      r.pair[e] = 0u;
    }
}

// Cosine and sine of the lane's dim 8 l + e; the partner's term has the sign of partner_sign.
template <int kMode>
__device__ __forceinline__ float partner_sign(const NormRopeArgs& a, int l, int e, float v) {
  if (kMode == kPairAdjacent) return e & 1 ? v : -v;
  if (kMode == kPairHalves) return v;  // one sign a lane, taken before (finish_row)
  int p, j;
  float sign;
  pair_of(a, 8 * l + e, p, j, sign);
  return sign * v;
}
template <int kMode, bool kFp32>
__device__ __forceinline__ void angle_of(const Angles<kMode, kFp32>& r, int e, float& c, float& s) {
  auto half_word = [](uint32_t w, int i) { return bf16_to_float(i & 1 ? w >> 16 : w & 0xffffu); };
  if constexpr (kMode == kPairAdjacent) {
    const int j = e >> 1;
    c = kFp32 ? __uint_as_float(r.c[0][j]) : half_word(r.c[0][j >> 1], j);
    s = kFp32 ? __uint_as_float(r.s[0][j]) : half_word(r.s[0][j >> 1], j);
  } else if constexpr (kMode == kPairHalves) {
    c = kFp32 ? __uint_as_float(r.c[e >> 2 & (r.kWords - 1)][e & 3]) : half_word(r.c[0][e >> 1], e);
    s = kFp32 ? __uint_as_float(r.s[e >> 2 & (r.kWords - 1)][e & 3]) : half_word(r.s[0][e >> 1], e);
  } else {
    c = __uint_as_float(r.c[e >> 2][e & 3]);
    s = __uint_as_float(r.s[e >> 2][e & 3]);
  }
}

template <int kMode>
__device__ __forceinline__ void load_row(const NormRopeArgs& a, const uint16_t* x, int l,
                                         RowLoads& r) {
  r.x = *reinterpret_cast<const u32x4*>(x + 8 * l);
  if (kMode == kPairAdjacent || 8 * l >= a.rotary) return;
  const int half = a.rotary >> 1;
  if (kMode == kPairHalves) {
    r.pair = *reinterpret_cast<const u32x4*>(x + (8 * l < half ? 8 * l + half : 8 * l - half));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (8 * l + e >= a.rotary) break;
      int p, j;
      float sign;
      pair_of(a, 8 * l + e, p, j, sign);
      const uint32_t bits = x[p];
      r.pair[e >> 1] = e & 1 ? (r.pair[e >> 1] & 0xffffu) | bits << 16
                             : (r.pair[e >> 1] & 0xffff0000u) | bits;
    }
  }
}

// The row's 8 dims of this lane as bf16: zeros past the live tokens, NaN at a position outside the
// table (never a row of wrong angles).
template <int kMode, bool kFp32>
__device__ __forceinline__ u32x4 finish_row(const NormRopeArgs& a, const float* s_weight,
                                            const Angles<kMode, kFp32>& t, const RowLoads& r,
                                            int l) {
  float own_w[8], pair_w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) own_w[e] = s_weight[8 * l + e];
  const int half = a.rotary >> 1;
  // Past the rotary dims: the zeros behind the weights.
  const int partner = 8 * l >= a.rotary ? kHeadDim : 8 * l < half ? 8 * l + half : 8 * l - half;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (kMode == kPairAdjacent) {
      pair_w[e] = own_w[e ^ 1];
    } else if (kMode == kPairHalves) {
      pair_w[e] = s_weight[partner + e];
    } else {
      int p = kHeadDim, j;
      float sign;
      if (8 * l + e < a.rotary) pair_of(a, 8 * l + e, p, j, sign);
      pair_w[e] = s_weight[p];
    }
  }
  u32x4 own = r.x, other = r.pair;
  auto mean_square = [&](float eps) {
    float v[8], sum = 0.f;
    unpack_eight(own, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
    sum += dpp<kDppQuadXor1>(sum);
    sum += dpp<kDppQuadXor2>(sum);
    sum += dpp<kDppRowHalfMirror>(sum);
    sum += dpp<kDppRowMirror>(sum);
    sum = sum_xor16(sum);
    return fmaf(sum, 1.0f / kHeadDim, eps);
  };
  float mean = mean_square(a.eps);
  if (const float by = range_scale(mean); __builtin_expect(__any(by != 1.f), 0)) {
    // The packed values are scaled, so that no register more is live across the branch.
    own = scale_eight(own, by);
    other = scale_eight(other, by);
    mean = mean_square(a.eps * by * by);
  }
  const float inv = inverse_root(mean, t.bad);
  float v[8], pair[8];
  unpack_eight(own, v);
  if (kMode == kPairAdjacent) {
#pragma unroll
    for (int e = 0; e < 8; ++e) pair[e] = v[e ^ 1];
  } else {
    unpack_eight(other, pair);
  }
  const float pair_inv = kMode == kPairHalves && 8 * l < half ? -inv : inv;
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = v[e] * inv * own_w[e], p = pair[e] * pair_inv * pair_w[e];
    float c, s;
    angle_of(t, e, c, s);
    const float turned = fmaf(y, c, partner_sign<kMode>(a, l, e, p) * s);
    o[e] = kMode == kPairHalves || 8 * l + e < a.rotary ? turned : y;
  }
  u32x4 bits;
#pragma unroll
  for (int e = 0; e < 4; ++e) bits[e] = t.live ? pack_bf16x2(o[2 * e], o[2 * e + 1]) : 0u;
  return bits;
}

__device__ __forceinline__ int64_t live_tokens(const NormRopeArgs& a) {
  return a.counts ? min(static_cast<int64_t>(max(a.counts[1], 0)), a.n) : a.n;
}

// ---- no rotation by R_k. Half a wavefront takes one token's rows of up to kRopeHeads heads: their
// loads and the token's angles are in flight together (one row per half wavefront, the angles read
// again for each, keeps half as many bytes in flight: 16384 tokens x 7 heads 30 us).
constexpr int kRopeHeads = 4;

template <int kMode, bool kFp32>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeArgs a,
                                                             int64_t q_blocks, FastDiv q_div,
                                                             FastDiv k_div) {
  __shared__ float s_weight[kHeadDim + 8];
  const int l = threadIdx.x & 31;
  const bool is_q = blockIdx.x < q_blocks;
  const NormArgs& t = is_q ? a.q : a.k;
  stage_weights(a, t.weight, s_weight, 0);
  __syncthreads();
  const FastDiv div = is_q ? q_div : k_div;  // items per token
  const uint32_t item =
      static_cast<uint32_t>((blockIdx.x - (is_q ? 0 : q_blocks)) * 8 + (threadIdx.x >> 5));
  const uint32_t index = fastdiv(item, div);
  if (index >= a.n) return;
  const int64_t token = index;
  const int h0 = static_cast<int>(item - index * div.divisor) * kRopeHeads;
  const int count = min(kRopeHeads, t.heads - h0);
  const int64_t active = live_tokens(a);
  const int64_t position = token < active ? a.positions[token] : 0;
  const uint16_t* x = t.x + token * t.s0 + h0 * t.s1;
  RowLoads r[kRopeHeads];
  Angles<kMode, kFp32> angles;
#pragma unroll
  for (int i = 0; i < kRopeHeads; ++i) start_row(angles, r[i]);
#pragma unroll
  for (int i = 0; i < kRopeHeads; ++i)
    if (i < count) load_row<kMode>(a, x + i * t.s1, l, r[i]);
  load_angles(a, token, position, active, l, angles);
  uint16_t* out = t.out + (token * t.heads + h0) * kHeadDim + 8 * l;
#pragma unroll
  for (int i = 0; i < kRopeHeads; ++i)
    if (i < count)
      *reinterpret_cast<u32x4*>(out + i * kHeadDim) = finish_row(a, s_weight, angles, r[i], l);
}

// ---- tokens with several positions, no rotation by R_k: half a wavefront takes up to eight of a token's
// rows, queries and keys in one list, since its angles cost more here: a position per axis, and a load of
// each axis' table row for the lanes that have a pair of it.
constexpr int kAxesHeads = 8;

template <int kMode, bool kFp32>
__global__ __launch_bounds__(kThreads) void norm_rope_axes_kernel(const NormRopeArgs a,
                                                                  FastDiv per_token) {
  static_assert(kMode != kPairGeneric, "pairs of eight dims");
  constexpr int kN = kMode == kPairHalves ? 8 : 4, kWords = kFp32 ? kN : kN / 2;
  __shared__ float s_weight[2][kHeadDim + 8];
  const int l = threadIdx.x & 31;
  const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t index = fastdiv(item, per_token);
  const int64_t token = index;
  const int h0 = static_cast<int>(item - index * per_token.divisor) * kAxesHeads;
  const int count = token < a.n ? min(kAxesHeads, a.q.heads + a.k.heads - h0) : 0;
  const int64_t active = live_tokens(a);
  const bool live = token < active;
  const int half = a.rotary >> 1;
  const int pair0 = kMode == kPairAdjacent ? 4 * l : 8 * l < half ? 8 * l : 8 * l - half;
  // The position on axis l, the pairs' axes, and the rows: in flight together.
  int64_t position = 0;
  if (live && l < a.axes.count) position = a.axes.positions[l * a.axes.position_stride + token];
  PairAxes<kN> pairs;
  if (8 * l < a.rotary) pairs = pair_axes<kN>(a.axes, pair0);
  RowLoads r[kAxesHeads];
  Angles<kMode, kFp32> angles;
  auto row_at = [&](int i, int64_t (&at)[2]) {  // source and output of row i of the list
    const int head = h0 + i;
    const bool is_k = head >= a.q.heads;
    const NormArgs& t = is_k ? a.k : a.q;
    const int h = is_k ? head - a.q.heads : head;
    at[0] = reinterpret_cast<int64_t>(t.x + token * t.s0 + h * t.s1);
    at[1] = reinterpret_cast<int64_t>(t.out + (token * t.heads + h) * kHeadDim + 8 * l);
    return is_k;
  };
#pragma unroll
  for (int i = 0; i < kAxesHeads; ++i) start_row(angles, r[i]);
#pragma unroll
  for (int i = 0; i < kAxesHeads; ++i)
    if (i < count) {
      int64_t at[2];
      row_at(i, at);
      load_row<kMode>(a, reinterpret_cast<const uint16_t*>(at[0]), l, r[i]);
    }
  stage_weights(a, a.q.weight, s_weight[0], 0);
  stage_weights(a, a.k.weight, s_weight[1], 32);
  angles.live = live;
  const bool outside = live && l < a.axes.count && (position < 0 || position >= a.axes.rows);
  angles.bad = a.rotary > 0 && (__ballot(outside) >> (threadIdx.x & 32) & 0xffffffffull) != 0;
  auto position_on = [&](int axis) {
    const int lo = __shfl(static_cast<int>(position), axis, 32);
    const int hi = __shfl(static_cast<int>(position >> 32), axis, 32);
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 |
                                static_cast<uint32_t>(lo));
  };
  // Every lane of the wavefront takes part (its exchanges read other lanes'); lanes past the rotary dims
  // keep their identity turn.
  if (8 * l >= a.rotary) {
#pragma unroll
    for (int e = 0; e < kN; ++e) pairs.axis[e] = 0;
    pairs.one = true;
  }
  uint32_t c[kWords], s[kWords];
  axis_words<kN, kFp32>(a.axes, position_on, 8 * l < a.rotary ? pair0 : 0, pairs, c, s);
  if (8 * l < a.rotary)
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      angles.c[w >> 2][w & 3] = c[w];
      angles.s[w >> 2][w & 3] = s[w];
    }
  __syncthreads();  // the weights
#pragma unroll
  for (int i = 0; i < kAxesHeads; ++i)
    if (i < count) {
      int64_t at[2];
      const bool is_k = row_at(i, at);
      *reinterpret_cast<u32x4*>(at[1]) = finish_row(a, s_weight[is_k], angles, r[i], l);
    }
}

// ---- with the rotation, few rows or pairs that lie further apart: workgroups of kWaves wavefronts
// walk blocks of 2 kWaves query rows, one per half wavefront. A wavefront keeps 16 columns of R_k in
// registers for the whole walk (32 a lane): 16 wavefronts hold all of R_k, 8 half of it (the rows of a
// decode step, few blocks: two workgroups share a block and each reads half as much of R_k). The
// block's rows go through LDS (16-byte piece p of row r at p ^ r % 16) as the B operand; the columns
// are the A operand, so that a lane ends with four consecutive columns of a row. While a block is
// multiplied, the next one's rows are normed and the loads of the one after are in flight, with its
// positions read a block earlier. The keys' blocks follow the queries' in the walk.
template <int kMode, bool kFp32, int kWaves>
__global__ __launch_bounds__(kWaves * kWave, 4) void norm_rope_rotate_kernel(const NormRopeArgs a) {
  constexpr int kRows = 2 * kWaves, kSets = kWaves / 8;
  __shared__ __attribute__((aligned(16))) uint8_t s_rows[2][kRows * kHeadDim * 2];
  __shared__ float s_weight[2][kHeadDim + 8];
  const int tid = threadIdx.x, l = tid & 31, mine = tid >> 5;
  const int64_t active = live_tokens(a);
  const int64_t q_blocks = (a.q.rows + kRows - 1) / kRows;
  const int64_t blocks = q_blocks + (a.k.rows + kRows - 1) / kRows;
  const int64_t first = blockIdx.x, step = gridDim.x;
  RowLoads r;
  Angles<kMode, kFp32> angles;
  start_row(angles, r);
  int64_t position;
  auto rows_of = [&](int64_t b) -> const NormArgs& { return b < q_blocks ? a.q : a.k; };
  auto my_row = [&](int64_t b) { return (b < q_blocks ? b : b - q_blocks) * kRows + mine; };
  // This half wavefront's row of block b; rows past the last are no live token's (and read row 0).
  auto load_position = [&](int64_t b) {
    const NormArgs& t = rows_of(b);
    const int64_t row = my_row(b);
    const int64_t token = row < t.rows ? fastdiv(static_cast<uint32_t>(row), t.h_div) : a.n;
    position = token < active ? a.positions[token] : 0;
  };
  auto load_block = [&](int64_t b) {
    const NormArgs& t = rows_of(b);
    const int64_t row = my_row(b);
    const uint32_t safe = row < t.rows ? static_cast<uint32_t>(row) : 0u;
    const uint32_t token = fastdiv(safe, t.h_div);
    load_row<kMode>(a, t.x + static_cast<int64_t>(token) * t.s0 +
                           static_cast<int64_t>(safe - token * static_cast<uint32_t>(t.heads)) * t.s1,
                    l, r);
    load_angles(a, row < t.rows ? static_cast<int64_t>(token) : a.n, position, active, l, angles);
  };
  auto finish_block = [&](int64_t b, int buf) {
    const NormArgs& t = rows_of(b);
    const int64_t row = my_row(b);
    const u32x4 bits = finish_row(a, s_weight[b < q_blocks ? 0 : 1], angles, r, l);
    *reinterpret_cast<u32x4*>(&s_rows[buf][mine * 512 + 16 * (l ^ (mine & 15))]) = bits;
    if (blockIdx.y == 0 && row < t.rows)
      *reinterpret_cast<u32x4*>(t.out + row * kHeadDim + 8 * l) = bits;
  };
  load_position(first);
  stage_weights(a, a.q.weight, s_weight[0], 0);
  stage_weights(a, a.k.weight, s_weight[1], 32);
  load_block(first);
  const int lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int base = 16 * (kWaves * blockIdx.y + wave);
  u32x4 rk[8];
  if (first < q_blocks) {
    const uint16_t* col = a.rk_t + static_cast<int64_t>(base + n) * kHeadDim + 8 * g;
#pragma unroll
    for (int m = 0; m < 8; ++m) rk[m] = *reinterpret_cast<const u32x4*>(col + 32 * m);
  }
  __syncthreads();  // the weights
  finish_block(first, 0);
  if (first + step < blocks) {
    load_position(first + step);
    load_block(first + step);
    load_position(first + 2 * step);
  }
  __syncthreads();
  int buf = 0;
  for (int64_t b = first; b < blocks; b += step, buf ^= 1) {
    if (b + step < blocks) {
      finish_block(b + step, buf ^ 1);
      if (b + 2 * step < blocks) {
        load_block(b + 2 * step);
        load_position(b + 3 * step);
      }
    }
    if (b < q_blocks) {
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 8; ++m)
          acc = mfma16x16x32(rk[m], *reinterpret_cast<const u32x4*>(
                                        &s_rows[buf][(16 * i + n) * 512 + 16 * ((4 * m + g) ^ n)]),
                             acc);
        const int64_t row = b * kRows + 16 * i + n;
        if (row < a.q.rows)
          *reinterpret_cast<uint2*>(a.q_rot + row * kHeadDim + base + 4 * g) =
              make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
      }
    }
    __syncthreads();  // this block's rows are read, the next one's are written
  }
}

// ---- with the rotation, many rows: workgroups of 8 wavefronts, one per CU, with all of R_k in LDS;
// each wavefront walks 16-row blocks of its own and needs no other. A lane loads the eight 16-byte
// pieces 32 m + 8 g of row lane % 16 (g = lane / 16), which is what the products read as B operand, so
// a row goes from memory to the matrix instruction in registers; pairs of halves 32 dims or a multiple
// of it apart, and adjacent ones, lie in one lane. Sums are added in the order of finish_row: the same
// bits in either kernel. 2048 tokens of 14 heads, us after the first workgroup's start: rows and R_k
// there 6.2, normed 7, first block's stores and products done 10 to 12.6 (R_k is read from LDS once per
// 16 rows, 1024 cycles a block at 128 bytes a cycle).
constexpr int kWalkWaves = 8;

template <int kMode, bool kFp32>
__global__ __launch_bounds__(kWalkWaves * kWave, 2) void norm_rope_walk_kernel(
    const NormRopeArgs a) {
  static_assert(kMode != kPairGeneric, "pairs lie in one lane");
  __shared__ __attribute__((aligned(16))) uint8_t s_rk[kHeadDim * kHeadDim * 2];
  __shared__ __attribute__((aligned(16))) float s_weight[2][kHeadDim];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int64_t active = live_tokens(a);
  const int64_t q_blocks = (a.q.rows + 15) / 16, blocks = q_blocks + (a.k.rows + 15) / 16;
  const int64_t first = static_cast<int64_t>(wave) * gridDim.x + blockIdx.x;
  const int64_t step = static_cast<int64_t>(kWalkWaves) * gridDim.x;
  const int half = a.rotary >> 1;
  u32x4 x[8];
  int64_t position = 0;
  bool live = false, bad = false;
  const char* turn = nullptr;  // the angles' table row, from the lane's first dim on
  constexpr int kBytes = kFp32 ? 4 : 2, kLoads = kFp32 ? 2 : 1;
  // Packed angles of eight consecutive dims of a half, or of the four pairs of eight adjacent dims.
  constexpr int kWords = kMode == kPairHalves ? 4 * kLoads : 2 * kLoads;
  auto load_words = [&](const char* at, uint32_t (&w)[kWords]) {
    if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(at);
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 v = reinterpret_cast<const u32x4*>(at)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
      }
    }
  };
  auto word_value = [](const uint32_t (&w)[kWords], int i) {
    if (kFp32) return __uint_as_float(w[i]);
    return bf16_to_float(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
  };
  uint32_t cos0[kWords], sin0[kWords];  // of the first group of dims, with the row's loads

  auto rows_of = [&](int64_t b) -> const NormArgs& { return b < q_blocks ? a.q : a.k; };
  auto my_row = [&](int64_t b) { return (b < q_blocks ? b : b - q_blocks) * 16 + n; };
  auto load_position = [&](int64_t b) {
    const NormArgs& t = rows_of(b);
    const int64_t row = my_row(b);
    const int64_t token = row < t.rows ? fastdiv(static_cast<uint32_t>(row), t.h_div) : a.n;
    position = token < active ? a.positions[token] : 0;
  };
  auto load_rows = [&](int64_t b) {
    const NormArgs& t = rows_of(b);
    const int64_t row = my_row(b);
    const uint32_t safe = row < t.rows ? static_cast<uint32_t>(row) : 0u;
    const uint32_t token = fastdiv(safe, t.h_div);
    const uint16_t* src = t.x + static_cast<int64_t>(token) * t.s0 +
                          static_cast<int64_t>(safe - token * static_cast<uint32_t>(t.heads)) * t.s1 +
                          8 * g;
#pragma unroll
    for (int m = 0; m < 8; ++m) x[m] = *reinterpret_cast<const u32x4*>(src + 32 * m);
    live = row < t.rows && token < active;
  };
  auto load_angles = [&]() {
    bad = a.rotary > 0 && (position < 0 || position >= a.table_rows);
    turn = static_cast<const char*>(a.table) +
           ((bad ? 0 : position) * a.table_stride + (kMode == kPairHalves ? 8 * g : 4 * g)) * kBytes;
    if (8 * g < a.rotary) {
      load_words(turn, cos0);
      load_words(turn + half * kBytes, sin0);
    }
  };
  u32x4 y[8];  // the finished rows
  auto finish = [&](int64_t b) {
    const float* w = s_weight[b < q_blocks ? 0 : 1] + 8 * g;
    float v[8][8];
    auto mean_square = [&](float eps) {
      float sums[8];
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        float sum = 0.f;
        unpack_eight(x[m], v[m]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[m][e], v[m][e], sum);
        sums[m] = sum_xor32(sum_xor16(sum));
      }
      const float sum = ((sums[0] + sums[1]) + (sums[2] + sums[3])) +
                        ((sums[4] + sums[5]) + (sums[6] + sums[7]));
      return fmaf(sum, 1.0f / kHeadDim, eps);
    };
    float mean = mean_square(a.eps);
    if (const float by = range_scale(mean); __any(by != 1.f)) {
#pragma unroll
      for (int m = 0; m < 8; ++m) x[m] = scale_eight(x[m], by);
      mean = mean_square(a.eps * by * by);
    }
    const float inv = inverse_root(mean, bad);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(w + 32 * m);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(w + 32 * m + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[m][e] = v[m][e] * inv * (e < 4 ? lo[e & 3] : hi[e & 3]);
    }
    if constexpr (kMode == kPairHalves) {
      const int apart = half >> 5;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= apart) break;
        uint32_t c[kWords], s[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          c[i] = cos0[i];
          s[i] = sin0[i];
        }
        if (j) {
          load_words(turn + 32 * j * kBytes, c);
          load_words(turn + (32 * j + half) * kBytes, s);
        }
        auto rotate_pair = [&](float (&lo)[8], float (&hi)[8]) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float co = word_value(c, e), si = word_value(s, e);
            const float l = lo[e], h = hi[e];
            lo[e] = fmaf(l, co, -h * si);
            hi[e] = fmaf(h, co, l * si);
          }
        };
        // The other half is 1 to 4 pieces on: constant indexes, so that the rows stay in registers.
        if (apart == 1)
          rotate_pair(v[j], v[j + 1]);
        else if (apart == 2)
          rotate_pair(v[j], v[j + 2]);
        else if (apart == 3)
          rotate_pair(v[j], v[j + 3]);
        else
          rotate_pair(v[j], v[j + 4]);
      }
    } else {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        if (32 * m + 8 * g < a.rotary) {
          uint32_t c[kWords], s[kWords];
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            c[i] = cos0[i];
            s[i] = sin0[i];
          }
          if (m) {
            load_words(turn + 16 * m * kBytes, c);
            load_words(turn + (16 * m + half) * kBytes, s);
          }
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float co = word_value(c, e >> 1), si = word_value(s, e >> 1);
            const float l = v[m][e], h = v[m][e + 1];
            v[m][e] = fmaf(l, co, -h * si);
            v[m][e + 1] = fmaf(h, co, l * si);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[m][e] = live ? pack_bf16x2(v[m][2 * e], v[m][2 * e + 1]) : 0u;
  };

  auto store = [&](int64_t b) {
    const NormArgs& t = rows_of(b);
    const int64_t row = my_row(b);
    uint16_t* out = t.out + row * kHeadDim + 8 * g;
    if (row < t.rows)
#pragma unroll
      for (int m = 0; m < 8; ++m) *reinterpret_cast<u32x4*>(out + 32 * m) = y[m];
  };

  // Everything that the first block waits for is in flight together: its rows, the weights, the
  // angles behind their position, and R_k.
  if (first < blocks) {
    load_position(first);
    load_rows(first);
  }
  float weight[8];
  const bool stages = tid < 64;
  if (stages) load_eight(tid < 32 ? a.q.weight : a.k.weight, 8 * (tid & 31), a.weight_fp32, weight);
  if (first < blocks) {
    load_angles();
    load_position(first + step);
  }
  // Row 16 t + i of the LDS copy is the column of R_k that lane i's A operand of tile t reads, 32 (t / 2)
  // + 8 (i / 4) + 4 (t % 2) + i % 4, so that a lane ends with eight consecutive columns of a row in two
  // tiles; its 16-byte piece p lies at p ^ i, so that 16 lanes read 256 bytes of all banks (p ^ i % 8: 4
  // cycles of conflicts a read, 0.2 us).
  if (blockIdx.x < q_blocks) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int r = 2 * (16 * wave + j) + (lane >> 5), t = r >> 4, i = r & 15;
      const int col = 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(a.rk_t + col * kHeadDim +
                                                          8 * ((lane & 31) ^ i)),
          (__attribute__((address_space(3))) void*)(s_rk + 1024 * (16 * wave + j)), 16, 0, 0);
    }
  }
  if (stages)
#pragma unroll
    for (int e = 0; e < 8; ++e) s_weight[tid >> 5][8 * (tid & 31) + e] = weight[e] + a.offset;
  barrier_lds();  // the weights
  if (first < blocks) finish(first);
  OSCAR_WAIT_VM0_SEEN();
  __syncthreads();  // R_k
  for (int64_t b = first; b < blocks;) {
    const int64_t next = b + step;
    if (next < blocks) {
      load_rows(next);
      load_angles();
      load_position(next + step);
    }
    store(b);
    if (b < q_blocks) {
      const int64_t row = 16 * b + n;
      uint16_t* out = a.q_rot + row * kHeadDim + 8 * g;
      // Eight operands (four products of two tiles) are read ahead of the eight in use.
      const uint8_t* from[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) from[m] = s_rk + 512 * n + 16 * ((4 * m + g) ^ n);
      u32x4 f[2][8];
      auto read = [&](int i, u32x4 (&w)[8]) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[k] = *reinterpret_cast<const u32x4*>(
              from[k >> 1] + 8192 * (2 * (i >> 1) + (k & 1)) + 256 * (i & 1));
      };
      read(0, f[0]);
      f32x4 acc[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (i < 15) read(i + 1, f[(i + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (!(i & 1)) acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; ++k)
          acc[k & 1] = mfma16x16x32(f[i & 1][k], y[4 * (i & 1) + (k >> 1)], acc[k & 1]);
        if ((i & 1) && row < a.q.rows)
          *reinterpret_cast<u32x4*>(out + 32 * (i >> 1)) =
              u32x4{pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3]),
                    pack_bf16x2(acc[1][0], acc[1][1]), pack_bf16x2(acc[1][2], acc[1][3])};
      }
    }
    b = next;
    if (b < blocks) finish(b);
  }
}

// With R_k: 16-row blocks up to which two workgroups of 8 wavefronts share each, all on CUs of their
// own (300 tokens of 7 heads: 5.9 us, 6.3 by norm_rope_walk_kernel; 340, more workgroups than CUs: 7.6
// and 6.4). Above, one workgroup per CU walks: wavefronts by themselves where a pair's dims lie in one
// lane (2048 tokens of 14 heads 14.1 us, 18.2 by blocks through LDS; 16384 of 7 heads 35.2 and 50.4),
// else blocks of 32 rows.
constexpr int64_t kFewBlocks = 128, kRotateGroups = 256;

template <int kMode, bool kFp32>
void launch_norm_rope(NormRopeArgs& a, hipStream_t s) {
  if (!a.rk_t) {
    const int64_t per_q = (a.q.heads + kRopeHeads - 1) / kRopeHeads;
    const int64_t per_k = (a.k.heads + kRopeHeads - 1) / kRopeHeads;
    const int64_t q_blocks = (a.n * per_q + 7) / 8, k_blocks = (a.n * per_k + 7) / 8;
    hipLaunchKernelGGL((norm_rope_kernel<kMode, kFp32>),
                       dim3(static_cast<unsigned>(q_blocks + k_blocks)), dim3(kThreads), 0, s, a,
                       q_blocks, make_fastdiv(static_cast<uint32_t>(per_q)),
                       make_fastdiv(static_cast<uint32_t>(per_k)));
    return;
  }
  const int64_t all = (a.q.rows + 15) / 16 + (a.k.rows + 15) / 16;
  const bool few = all <= kFewBlocks;
  const int64_t rows = few ? 16 : 32;
  const int64_t blocks = (a.q.rows + rows - 1) / rows + (a.k.rows + rows - 1) / rows;
  if constexpr (kMode != kPairGeneric) {
    if (!few && (kMode == kPairAdjacent || a.rotary % 64 == 0)) {
      hipLaunchKernelGGL((norm_rope_walk_kernel<kMode, kFp32>),
                         dim3(static_cast<unsigned>(all < kRotateGroups ? all : kRotateGroups)),
                         dim3(kWalkWaves * kWave), 0, s, a);
      return;
    }
  }
  const unsigned x = static_cast<unsigned>(few || blocks < kRotateGroups ? blocks : kRotateGroups);
  if (few)
    hipLaunchKernelGGL((norm_rope_rotate_kernel<kMode, kFp32, 8>), dim3(x, 2), dim3(8 * kWave), 0, s,
                       a);
  else if constexpr (kMode != kPairAdjacent)  // of adjacent pairs the few rows alone get here
    hipLaunchKernelGGL((norm_rope_rotate_kernel<kMode, kFp32, 16>), dim3(x, 1), dim3(16 * kWave), 0,
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
  // Rows are 32-bit, and a launch holds fewer than 2^32 threads (32 for a token's four heads).
  if (hq > 0x7fffffffll / n || hk > 0x7fffffffll / n ||
      (hq + 3) / 4 + (hk + 3) / 4 > 0xffffff00ll / 32 / n)
    return OSCAR_E_SHAPE;
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
  a.adjacent = interleaved ? 1 : 0;
  a.offset = unit_offset ? 1.f : 0.f;
  a.eps = eps;
  a.rk_t = static_cast<const uint16_t*>(rk_t);
  a.q_rot = static_cast<uint16_t*>(q_rot);
  hipStream_t s = as_stream(stream);
  const bool rows16 = aligned16(cos_sin) && table_stride % 8 == 0;
  auto launch = [&](auto mode) {
    constexpr int kMode = decltype(mode)::value;
    if (table_fp32)
      launch_norm_rope<kMode, true>(a, s);
    else
      launch_norm_rope<kMode, false>(a, s);
  };
  if (interleaved && rotary_dim % 8 == 0 && rows16)
    launch(std::integral_constant<int, kPairAdjacent>());
  else if (!interleaved && rotary_dim % 16 == 0 && rows16)
    launch(std::integral_constant<int, kPairHalves>());
  else
    launch(std::integral_constant<int, kPairGeneric>());
  return static_cast<int>(hipGetLastError());
}

namespace oscar {

// The form for tokens with several positions, without R_k: oscar_rope_append has checked the arguments.
// False where its pairs do not lie eight dims a lane (then it takes another kernel).
bool launch_norm_rope_axes(const void* query, int64_t q_s0, int64_t q_s1, const void* key, int64_t k_s0,
                           int64_t k_s1, int64_t n, int64_t hq, int64_t hk, const void* q_weight,
                           const void* k_weight, bool weight_fp32, bool unit_offset, float eps,
                           bool table_fp32, bool interleaved, const int32_t* counts, void* q_out,
                           void* k_out, const AxisTable& axes, hipStream_t s) {
  if (axes.rotary % (interleaved ? 8 : 16) || !aligned16(axes.table) || axes.stride % 8 ||
      !aligned16(axes.axes))
    return false;
  NormRopeArgs a{};
  a.q = {static_cast<const uint16_t*>(query), q_s0, q_s1, q_weight, static_cast<uint16_t*>(q_out),
         n * hq, static_cast<int32_t>(hq), make_fastdiv(static_cast<uint32_t>(hq))};
  a.k = {static_cast<const uint16_t*>(key), k_s0, k_s1, k_weight, static_cast<uint16_t*>(k_out),
         n * hk, static_cast<int32_t>(hk), make_fastdiv(static_cast<uint32_t>(hk))};
  a.axes = axes;
  a.counts = counts;
  a.n = n;
  a.rotary = axes.rotary;
  a.weight_fp32 = weight_fp32 ? 1 : 0;
  a.adjacent = interleaved ? 1 : 0;
  a.offset = unit_offset ? 1.f : 0.f;
  a.eps = eps;
  const int64_t per = (hq + hk + kAxesHeads - 1) / kAxesHeads;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n * per + 7) / 8)), dim3(kThreads), 0, s, a,
                       make_fastdiv(static_cast<uint32_t>(per)));
  };
  if (interleaved)
    table_fp32 ? launch(norm_rope_axes_kernel<kPairAdjacent, true>)
               : launch(norm_rope_axes_kernel<kPairAdjacent, false>);
  else
    table_fp32 ? launch(norm_rope_axes_kernel<kPairHalves, true>)
               : launch(norm_rope_axes_kernel<kPairHalves, false>);
  return true;
}

}  // namespace oscar
