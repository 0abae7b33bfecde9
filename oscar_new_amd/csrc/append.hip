// Rows of a packed projection on their way into the paged cache, in one launch: optional norms of the
// queries and keys, the position rotation (one or several position axes), the rotation of the queries
// and keys by R_k and of the values by R_v, and the records of the rotated keys and values.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (w, 1 + w with a unit offset, or no norm: y = x)
//   (a, b) -> (a cos - b sin, b cos + a sin)     pair j by the angle at the position of its axis
//   q, k = bf16(y);  q_rot = bf16(q R_k);  record of bf16(k R_k) and bf16(v R_v) (quant.h, quant4.h)
//
// No reference counterpart as one call: kernels.py:51-66 and 175-202 (oscar_ascend) behind a model's
// norms and rotary embedding. The rows have the bits of oscar_qk_norm_rope (norm_rope.hip), the rotated
// ones those of oscar_rotate and 2-bit records the bytes of oscar_store_int2.
//
// Three forms. Few rows: blocks of 16 (token, head) rows on as many CUs as there are blocks, bound by the
// chain counts - positions - angles - norm - product - quantile - record (11.6 us for 32 tokens of 6 + 1
// heads, 12.2 for 512; kernel times here and below). Many rows of 4-bit layouts: wavefronts that walk 16-row
// blocks (15.7 us for 2048 tokens, 50 to 52 for 16384, 181 MB). Rows that are turned only: no product, the
// rows' bytes.
#include "dma.h"
#include "norm_row.h"
#include "quant4.h"
#include "rotate.h"

namespace oscar {

bool launch_norm_rope_axes(const void* query, int64_t q_s0, int64_t q_s1, const void* key, int64_t k_s0,
                           int64_t k_s1, int64_t n, int64_t hq, int64_t hk, const void* q_weight,
                           const void* k_weight, bool weight_fp32, bool unit_offset, float eps,
                           bool table_fp32, bool interleaved, const int32_t* counts, void* q_out,
                           void* k_out, const AxisTable& axes, hipStream_t s);  // norm_rope.hip

namespace {

constexpr int kMostAxes = 32;  // a lane of the half wavefront checks an axis' position

struct RowSet {
  const uint16_t* x;
  int64_t s0, s1;      // token and head strides, elements
  const void* weight;  // null: no norm
  uint16_t* out;       // [tokens][heads][256], null for the values
  int64_t rows;
  int32_t heads;
  FastDiv h_div;
};

struct AppendArgs {
  RowSet set[3];      // queries, keys, values
  AxisTable angles;   // axes null: axis 0 of every pair
  const int32_t* counts;
  int64_t n;
  int32_t rotary, table_fp32, weight_fp32, adjacent;
  FastDiv rotary_div;
  float offset, eps;
  const uint16_t* rt[3];  // R^T of each set, contiguous [256][256]; null: no rotation
  uint16_t* q_rot;
  uint8_t* history;
  int64_t history_bytes;
  const int64_t* slots;
  Layout L;
  int32_t mode;
  float ratio[3], factor[3];
};

__device__ __forceinline__ int64_t live_tokens(const AppendArgs& a) {
  return a.counts ? min(static_cast<int64_t>(max(a.counts[1], 0)), a.n) : a.n;
}

// The angles of the tokens of rows r0 .. r0 + rows - 1, cosines then sines of a token, to s_turn
// [token][rotary] by the workgroup's kThreadsA threads. A pair whose axis is none of the positions'
// turns to NaN (as a token's rows do whose position is outside the table: finish_row).
template <int kThreadsA>
__device__ __forceinline__ void gather_angles(const AppendArgs& a, int64_t first_token, int tokens,
                                              int64_t active, float* s_turn) {
  const int half = a.rotary >> 1;
  for (int i = threadIdx.x; i < tokens * a.rotary; i += kThreadsA) {
    const int t = static_cast<int>(fastdiv(static_cast<uint32_t>(i), a.rotary_div));
    const int e = i - t * a.rotary;
    const AxisTable& table = a.angles;
    const int axis = table.axes ? table.axes[e < half ? e : e - half] : 0;
    const int64_t token = first_token + t;
    float v = __uint_as_float(0x7fc00000u);
    if (token < active && axis >= 0 && axis < table.count) {
      const int64_t p = table.positions[axis * table.position_stride + token];
      if (p >= 0 && p < table.rows) v = load_value(table.table, p * table.stride + e, a.table_fp32);
    }
    s_turn[i] = v;
  }
}

// The lane's 8 dims of a row (l = lane % 32) as bf16, with the arithmetic of norm_rope.hip's
// finish_row. `turn`: the token's angles; `s_y`: the row's part of an LDS area of `rotary` floats, from
// which pairs of halves read their partners. Zeros past the live tokens; NaN where bad.
__device__ __forceinline__ u32x4 finish_row(const AppendArgs& a, u32x4 x, const float (&w)[8],
                                            bool norm, const float* turn, float* s_y, bool live,
                                            bool bad, int l) {
  float v[8], y[8];
  float inv = bad ? __uint_as_float(0x7fc00000u) : 1.f;
  if (norm) {
    auto mean_square = [&](float eps) {
      float sum = 0.f;
      unpack_eight(x, v);
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
      x = scale_eight(x, by);
      mean = mean_square(a.eps * by * by);
    }
    inv = inverse_root(mean, bad);
  }
  unpack_eight(x, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = norm ? v[e] * inv * w[e] : v[e] * inv;
  const int half = a.rotary >> 1, d0 = 8 * l;
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = y[e];
  if (d0 < a.rotary) {
    if (a.adjacent) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if (d0 + e >= a.rotary) break;
        const float c = turn[(d0 + e) >> 1], s = turn[half + ((d0 + e) >> 1)];
        o[e] = fmaf(y[e], c, -y[e + 1] * s);
        o[e + 1] = fmaf(y[e + 1], c, y[e] * s);
      }
    } else if (half % 8 == 0) {
      // A lane's dims and their partners are two runs of eight.
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(s_y + d0 + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
      const bool low = d0 < half;
      const float* other = s_y + (low ? d0 + half : d0 - half);
      const float* c = turn + (low ? d0 : d0 - half);
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f32x4 ov = *reinterpret_cast<const f32x4*>(other + e);
        const f32x4 cv = *reinterpret_cast<const f32x4*>(c + e);
        const f32x4 sv = *reinterpret_cast<const f32x4*>(c + half + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[e + i] = fmaf(y[e + i], cv[i], (low ? -ov[i] : ov[i]) * sv[i]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < a.rotary) s_y[d0 + e] = y[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        if (d >= a.rotary) break;
        const int j = d < half ? d : d - half;
        const float p = d < half ? -s_y[d + half] : s_y[j];
        o[e] = fmaf(y[e], turn[j], p * turn[half + j]);
      }
    }
  }
  u32x4 bits;
#pragma unroll
  for (int e = 0; e < 4; ++e) bits[e] = live ? pack_bf16x2(o[2 * e], o[2 * e + 1]) : 0u;
  return bits;
}

// The norm weights of the lane's dims, with the offset.
__device__ __forceinline__ void load_weights(const AppendArgs& a, const RowSet& t, int l,
                                             float (&w)[8]) {
  if (!t.weight) return;
  load_eight(t.weight, 8 * l, a.weight_fp32, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] += a.offset;
}

// Whether some position of the token lies outside the table (the same for the half wavefront).
__device__ __forceinline__ bool bad_token(const AppendArgs& a, int64_t token, bool live, int l) {
  const bool out = a.rotary && live && l < a.angles.count && bad_position(a.angles, token, l);
  const uint64_t any = __ballot(out);
  return ((any >> (threadIdx.x & 32)) & 0xffffffffull) != 0;
}

// ---- rows that are turned only: each half wavefront takes kTurnPerHalf rows, 32 lanes of 8 dims each. The
// block's angles are gathered into LDS first, each pair from the table row of its axis' position, in flight
// with the rows: so several axes, any table type, any rotary size and any pair order cost the rows nothing.
constexpr int kTurnPerHalf = 4, kTurnRows = 8 * kTurnPerHalf;

__global__ __launch_bounds__(kThreads) void turn_rows_kernel(const AppendArgs a, int64_t q_blocks) {
  extern __shared__ __attribute__((aligned(16))) float s_angles[];  // [rows][rotary], then partners
  const int l = threadIdx.x & 31, mine = threadIdx.x >> 5;
  const bool is_q = blockIdx.x < q_blocks;
  const RowSet& t = a.set[is_q ? 0 : 1];
  const int64_t r0 = (blockIdx.x - (is_q ? 0 : q_blocks)) * kTurnRows;
  const int64_t active = live_tokens(a);
  float w[8];
  load_weights(a, t, l, w);
  u32x4 x[kTurnPerHalf];
  bool bad[kTurnPerHalf];
  uint32_t token[kTurnPerHalf];
#pragma unroll
  for (int i = 0; i < kTurnPerHalf; ++i) {
    const int64_t row = r0 + 8 * i + mine;
    const uint32_t safe = static_cast<uint32_t>(row < t.rows ? row : 0);
    token[i] = fastdiv(safe, t.h_div);
    x[i] = *reinterpret_cast<const u32x4*>(
        t.x + static_cast<int64_t>(token[i]) * t.s0 +
        static_cast<int64_t>(safe - token[i] * static_cast<uint32_t>(t.heads)) * t.s1 + 8 * l);
  }
  const uint32_t first = fastdiv(static_cast<uint32_t>(r0), t.h_div);
  const int64_t last_row = min(r0 + kTurnRows, t.rows) - 1;
  const int tokens = static_cast<int>(fastdiv(static_cast<uint32_t>(last_row), t.h_div) - first) + 1;
#pragma unroll
  for (int i = 0; i < kTurnPerHalf; ++i)
    bad[i] = bad_token(a, token[i], token[i] < active, l);
  gather_angles<kThreads>(a, first, tokens, active, s_angles);
  __syncthreads();
  float* s_y = s_angles + kTurnRows * a.rotary + mine * a.rotary;
#pragma unroll
  for (int i = 0; i < kTurnPerHalf; ++i) {
    const int64_t row = r0 + 8 * i + mine;
    if (row >= t.rows) break;
    const u32x4 bits = finish_row(a, x[i], w, t.weight != nullptr,
                                  s_angles + (token[i] - first) * a.rotary, s_y, token[i] < active,
                                  bad[i], l);
    *reinterpret_cast<u32x4*>(t.out + row * kHeadDim + 8 * l) = bits;
  }
}

// ---- rows that are rotated by R too: blocks of 16 kTiles rows by 16 wavefronts, each with 16 columns
// of R in registers. The finished rows go through LDS as the products' B operand (16-byte piece p of
// row r at p ^ r % 16), so that a lane ends with four consecutive columns of a row. Rotated queries
// leave from there; rotated keys and values go through LDS again (8-byte piece p of row r at p ^ r % 16)
// to the wavefronts that quantize a row each, whose chain of exchanges hides behind the other fifteen's.
constexpr int kAppendWaves = 16, kAppendThreads = kAppendWaves * kWave;

template <int kTiles>
__global__ __launch_bounds__(kAppendThreads) __attribute__((amdgpu_waves_per_eu(4)))
void append_kernel(const AppendArgs a, int64_t q_blocks, int64_t k_blocks) {
  constexpr int kRows = 16 * kTiles;
  extern __shared__ __attribute__((aligned(16))) float s_angles[];  // [rows][rotary], then partners
  __shared__ __attribute__((aligned(16))) uint8_t s_x[kRows * kHeadDim * 2];
  __shared__ __attribute__((aligned(16))) uint8_t s_rot[kRows * kHeadDim * 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l = tid & 31, mine = tid >> 5, n = lane & 15, g = lane >> 4;
  const int64_t b = blockIdx.x;
  const int which = b < q_blocks ? 0 : b < q_blocks + k_blocks ? 1 : 2;
  const RowSet& t = a.set[which];
  const int64_t r0 = (b - (which == 0 ? 0 : which == 1 ? q_blocks : q_blocks + k_blocks)) * kRows;
  const int64_t active = live_tokens(a);
  const uint16_t* rt = a.rt[which];

  // ---- everything that the block waits for, in flight together.
  const int64_t row = r0 + mine;
  const bool has_row = mine < kRows && row < t.rows;
  const uint32_t safe = static_cast<uint32_t>(has_row ? row : 0);
  const uint32_t token = fastdiv(safe, t.h_div);
  u32x4 x = {0u, 0u, 0u, 0u};
  if (has_row)
    x = *reinterpret_cast<const u32x4*>(
        t.x + static_cast<int64_t>(token) * t.s0 +
        static_cast<int64_t>(safe - token * static_cast<uint32_t>(t.heads)) * t.s1 + 8 * l);
  float w[8];
  if (which < 2) load_weights(a, t, l, w);
  int64_t slot[kTiles];
  int head[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int64_t mine_row = r0 + 16 * i + wave;
    slot[i] = -1;
    head[i] = 0;
    if (which && rt && mine_row < t.rows) {  // slots are read where records are written only
      const uint32_t at = fastdiv(static_cast<uint32_t>(mine_row), t.h_div);
      head[i] = static_cast<int>(mine_row - static_cast<int64_t>(at) * t.heads);
      if (at < active) slot[i] = a.slots[at];
    }
  }
  const int base = 16 * wave;
  u32x4 r[8];
  if (rt) {
    const uint16_t* col = rt + static_cast<int64_t>(base + n) * kHeadDim + 8 * g;
#pragma unroll
    for (int m = 0; m < 8; ++m) r[m] = *reinterpret_cast<const u32x4*>(col + 32 * m);
  }
  if (which < 2) {
    bool bad = false;
    uint32_t first = 0;
    if (a.rotary) {
      first = fastdiv(static_cast<uint32_t>(r0), t.h_div);
      const int64_t last_row = min(r0 + kRows, t.rows) - 1;
      const int tokens =
          static_cast<int>(fastdiv(static_cast<uint32_t>(last_row), t.h_div) - first) + 1;
      bad = bad_token(a, token, has_row && token < active, l);
      gather_angles<kAppendThreads>(a, first, tokens, active, s_angles);
      __syncthreads();
    }
    if (mine < kRows) {
      const int place = has_row ? static_cast<int>(token - first) : 0;
      x = finish_row(a, x, w, t.weight != nullptr, s_angles + place * a.rotary,
                     s_angles + kRows * a.rotary + mine * a.rotary,
                     has_row && token < active, bad, l);
      if (has_row) *reinterpret_cast<u32x4*>(t.out + row * kHeadDim + 8 * l) = x;
    }
  }
  if (!rt) return;
  if (mine < kRows) *reinterpret_cast<u32x4*>(s_x + mine * 512 + 16 * (l ^ (mine & 15))) = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 8; ++m)
      acc = mfma16x16x32(
          r[m], *reinterpret_cast<const u32x4*>(s_x + (16 * i + n) * 512 + 16 * ((4 * m + g) ^ n)),
          acc);
    const uint2 out = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
    if (which)
      *reinterpret_cast<uint2*>(s_rot + (16 * i + n) * 512 + 8 * ((4 * wave + g) ^ n)) = out;
    else if (r0 + 16 * i + n < t.rows)
      *reinterpret_cast<uint2*>(a.q_rot + (r0 + 16 * i + n) * kHeadDim + base + 4 * g) = out;
  }
  if (!which) return;
  __syncthreads();
  const int is_v = which - 1;
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    // A buffer holds fewer slots than bytes: no larger one's offset is formed (it could wrap).
    if (slot[i] < 0 || slot[i] >= a.history_bytes) continue;
    const int64_t at = slot_offset(a.L, slot[i], head[i]);
    if (at + a.L.slot_bytes > a.history_bytes) continue;
    const uint2 raw = *reinterpret_cast<const uint2*>(s_rot + (16 * i + wave) * 512 +
                                                      8 * (lane ^ wave));
    const float v[4] = {bf16_to_float(raw.x & 0xffffu), bf16_to_float(raw.x >> 16),
                        bf16_to_float(raw.y & 0xffffu), bf16_to_float(raw.y >> 16)};
    uint8_t* record = a.history + at;
    if (a.L.bits == 4)
      quantize_store4(v, a.mode, a.ratio[which], a.factor[which], record + is_v * kCodes4,
                      record + kSide4 + 4 * is_v);
    else
      quantize_store(v, a.mode, a.ratio[which], a.factor[which], record + is_v * a.L.vector_bytes);
  }
}

// Rows up to which blocks of 16 find a CU each. 512 tokens of 8 rows: 12.2 us, against 15.9 in blocks of 32
// and 13.0 by walking wavefronts; 768: 18.5, 16.3 and 13.4; 2048: 33, 25.9 and 15.7. Blocks of 32 remain for
// what the walk does not serve (`walks`), and load R anew each: 16384 tokens with 96 rotary dims in halves
// 149 us, with 2-bit records 145.
constexpr int64_t kSmallAppendRows = 16 * 256;
constexpr unsigned kWalkGroups = 256;  // one per CU

// ---- the same for many rows of 4-bit layouts: workgroups of 8 wavefronts, one per CU, with one of the
// rotations in LDS (queries and keys by R_k, values by R_v, the CUs divided by their work); each wavefront
// walks 16-row blocks of its own and needs no other. A lane loads the eight 16-byte pieces 32 m + 8 g of
// row lane % 16 (g = lane / 16), which is what the products read as B operand, and ends with the same
// pieces of the rotated row, so that a row goes from memory to its record in registers: 16 rows are
// quantized at a time, four lanes each. Pairs of halves 32 dims or a multiple of it apart, and adjacent
// ones, lie in one lane. 2048 tokens of 8 rows, one block a wavefront, are bound by what a block takes: 5 to
// 7 us until R and the angles are there, 4 for the norm and the turn, 3 for the products (whose operands,
// 128 KB a block, LDS hands over in 2), 4 for the records. 16384 move their bytes at 60 to 70 % of a copy's
// rate: a wavefront's next rows are on the way while it works on a block, and no more fit its registers.
constexpr int kWalkWaves = 8, kWalkThreads = kWalkWaves * kWave;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 as_u16x2(uint32_t v) { return __builtin_bit_cast(u16x2, v); }
__device__ __forceinline__ i16x2 as_i16x2(uint32_t v) { return __builtin_bit_cast(i16x2, v); }
__device__ __forceinline__ uint32_t as_u32(u16x2 v) { return __builtin_bit_cast(uint32_t, v); }

// Sum and maximum over the four lanes of a row.
__device__ __forceinline__ uint32_t row_sum(uint32_t v) {
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] + r[1];
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return r[0] + r[1];
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}

// The kLargest largest magnitudes of a row whose lanes hold z, in descending order. A lane sorts its words
// eight at a time, either half word apart (19 compares of a network), and joins the lists: the largest of
// two descending lists are the larger ones of a[i] and b[7 - i], which three steps of compares put in order;
// then lanes' lists and the half words' are joined the same way: 390 instructions.
constexpr uint32_t kLargest = 8;
template <class T>
__device__ __forceinline__ void in_order(T& a, T& b) {
  const T larger = __builtin_elementwise_max(a, b);
  b = __builtin_elementwise_min(a, b);
  a = larger;
}
template <class T>
__device__ __forceinline__ void join_lists(T (&a)[kLargest], const T (&b)[kLargest]) {
#pragma unroll
  for (uint32_t i = 0; i < kLargest; ++i) a[i] = __builtin_elementwise_max(a[i], b[kLargest - 1 - i]);
#pragma unroll
  for (uint32_t d = kLargest / 2; d; d >>= 1)
#pragma unroll
    for (uint32_t i = 0; i < kLargest; ++i)
      if (!(i & d)) in_order(a[i], a[i + d]);
}
__device__ __forceinline__ void largest_of_row(const u32x4 (&z)[8], uint32_t (&most)[kLargest]) {
  u16x2 s[kLargest];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    u16x2 t[kLargest];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = as_u16x2(z[2 * k + (i >> 2)][i & 3] & 0x7fff7fffu);
    constexpr int kFirst[19] = {0, 1, 4, 5, 0, 1, 2, 3, 0, 2, 4, 6, 2, 3, 1, 3, 1, 3, 5};
    constexpr int kSecond[19] = {2, 3, 6, 7, 4, 5, 6, 7, 1, 3, 5, 7, 4, 5, 4, 6, 2, 4, 6};
#pragma unroll
    for (int i = 0; i < 19; ++i) in_order(t[kFirst[i]], t[kSecond[i]]);
    if (k) {
      join_lists(s, t);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kLargest; ++i) s[i] = t[i];
    }
  }
  u16x2 other[kLargest];
#pragma unroll
  for (uint32_t i = 0; i < kLargest; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(as_u32(s[i]), as_u32(s[i]), false, false);
    s[i] = as_u16x2(r[0]);
    other[i] = as_u16x2(r[1]);
  }
  join_lists(s, other);
#pragma unroll
  for (uint32_t i = 0; i < kLargest; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(as_u32(s[i]), as_u32(s[i]), false, false);
    s[i] = as_u16x2(r[0]);
    other[i] = as_u16x2(r[1]);
  }
  join_lists(s, other);
  uint32_t high[kLargest];
#pragma unroll
  for (uint32_t i = 0; i < kLargest; ++i) {
    most[i] = s[i][0];
    high[i] = s[i][1];
  }
  join_lists(most, high);
}

// The need-th largest magnitude of a row and the one before it (need >= 2): first in bins of four below the
// row's largest, `top`, a byte each (127: a bin of all that lie 508, four powers of two, below), whose
// number is bisected four values at a time, then inside the bin that holds it.
__device__ __forceinline__ void statistics_of_row(const u32x4 (&z)[8], uint32_t top, uint32_t need,
                                                  uint32_t& below, uint32_t& above) {
  u16x2 mag[32];
  uint32_t bins[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    u16x2 b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mag[2 * k + i] = as_u16x2(z[k >> 1][2 * (k & 1) + i] & 0x7fff7fffu);
      b[i] = __builtin_elementwise_min((as_u16x2(top * 0x10001u) - mag[2 * k + i]) >> u16x2{2, 2},
                                       u16x2{127, 127});
    }
    bins[k] = as_u32(b[0]) | as_u32(b[1]) << 8;
  }
  // Up to bin `low` there are `larger` < need values, up to bin `high` at least need.
  int low = -1, high = 127;
  uint32_t larger = 0;
#pragma unroll 1
  for (int i = 0; i < 7; ++i) {
    const int mid = (low + high) >> 1;
    const uint32_t add = static_cast<uint32_t>(127 - mid) * 0x01010101u;
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) c += __builtin_popcount((bins[k] + add) & 0x80808080u);
    const uint32_t upto = kHeadDim - row_sum(c);
    const bool enough = upto >= need;
    high = enough ? mid : high;
    low = enough ? low : mid;
    larger = enough ? larger : upto;
  }
  // At or above `lo` there are at least need, at or above `hi` `larger` < need.
  uint32_t hi = top - 4 * high + 1;
  uint32_t lo = high == 127 || hi < 4 ? 0 : hi - 4;
  while (__any(hi - lo > 1)) {
    const uint32_t mid = (lo + hi) >> 1;  // lo where they are next to each other: it stays
    const u16x2 add = as_u16x2((0x8000u - mid) * 0x10001u);
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) c += __builtin_popcount(as_u32(mag[k] + add) & 0x80008000u);
    c = row_sum(c);
    const bool enough = c >= need || mid == lo;
    lo = enough ? mid : lo;
    hi = enough ? hi : mid;
    larger = enough ? larger : c;
  }
  u16x2 next = as_u16x2(0xffffffffu);
  const u16x2 sub = as_u16x2((lo + 1) * 0x10001u);
#pragma unroll
  for (int k = 0; k < 32; ++k) next = __builtin_elementwise_min(next, mag[k] - sub);
  const uint32_t least = 0xffffu - row_max(0xffffu - min(uint32_t{next[0]}, uint32_t{next[1]}));
  below = lo;
  above = larger == need - 1 ? least + lo + 1 : lo;
}

// quantize_store4 (percentile or factor) of 16 rows, four lanes each: z[m] holds dims 32 m + 8 g .. + 7 as
// bf16. The quantile's two order statistics are among the kLargest largest magnitudes where it is near 1
// (0.9726 on).
// `record_of`: the row's record or null, asked for when the statistics are known (its slot is on the way
// until then).
template <class Record>
__device__ __forceinline__ void quantize_rows4(const u32x4 (&z)[8], int mode, float ratio, float factor,
                                               bool is_v, int g, Record record_of) {
#pragma clang fp contract(off)
  // Two bf16 values a word: as signed numbers the largest is the row's maximum unless all are negative, as
  // unsigned ones the largest is its minimum unless none is.
  i16x2 largest2 = {INT16_MIN, INT16_MIN};
  u16x2 most2 = as_u16x2(0u), least2 = as_u16x2(0xffffffffu);
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      largest2 = __builtin_elementwise_max(largest2, as_i16x2(z[m][e]));
      most2 = __builtin_elementwise_max(most2, as_u16x2(z[m][e]));
      least2 = __builtin_elementwise_min(least2, as_u16x2(z[m][e]));
    }
  const int largest = static_cast<int>(row_max(static_cast<uint32_t>(
                          max(int{largest2[0]}, int{largest2[1]}) + 0x8000))) - 0x8000;
  const uint32_t most = row_max(max(uint32_t{most2[0]}, uint32_t{most2[1]}));
  const uint32_t least = 0xffffu - row_max(0xffffu - min(uint32_t{least2[0]}, uint32_t{least2[1]}));
  const uint32_t top = max(static_cast<uint32_t>(max(largest, 0)), most & 0x8000u ? most & 0x7fffu : 0u);
  float mx = __uint_as_float((largest >= 0 ? static_cast<uint32_t>(largest) : least) << 16);
  float mn = __uint_as_float((most & 0x8000u ? most : least) << 16);
  float thr = INFINITY;
  if (mode == OSCAR_CLIP_FACTOR) {
    thr = __uint_as_float(top << 16) * factor;
  } else if (ratio != 0.0f) {
    const float rank = ratio * 255.0f;
    const int lo_idx = static_cast<int>(floorf(rank)), hi_idx = static_cast<int>(ceilf(rank));
    const float weight = rank - static_cast<float>(lo_idx);
    const uint32_t need = static_cast<uint32_t>(kHeadDim - lo_idx);
    uint32_t below, above;
    if (need <= kLargest) {
      uint32_t first[kLargest];
      largest_of_row(z, first);
      const uint32_t more = static_cast<uint32_t>(kHeadDim - hi_idx);  // need or one less
      below = above = first[0];
#pragma unroll
      for (uint32_t i = 1; i < kLargest; ++i) {
        below = need == i + 1 ? first[i] : below;
        above = more == i + 1 ? first[i] : above;
      }
    } else {
      statistics_of_row(z, top, need, below, above);
      if (hi_idx == lo_idx) above = below;
    }
    const float under = __uint_as_float(below << 16);
    thr = __fmaf_rn(weight, __uint_as_float(above << 16) - under, under);
  }
  if (thr != INFINITY) {
    mn = clamp1(mn, thr);
    mx = clamp1(mx, thr);
  }
  float spread = (mx - mn) / 15.0f;
  spread = spread < 6.103515625e-05f ? 6.103515625e-05f : spread;
  if (top > 0x7f80u) spread = mn = __uint_as_float(0x7fc00000u);  // a NaN: so are the record's values
  const uint32_t zero = float_to_f16_bits(mn), scale = float_to_f16_bits(spread);
  const float zf = f16_bits_to_float(zero), sf = f16_bits_to_float(scale);
  const float r = scale_rcp(sf);
  uint8_t* const record = record_of();
  uint8_t* const codes = record + is_v * kCodes4;
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    float d[8], y[8];
    bool near = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = z[m][e >> 1];
      float x = __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
      x = __builtin_amdgcn_fmed3f(x, -thr, thr);
      d[e] = x - zf;
      y[e] = __builtin_fmaf(d[e], r, 0.5f);
      near |= fabsf(y[e] - rintf(y[e])) < 1.52587890625e-05f;  // quant4.h
    }
    if (__any(near)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = d[e] / sf + 0.5f;
    }
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int c = static_cast<int>(y[e]);
      c = c < 0 ? 0 : (c > 15 ? 15 : c);
      packed |= static_cast<uint32_t>(c) << (4 * e);
    }
    if (record) *reinterpret_cast<uint32_t*>(codes + 16 * m + 4 * g) = packed;
  }
  if (record && g == 0)
    *reinterpret_cast<uint32_t*>(record + kSide4 + 4 * is_v) = scale | (zero << 16);
}

template <bool kAdjacent, bool kFp32, bool kAxes>
__global__ __launch_bounds__(kWalkThreads, 2) void append_walk_kernel(const AppendArgs a,
                                                                      int value_groups) {
  __shared__ __attribute__((aligned(16))) uint8_t s_r[kHeadDim * kHeadDim * 2];
  __shared__ __attribute__((aligned(16))) float s_weight[2][kHeadDim];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int64_t active = live_tokens(a);
  // The last workgroups take the values, the others the keys and then the queries.
  const int groups = static_cast<int>(gridDim.x);
  const bool is_v = static_cast<int>(blockIdx.x) >= groups - value_groups;
  const int mine = is_v ? groups - value_groups : 0;
  const int64_t k_blocks = is_v ? 0 : (a.set[1].rows + 15) / 16;
  const int64_t blocks = is_v ? (a.set[2].rows + 15) / 16 : k_blocks + (a.set[0].rows + 15) / 16;
  const int64_t width = is_v ? value_groups : groups - value_groups;
  const int64_t first = static_cast<int64_t>(wave) * width + (blockIdx.x - mine);
  const int64_t step = kWalkWaves * width;
  const int half = a.rotary >> 1;
  auto set_of = [&](int64_t b) { return is_v ? 2 : b < k_blocks ? 1 : 0; };

  u32x4 x[8];
  int64_t row = 0, position = 0;
  uint32_t token = 0;
  int head = 0;
  bool live = false, bad = false;
  constexpr int kBytes = kFp32 ? 4 : 2, kLoads = kFp32 ? 2 : 1;
  // Packed angles of eight consecutive dims of a half, or of the four pairs of eight adjacent dims.
  constexpr int kWords = kAdjacent ? 2 * kLoads : 4 * kLoads;
  const char* turn = nullptr;  // the angles' table row
  uint32_t turn_token = 0;     // or the token that has several
  // Angles of the lane's group j of dims (32 j + 8 g on).
  auto load_words = [&](int j, uint32_t (&c)[kWords], uint32_t (&sn)[kWords]) {
    const int pair = kAdjacent ? 16 * j + 4 * g : 32 * j + 8 * g;
    if constexpr (kAxes) {
      constexpr int kN = kAdjacent ? 4 : 8;
      axis_words<kN, kFp32>(
          a.angles,
          [&](int axis) { return a.angles.positions[axis * a.angles.position_stride + turn_token]; },
          pair, pair_axes<kN>(a.angles, pair), c, sn);
    } else {
      auto load = [](const char* at, uint32_t (&w)[kWords]) {
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
      load(turn + pair * kBytes, c);
      load(turn + (pair + half) * kBytes, sn);
    }
  };
  auto word_value = [](const uint32_t (&w)[kWords], int i) {
    if (kFp32) return __uint_as_float(w[i]);
    return bf16_to_float(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
  };
  uint32_t cos0[kWords], sin0[kWords];  // of the first group of dims, with the row's loads

  // The lane's row of block b: its token (and position), then its values.
  auto place = [&](int64_t b) {
    const int which = set_of(b);
    const RowSet& t = a.set[which];
    row = (which == 0 ? b - k_blocks : b) * 16 + n;
    const uint32_t safe = row < t.rows ? static_cast<uint32_t>(row) : 0u;
    token = fastdiv(safe, t.h_div);
    head = static_cast<int>(safe - token * static_cast<uint32_t>(t.heads));
    live = row < t.rows && token < active;
    position = !kAxes && which < 2 && a.rotary && live ? a.angles.positions[token] : 0;
    const uint16_t* src = t.x + static_cast<int64_t>(token) * t.s0 + static_cast<int64_t>(head) * t.s1 + 8 * g;
#pragma unroll
    for (int m = 0; m < 8; ++m) x[m] = *reinterpret_cast<const u32x4*>(src + 32 * m);
  };
  auto load_angles = [&](int64_t b) {
    if (set_of(b) == 2) return;
    if constexpr (kAxes) {
      bad = false;
      for (int k = g; live && k < a.angles.count; k += 4) bad |= bad_position(a.angles, token, k);
      bad = row_max(bad) != 0;
      turn_token = live ? token : 0;  // a dead row's angles are those of a token that exists
    } else {
      bad = a.rotary > 0 && (position < 0 || position >= a.angles.rows);
      turn = static_cast<const char*>(a.angles.table) + (bad ? 0 : position) * a.angles.stride * kBytes;
    }
    if (8 * g < a.rotary) load_words(0, cos0, sin0);
  };

  u32x4 y[8];  // the finished rows
  // The arithmetic of norm_rope.hip's walking kernel.
  auto finish = [&](int which) {
    if (which == 2) {
#pragma unroll
      for (int m = 0; m < 8; ++m) y[m] = x[m];
      return;
    }
    const float* w = s_weight[which] + 8 * g;
    float v[8][8];
    float inv = bad ? __uint_as_float(0x7fc00000u) : 1.f;
    const bool norm = a.set[which].weight != nullptr;
    if (norm) {
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
      inv = inverse_root(mean, bad);
    }
    if (norm) {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        unpack_eight(x[m], v[m]);
        const f32x4 lo = *reinterpret_cast<const f32x4*>(w + 32 * m);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(w + 32 * m + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[m][e] = v[m][e] * inv * (e < 4 ? lo[e & 3] : hi[e & 3]);
      }
    } else {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        unpack_eight(x[m], v[m]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[m][e] *= inv;
      }
    }
    if constexpr (!kAdjacent) {
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
        if (j) load_words(j, c, s);
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
          if (m) load_words(m, c, s);
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
      for (int e = 0; e < 4; ++e) y[m][e] = pack_bf16x2(v[m][2 * e], v[m][2 * e + 1]);
    if (!__all(live)) {
#pragma unroll
      for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[m][e] = live ? y[m][e] : 0u;
    }
  };

  if (first < blocks) place(first);
  float weight[8];
  const bool stages = tid < 64 && a.set[tid >> 5].weight;
  if (stages) load_eight(a.set[tid >> 5].weight, 8 * (tid & 31), a.weight_fp32, weight);
  if (first < blocks) load_angles(first);
  // Row 16 t + i of the LDS copy is the column of R that lane i's A operand of tile t reads, 32 (t / 2)
  // + 8 (i / 4) + 4 (t % 2) + i % 4, so that a lane ends with eight consecutive columns of a row in two
  // tiles; its 16-byte piece p lies at p ^ i (norm_rope.hip).
  const uint16_t* rt = a.rt[is_v ? 2 : 1];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int q = 2 * (16 * wave + j) + (lane >> 5), t = q >> 4, i = q & 15;
    const int col = 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(rt + col * kHeadDim + 8 * ((lane & 31) ^ i)),
        (__attribute__((address_space(3))) void*)(s_r + 1024 * (16 * wave + j)), 16, 0, 0);
  }
  if (stages)
#pragma unroll
    for (int e = 0; e < 8; ++e) s_weight[tid >> 5][8 * (tid & 31) + e] = weight[e] + a.offset;
  OSCAR_WAIT_VM0_SEEN();
  __syncthreads();  // R and the weights
  for (int64_t b = first; b < blocks; b += step) {
    const int which = set_of(b);
    finish(which);
    const int64_t my_row = row;
    const uint32_t my_token = token;
    const bool my_live = live;
    const int my_head = head;
    if (b + step < blocks) {
      place(b + step);
      load_angles(b + step);
    }
    const RowSet& t = a.set[which];
    const bool in = my_row < t.rows;
    if (which < 2 && in) {
      uint16_t* out = t.out + my_row * kHeadDim + 8 * g;
#pragma unroll
      for (int m = 0; m < 8; ++m) *reinterpret_cast<u32x4*>(out + 32 * m) = y[m];
    }
    if (!which && !a.q_rot) continue;
    u32x4 z[8];
    const uint8_t* from[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) from[m] = s_r + 512 * n + 16 * ((4 * m + g) ^ n);
    // Eight operands (four products of two tiles) are read ahead of the eight in use.
    u32x4 f[2][8];
    auto read = [&](int i, u32x4 (&w)[8]) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        w[k] = *reinterpret_cast<const u32x4*>(from[k >> 1] + 8192 * (2 * (i >> 1) + (k & 1)) +
                                               256 * (i & 1));
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
      if (i & 1)
        z[i >> 1] = u32x4{pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3]),
                          pack_bf16x2(acc[1][0], acc[1][1]), pack_bf16x2(acc[1][2], acc[1][3])};
    }
    if (!which) {
      uint16_t* out = a.q_rot + my_row * kHeadDim + 8 * g;
      if (in)
#pragma unroll
        for (int m = 0; m < 8; ++m) *reinterpret_cast<u32x4*>(out + 32 * m) = z[m];
      continue;
    }
    const int64_t slot = my_live ? a.slots[my_token] : -1;
    quantize_rows4(z, a.mode, a.ratio[which], a.factor[which], is_v, g, [&]() -> uint8_t* {
      if (slot < 0 || slot >= a.history_bytes) return nullptr;
      const int64_t at = slot_offset(a.L, slot, my_head);
      return at + a.L.slot_bytes <= a.history_bytes ? a.history + at : nullptr;
    });
  }
}

// ---- records back to values: half a wavefront per record, 8 dims a lane of either vector, two records in
// flight. 2048 records take 3.4 us, 16384 6.0 (21 MB, 3.5 TB/s) to 6.8.
struct ReadArgs {
  const uint8_t* history;
  int64_t history_bytes;
  const int64_t* slots;
  int64_t items;  // (token, head) pairs
  FastDiv h_div;
  Layout L;
  uint16_t* out[2];
};
constexpr int kReadPer = 2, kReadItems = 8 * kReadPer;  // records of a half wavefront, of a workgroup

template <int kBits>
__global__ __launch_bounds__(kThreads) void read_records_kernel(const ReadArgs a) {
  const int l = threadIdx.x & 31, mine = threadIdx.x >> 5;
  const int64_t item0 = static_cast<int64_t>(blockIdx.x) * kReadItems + mine;
  uint32_t codes[kReadPer][2] = {}, side[kReadPer][2] = {};  // no record: zeros
#pragma unroll
  for (int i = 0; i < kReadPer; ++i) {
    const int64_t item = item0 + 8 * i;
    if (item >= a.items) break;
    const uint32_t token = fastdiv(static_cast<uint32_t>(item), a.h_div);
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= a.history_bytes) continue;
    const int64_t at = slot_offset(
        a.L, slot, static_cast<int>(item - static_cast<int64_t>(token) * a.L.kv_heads));
    if (at + a.L.slot_bytes > a.history_bytes) continue;
    const uint8_t* p = a.history + at;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (kBits == 4) {
        codes[i][v] = reinterpret_cast<const uint32_t*>(p + v * kCodes4)[l];
        side[i][v] = *reinterpret_cast<const uint32_t*>(p + kSide4 + 4 * v);
      } else {
        codes[i][v] = reinterpret_cast<const uint16_t*>(p + v * a.L.vector_bytes)[l];
        side[i][v] = *reinterpret_cast<const uint32_t*>(p + v * a.L.vector_bytes + kHeadDim / 4);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kReadPer; ++i) {
    const int64_t item = item0 + 8 * i;
    if (item >= a.items) break;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const float scale = half_lo_to_float(side[i][v]), zero = half_hi_to_float(side[i][v]);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = codes[i][v] >> (kBits * e) & ((1u << kBits) - 1);
        // As the oracle decodes: the product is rounded before the sum.
        x[e] = __fadd_rn(__fmul_rn(static_cast<float>(c), scale), zero);
      }
      *reinterpret_cast<u32x4*>(a.out[v] + item * kHeadDim + 8 * l) =
          u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                pack_bf16x2(x[6], x[7])};
    }
  }
}

inline bool aligned(const void* p, uintptr_t by) { return reinterpret_cast<uintptr_t>(p) % by == 0; }

RowSet row_set(const void* x, int64_t s0, int64_t s1, const void* weight, void* out, int64_t n,
               int64_t heads) {
  return {static_cast<const uint16_t*>(x), s0, s1, weight, static_cast<uint16_t*>(out), n * heads,
          static_cast<int32_t>(heads), make_fastdiv(static_cast<uint32_t>(heads))};
}

// The workgroups for the values such that the longer of both kinds' walks is shortest. A CU's wavefronts
// share its four SIMDs, so the largest number of blocks of a SIMD counts, each at its cost in units of about
// 1 us: a value 6 (product and quantizer), a key 6, a query 3, a norm 2 more, a query's product 3. 16384
// tokens of 6 heads, normed and rotated: 32 workgroups 50.6 us, 28 55.9, 40 52.8, 64 56.0; 4 heads that are only
// turned: 64 27.8, 52 29.8, 44 35.5, 80 29.0; 2048 tokens of 12: 32 19.7, 28 22.0, 36 21.7. The 255
// trials take the host 2.7 us a call.
int value_groups_of(int64_t q_blocks, int64_t kv_blocks, bool rotated, bool normed) {
  const int64_t k_cost = normed ? 8 : 6, q_cost = 3 + (normed ? 2 : 0) + (rotated ? 3 : 0);
  auto of_simd = [](int64_t blocks, int64_t groups) { return (blocks + 4 * groups - 1) / (4 * groups); };
  int best = 1;
  int64_t least = INT64_MAX;
  for (int g = 1; g < static_cast<int>(kWalkGroups); ++g) {
    const int64_t rest = kWalkGroups - g, keys = of_simd(kv_blocks, rest);
    const int64_t qk = k_cost * keys + q_cost * (of_simd(q_blocks + kv_blocks, rest) - keys);
    const int64_t v = 6 * of_simd(kv_blocks, g), time = v > qk ? v : qk;
    if (time <= least) {
      least = time;
      best = g;
    }
  }
  return best;
}

// Whether append_walk_kernel serves the call: 4-bit records, no clip search, and pairs in one lane.
bool walks(const AppendArgs& a) {
  const bool rows16 = !a.rotary || (aligned(a.angles.table, 16) && a.angles.stride % 8 == 0 &&
                                    aligned(a.angles.axes, 16));
  return a.set[2].rows && a.L.bits == 4 && a.mode != OSCAR_CLIP_SEARCH && rows16 &&
         (a.adjacent ? a.rotary % 8 == 0 : a.rotary % 64 == 0);
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_rope_append(
    const void* query, int64_t q_s0, int64_t q_s1, const void* key, int64_t k_s0, int64_t k_s1,
    const void* value, int64_t v_s0, int64_t v_s1, int64_t n, int64_t hq, int64_t hk,
    const void* q_weight, const void* k_weight, int32_t weight_fp32, int32_t unit_offset, float eps,
    const void* cos_sin, int64_t table_rows, int64_t table_stride, int32_t table_fp32,
    int32_t rotary_dim, int32_t interleaved, const int64_t* positions, int64_t position_stride,
    int32_t axis_count, const int32_t* axes, const int32_t* counts, void* q_out, void* k_out,
    const void* rk_t, const void* rv_t, void* q_rot, void* history, int64_t history_bytes,
    const int64_t* slots, const oscar_layout* layout, const oscar_clip* clip, void* stream) {
  using namespace oscar;
  const bool store = value != nullptr;
  AppendArgs a{};
  if (n < 0 || hq < 0 || hk <= 0 || rotary_dim < 0 || rotary_dim > kHeadDim || rotary_dim % 2)
    return OSCAR_E_SHAPE;
  if (rotary_dim && (table_rows < 1 || table_stride < rotary_dim || axis_count < 1 ||
                     axis_count > kMostAxes || (axis_count > 1 && position_stride < n)))
    return OSCAR_E_SHAPE;
  if (!(eps >= 0.f) || !(eps < INFINITY)) return OSCAR_E_UNSUPPORTED;
  if (store) {
    const int st = make_any_layout(layout, &a.L);
    if (st != OSCAR_OK) return st;
    if (!clip) return OSCAR_E_NULL;
    if (clip->mode < OSCAR_CLIP_PERCENTILE || clip->mode > OSCAR_CLIP_SEARCH || history_bytes < 0 ||
        hk != a.L.kv_heads)
      return OSCAR_E_SHAPE;
  }
  if (n == 0) return OSCAR_OK;
  if (!key || !k_out || !query != !hq || !query != !q_out || (rotary_dim && (!positions || !cos_sin)) ||
      (rotary_dim && axis_count > 1 && !axes) || (!query && q_rot) || !q_weight != !(k_weight && query))
    return OSCAR_E_NULL;
  if ((q_rot || store) && !rk_t) return OSCAR_E_NULL;
  if (store && (!rv_t || !history || !slots || !counts)) return OSCAR_E_NULL;
  // A launch holds fewer than 2^32 threads: 64 a row, and each set's last block.
  if (hq > (1ll << 26) || hk > (1ll << 26) || hq + 2 * hk > ((1ll << 26) - 64) / n)
    return OSCAR_E_SHAPE;
  if ((query && (q_s0 % 8 || q_s1 % 8 || !aligned(query, 16) || !aligned(q_out, 16))) || k_s0 % 8 ||
      k_s1 % 8 || !aligned(key, 16) || !aligned(k_out, 16) || !aligned(q_weight, 16) ||
      !aligned(k_weight, 16) || !aligned(rk_t, 16) || !aligned(q_rot, 16) ||
      !aligned(cos_sin, table_fp32 ? 4 : 2))
    return OSCAR_E_ALIGN;
  if (store && (v_s0 % 8 || v_s1 % 8 || !aligned(value, 16) || !aligned(rv_t, 16) ||
                !aligned(history, 16)))
    return OSCAR_E_ALIGN;
  hipStream_t s = as_stream(stream);
  const int64_t all = n * (hq + hk + (store ? hk : 0));
  // Rows of several positions without R_k: norm_rope.hip's streaming kernel.
  if (axes && !store && !q_rot && query && q_weight && rotary_dim &&
      launch_norm_rope_axes(query, q_s0, q_s1, key, k_s0, k_s1, n, hq, hk, q_weight, k_weight,
                            weight_fp32, unit_offset, eps, table_fp32, interleaved, counts, q_out,
                            k_out, {cos_sin, table_rows, table_stride, positions, position_stride, axes,
                                    axis_count, rotary_dim}, s))
    return static_cast<int>(hipGetLastError());
  if (query) a.set[0] = row_set(query, q_s0, q_s1, q_weight, q_out, n, hq);
  a.set[1] = row_set(key, k_s0, k_s1, k_weight, k_out, n, hk);
  if (store) a.set[2] = row_set(value, v_s0, v_s1, nullptr, nullptr, n, hk);
  a.angles = {cos_sin, table_rows, table_stride, positions, position_stride,
              rotary_dim ? axes : nullptr, axis_count, rotary_dim};
  a.counts = counts;
  a.n = n;
  a.rotary = rotary_dim;
  a.rotary_div = make_fastdiv(static_cast<uint32_t>(rotary_dim ? rotary_dim : 1));
  a.table_fp32 = table_fp32 ? 1 : 0;
  a.weight_fp32 = weight_fp32 ? 1 : 0;
  a.adjacent = interleaved ? 1 : 0;
  a.offset = unit_offset ? 1.f : 0.f;
  a.eps = eps;
  a.rt[0] = q_rot ? static_cast<const uint16_t*>(rk_t) : nullptr;
  a.rt[1] = store ? static_cast<const uint16_t*>(rk_t) : nullptr;
  a.rt[2] = static_cast<const uint16_t*>(rv_t);
  a.q_rot = static_cast<uint16_t*>(q_rot);
  a.history = static_cast<uint8_t*>(history);
  a.history_bytes = history_bytes;
  a.slots = slots;
  if (store) {
    a.mode = clip->mode;
    a.ratio[1] = clip->k_ratio;
    a.ratio[2] = clip->v_ratio;
    a.factor[1] = clip->k_factor;
    a.factor[2] = clip->v_factor;
  }
  auto blocks = [&](int i, int64_t rows) { return (a.set[i].rows + rows - 1) / rows; };
  auto lds = [&](int rows) { return static_cast<uint32_t>(rows * rotary_dim * sizeof(float)); };
  if (!q_rot && !store) {
    const int64_t q = blocks(0, kTurnRows), grid = q + blocks(1, kTurnRows);
    hipLaunchKernelGGL(turn_rows_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                       lds(kTurnRows + 8), s, a, q);
  } else if (all > kSmallAppendRows && walks(a)) {
    const int value_groups = value_groups_of(blocks(0, 16), blocks(1, 16), q_rot != nullptr,
                                             k_weight != nullptr);
    auto walk = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(kWalkGroups), dim3(kWalkThreads), 0, s, a, value_groups);
    };
    auto by_axes = [&](auto adjacent, auto fp32) {
      constexpr bool kAdjacent = decltype(adjacent)::value, kFp32 = decltype(fp32)::value;
      if (a.angles.axes)
        walk(append_walk_kernel<kAdjacent, kFp32, true>);
      else
        walk(append_walk_kernel<kAdjacent, kFp32, false>);
    };
    if (a.adjacent || !rotary_dim)
      table_fp32 ? by_axes(std::true_type(), std::true_type())
                 : by_axes(std::true_type(), std::false_type());
    else
      table_fp32 ? by_axes(std::false_type(), std::true_type())
                 : by_axes(std::false_type(), std::false_type());
  } else if (all <= kSmallAppendRows) {
    const int64_t q = blocks(0, 16), k = blocks(1, 16);
    hipLaunchKernelGGL(append_kernel<1>, dim3(static_cast<unsigned>(q + k + blocks(2, 16))),
                       dim3(kAppendThreads), lds(2 * 16), s, a, q, k);
  } else {
    const int64_t q = blocks(0, 32), k = blocks(1, 32);
    hipLaunchKernelGGL(append_kernel<2>, dim3(static_cast<unsigned>(q + k + blocks(2, 32))),
                       dim3(kAppendThreads), lds(2 * 32), s, a, q, k);
  }
  return static_cast<int>(hipGetLastError());
}

extern "C" int oscar_read_records(const void* history, int64_t history_bytes, const int64_t* slots,
                                  int64_t n, const oscar_layout* layout, void* key_out,
                                  void* value_out, void* stream) {
  using namespace oscar;
  if (n < 0 || history_bytes < 0) return OSCAR_E_SHAPE;
  ReadArgs a{};
  const int st = make_any_layout(layout, &a.L);
  if (st != OSCAR_OK) return st;
  if (n == 0) return OSCAR_OK;
  if (!history || !slots || !key_out || !value_out) return OSCAR_E_NULL;
  // 16 threads an item, fewer than 2^32 a launch.
  if (a.L.kv_heads > 0x7ffffffll / n) return OSCAR_E_SHAPE;
  if (!aligned(history, 4) || !aligned(key_out, 16) || !aligned(value_out, 16)) return OSCAR_E_ALIGN;
  a.history = static_cast<const uint8_t*>(history);
  a.history_bytes = history_bytes;
  a.slots = slots;
  a.items = n * a.L.kv_heads;
  a.h_div = make_fastdiv(static_cast<uint32_t>(a.L.kv_heads));
  a.out[0] = static_cast<uint16_t*>(key_out);
  a.out[1] = static_cast<uint16_t*>(value_out);
  const dim3 grid(static_cast<unsigned>((a.items + kReadItems - 1) / kReadItems));
  if (a.L.bits == 4)
    hipLaunchKernelGGL(read_records_kernel<4>, grid, dim3(kThreads), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(read_records_kernel<2>, grid, dim3(kThreads), 0, as_stream(stream), a);
  return static_cast<int>(hipGetLastError());
}
