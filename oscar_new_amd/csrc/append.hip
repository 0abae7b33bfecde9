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
// A block of rows (token, head) is one workgroup: half a wavefront per row, 32 lanes of 8 dims. The
// block's angles are gathered into LDS first, each pair from the table row of its axis' position, in
// flight with the rows: so several axes, any table type and any pair order cost the rows nothing.
#include "norm_row.h"
#include "quant4.h"
#include "rotate.h"

namespace oscar {
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
  const void* table;  // [table_rows][rotary]: cos of every pair, then sin
  int64_t table_rows, table_stride;
  const int64_t* positions;  // axis a of token t at a * position_stride + t
  int64_t position_stride;
  const int32_t* axes;  // axis of every pair; null: axis 0
  const int32_t* counts;
  int64_t n;
  int32_t axis_count, rotary, table_fp32, weight_fp32, adjacent;
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
    const int axis = a.axes ? a.axes[e < half ? e : e - half] : 0;
    const int64_t token = first_token + t;
    float v = __uint_as_float(0x7fc00000u);
    if (token < active && axis >= 0 && axis < a.axis_count) {
      const int64_t p = a.positions[axis * a.position_stride + token];
      if (p >= 0 && p < a.table_rows) v = load_value(a.table, p * a.table_stride + e, a.table_fp32);
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
__device__ __forceinline__ bool bad_position(const AppendArgs& a, int64_t token, bool live, int l) {
  bool out = false;
  if (a.rotary && live && l < a.axis_count) {
    const int64_t p = a.positions[l * a.position_stride + token];
    out = p < 0 || p >= a.table_rows;
  }
  const uint64_t any = __ballot(out);
  return ((any >> (threadIdx.x & 32)) & 0xffffffffull) != 0;
}

// ---- rows that are turned only: each half wavefront takes kPerHalf rows, whose loads are in flight
// together with the block's angles.
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
    bad[i] = bad_position(a, token[i], token[i] < active, l);
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
// to the wavefronts that quantize a row each.
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
      bad = bad_position(a, token, has_row && token < active, l);
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

// Rows up to which blocks hold 16 of them instead of 32, so that the blocks of a decode step lie on as
// many CUs as they can.
constexpr int64_t kSmallAppendRows = 16 * 256;

// ---- records back to values: a wavefront per vector.
struct ReadArgs {
  const uint8_t* history;
  int64_t history_bytes;
  const int64_t* slots;
  int64_t items;  // (token, head) pairs
  FastDiv h_div;
  Layout L;
  uint16_t* out[2];
};

__global__ __launch_bounds__(kThreads) void read_records_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 2 + (wave >> 1);
  const int is_v = wave & 1;
  if (item >= a.items) return;
  const uint32_t token = fastdiv(static_cast<uint32_t>(item), a.h_div);
  const int head = static_cast<int>(item - static_cast<int64_t>(token) * a.L.kv_heads);
  const int64_t slot = a.slots[token];
  uint2 bits = make_uint2(0u, 0u);
  if (slot >= 0 && slot < a.history_bytes) {
    const int64_t at = slot_offset(a.L, slot, head);
    if (at + a.L.slot_bytes <= a.history_bytes) {
      const uint8_t* p = a.history + at;
      uint32_t codes, side;
      float value[4];
      if (a.L.bits == 4) {
        codes = reinterpret_cast<const uint16_t*>(p + is_v * kCodes4)[lane];
        side = *reinterpret_cast<const uint32_t*>(p + kSide4 + 4 * is_v);
      } else {
        codes = p[is_v * a.L.vector_bytes + lane];
        side = *reinterpret_cast<const uint32_t*>(p + is_v * a.L.vector_bytes + kHeadDim / 4);
      }
      const float scale = half_lo_to_float(side), zero = half_hi_to_float(side);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t c = a.L.bits == 4 ? codes >> (4 * e) & 15u : codes >> (2 * e) & 3u;
        // As the oracle decodes: the product is rounded before the sum.
        value[e] = __fadd_rn(__fmul_rn(static_cast<float>(c), scale), zero);
      }
      bits = make_uint2(pack_bf16x2(value[0], value[1]), pack_bf16x2(value[2], value[3]));
    }
  }
  *reinterpret_cast<uint2*>(a.out[is_v] + item * kHeadDim + 4 * lane) = bits;
}

inline bool aligned(const void* p, uintptr_t by) { return reinterpret_cast<uintptr_t>(p) % by == 0; }

RowSet row_set(const void* x, int64_t s0, int64_t s1, const void* weight, void* out, int64_t n,
               int64_t heads) {
  return {static_cast<const uint16_t*>(x), s0, s1, weight, static_cast<uint16_t*>(out), n * heads,
          static_cast<int32_t>(heads), make_fastdiv(static_cast<uint32_t>(heads))};
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
  if (query) a.set[0] = row_set(query, q_s0, q_s1, q_weight, q_out, n, hq);
  a.set[1] = row_set(key, k_s0, k_s1, k_weight, k_out, n, hk);
  if (store) a.set[2] = row_set(value, v_s0, v_s1, nullptr, nullptr, n, hk);
  a.table = cos_sin;
  a.table_rows = table_rows;
  a.table_stride = table_stride;
  a.positions = positions;
  a.position_stride = position_stride;
  a.axes = axis_count > 1 ? axes : nullptr;
  a.axis_count = axis_count;
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
  hipStream_t s = as_stream(stream);
  const int64_t all = a.set[0].rows + a.set[1].rows + a.set[2].rows;
  auto blocks = [&](int i, int64_t rows) { return (a.set[i].rows + rows - 1) / rows; };
  auto lds = [&](int rows) { return static_cast<uint32_t>(rows * rotary_dim * sizeof(float)); };
  if (!q_rot && !store) {
    const int64_t q = blocks(0, kTurnRows), grid = q + blocks(1, kTurnRows);
    hipLaunchKernelGGL(turn_rows_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                       lds(kTurnRows + 8), s, a, q);
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
  // 128 threads an item, fewer than 2^32 a launch.
  if (a.L.kv_heads > 0x1ffffffll / n) return OSCAR_E_SHAPE;
  if (!aligned(history, 4) || !aligned(key_out, 8) || !aligned(value_out, 8)) return OSCAR_E_ALIGN;
  a.history = static_cast<const uint8_t*>(history);
  a.history_bytes = history_bytes;
  a.slots = slots;
  a.items = n * a.L.kv_heads;
  a.h_div = make_fastdiv(static_cast<uint32_t>(a.L.kv_heads));
  a.out[0] = static_cast<uint16_t*>(key_out);
  a.out[1] = static_cast<uint16_t*>(value_out);
  hipLaunchKernelGGL(read_records_kernel, dim3(static_cast<unsigned>((a.items + 1) / 2)),
                     dim3(kThreads), 0, as_stream(stream), a);
  return static_cast<int>(hipGetLastError());
}
