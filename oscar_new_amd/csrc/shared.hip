// INT2 history attention of a batch whose requests share long prefixes (samples of one prompt): the
// shared positions are computed once for all rows of a group instead of once per request.
//
//   out[row] = sum_p e^{s_p} v_p / sum_p e^{s_p},  s_p = scale q . k_p,  p in [sink_len, recent_begin)
//
// of the row's request: the history branch of oscar_ascend/kernels.py:290-482 followed by its split
// merge (485-511); the reference shares nothing between requests (oscar_ascend/metadata.py:82-95).
// History positions are masked by no row of a step, so every row of a group sees all positions
// before E, the first one that some member does not share, rounded down to a chunk. They form one
// long matrix product: `rows` is the members' query tokens times the heads of a KV head.
//
// Units. A step's work is (row tile, position range) units: the group's rows against [sink, E)
// through its first member's pages, and each request's own rows against [E, recent_begin) through
// its own. Up to kSmallRows rows a tile is 16 rows whose positions the wavefronts of a workgroup
// divide (row_tile.h), above that 128 rows that share the codes (chunk_tile.h). The plan kernel cuts
// every tile's positions into pieces from the whole step's lengths, so that the launch ends early on
// 256 CUs, and writes the list, once per step and before every layer's launch. Partial rows of a
// tile's pieces go to slots that the merge kernel joins by their LSEs, as many as the plan says for
// each token.
#include "merge.h"
#include "row_tile.h"

namespace oscar {
namespace {

constexpr int kSharedThreads = 1024;
constexpr int kSharedEntries = 4096;  // groups and requests whose counts live in LDS
constexpr int kSharedSlots = 256;     // partial rows of a row: four per lane of a merging wavefront
constexpr int kUnitWords = 8;
// Rows up to which a tile is 16 rows; 128-token chunks such a unit takes at least.
constexpr int kSmallRows = 48, kSmallPiece = 4;
// A unit's time in us: its start and end, and each 128-token chunk.
constexpr float kTileStart = 11.f, kTileChunk = 4.1f, kSmallStart = 11.f, kSmallChunk = 0.8f;

// A unit: rows [row_base, row_end) of tokens token0 .. (row r is token token0 + r / g), positions
// [p_lo, p_hi) through block-table row req, partials to `slot`; small: at most 16 rows, row_tile.h.
struct Unit {
  int32_t req, token0, row_end, row_base, p_lo, p_hi, slot, small;
};
static_assert(sizeof(Unit) == kUnitWords * 4, "one unit is eight words");

struct SharedPlanArgs {
  const int32_t* qstarts;
  const int32_t* seq_lens;
  const int32_t* counts;
  const int32_t* group_starts;   // [groups + 1] request indexes
  const int32_t* prefix_tokens;  // [groups]
  Unit* units;
  int32_t* unit_count;
  int32_t* token_slots;
  int32_t groups, max_reqs, sink, recent, g, budget, capacity, slots;
  int64_t tokens;
};

// Sums of two counts and a maximum over the workgroup (every thread gets them).
__device__ __forceinline__ void plan_reduce(int64_t (&sum)[2], int& most) {
  __shared__ int64_t s_sum[2][kSharedThreads / kWave];
  __shared__ int s_most[kSharedThreads / kWave];
  const int wave = threadIdx.x >> 6;
  for (int i = 0; i < 2; ++i) sum[i] = wave_sum_i64(sum[i]);
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) most = max(most, __shfl_xor(most, m, kWave));
  if ((threadIdx.x & 63) == 0) {
    s_sum[0][wave] = sum[0];
    s_sum[1][wave] = sum[1];
    s_most[wave] = most;
  }
  __syncthreads();
  sum[0] = sum[1] = 0;
#pragma unroll
  for (int w = 0; w < kSharedThreads / kWave; ++w) {
    sum[0] += s_sum[0][w];
    sum[1] += s_sum[1][w];
    most = max(most, s_most[w]);
  }
}

// Tiles of an entry of `rows` rows (small entries: 16-row tiles, kept negative).
__device__ __forceinline__ int tiles_of(int rows) {
  return rows <= kSmallRows ? -((rows + 15) / 16) : (rows + kRowsC - 1) / kRowsC;
}
__device__ __forceinline__ int chunks_of(int lo, int hi) {
  return lo < hi ? ((hi - 1) >> 7) - (lo >> 7) + 1 : 0;
}

__global__ __launch_bounds__(kSharedThreads) void shared_plan_kernel(const SharedPlanArgs a) {
  // Entries: the groups, then the requests.
  __shared__ int s_chunks[kSharedEntries], s_tiles[kSharedEntries], s_start[kSharedEntries + 1];
  // Requests: first token, end of the history, first position of the request's own part, and the
  // group whose positions it shares, or -1.
  __shared__ int s_token[kSharedEntries + 1], s_end[kSharedEntries], s_own[kSharedEntries];
  __shared__ int s_group[kSharedEntries];
  __shared__ int s_wave[kSharedThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int reqs = max(min(a.counts[0], a.max_reqs), 0);
  const int active = static_cast<int>(
      min(static_cast<int64_t>(max(a.counts[1], 0)), a.tokens));
  for (int r = tid; r < reqs; r += kSharedThreads) {
    const int t0 = min(max(a.qstarts[r], 0), active), t1 = min(max(a.qstarts[r + 1], 0), active);
    const int prefix = a.seq_lens[r] - max(t1 - t0, 0);
    const int sink_len = max(min(a.sink, prefix), 0);
    s_token[r] = t0;
    if (r + 1 == reqs) s_token[reqs] = t1;
    s_end[r] = max(sink_len, prefix - a.recent);
    s_own[r] = sink_len;
    s_group[r] = -1;
  }
  // Starts that descend are no partition: then nothing is shared.
  bool bad = false;
  for (int i = tid; i < a.groups; i += kSharedThreads)
    bad |= a.group_starts[i + 1] < a.group_starts[i];
  const int groups = __syncthreads_or(bad) ? 0 : a.groups;
  const int entries = groups + reqs;
  auto rows_of = [&](int r0, int r1) { return max(s_token[r1] - s_token[r0], 0) * a.g; };
  auto clip = [&](int r) { return min(max(r, 0), reqs); };

  for (int i = wave; i < groups; i += kSharedThreads / kWave) {
    const int r0 = clip(a.group_starts[i]), r1 = clip(a.group_starts[i + 1]);
    int end = a.prefix_tokens[i];
    for (int r = r0 + lane; r < r1; r += kWave) end = min(end, s_end[r]);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) end = min(end, __shfl_xor(end, m, kWave));
    end &= ~(kTokC - 1);
    // Past the sink every member's recent part starts behind it, so all begin at `sink`.
    const bool shared = r1 - r0 > 1 && end > a.sink;
    if (shared)
      for (int r = r0 + lane; r < r1; r += kWave) {
        s_own[r] = end;
        s_group[r] = i;
      }
    if (lane == 0) {
      s_chunks[i] = shared ? chunks_of(a.sink, end) : 0;
      s_tiles[i] = tiles_of(shared ? rows_of(r0, r1) : 0);
    }
  }
  __syncthreads();
  int most = 0;  // chunks of one row's positions
  for (int r = tid; r < reqs; r += kSharedThreads) {
    const int rows = rows_of(r, r + 1);
    s_chunks[groups + r] = chunks_of(s_own[r], s_end[r]);
    s_tiles[groups + r] = tiles_of(rows);
    if (rows > 0)
      most = max(most, s_chunks[groups + r] + (s_group[r] >= 0 ? s_chunks[s_group[r]] : 0));
  }
  __syncthreads();
  int64_t work = 0, small = 0;  // chunks of 128-row tiles and of 16-row tiles
  for (int e = tid; e < entries; e += kSharedThreads) {
    const int64_t w = static_cast<int64_t>(abs(s_tiles[e])) * s_chunks[e];
    work += s_tiles[e] > 0 ? w : 0;
    small += s_tiles[e] < 0 ? w : 0;
  }
  int64_t sums[2] = {work, small};
  plan_reduce(sums, most);
  work = sums[0];
  small = sums[1];
  // Chunks of a piece: no row in more than `slots` pieces (a row's positions are two ranges, each
  // with one uneven piece), at most `budget` units by the average, and then the first count, of 16
  // tried by the wavefronts at once, with which the 128-row units and the others' load, in units of
  // the same time, fit the budget: they run side by side, one per CU, and a second round would
  // cost more than longer units do.
  const int least = (most + a.slots - 3) / (a.slots - 2);
  const int small_least = max(max(kSmallPiece, least),
                              static_cast<int>((small + a.budget - 1) / a.budget));
  int per = max(max(1, least), static_cast<int>((work + a.budget - 1) / a.budget));
  auto small_per = [&](int t) {
    return max(small_least, static_cast<int>(t * (kTileChunk / kSmallChunk)));
  };
  __shared__ int s_fits;
  for (int round = 0; round < 16; ++round) {
    const int t = per + wave;
    const int t_small = small_per(t);
    int64_t units = 0, small_units = 0;
    for (int e = lane; e < entries; e += kWave) {
      const int64_t count = abs(s_tiles[e]);
      if (s_tiles[e] > 0)
        units += count * cdiv(s_chunks[e], t);
      else
        small_units += count * cdiv(s_chunks[e], t_small);
    }
    units = wave_sum_i64(units);
    small_units = wave_sum_i64(small_units);
    const float load = small_units * kSmallStart + small * kSmallChunk;
    if (tid == 0) s_fits = kSharedThreads / kWave;
    __syncthreads();
    if (lane == 0 && units + load / (kTileStart + kTileChunk * t) <= a.budget)
      atomicMin(&s_fits, wave);
    __syncthreads();
    const int fits = s_fits;
    __syncthreads();
    per += fits;
    if (fits < kSharedThreads / kWave || per >= most) break;
  }
  per = max(1, min(per, most));
  const int per_small = small_per(per);
  auto pieces = [&](int e) {
    return cdiv(s_chunks[e], s_tiles[e] < 0 ? per_small : per);
  };
  auto units_of = [&](int e) { return abs(s_tiles[e]) * pieces(e); };

  // Exclusive scan of the entries' units, eight entries a thread.
  constexpr int kPer = kSharedEntries / kSharedThreads;
  int mine = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int e = kPer * tid + k;
    if (e < entries) mine += units_of(e);
  }
  int incl = mine;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int y = __shfl_up(incl, d, kWave);
    incl += lane >= d ? y : 0;
  }
  if (lane == kWave - 1) s_wave[wave] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < wave; ++w) at += s_wave[w];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int e = kPer * tid + k;
    if (e >= entries) break;
    s_start[e] = at;
    at += units_of(e);
  }
  int total = 0;
#pragma unroll
  for (int w = 0; w < kSharedThreads / kWave; ++w) total += s_wave[w];
  if (tid == 0) s_start[entries] = total;
  __syncthreads();
  const int units = min(total, a.capacity);
  if (tid == 0) a.unit_count[0] = units;
  for (int u = tid; u < units; u += kSharedThreads) {
    int lo = 0, hi = entries;  // the last entry that starts at or before u
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_start[mid] <= u)
        lo = mid;
      else
        hi = mid;
    }
    const int e = lo, tile_count = abs(s_tiles[e]);
    const int64_t count = pieces(e);
    const int local = u - s_start[e], piece = local / tile_count, tile = local - piece * tile_count;
    Unit x;
    int begin, end, rows;
    if (e < groups) {
      const int r0 = clip(a.group_starts[e]), r1 = clip(a.group_starts[e + 1]);
      x.req = r0;
      rows = rows_of(r0, r1);
      begin = a.sink;
      end = s_own[r0];
      x.slot = piece;
    } else {
      const int r = e - groups;
      x.req = r;
      rows = rows_of(r, r + 1);
      begin = s_own[r];
      end = s_end[r];
      x.slot = piece + (s_group[r] >= 0 ? pieces(s_group[r]) : 0);
    }
    x.token0 = s_token[x.req];
    // Tiles of equal numbers of 16-row groups, pieces of equal numbers of chunks.
    const int share = ((rows + 15) / 16 + tile_count - 1) / tile_count * 16;
    x.row_base = tile * share;
    x.row_end = min(x.row_base + share, rows);
    const int c0 = (begin >> 7) + static_cast<int>(static_cast<int64_t>(piece) * s_chunks[e] / count);
    const int c1 =
        (begin >> 7) + static_cast<int>(static_cast<int64_t>(piece + 1) * s_chunks[e] / count);
    x.p_lo = max(begin, c0 << 7);
    x.p_hi = min(end, c1 << 7);
    x.small = s_tiles[e] < 0;
    a.units[u] = x;
  }
  // Eight threads per request.
  for (int r = tid >> 3; r < reqs; r += kSharedThreads / 8) {
    const int used = pieces(groups + r) + (s_group[r] >= 0 ? pieces(s_group[r]) : 0);
    for (int t = s_token[r] + (tid & 7); t < s_token[r + 1]; t += 8) a.token_slots[t] = used;
  }
}

__global__ __launch_bounds__(kThreadsC, 2) void shared_history_kernel(const AttnArgs a) {
  __shared__ union {
    ChunkLds chunk;
    RowTileLds row;
  } lds;
  const int heads = a.L.kv_heads;
  const int index = static_cast<int>(blockIdx.x) / heads;
  const int count = a.task_count[0];
  const Unit u = reinterpret_cast<const Unit*>(a.tasks)[index];  // below the capacity: one wait for both
  if (index >= count || u.row_base >= u.row_end) return;
  Task t{};
  t.req = u.req;
  t.qstart = u.token0;
  const int head = static_cast<int>(blockIdx.x) - index * heads;
  if (u.small)
    row_tile(a, t, head, u.row_end, u.row_base, u.p_lo, u.p_hi, u.slot, lds.row);
  else
    chunk_tile<true>(a, t, head, u.row_end, u.row_base, u.p_lo, u.p_hi, u.slot, lds.chunk);
}

struct SharedMergeArgs {
  const float* partials;  // [rows][slots][256]
  const float* lse;       // [rows][slots]
  const int32_t* token_slots;
  const int32_t* counts;
  void* out;  // bf16 [rows][256], or fp32 with kFloat
  float* out_lse;
  int32_t hq, slots;
};

// One workgroup per row: every wavefront holds all LSEs (four per lane) and adds every fourth slot,
// eight loads in flight; the four sums are added in wavefront order.
template <bool kFloat>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(const SharedMergeArgs a) {
  __shared__ f32x4 s_sum[3][kWave];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t row = blockIdx.x, token = row / a.hq;
  const int used = token < a.counts[1] ? min(max(a.token_slots[token], 0), a.slots) : 0;
  float w[kSharedSlots / kWave];
  float mx = -INFINITY, den = 0.f;
#pragma unroll
  for (int i = 0; i < kSharedSlots / kWave; ++i) {
    w[i] = kWave * i + lane < used ? a.lse[row * a.slots + kWave * i + lane] : -INFINITY;
    mx = fmaxf(mx, w[i]);
  }
  mx = wave_max_dpp(mx);
#pragma unroll
  for (int i = 0; i < kSharedSlots / kWave; ++i) {
    w[i] = w[i] == -INFINITY ? 0.f : expf(w[i] - mx);
    den += w[i];
  }
  den = wave_tree_sum_dpp(den);
  const f32x4* part = reinterpret_cast<const f32x4*>(a.partials + row * a.slots * kHeadDim) + lane;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kSharedSlots / kWave; ++i)
    for (int s0 = wave; s0 < min(used - kWave * i, kWave); s0 += 32) {
      f32x4 v[8];
      float ws[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = s0 + 4 * k;
        const bool in = kWave * i + s < used;
        v[k] = in ? part[static_cast<int64_t>(kWave * i + s) * (kHeadDim / 4)]
                  : f32x4{0.f, 0.f, 0.f, 0.f};
        ws[k] = in ? lane_value(w[i], s) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(ws[k], v[k][e], sum[e]);
    }
  if (wave) s_sum[wave - 1][lane] = sum;
  __syncthreads();
  if (wave) return;
  const float dn = fmaxf(den, kDenFloor);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    sum[e] = (((sum[e] + s_sum[0][lane][e]) + s_sum[1][lane][e]) + s_sum[2][lane][e]) / dn;
  if (kFloat)
    reinterpret_cast<f32x4*>(a.out)[row * (kHeadDim / 4) + lane] = sum;
  else
    reinterpret_cast<uint2*>(a.out)[row * (kHeadDim / 4) + lane] =
        make_uint2(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]));
  if (lane == 0) a.out_lse[row] = den > 0.f ? mx + logf(den) : -INFINITY;
}

// Units that a plan may hold: a tile's pieces pass its share of the budget by less than one, for
// 128-row tiles (one per 128 rows and one more per entry) and for 16-row tiles (at most three per
// entry, and one per 16 rows and one more per entry).
int64_t shared_capacity(int64_t tokens, int64_t g, int64_t groups, int64_t max_reqs,
                        int64_t budget) {
  const int64_t entries = groups + (max_reqs < tokens ? max_reqs : tokens);
  const int64_t tiles = 2 * (tokens * g / kRowsC) + entries;
  const int64_t by_rows = 2 * (tokens * g / 16) + entries;
  return 2 * budget + tiles + (by_rows < 3 * entries ? by_rows : 3 * entries);
}

}  // namespace
}  // namespace oscar

extern "C" int64_t oscar_shared_capacity(int64_t tokens, int64_t hq, int64_t groups,
                                         int64_t max_reqs, int32_t kv_heads) {
  if (tokens < 0 || hq <= 0 || kv_heads <= 0 || groups < 0 || max_reqs < 0) return -1;
  return oscar::shared_capacity(tokens, hq / kv_heads, groups, max_reqs,
                                kv_heads < 256 ? 256 / kv_heads : 1);
}

extern "C" int oscar_shared_plan(const int32_t* qstarts, const int32_t* seq_lens,
                                 const int32_t* counts, const int32_t* group_starts,
                                 const int32_t* prefix_tokens, int64_t groups, int64_t max_reqs,
                                 int64_t tokens, int64_t hq, int32_t slots,
                                 const oscar_layout* layout, int32_t* units, int64_t capacity,
                                 int32_t* unit_count, int32_t* token_slots, void* stream) {
  using namespace oscar;
  Layout L;
  const int st = make_layout(layout, &L);
  if (st != OSCAR_OK) return st;
  if (groups < 0 || max_reqs < 1 || tokens < 0 || tokens > 0x7fffffffll || hq <= 0 ||
      hq % L.kv_heads || hq > 0x7fffffffll / (tokens > 0 ? tokens : 1))
    return OSCAR_E_SHAPE;
  if (groups + max_reqs > kSharedEntries || hq / L.kv_heads > 32) return OSCAR_E_UNSUPPORTED;
  if (slots < 4 || slots > kSharedSlots) return OSCAR_E_SHAPE;
  const int64_t g = hq / L.kv_heads, budget = L.kv_heads < 256 ? 256 / L.kv_heads : 1;
  if (capacity < shared_capacity(tokens, g, groups, max_reqs, budget) || capacity > 0x7fffffffll)
    return OSCAR_E_SHAPE;
  if (!qstarts || !seq_lens || !counts || !units || !unit_count || !token_slots ||
      (groups && (!group_starts || !prefix_tokens)))
    return OSCAR_E_NULL;
  if (reinterpret_cast<uintptr_t>(units) % 16) return OSCAR_E_ALIGN;
  const SharedPlanArgs a{qstarts, seq_lens, counts, group_starts, prefix_tokens,
                         reinterpret_cast<Unit*>(units), unit_count, token_slots,
                         static_cast<int32_t>(groups), static_cast<int32_t>(max_reqs), L.sink,
                         L.recent, static_cast<int32_t>(g), static_cast<int32_t>(budget),
                         static_cast<int32_t>(capacity), slots, tokens};
  hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kSharedThreads), 0, as_stream(stream), a);
  return static_cast<int>(hipGetLastError());
}

extern "C" int oscar_shared_history(const void* query, int64_t q_s0, int64_t q_s1, int64_t q_s2,
                                    const void* history, int64_t history_bytes,
                                    const int32_t* block_tables, int64_t table_stride,
                                    int64_t table_columns, const int32_t* counts,
                                    const int32_t* units, int64_t capacity,
                                    const int32_t* unit_count, const int32_t* token_slots,
                                    int64_t n, int64_t hq, int32_t slots, float scale,
                                    const oscar_layout* layout, float* partials, float* lse,
                                    int32_t fp32_out, void* out, float* out_lse, void* stream) {
  using namespace oscar;
  if (slots < 4 || slots > kSharedSlots || capacity < 1) return OSCAR_E_SHAPE;
  AttnArgs a;
  int64_t qrows = 0;
  // The unit list stands where the task table does; lengths and query starts are in the units.
  const int st = make_attn_args(query, q_s0, q_s1, q_s2, nullptr, 0, 0, 1, nullptr, 0, 0, 1, history,
                                history_bytes, nullptr, 0, units, units, block_tables, table_stride,
                                table_columns, counts, units, unit_count, n, hq, capacity, slots, 1,
                                1, 1, scale, 0, 0, layout, partials, lse, &a, &qrows);
  if (st != OSCAR_OK || n == 0) return st;
  if (!token_slots || !out || !out_lse) return OSCAR_E_NULL;
  if (reinterpret_cast<uintptr_t>(out) % 16) return OSCAR_E_ALIGN;
  if (hq > 0x7fffffffll / n || capacity > 0x7fffffffll / a.L.kv_heads) return OSCAR_E_SHAPE;
  hipStream_t s = as_stream(stream);
  hipLaunchKernelGGL(shared_history_kernel, dim3(static_cast<unsigned>(capacity * a.L.kv_heads)),
                     dim3(kThreadsC), 0, s, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return static_cast<int>(err);
  const SharedMergeArgs m{partials, lse, token_slots, counts, out, out_lse,
                          static_cast<int32_t>(hq), slots};
  if (fp32_out)
    hipLaunchKernelGGL(shared_merge_kernel<true>, dim3(static_cast<unsigned>(n * hq)),
                       dim3(kThreads), 0, s, m);
  else
    hipLaunchKernelGGL(shared_merge_kernel<false>, dim3(static_cast<unsigned>(n * hq)),
                       dim3(kThreads), 0, s, m);
  return static_cast<int>(hipGetLastError());
}
