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
// Units. A step's work is (row tile, position range) units of the 128-row tile of chunk_tile.h:
// the group's rows against [sink, E) through its first member's pages, and each request's own rows
// against [E, recent_begin) through its own. The plan kernel cuts every tile's positions into pieces
// of about T chunks, T from the whole step's lengths so that the units fill the CUs once, and writes
// the list; it runs once per step, before every layer's launch. Partial rows of a tile's pieces go to
// slots that the merge kernel joins by their LSEs, as many as the plan says for each token.
#include "chunk_tile.h"
#include "merge.h"

namespace oscar {
namespace {

constexpr int kSharedThreads = 1024;
constexpr int kSharedEntries = 8192;  // groups and requests whose counts live in LDS
constexpr int kSharedSlots = 64;      // partial rows of a row: one per lane of the merging wavefront
constexpr int kUnitWords = 8;

// A unit: rows [row_base, row_end) of tokens token0 .. (row r is token token0 + r / g), positions
// [p_lo, p_hi) through block-table row req, partials to `slot`.
struct Unit {
  int32_t req, token0, row_end, row_base, p_lo, p_hi, slot, reserved;
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

// Sum and maximum over the workgroup (every thread gets both).
__device__ __forceinline__ void plan_reduce(int64_t& sum, int& most) {
  __shared__ int64_t s_sum[kSharedThreads / kWave];
  __shared__ int s_most[kSharedThreads / kWave];
  sum = wave_sum_i64(sum);
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) most = max(most, __shfl_xor(most, m, kWave));
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    s_sum[wave] = sum;
    s_most[wave] = most;
  }
  __syncthreads();
  sum = 0;
  most = 0;
#pragma unroll
  for (int w = 0; w < kSharedThreads / kWave; ++w) {
    sum += s_sum[w];
    most = max(most, s_most[w]);
  }
}

__device__ __forceinline__ int chunks_of(int lo, int hi) {
  return lo < hi ? ((hi - 1) >> 7) - (lo >> 7) + 1 : 0;
}

__global__ __launch_bounds__(kSharedThreads) void shared_plan_kernel(const SharedPlanArgs a) {
  // Entries: the groups, then the requests.
  __shared__ int s_chunks[kSharedEntries], s_tiles[kSharedEntries], s_start[kSharedEntries + 1];
  __shared__ int s_own[kSharedEntries];  // first history position of a request's own part
  __shared__ int s_wave[kSharedThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int reqs = max(min(a.counts[0], a.max_reqs), 0);
  const int active = static_cast<int>(
      min(static_cast<int64_t>(max(a.counts[1], 0)), a.tokens));
  // Starts that descend are no partition: then nothing is shared.
  bool bad = false;
  for (int i = tid; i < a.groups; i += kSharedThreads)
    bad |= a.group_starts[i + 1] < a.group_starts[i];
  const int groups = __syncthreads_or(bad) ? 0 : a.groups;
  const int entries = groups + reqs;

  struct Span {
    int prefix, sink_len, recent, rows;
  };
  auto token = [&](int r) { return min(max(a.qstarts[r], 0), active); };
  auto span = [&](int r) {
    Span s;
    const int qlen = max(token(r + 1) - token(r), 0);
    s.prefix = a.seq_lens[r] - qlen;
    s.sink_len = max(min(a.sink, s.prefix), 0);
    s.recent = max(s.sink_len, s.prefix - a.recent);
    s.rows = qlen * a.g;
    return s;
  };
  auto clip = [&](int r) { return min(max(r, 0), reqs); };

  for (int r = tid; r < reqs; r += kSharedThreads) s_own[r] = -1;
  __syncthreads();
  for (int i = wave; i < groups; i += kSharedThreads / kWave) {
    const int r0 = clip(a.group_starts[i]), r1 = clip(a.group_starts[i + 1]);
    int end = a.prefix_tokens[i];
    for (int r = r0 + lane; r < r1; r += kWave) end = min(end, span(r).recent);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) end = min(end, __shfl_xor(end, m, kWave));
    end &= ~(kTokC - 1);
    // Past the sink every member's recent part starts behind it, so all begin at `sink`.
    const bool shared = r1 - r0 > 1 && end > a.sink;
    if (shared)
      for (int r = r0 + lane; r < r1; r += kWave) s_own[r] = end;
    if (lane == 0) {
      const int rows = shared ? max(token(r1) - token(r0), 0) * a.g : 0;
      s_chunks[i] = shared ? chunks_of(a.sink, end) : 0;
      s_tiles[i] = (rows + kRowsC - 1) / kRowsC;
    }
  }
  __syncthreads();
  int64_t work = 0;
  int most = 0;  // chunks of one row's positions
  for (int r = tid; r < reqs; r += kSharedThreads) {
    const Span s = span(r);
    const int own = s_own[r];
    const int lo = own >= 0 ? own : s.sink_len;
    s_own[r] = lo;
    s_chunks[groups + r] = chunks_of(lo, s.recent);
    s_tiles[groups + r] = (s.rows + kRowsC - 1) / kRowsC;
    if (s.rows > 0)
      most = max(most, s_chunks[groups + r] + (lo > a.sink ? chunks_of(a.sink, lo) : 0));
  }
  __syncthreads();
  int64_t tiles = 0;
  for (int e = tid; e < entries; e += kSharedThreads) {
    work += static_cast<int64_t>(s_tiles[e]) * s_chunks[e];
    tiles += s_chunks[e] ? s_tiles[e] : 0;
  }
  int none = 0;
  plan_reduce(work, most);
  plan_reduce(tiles, none);
  // Chunks per unit: at most about `budget` units, and no row in more than `slots` pieces (a row's
  // positions are two ranges, each with one uneven piece).
  int per = static_cast<int>(max(static_cast<int64_t>(1), (work + a.budget - 1) / a.budget));
  per = max(per, (most + a.slots - 3) / (a.slots - 2));
  auto count_units = [&](int t) {
    int64_t units = 0;
    for (int e = tid; e < entries; e += kSharedThreads)
      units += static_cast<int64_t>(s_tiles[e]) * cdiv(s_chunks[e], t);
    int unused = 0;
    plan_reduce(units, unused);
    return units;
  };
  // Uneven pieces may pass the budget: a second round of workgroups costs more than longer units.
  for (int i = 0; i < 8 && tiles < a.budget && count_units(per) > a.budget; ++i) ++per;

  // Exclusive scan of the entries' units, eight entries a thread.
  constexpr int kPer = kSharedEntries / kSharedThreads;
  int mine = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int e = kPer * tid + k;
    if (e < entries) mine += s_tiles[e] * cdiv(s_chunks[e], per);
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
    at += s_tiles[e] * cdiv(s_chunks[e], per);
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
    const int e = lo, tile_count = s_tiles[e], pieces = cdiv(s_chunks[e], per);
    const int local = u - s_start[e], piece = local / tile_count, tile = local - piece * tile_count;
    Unit x;
    int begin, end, rows;
    if (e < groups) {
      const int r0 = clip(a.group_starts[e]), r1 = clip(a.group_starts[e + 1]);
      x.req = r0;
      x.token0 = token(r0);
      rows = max(token(r1) - x.token0, 0) * a.g;
      begin = a.sink;
      end = s_own[r0];
      x.slot = piece;
    } else {
      const int r = e - groups;
      const Span s = span(r);
      x.req = r;
      x.token0 = token(r);
      rows = s.rows;
      begin = s_own[r];
      end = s.recent;
      x.slot = piece + (begin > a.sink ? cdiv(chunks_of(a.sink, begin), per) : 0);
    }
    // Tiles of equal numbers of 16-row groups, pieces of equal numbers of chunks.
    const int share = ((rows + 15) / 16 + tile_count - 1) / tile_count * 16;
    x.row_base = tile * share;
    x.row_end = min(x.row_base + share, rows);
    const int c0 = (begin >> 7) + static_cast<int>(static_cast<int64_t>(piece) * s_chunks[e] / pieces);
    const int c1 =
        (begin >> 7) + static_cast<int>(static_cast<int64_t>(piece + 1) * s_chunks[e] / pieces);
    x.p_lo = max(begin, c0 << 7);
    x.p_hi = min(end, c1 << 7);
    x.reserved = 0;
    a.units[u] = x;
  }
  for (int r = wave; r < reqs; r += kSharedThreads / kWave) {
    const int own = s_own[r];
    const int used = cdiv(s_chunks[groups + r], per) +
                     (own > a.sink ? cdiv(chunks_of(a.sink, own), per) : 0);
    const int t1 = token(r + 1);
    for (int t = token(r) + lane; t < t1; t += kWave) a.token_slots[t] = used;
  }
}

__global__ __launch_bounds__(kThreadsC, 2) void shared_history_kernel(const AttnArgs a) {
  __shared__ ChunkLds lds;
  const int heads = a.L.kv_heads;
  const int index = static_cast<int>(blockIdx.x) / heads;
  if (index >= a.task_count[0]) return;
  const Unit u = reinterpret_cast<const Unit*>(a.tasks)[index];
  if (u.row_base >= u.row_end) return;
  Task t{};
  t.req = u.req;
  t.qstart = u.token0;
  chunk_tile(a, t, static_cast<int>(blockIdx.x) - index * heads, u.row_end, u.row_base, u.p_lo,
             u.p_hi, u.slot, lds);
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

// One workgroup per row: every wavefront holds all LSEs (one per lane) and adds every fourth slot,
// eight loads in flight; the four sums are added in wavefront order.
template <bool kFloat>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(const SharedMergeArgs a) {
  __shared__ f32x4 s_sum[3][kWave];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t row = blockIdx.x, token = row / a.hq;
  const int used = token < a.counts[1] ? min(max(a.token_slots[token], 0), a.slots) : 0;
  const float l = lane < used ? a.lse[row * a.slots + lane] : -INFINITY;
  const float mx = wave_max_dpp(l);
  const float w = l == -INFINITY ? 0.f : expf(l - mx);
  const float den = wave_tree_sum_dpp(w);
  const f32x4* part = reinterpret_cast<const f32x4*>(a.partials + row * a.slots * kHeadDim) + lane;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = wave; s0 < used; s0 += 32) {
    f32x4 v[8];
    float ws[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = s0 + 4 * k;
      v[k] = s < used ? part[static_cast<int64_t>(s) * (kHeadDim / 4)] : f32x4{0.f, 0.f, 0.f, 0.f};
      ws[k] = lane_value(w, min(s, kWave - 1));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s0 + 4 * k < used)
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

}  // namespace
}  // namespace oscar

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
  const int64_t reqs = max_reqs < tokens ? max_reqs : tokens;
  // A tile per 128 rows and one more per group or request, a piece more than its share per tile.
  if (capacity < budget + 2 * (tokens * g / kRowsC) + groups + reqs || capacity > 0x7fffffffll)
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
