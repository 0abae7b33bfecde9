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
// its own. A tile is 16 rows whose positions the wavefronts of a workgroup divide
// (row_tile.h), or of many rows 128 that share the codes (chunk_tile.h). The plan kernel cuts
// every tile's positions into pieces from the whole step's lengths, so that the launch ends early on
// 256 CUs, and writes the list, once per step and before every layer's launch. Partial rows of a
// tile's pieces go to slots that the merge kernel joins by their LSEs, as many as the plan says for
// each token.
//
// What bounds it (history launch and merge of a layer, us, replayed back to back in a graph; the two
// kernels' times in a trace add up to 1 to 5 us more; unshared: the launches of history.hip and their
// merge, in a graph): a few samples of a short prompt their chain of loads, 6 of 2000 tokens 13.7 (unshared
// 19.5); 16-row tiles vector issue, the rounds of their wavefronts and the start of a unit, about half
// of its time, 32 of 32000 26.4 (38.3), three prompts of 9 samples with 4 query tokens 27.2 (48.6);
// 128-row tiles the pipeline of chunk_tile.h, 4.2 a chunk, 256 of 32500 84 to 88 (261). Which layer
// steps take it, in place of a history launch that carries more: config.shared_prefix_pays.
#include "merge.h"
#include "row_tile.h"

namespace oscar {
namespace {

constexpr int kSharedThreads = 1024;
constexpr int kSharedEntries = 4096;  // groups and requests whose counts live in LDS
constexpr int kSharedSlots = 256;     // partial rows of a row: four per lane of a merging wavefront
constexpr int kUnitWords = 8;
// Rows up to which an entry's tiles are 16 rows: always, and where the plan finds that faster for the
// step (in a graph, 32 samples of 32000 tokens, 192 rows: 26.7 us a layer against 34.4 with 128-row
// tiles, 96 of 16000: 36.6 and 40.3, 128 of 32000: 58.6 and 55.6).
constexpr int kSmallRows[2] = {48, 1024};
// A unit's time in us: its start and end, a 128-token chunk of a 128-row tile, and a round of a 16-row
// tile, in which each of the eight wavefronts takes 64 tokens (kRound chunks); what a short unit
// behind another on its CU adds, and a partial row that is written and merged.
constexpr float kUnitStart = 11.f, kTileChunk = 4.2f, kSmallRound = 3.0f, kSecond = 7.f;
constexpr float kUnitGap = 6.f;  // between two units of a CU, and a short one's uneven rounds
constexpr float kPartialRow = 5.5e-4f;
constexpr int kRound = kWavesC * 64 / kTokC;

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
  int32_t groups, max_reqs, sink, recent, g, heads, budget, capacity, slots;
  int64_t tokens;
};

__device__ __forceinline__ int tiles_of(int rows, bool small) {
  return small ? (rows + 15) / 16 : (rows + kRowsC - 1) / kRowsC;
}
__device__ __forceinline__ int chunks_of(int lo, int hi) {
  return lo < hi ? ((hi - 1) >> 7) - (lo >> 7) + 1 : 0;
}

__global__ __launch_bounds__(kSharedThreads) void shared_plan_kernel(const SharedPlanArgs a) {
  // Entries: the groups, then the requests.
  __shared__ int s_chunks[kSharedEntries], s_rows[kSharedEntries], s_start[kSharedEntries + 1];
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
      s_rows[i] = shared ? rows_of(r0, r1) : 0;
    }
  }
  __syncthreads();
  for (int r = tid; r < reqs; r += kSharedThreads) {
    s_chunks[groups + r] = chunks_of(s_own[r], s_end[r]);
    s_rows[groups + r] = rows_of(r, r + 1);
  }
  __syncthreads();
  // Tiles times chunks of either kind of tile, with the one and the other limit of small entries, and
  // the most chunks of one row's positions: a wavefront each.
  __shared__ int64_t s_sum[5];
  if (wave < 5) {
    int64_t sum = 0;
    int most = 0;
    if (wave < 4) {
      for (int e = lane; e < entries; e += kWave) {
        const bool small = s_rows[e] <= kSmallRows[wave >> 1];
        if (small == ((wave & 1) != 0))
          sum += static_cast<int64_t>(tiles_of(s_rows[e], small)) * s_chunks[e];
      }
      sum = wave_sum_i64(sum);
    } else {
      for (int r = lane; r < reqs; r += kWave)
        if (s_rows[groups + r] > 0)
          most = max(most, s_chunks[groups + r] + (s_group[r] >= 0 ? s_chunks[s_group[r]] : 0));
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) most = max(most, __shfl_xor(most, m, kWave));
      sum = most;
    }
    if (lane == 0) s_sum[wave] = sum;
  }
  __shared__ uint64_t s_best;  // the least estimate's bits, then 2 i + k
  if (tid == 0) s_best = ~0ull;
  __syncthreads();
  const int64_t sums[4] = {s_sum[0], s_sum[1], s_sum[2], s_sum[3]};
  const int most = static_cast<int>(s_sum[4]);
  // Chunks of a piece of either kind of tile, from a time that grows by half chunks: no row in more
  // than `slots` pieces (its positions are two ranges, each with one uneven piece), and neither kind
  // in more than `budget` units by the average.
  const int least = max(1, (most + a.slots - 3) / (a.slots - 2));
  int average[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    average[k] = max(least, static_cast<int>((sums[k] + a.budget - 1) / a.budget));
  auto tile_piece = [&](int k, int i) { return max(average[2 * k], i >> 1); };
  auto small_piece = [&](int k, int i) {
    const int rounds = max(1, static_cast<int>(i * (0.5f * kTileChunk / kSmallRound)));
    return (max(average[2 * k + 1], kRound * rounds) + kRound - 1) / kRound * kRound;
  };
  // The choice of least estimated time; the wavefronts estimate 16 at once, until the growing time
  // itself passes the best. Units that fit the CUs run side by side, one per CU, in the time of the
  // longest; more of them take their load and a short one's time behind another.
  const int kinds = sums[0] == sums[2] ? 1 : 2;  // no entry between the two limits
  for (int i0 = max(1, 2 * min(average[0], average[2]) - 6), end = i0 + 4096; i0 < end;
       i0 += kSharedThreads / kWave) {
    const int i = i0 + wave;
    for (int k = 0; k < kinds; ++k) {
      const int t = tile_piece(k, i), ts = small_piece(k, i);
      float tiles = 0.f, smalls = 0.f, rows = 0.f;
      const float per_t = __builtin_amdgcn_rcpf(t), per_ts = __builtin_amdgcn_rcpf(ts);
      for (int e = lane; e < entries; e += kWave) {
        const bool small = s_rows[e] <= kSmallRows[k];
        const float pieces = ceilf(s_chunks[e] * (small ? per_ts : per_t) - 1e-3f);
        const float units = tiles_of(s_rows[e], small) * pieces;
        tiles += small ? 0.f : units;
        smalls += small ? units : 0.f;
        rows += s_rows[e] * pieces;
      }
      tiles = wave_tree_sum_dpp(tiles);
      smalls = wave_tree_sum_dpp(smalls);
      rows = wave_tree_sum_dpp(rows) * a.heads;
      const float time = kUnitStart + fmaxf(tiles > 0.f ? kTileChunk * t : 0.f,
                                            smalls > 0.f ? kSmallRound / kRound * ts : 0.f);
      const float load = tiles * (kUnitStart + kTileChunk * t) + smalls * (kUnitStart + kUnitGap) +
                         sums[2 * k + 1] * (kSmallRound / kRound);
      const float estimate =
          (tiles + smalls <= a.budget ? time : fmaxf(time, load / a.budget) + kSecond) +
          kPartialRow * rows;
      if (lane == 0)
        atomicMin(reinterpret_cast<unsigned long long*>(&s_best),
                  static_cast<unsigned long long>(__float_as_uint(estimate)) << 32 | (2 * i + k));
    }
    __syncthreads();
    const float best = __uint_as_float(static_cast<uint32_t>(s_best >> 32));
    __syncthreads();
    if (kUnitStart + 0.5f * kTileChunk * (i0 + kSharedThreads / kWave) >= best) break;
  }
  const int choice = static_cast<int>(s_best & 0xffffffffu), kind = choice & 1;
  const int per = tile_piece(kind, choice >> 1), per_small = small_piece(kind, choice >> 1);
  auto small_entry = [&](int e) { return s_rows[e] <= kSmallRows[kind]; };
  auto tiles_in = [&](int e) { return tiles_of(s_rows[e], small_entry(e)); };
  auto pieces = [&](int e) { return cdiv(s_chunks[e], small_entry(e) ? per_small : per); };
  auto units_of = [&](int e) { return tiles_in(e) * pieces(e); };

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
    const int e = lo, tile_count = tiles_in(e);
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
    x.small = small_entry(e);
    a.units[u] = x;
  }
  // Eight threads per request.
  for (int r = tid >> 3; r < reqs; r += kSharedThreads / 8) {
    const int used = pieces(groups + r) + (s_group[r] >= 0 ? pieces(s_group[r]) : 0);
    for (int t = s_token[r] + (tid & 7); t < s_token[r + 1]; t += 8) a.token_slots[t] = used;
  }
  // Tokens behind the last request's hold nothing.
  for (int t = (reqs ? s_token[reqs] : 0) + tid; t < active; t += kSharedThreads)
    a.token_slots[t] = 0;
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
  // The LSEs of every slot are read beside the count of those in use, not behind it.
  float w[kSharedSlots / kWave];
#pragma unroll
  for (int i = 0; i < kSharedSlots / kWave; ++i)
    w[i] = kWave * i + lane < a.slots ? a.lse[row * a.slots + kWave * i + lane] : -INFINITY;
  const int live = a.counts[1], held = a.token_slots[token];
  const int used = token < live ? min(max(held, 0), a.slots) : 0;
  float mx = -INFINITY, den = 0.f;
#pragma unroll
  for (int i = 0; i < kSharedSlots / kWave; ++i) {
    w[i] = kWave * i + lane < used ? w[i] : -INFINITY;
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
  if (lane == 0) a.out_lse[row] = den == 0.f ? -INFINITY : mx + logf(den);  // NaN stays NaN
}

// Units that a plan may hold: a tile's pieces pass its share of the budget by less than one, for the
// tiles of either kind, of which there is one per 128 or 16 rows and one more per entry.
int64_t shared_capacity(int64_t tokens, int64_t g, int64_t groups, int64_t max_reqs,
                        int64_t budget) {
  const int64_t entries = groups + (max_reqs < tokens ? max_reqs : tokens);
  return 2 * budget + 2 * (tokens * g / kRowsC) + 2 * (tokens * g / 16) + 2 * entries;
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
                         L.recent, static_cast<int32_t>(g), L.kv_heads, static_cast<int32_t>(budget),
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
  // A launch holds fewer than 2^32 threads.
  if (hq > 0xffffffffll / kThreads / n || capacity > 0xffffffffll / kThreadsC / a.L.kv_heads)
    return OSCAR_E_SHAPE;
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
