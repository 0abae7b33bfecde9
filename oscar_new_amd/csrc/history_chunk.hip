// INT2 history branch of continuation chunks (more than 16 query tokens per request): 128
// (query, head) rows of one request and KV head per workgroup share every spread code.
//
// Reference: oscar_ascend/kernels.py:290-482 (`_attention_kernel` with IS_RAW false), split
// ranges kernels.py:368-370. Scores, masks, per-split normalization and LSE as in history.hip.
//
// The task-shaped kernel of history.hip serves the rows of four query tokens per workgroup, so
// a chunk's 2-bit codes are spread into FP4 operands once per 16 rows (a third of its vector
// instructions), a quarter of its rows are padding with six heads, and one split per request
// leaves a short chunk on a few CUs. Here eight wavefronts of 16 rows each take 128 consecutive
// rows (any number of heads, padding only in a request's last tile) and share the codes
// (chunk_tile.h).
//
// What bounds it: vector issue, and the waits of a wavefront for the others of its workgroup. A
// chunk takes a SIMD's two wavefronts 9100 cycles: their vector instructions (about 460 per
// wavefront, beside 64 MFMAs) hold its issue for 58 % of them, the matrix pipe is busy for 45 %, and
// a wavefront spends 38 % of its cycles at an s_waitcnt or the barrier (counters, 2048 tokens x 6
// heads over 32768). That chunk: 654 us (task-shaped kernel, one split) -> 415 us with five splits;
// 389 tokens over 20011 beside 15 decodes: 254 -> 102 us. Which steps take it:
// config.chunk_kernel_pays.
#include "chunk_tile.h"

namespace oscar {
namespace {

// Tile `x` of the step: the tiles of 128 rows of all requests, in task order. A tile starts in
// the task whose rows hold its first row (a task holds at most 32 rows, so at most one start).
// Every thread calls it; false past the last tile.
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int programs, int x, ChunkLds& lds,
                                          int& req, int& tile) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int count = max(min(a.task_count[0], programs), 0);
  const int task_rows = a.qt * a.g;
  if (threadIdx.x == 0) lds.found[0] = -1;
  __syncthreads();
  int before = 0;
  for (int c0 = 0; c0 < count && before <= x; c0 += kThreadsC) {
    const int i = c0 + static_cast<int>(threadIdx.x);
    int r = -1, b = 0;
    bool start = false;
    if (i < count) {
      r = a.tasks[2 * i];
      const int row0 = a.tasks[2 * i + 1] * a.g;
      b = (row0 + kRowsC - 1) / kRowsC;
      start = b * kRowsC < row0 + task_rows;
    }
    const uint64_t mask = __ballot(start);
    if (lane == 0) lds.count[wave] = __popcll(mask);
    __syncthreads();
    int at = before + __popcll(mask & ((1ull << lane) - 1));
    int all = 0;
#pragma unroll
    for (int w = 0; w < kWavesC; ++w) {
      at += w < wave ? lds.count[w] : 0;
      all += lds.count[w];
    }
    if (start && at == x) {
      lds.found[0] = r;
      lds.found[1] = b;
    }
    before += all;
    __syncthreads();  // counts are read, the tile is published
  }
  req = uniform(lds.found[0]);
  tile = uniform(lds.found[1]);
  return req >= 0;
}

__global__ __launch_bounds__(kThreadsC, 2) void history_chunk_kernel(const AttnArgs a,
                                                                     int32_t programs) {
  __shared__ ChunkLds lds;
  Task t;
  int tile;
  // Workgroup ((tile, kv head), split): the tiles that exist dispatch first. Their bound grows with
  // the engine's request capacity, and a workgroup past the last tile, too, holds a whole CU while
  // it looks for its tile; with the tiles varying fastest these came between the others (64 tokens
  // over 16000, capacity 256, 16 splits: 94 us, this order 49; 300 tokens and three decodes over
  // 30000, 11 splits: 182 and 108).
  const int unit = static_cast<int>(blockIdx.x) / a.splits, h = a.L.kv_heads;
  const int split = static_cast<int>(blockIdx.x) - unit * a.splits, head = unit % h;
  if (!find_tile(a, programs, unit / h, lds, t.req, tile)) return;
  t.qoff = 0;
  t.qstart = a.qstarts[t.req];
  t.qlen = min(a.qstarts[t.req + 1], a.counts[1]) - t.qstart;
  t.prefix = a.seq_lens[t.req] - t.qlen;
  t.sink_len = min(a.L.sink, t.prefix);
  t.recent_begin = max(t.sink_len, t.prefix - a.L.recent);
  const int rows = t.qlen * a.g;  // rows of this request and KV head
  const int row_base = tile * kRowsC;
  if (row_base >= rows) return;
  int begin, end;
  split_range(t.recent_begin - t.sink_len, a.block_n, a.splits, split, begin, end);
  const int p_lo = max(t.sink_len + begin, 0), p_hi = t.sink_len + end;
  chunk_tile<false>(a, t, head, rows, row_base, p_lo, p_hi, split, lds);
}

}  // namespace

// Grid x of the launch: at least the tiles find_tile can find. A request of q query tokens holds
// ceil(q / qt) task rows of qt g <= 32 rows, x rows in all, and starts ceil(x / 128) <= (x + 127) /
// 128 tiles; over at most `reqs` requests of n tokens and `programs` task rows, x sums to at most
// the smaller of programs qt g and (n + (qt - 1) reqs) g. A task row starts at most one tile.
int64_t history_chunk_tiles(int64_t n, int64_t max_reqs, int64_t programs, int64_t qt, int64_t g) {
  const int64_t reqs = n < max_reqs ? n : max_reqs;
  const int64_t by_tasks = programs * qt * g, by_tokens = (n + (qt - 1) * reqs) * g;
  const int64_t rows = by_tasks < by_tokens ? by_tasks : by_tokens;
  const int64_t tiles = (rows + (kRowsC - 1) * reqs) / kRowsC;
  return tiles < programs ? tiles : programs;
}

}  // namespace oscar

extern "C" int64_t oscar_history_chunk_tiles(int64_t n, int64_t max_reqs, int64_t programs,
                                             int32_t query_tile, int32_t group) {
  return oscar::history_chunk_tiles(n, max_reqs, programs, query_tile, group);
}

extern "C" int oscar_history_chunk(
    const void* query, int64_t q_s0, int64_t q_s1, int64_t q_s2, const void* history,
    int64_t history_bytes, const int32_t* qstarts, const int32_t* seq_lens,
    const int32_t* block_tables, int64_t table_stride, int64_t table_columns,
    const int32_t* counts, const int32_t* tasks, const int32_t* task_count, int64_t n, int64_t hq,
    int64_t programs, int64_t max_reqs, int32_t splits, int32_t block_n, int32_t query_tile,
    float scale, const oscar_layout* layout, float* partials, float* lse, void* stream) {
  using namespace oscar;
  if (max_reqs < 1 || max_reqs > 0x7fffffffll) return OSCAR_E_SHAPE;
  AttnArgs a;
  int64_t qrows = 0;
  const int st = make_attn_args(query, q_s0, q_s1, q_s2, nullptr, 0, 0, 1, nullptr, 0, 0, 1,
                                history, history_bytes, nullptr, 0, qstarts, seq_lens,
                                block_tables, table_stride, table_columns, counts, tasks,
                                task_count, n, hq, programs, splits, block_n, query_tile, 0, scale,
                                0, 0, layout, partials, lse, &a, &qrows);
  if (st != OSCAR_OK || n == 0) return st;
  const int64_t tiles = history_chunk_tiles(n, max_reqs, programs, query_tile, a.g);
  if (tiles * a.L.kv_heads > 0x7fffffffll / splits) return OSCAR_E_SHAPE;
  const dim3 grid(static_cast<unsigned>(tiles * a.L.kv_heads * splits));
  hipLaunchKernelGGL(history_chunk_kernel, grid, dim3(kThreadsC), 0, as_stream(stream), a,
                     static_cast<int32_t>(programs));
  return static_cast<int>(hipGetLastError());
}
