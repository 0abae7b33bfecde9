// Pages of a cache: which ones are free, requests that continue a parent's tokens (fork), and live
// pages moved to the pool's start (compact), in the caches of every layer of a model at once.
//
// No reference counterpart (the reference refuses page copies, oscar_ascend/backend.py:30-38: a
// request's BF16 window lies in the V stripe of its first page, so that page has one owner). The
// other pages hold INT2 records that are never written again once full, and several requests may
// map them: a fork shares a parent's full pages and copies the first page, with the window, and an
// unfinished last page.
//
// Copies are bounded by memory: 16 bytes a lane, only live records (a request's last page ends
// inside) and live window rows. 96 forks in six layers, 356 MB read and written: 75.7 us, 4.7 TB/s of
// the 5.0 that a large copy reaches; 8 forks of one parent in 16 layers 16.1 us (77 MB, the parent's
// rows from the caches); 174 MB of moved pages 34.2 us, about 45 where nothing of them is in the
// last-level cache. The bookkeeping is a few integers per page and runs in one workgroup, or in every
// workgroup of a fork again, so that a call is one or two launches. It grows with the pool (us, free
// pages and a compaction in which nothing moves): 3.7 and 7.9 at 100 pages and 8 requests, 6.8 and 10.9
// at 1000 and 60, 16 and 23 at 4000 and 200, 58 and 75 at 16000 and 800.
#include "common.h"

namespace oscar {
namespace {

struct Stripes {
  uint8_t* history;
  uint8_t* window;
};

struct PoolArgs {
  const Stripes* layers;
  int32_t layer_count, num_pages;
  Layout L;
};

constexpr int kUnitBytes = 32 << 10;  // bytes of one page copy that a workgroup moves

// ---------------------------------------------------------------- copying a page

// `bytes` from src + lo .. to dst + lo .., the part that lies in [from, to) of a run that starts at
// `at`; everything is a multiple of 16 (records are 160 bytes, window rows 512).
__device__ __forceinline__ void copy_run(const uint8_t* src, uint8_t* dst, int64_t at, int64_t bytes,
                                         int64_t from, int64_t to) {
  const int64_t lo = max(from - at, static_cast<int64_t>(0)), hi = min(to - at, bytes);
  const u32x4* s = reinterpret_cast<const u32x4*>(src);
  u32x4* d = reinterpret_cast<u32x4*>(dst);
  int64_t i = lo / 16 + threadIdx.x;
  const int64_t end = hi / 16;
  for (; i + 3 * kThreads < end; i += 4 * kThreads) {
    u32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = s[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < 4; ++k) d[i + k * kThreads] = v[k];
  }
  for (; i < end; i += kThreads) d[i] = s[i];
}

// What a copied page holds: `slots` records and the window rows of a request of `length` tokens
// (0: not a first page).
__device__ __forceinline__ int64_t record_bytes(const Layout& L, int slots) {
  return static_cast<int64_t>(slots) * L.kv_heads * L.slot_bytes;
}
__device__ __forceinline__ int64_t window_row(const Layout& L) {
  return static_cast<int64_t>(L.kv_heads) * L.head_dim * 4;  // K and V rows of one position
}
__device__ __forceinline__ int64_t page_copy_bytes(const Layout& L, int slots, int length) {
  return record_bytes(L, slots) + min(length, L.sink + L.ring) * window_row(L);
}

// Bytes [from, to) of the copy of one layer's page: records, sink rows, then the ring rows of
// positions max(sink, length - ring) .. length - 1 (position p at row sink + p % ring).
__device__ __forceinline__ void copy_page(const Layout& L, const Stripes& layer, int src, int dst,
                                          int slots, int length, int64_t from, int64_t to) {
  const int64_t ps = src * L.page_bytes, pd = dst * L.page_bytes, row = window_row(L);
  const int64_t records = record_bytes(L, slots);
  copy_run(layer.history + ps, layer.history + pd, 0, records, from, to);
  if (length <= 0 || to <= records) return;
  const uint8_t* ws = layer.window + ps;
  uint8_t* wd = layer.window + pd;
  const int sinks = min(length, L.sink);
  int64_t at = records;
  copy_run(ws, wd, at, sinks * row, from, to);
  at += sinks * row;
  const int count = min(length - sinks, L.ring);
  const int start = count == L.ring ? 0 : L.sink % L.ring;  // a ring not yet full starts at `sink`
  const int first = min(count, L.ring - start);
  copy_run(ws + (L.sink + start) * row, wd + (L.sink + start) * row, at, first * row, from, to);
  at += first * row;
  copy_run(ws + L.sink * row, wd + L.sink * row, at, (count - first) * row, from, to);
}

// ---------------------------------------------------------------- which pages are in use

// One workgroup: used[p] = most tokens of page p that a live request holds, owner[p] = length of
// the request whose first page it is (0: none; null: not asked for). The counters are written and
// read where atomics act (the device's point of coherence), each phase complete before the next.
constexpr int kPlanThreads = 1024;

struct TableArgs {
  const int32_t* table;
  int64_t stride, columns;
  const int32_t* seq_lens;
  const int32_t* counts;
  int64_t rows;
};

__device__ __forceinline__ int32_t load_shared_i32(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared_i32(int32_t* p, int32_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void phase_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

__device__ void mark_pages(const TableArgs& t, const Layout& L, int num_pages, int32_t* used,
                           int32_t* owner) {
  for (int p = threadIdx.x; p < num_pages; p += kPlanThreads) {
    store_shared_i32(used + p, 0);
    if (owner) store_shared_i32(owner + p, 0);
  }
  phase_barrier();
  const int live = static_cast<int>(min(static_cast<int64_t>(max(t.counts[0], 0)), t.rows));
  const int lane = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < live; r += kPlanThreads / kWave) {
    const int length = t.seq_lens[r];
    const int pages = length > 0 ? (length - 1) / L.bp + 1 : 0;
    for (int j = lane; j < pages; j += kWave) {
      const int64_t c = static_cast<int64_t>(j) * L.bpp;
      if (c >= t.columns) break;
      const int block = t.table[r * t.stride + c];
      const int page = block >= 0 ? block / L.bpp : -1;
      if (page < 0 || page >= num_pages) continue;
      atomicMax(used + page, min(length - j * L.bp, L.bp));
      if (owner && j == 0) atomicMax(owner + page, length);
    }
  }
  phase_barrier();
}

// Exclusive scan of one value per thread over the workgroup, and the total.
__device__ __forceinline__ int plan_scan(int v, int& total) {
  __shared__ int s_wave[kPlanThreads / kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int y = __shfl_up(incl, d, kWave);
    incl += lane >= d ? y : 0;
  }
  if (lane == kWave - 1) s_wave[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    before += w < wave ? s_wave[w] : 0;
    total += s_wave[w];
  }
  __syncthreads();
  return before + incl - v;
}

// Free pages in ascending order, -1 behind them, and their number.
__global__ __launch_bounds__(kPlanThreads) void free_pages_kernel(const TableArgs t, const Layout L,
                                                                  int32_t num_pages, int32_t* used,
                                                                  int32_t* pages, int32_t* count) {
  mark_pages(t, L, num_pages, used, nullptr);
  int base = 0;
  for (int p0 = 0; p0 < num_pages; p0 += kPlanThreads) {
    const int p = p0 + static_cast<int>(threadIdx.x);
    const bool free = p < num_pages && load_shared_i32(used + p) == 0;
    int found;
    const int at = base + plan_scan(free ? 1 : 0, found);
    if (free) pages[at] = p;
    base += found;
  }
  for (int i = base + threadIdx.x; i < num_pages; i += kPlanThreads) pages[i] = -1;
  if (threadIdx.x == 0) count[0] = base;
}

// ---------------------------------------------------------------- fork

constexpr int64_t kMaxForks = 4096;  // every workgroup looks through the call's lists

struct ForkArgs {
  PoolArgs pool;
  int32_t* table;
  int64_t stride, columns, rows;
  int32_t* seq_lens;
  const int32_t* parents;
  const int32_t* children;
  const int32_t* fresh;  // [forks][2]
  int32_t* status;
  int32_t forks, units;  // units: workgroups per (fork, layer)
};

// Workgroup (unit, layer, fork). Every workgroup of a fork checks it by itself, in the same way:
// a row that this call writes (a child) is never read as a parent by a fork that is carried out.
__global__ __launch_bounds__(kThreads) void fork_kernel(const ForkArgs a) {
  const Layout& L = a.pool.L;
  const int f = blockIdx.z, tid = threadIdx.x;
  const int parent = a.parents[f], child = a.children[f];
  const int p0 = a.fresh[2 * f], p1 = a.fresh[2 * f + 1];
  bool bad = parent < 0 || parent >= a.rows || child < 0 || child >= a.rows;
  const int length = bad ? 0 : max(a.seq_lens[parent], 0);
  const int pages = length > 0 ? (length - 1) / L.bp + 1 : 0;
  const int tail = length - (pages - 1) * L.bp;
  const bool first = pages > 0, second = pages > 1 && tail < L.bp;
  bad |= length > 0 && (length - 1) / L.bk >= a.columns;  // a block of tokens without a column
  bad |= first && (p0 < 0 || p0 >= a.pool.num_pages);
  bad |= second && (p1 < 0 || p1 >= a.pool.num_pages || p1 == p0);
  for (int i = tid; i < a.forks; i += kThreads) {
    const int c = a.children[i];
    bad |= c == parent || (i < f && c == child);
    if (i < f) {
      const int x = a.fresh[2 * i], y = a.fresh[2 * i + 1];
      bad |= first && (x == p0 || y == p0);
      bad |= second && (x == p1 || y == p1);
    }
  }
  const int32_t* row = a.table + static_cast<int64_t>(parent) * a.stride;
  int src_first = 0, src_last = 0;
  if (!__syncthreads_or(bad)) {
    for (int j = tid; j < pages; j += kThreads) {
      const int block = row[static_cast<int64_t>(j) * L.bpp];
      const int page = block >= 0 ? block / L.bpp : -1;
      bad |= page < 0 || page >= a.pool.num_pages || (first && page == p0) ||
             (second && page == p1);
    }
    if (first) {
      src_first = row[0] / L.bpp;
      src_last = row[static_cast<int64_t>(pages - 1) * L.bpp] / L.bpp;
    }
  }
  const bool refused = __syncthreads_or(bad);
  const bool lead = blockIdx.x == 0 && blockIdx.y == 0;
  if (lead && tid == 0) a.status[f] = refused ? 0 : 1;
  if (refused) return;
  if (lead) {
    int32_t* out = a.table + static_cast<int64_t>(child) * a.stride;
    // The last page's blocks behind the tokens may have no columns.
    const int columns = static_cast<int>(min(static_cast<int64_t>(pages) * L.bpp, a.columns));
    for (int c = tid; c < columns; c += kThreads) {
      const int j = c / L.bpp, b = c - j * L.bpp;
      out[c] = j == 0 ? p0 * L.bpp + b
                      : (second && j == pages - 1 ? p1 * L.bpp + b : row[c]);
    }
    if (tid == 0) a.seq_lens[child] = length;
  }
  if (!first) return;
  const Stripes layer = a.pool.layers[blockIdx.y];
  const int64_t from = static_cast<int64_t>(blockIdx.x) * kUnitBytes, to = from + kUnitBytes;
  const int slots = min(length, L.bp);
  const int64_t all = page_copy_bytes(L, slots, length);
  if (from < all) copy_page(L, layer, src_first, p0, slots, length, from, to);
  if (second && to > all)
    copy_page(L, layer, src_last, p1, tail, 0, max(from - all, static_cast<int64_t>(0)), to - all);
}

// ---------------------------------------------------------------- compaction

struct CompactArgs {
  PoolArgs pool;
  TableArgs t;
  int32_t* new_table;  // [rows][columns]
  int32_t* live;       // [1]
  int32_t* used;       // scratch: num_pages each
  int32_t* owner;
  int32_t* place;  // new page of each page
  int32_t* moves;  // the pages that move, ascending
  int32_t* count;  // [1] number of moves
};

// One workgroup: pages below the number of live pages stay; the k-th live page above moves to the
// k-th free page below.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(const CompactArgs a) {
  const int n = a.pool.num_pages;
  mark_pages(a.t, a.pool.L, n, a.used, a.owner);
  int live = 0;
  for (int p = threadIdx.x; p < n; p += kPlanThreads) live += load_shared_i32(a.used + p) > 0;
  int total;
  plan_scan(live, total);
  int32_t* holes = a.moves + n;  // the free pages below `total`, ascending
  int found_holes = 0, found_moves = 0;
  for (int p0 = 0; p0 < n; p0 += kPlanThreads) {
    const int p = p0 + static_cast<int>(threadIdx.x);
    const bool in = p < n, used = in && load_shared_i32(a.used + p) > 0;
    const bool hole = in && !used && p < total, move = used && p >= total;
    int step;
    const int h = found_holes + plan_scan(hole ? 1 : 0, step);
    found_holes += step;
    const int m = found_moves + plan_scan(move ? 1 : 0, step);
    found_moves += step;
    if (hole) store_shared_i32(holes + h, p);
    if (move) store_shared_i32(a.moves + m, p);
    if (in && !move) a.place[p] = p;
  }
  phase_barrier();
  for (int m = threadIdx.x; m < found_moves; m += kPlanThreads)
    a.place[load_shared_i32(a.moves + m)] = load_shared_i32(holes + m);
  if (threadIdx.x == 0) {
    a.live[0] = total;
    a.count[0] = found_moves;
  }
}

// Persistent workgroups: units of (move, layer, 32 KB), then rows of the new table.
__global__ __launch_bounds__(kThreads) void compact_move_kernel(const CompactArgs a, int32_t units) {
  const Layout& L = a.pool.L;
  const int64_t work = static_cast<int64_t>(a.count[0]) * a.pool.layer_count * units;
  for (int64_t i = blockIdx.x; i < work; i += gridDim.x) {
    const int64_t pair = i / units;
    const int64_t from = (i - pair * units) * kUnitBytes;
    const int move = static_cast<int>(pair / a.pool.layer_count);
    const int layer = static_cast<int>(pair - static_cast<int64_t>(move) * a.pool.layer_count);
    const int src = a.moves[move], slots = a.used[src], length = a.owner[src];
    if (from >= page_copy_bytes(L, slots, length)) continue;
    copy_page(L, a.pool.layers[layer], src, a.place[src], slots, length, from, from + kUnitBytes);
  }
  const int live = static_cast<int>(min(static_cast<int64_t>(max(a.t.counts[0], 0)), a.t.rows));
  for (int64_t r = blockIdx.x; r < a.t.rows; r += gridDim.x) {
    const int length = r < live ? a.t.seq_lens[r] : 0;
    const int64_t held = static_cast<int64_t>(length > 0 ? (length - 1) / L.bp + 1 : 0) * L.bpp;
    for (int64_t c = threadIdx.x; c < a.t.columns; c += kThreads) {
      int block = a.t.table[r * a.t.stride + c];
      const int page = block >= 0 ? block / L.bpp : -1;
      if (c < held) {
        if (page >= 0 && page < a.pool.num_pages) block += (a.place[page] - page) * L.bpp;
      } else if (r < live) {
        block = -1;  // a free page, in which another row's may lie now
      }
      a.new_table[r * a.t.columns + c] = block;
    }
  }
}

int make_pool(const void* stripes, int64_t layers, int64_t num_pages, const oscar_layout* layout,
              PoolArgs* out) {
  const int st = make_layout(layout, &out->L);
  if (st != OSCAR_OK) return st;
  if (layers <= 0 || layers > 65535 || num_pages <= 0) return OSCAR_E_SHAPE;
  if (num_pages > 0x7fffffffll / out->L.bpp) return OSCAR_E_SHAPE;
  if (!stripes) return OSCAR_E_NULL;
  out->layers = static_cast<const Stripes*>(stripes);
  out->layer_count = static_cast<int32_t>(layers);
  out->num_pages = static_cast<int32_t>(num_pages);
  return OSCAR_OK;
}

int make_table(const int32_t* table, int64_t stride, int64_t columns, int64_t rows,
               const int32_t* seq_lens, const int32_t* counts, TableArgs* out) {
  if (rows <= 0 || columns <= 0 || stride < columns || rows > 0x7fffffffll ||
      columns > 0x7fffffffll)
    return OSCAR_E_SHAPE;
  if (!table || !seq_lens || !counts) return OSCAR_E_NULL;
  *out = {table, stride, columns, seq_lens, counts, rows};
  return OSCAR_OK;
}

// Most bytes of one page copy: every record, and every window row of a first page.
int64_t most_bytes(const Layout& L) {
  return (static_cast<int64_t>(L.bp) * L.slot_bytes +
          static_cast<int64_t>(L.sink + L.ring) * L.head_dim * 4) * L.kv_heads;
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_free_pages(int64_t num_pages, const int32_t* table, int64_t table_stride,
                                int64_t table_columns, int64_t rows, const int32_t* seq_lens,
                                const int32_t* counts, const oscar_layout* layout, int32_t* used,
                                int32_t* pages, int32_t* count, void* stream) {
  using namespace oscar;
  Layout L;
  int st = make_layout(layout, &L);
  if (st != OSCAR_OK) return st;
  if (num_pages <= 0 || num_pages > 0x7fffffffll / L.bpp) return OSCAR_E_SHAPE;
  TableArgs t;
  st = make_table(table, table_stride, table_columns, rows, seq_lens, counts, &t);
  if (st != OSCAR_OK) return st;
  if (!used || !pages || !count) return OSCAR_E_NULL;
  hipLaunchKernelGGL(free_pages_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), t, L,
                     static_cast<int32_t>(num_pages), used, pages, count);
  return static_cast<int>(hipGetLastError());
}

extern "C" int oscar_fork_requests(const void* stripes, int64_t layers, int64_t num_pages,
                                   int32_t* table, int64_t table_stride, int64_t table_columns,
                                   int64_t rows, int32_t* seq_lens, const int32_t* parents,
                                   const int32_t* children, const int32_t* fresh, int64_t forks,
                                   const oscar_layout* layout, int32_t* status, void* stream) {
  using namespace oscar;
  ForkArgs a;
  const int st = make_pool(stripes, layers, num_pages, layout, &a.pool);
  if (st != OSCAR_OK) return st;
  if (rows <= 0 || rows > 0x7fffffffll || table_columns <= 0 || table_columns > 0x7fffffffll ||
      table_stride < table_columns || forks < 0 || forks > kMaxForks)
    return OSCAR_E_SHAPE;
  if (forks == 0) return OSCAR_OK;
  if (!table || !seq_lens || !parents || !children || !fresh || !status) return OSCAR_E_NULL;
  a.table = table;
  a.stride = table_stride;
  a.columns = table_columns;
  a.rows = rows;
  a.seq_lens = seq_lens;
  a.parents = parents;
  a.children = children;
  a.fresh = fresh;
  a.status = status;
  a.forks = static_cast<int32_t>(forks);
  // The first page's bytes and an unfinished last page's.
  const int64_t most = most_bytes(a.pool.L) +
                       static_cast<int64_t>(a.pool.L.bp) * a.pool.L.kv_heads * a.pool.L.slot_bytes;
  a.units = static_cast<int32_t>((most + kUnitBytes - 1) / kUnitBytes);
  hipLaunchKernelGGL(fork_kernel, dim3(static_cast<unsigned>(a.units),
                                       static_cast<unsigned>(layers), static_cast<unsigned>(forks)),
                     dim3(kThreads), 0, as_stream(stream), a);
  return static_cast<int>(hipGetLastError());
}

extern "C" int oscar_compact_pages(const void* stripes, int64_t layers, int64_t num_pages,
                                   const int32_t* table, int64_t table_stride,
                                   int64_t table_columns, int64_t rows, const int32_t* seq_lens,
                                   const int32_t* counts, const oscar_layout* layout,
                                   int32_t* scratch, int32_t* new_table, int32_t* live,
                                   void* stream) {
  using namespace oscar;
  CompactArgs a;
  int st = make_pool(stripes, layers, num_pages, layout, &a.pool);
  if (st != OSCAR_OK) return st;
  st = make_table(table, table_stride, table_columns, rows, seq_lens, counts, &a.t);
  if (st != OSCAR_OK) return st;
  if (!scratch || !new_table || !live) return OSCAR_E_NULL;
  a.used = scratch;
  a.owner = scratch + num_pages;
  a.place = scratch + 2 * num_pages;
  a.moves = scratch + 3 * num_pages;  // and the free pages behind them
  a.count = scratch + 5 * num_pages;
  a.new_table = new_table;
  a.live = live;
  hipStream_t s = as_stream(stream);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return static_cast<int>(err);
  const int32_t units = static_cast<int32_t>((most_bytes(a.pool.L) + kUnitBytes - 1) / kUnitBytes);
  hipLaunchKernelGGL(compact_move_kernel, dim3(2048), dim3(kThreads), 0, s, a, units);
  return static_cast<int>(hipGetLastError());
}
