// Attention of a step's tasks over the 4-bit history (the history branch of a layer whose cache holds
// 4-bit records): per (task, KV head, split)
//
//   out[row] = sum_p e^{s_p} v_p / sum_p e^{s_p},  s_p = scale q . k_p,  k_p = z + s c  (record4.h)
//
// over the split's share of the positions [sink_len, recent_begin), with the rows' LSEs, for the split
// merges of merge.h. The task table, splits and masks are those of history.hip; the reference has 2-bit
// records only (oscar_ascend/kernels.py:290-482).
//
// Scale and zero fold out of the products: q . k = s (q . c) + z sum q, and sum p v = sum (p s) c + sum p z,
// so that the matrix instructions run over codes as they unpack. K's are exact in bf16, as the queries
// are; V's in fp16, and p s is rounded to fp16: by 2^-11 of itself (bf16's 2^-8 made the error against 64
// bits 0.0023 of the output's norm; now it is the 0.0017 of the output's own rounding), or, the smallest,
// by 2^-24 of the largest V scale of a wavefront's first chunk (see v_by). Sums are fp32.
//
// A workgroup of eight wavefronts, one per CU, takes up to 32 query rows. Wavefront w streams chunks of
// 32 positions w, w + 8, ... of the split through an LDS ring of its own (direct-to-LDS copies, no barrier
// in the loop); scores are computed transposed (positions by rows), so that a lane holds one row's
// scores of eight positions and its probabilities are the P operand of the second product, whose other
// operand comes from transposed LDS reads of 4-bit codes. The eight states are joined at the end.
//
// Up to 16 rows the records' bytes bound it: 32 requests of 32636 positions (284 MB) take 52 us, 5.5 TB/s
// where a large copy moves 5.2 (reads alone reach 7); a small step its chain (one request of 579 positions 10.1
// us: 2.5 until the unit is known, 1.6 until its records are there, 0.6 for the query operands, 1.7 for a
// wavefront's chunk, 2.6 for the join). Tiles of 32 rows are bound by the vector units, which
// issue in 78 % of the cycles (the matrix units' share is 38 %): a wavefront's 32 positions cost 400 vector
// instructions, of which the unpacking, 224, is paid once per tile, and 64 matrix instructions: 2048 tokens
// of 6 heads against 30400 positions take 456 us, 0.84 PFLOP/s. Tiles of 48 or 64 rows, on one wavefront a
// SIMD with 512 registers, halve the unpacking's share but have no second wavefront that fills the waits:
// 617 and 632 us. Codes as fp16 subnormals (five instructions for eight instead of seven) lose the low bits
// of the products (errors 2.5e-5 of the sum of magnitudes, which the matrix instruction aligns as if the
// codes were normal).
#include "dma.h"
#include "history4.h"

namespace oscar {
namespace {

constexpr int kChunk4 = 32;
constexpr int kPieces4 = kSlot4 / 16;               // 17 pieces of a record
constexpr int kStage4 = kChunk4 * kSlot4;           // 8704 bytes
constexpr int kDma4 = (kChunk4 * kPieces4 + 63) / 64;  // 9 copies of a chunk, the last of 32 lanes
constexpr int kTable4 = 512;                        // kernel blocks whose offsets live in LDS
constexpr float kRoom4 = 13.0f;                     // of scores above a row's reference, log2 units
constexpr float kScaleRoom4 = 4.0f;                 // of scaled V scales
constexpr int kMaxTasks4 = 16384;                   // task rows of the device rule

// A workgroup's form: RG groups of 16 query rows, W wavefronts with S ring stages each.
template <int kRowGroups, int kWavesW, int kStagesS>
struct Form4 {
  static constexpr int RG = kRowGroups, W = kWavesW, S = kStagesS, kThreads = W * kWave;
  struct Lds {
    uint8_t ring[W][S][kStage4] __attribute__((aligned(16)));
    uint8_t q[RG * 16 * kHeadDim * 2] __attribute__((aligned(16)));
    uint32_t off[kTable4];
    float red[3][W][16 * RG];  // per wavefront: reference score, sum p, sum p z
  };
  static_assert(S == 2);  // wait_chunks
  static_assert(W * 16 * kHeadDim * 4 <= sizeof(Lds::ring), "a row group's merge fits the ring");
};

// Waits until at most `chunks` chunks' copies (0 or 1) are in flight.
__device__ __forceinline__ void wait_chunks(int chunks) {
  if (chunks)
    OSCAR_WAIT_VM(kDma4);
  else
    OSCAR_WAIT_VM(0);
}

// Sum over the wavefront and inclusive sums of its lanes, through data-parallel primitives: a launch waits for
// these chains (with exchanges through LDS one request of 579 positions took 0.7 us more).
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
  v += dpp_u32<kDppQuadXor1>(v);
  v += dpp_u32<kDppQuadXor2>(v);
  v += dpp_u32<kDppRowHalfMirror>(v);
  v += dpp_u32<kDppRowMirror>(v);
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] + r[1];
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return r[0] + r[1];
}
__device__ __forceinline__ int wave_scan(int v) {
  constexpr int kShr1 = 0x111, kBcast15 = 0x142, kBcast31 = 0x143;
  v += __builtin_amdgcn_update_dpp(0, v, kShr1, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kShr1 + 1, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kShr1 + 3, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kShr1 + 7, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kBcast15, 0xa, 0xf, false);  // rows 1 and 3: the row below's last
  return v + __builtin_amdgcn_update_dpp(0, v, kBcast31, 0xc, 0xf, false);  // the upper half: lane 31's
}

// The unit of workgroup slot u under the device rule: split lengths T such that the tasks' splits,
// ceil(length / T) each, fit the budget's slots of one KV head (or one a task where it is smaller).
// All splits run at once, one per CU, so the launch takes as long as T: eight lengths between the mean
// share and the one that always fits are tried, one by each wavefront, and the least that fits is
// taken (32 requests of 32636 positions on 256 slots: 8 splits of 4096 each). Multiples of kStep4, at
// least kMinSplit4, one chunk for a wavefront of each SIMD (one request of 579 positions with its merge: 0.9
// us less than in splits of 256).
constexpr int kMinSplit4 = 128, kStep4 = 64, kTried4 = 8;

struct Unit4 {
  Task t;
  int split, nsplit, split_tokens;
};

template <int W>
__device__ bool unit_of_slot(const AttnArgs& a, int programs, int u, int* lengths, Unit4& out) {
  constexpr int kThreads4 = W * kWave;
  __shared__ int64_t s_total[W];
  __shared__ int s_fit[kTried4], s_carry[W], s_found[10];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t sum = 0;
  Task mine{};  // of the thread's last task: with at most one a thread, its owner has the row of the unit's
  int mine_task = -1;
  for (int i = tid; i < programs; i += kThreads4) {
    Task t;
    const bool live = read_task(a, t, i);
    const int len = live ? max(t.recent_begin - t.sink_len, 0) : -1;
    lengths[i] = len;
    sum += max(len, 0);
    mine = t;
    mine_task = i;
  }
  // A thread has at most 32 lengths below 2^31.
  sum = (static_cast<int64_t>(wave_sum_u32(static_cast<uint32_t>(sum >> 20))) << 20) +
        wave_sum_u32(static_cast<uint32_t>(sum) & 0xfffffu);
  if (lane == 0) s_total[wave] = sum;
  if (tid == 0) s_found[0] = -1;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) total += s_total[w];
  const int count = max(min(a.task_count[0], programs), 0);
  const int slots = max(-a.split_tokens / a.L.kv_heads, 1);
  auto rounded = [](uint32_t per) {
    return static_cast<int>(min(max((per + kStep4 - 1) / kStep4 * kStep4, uint32_t{kMinSplit4}),
                                uint32_t{1} << 30));
  };
  // A 32-bit division where the batch allows it (its tokens are below 2^32 in all but absurd ones).
  auto share = [&](uint32_t by) {
    const uint64_t per = total >> 32 ? static_cast<uint64_t>(total) / by
                                     : static_cast<uint32_t>(total) / by;
    return static_cast<uint32_t>(min(per, uint64_t{1} << 30)) + 1;
  };
  const int least = rounded(share(slots));
  const int most = rounded(share(max(slots - count, 1)));
  auto tried = [&](int w) {
    return w == kTried4 - 1 ? most : rounded(least + (most - least) / (kTried4 - 1) * w);
  };
  for (int k = wave; k < kTried4; k += W) {
    const int t = tried(k);
    int units = 0;
    for (int i = lane; i < count; i += kWave) units += history_splits(a, max(lengths[i], 0), t);
    units = static_cast<int>(wave_sum_u32(static_cast<uint32_t>(units)));
    if (lane == 0) s_fit[k] = units <= slots;
  }
  __syncthreads();
  int st = most;
#pragma unroll
  for (int k = kTried4 - 1; k >= 0; --k)
    if (s_fit[k]) st = tried(k);
  // Exclusive scan of the split counts; the thread whose task holds slot u says so.
  int carry = 0;
  for (int c0 = 0; c0 < programs; c0 += kThreads4) {
    const int i = c0 + tid;
    const int ns = i < count && lengths[i] >= 0 ? history_splits(a, lengths[i], st) : 0;
    const int incl = wave_scan(ns);
    if (lane == kWave - 1) s_carry[wave] = incl;
    __syncthreads();
    int before = carry, chunk = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      before += w < wave ? s_carry[w] : 0;
      chunk += s_carry[w];
    }
    const int base = before + incl - ns;
    if (ns > 0 && u >= base && u < base + ns) {
      Task t = mine;
      if (i != mine_task) read_task(a, t, i);
      const int row[10] = {i, u - base, ns, t.req, t.qoff, t.qstart, t.qlen, t.prefix, t.sink_len,
                           t.recent_begin};
#pragma unroll
      for (int k = 0; k < 10; ++k) s_found[k] = row[k];
    }
    carry += chunk;
    __syncthreads();  // s_carry is read before the next round writes it
  }
  if (uniform(s_found[0]) < 0) return false;
  out.split = uniform(s_found[1]);
  out.nsplit = uniform(s_found[2]);
  out.split_tokens = st;
  out.t.req = uniform(s_found[3]);
  out.t.qoff = uniform(s_found[4]);
  out.t.qstart = uniform(s_found[5]);
  out.t.qlen = uniform(s_found[6]);
  out.t.prefix = uniform(s_found[7]);
  out.t.sink_len = uniform(s_found[8]);
  out.t.recent_begin = uniform(s_found[9]);
  return true;
}

// fmaxf keeps its operands quiet with an instruction each where it does not know them to be.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

__device__ __forceinline__ f32x4 splat(float v) { return f32x4{v, v, v, v}; }

// A workgroup's rows: row r (of 16 RG) is row base + r of the query tokens from token0 on times the group's
// heads, where that lies below `end`.
struct Rows4 {
  int64_t token0;
  int base, end;
};
__device__ __forceinline__ RowInfo row_of(const AttnArgs& a, const Rows4& rows, int head, int r) {
  const int row = rows.base + r, qi = static_cast<int>(fastdiv(static_cast<uint32_t>(row), a.g_div));
  RowInfo ri;
  ri.qi = qi;
  ri.token = rows.token0 + qi;
  ri.valid = row < rows.end && ri.token >= 0 && ri.token < a.n;
  ri.qhead = head * a.g + (row - qi * a.g);
  return ri;
}

// The rows against positions [p_lo, p_hi) of request t.req, partial rows to `split`.
template <class F>
__device__ __forceinline__ void history_rows4(const AttnArgs& a, const Task& t, const Rows4& rows,
                                              int head, int p_lo, int p_hi, int split,
                                              typename F::Lds& lds) {
  constexpr int RG = F::RG, W = F::W, S = F::S;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int first = p_lo / kChunk4;
  const int nchunk = p_lo < p_hi ? (p_hi - 1) / kChunk4 - first + 1 : 0;
  const int nmine = nchunk > wave ? (nchunk - wave + W - 1) / W : 0;
  const int kb_first = p_lo >> a.L.bk_shift;
  if (nchunk > 0) {
    const int nkb = min(((p_hi - 1) >> a.L.bk_shift) - kb_first + 1, kTable4);
    for (int j = tid; j < nkb; j += F::kThreads) lds.off[j] = block_offset4(a, t, head, kb_first + j);
  }
  // Query rows as they are, two rows a copy; 16-byte piece 8 g + m of row r at (16 (g % 2) + 8 (g / 2) + m)
  // ^ r % 16, for the banks of the reads below, in which a quarter of a wavefront is lanes of two g. A row past
  // the task's reads the buffer's first row and is zeroed below.
  const uint32_t q_area = lds_addr(lds.q);
#pragma unroll
  for (int i = 0; i < RG * 8 / W; ++i) {
    const int row0 = 2 * (i * W + wave), row = row0 + (lane >> 5);
    const RowInfo ri = row_of(a, rows, head, row);
    const int at = (lane & 31) ^ (row & 15);
    const uint16_t* src = a.query + (ri.valid ? ri.token * a.qs0 + ri.qhead * a.qs1 : 0) +
                          8 * ((at >> 1 & 8) | (at << 1 & 16) | (at & 7));
    dma_dwordx4(src, q_area + row0 * kHeadDim * 2);
  }
  barrier_lds();  // the offsets

  // 16-byte piece c = 64 i + lane of a chunk is record c / 17, bytes 16 (c % 17).
  const uint32_t tok_bytes = static_cast<uint32_t>(a.L.kv_heads) * kSlot4;
  uint32_t voff[kDma4];
#pragma unroll
  for (int i = 0; i < kDma4; ++i) {
    const int c = 64 * i + lane;
    voff[i] = static_cast<uint32_t>(c / kPieces4) * tok_bytes + 16 * (c % kPieces4);
  }
  const uint32_t my_ring = lds_addr(lds.ring[wave][0]);
  const uint32_t in_kb_mask = static_cast<uint32_t>(a.L.bk - 1);
  uint32_t mapped = 0;  // bit s: stage s holds a mapped block's positions
  auto issue = [&](int j, int s) {
    const int t0 = (first + wave + W * j) * kChunk4;
    const int local = (t0 >> a.L.bk_shift) - kb_first;
    uint32_t off16 = lds.off[min(local, kTable4 - 1)];
    if (local >= kTable4) off16 = block_offset4(a, t, head, t0 >> a.L.bk_shift);
    off16 = uniform(off16);
    const bool ok = off16 != kNoBlock4;  // an unmapped block copies the buffer's first records
    const uint8_t* base = a.history;
    if (ok)
      base += (static_cast<uint64_t>(off16) << 4) + (static_cast<uint32_t>(t0) & in_kb_mask) * tok_bytes;
    mapped = ok ? (mapped | 1u << s) : (mapped & ~(1u << s));
    const uint32_t at = my_ring + s * kStage4;
#pragma unroll
    for (int i = 0; i < kDma4 - 1; ++i) dma_x4_stream(base, voff[i], at + 1024 * i);
    if (lane < 32) dma_x4_stream(base, voff[kDma4 - 1], at + 1024 * (kDma4 - 1));
  };
  // The first chunks on their way, behind the query rows' copies.
  auto start = [&]() {
#pragma unroll
    for (int s = 0; s < S - 1; ++s)
      if (s < nmine) issue(s, s);
  };
  start();
  wait_chunks(min(nmine, S - 1));
  barrier_lds();  // the query rows

  // The rows' values in the order of the unpacked codes, in place.
#pragma unroll
  for (int i = 0; i < RG * 16; i += F::kThreads / 32) {
    const int row = i + (tid >> 5);
    u32x4* at = reinterpret_cast<u32x4*>(lds.q + row * kHeadDim * 2 + 16 * (tid & 31));
    *at = row_of(a, rows, head, row).valid ? code_order(*at) : u32x4{0u, 0u, 0u, 0u};
  }
  barrier_lds();
  // B operand of k-step m: dims 64 g + 8 m .. + 7 of row n. One row group's stay in registers; two
  // groups' are read from LDS as they are used (256 registers a lane hold the accumulators and no more).
  auto q_operand = [&](int i, int m) {
    return *reinterpret_cast<const u32x4*>(lds.q + (16 * i + n) * kHeadDim * 2 +
                                           16 * ((16 * (g & 1) + 8 * (g >> 1) + m) ^ n));
  };
  const float fq = a.scale_log2;
  float qs[RG];
  u32x4 qb[8];
#pragma unroll
  for (int i = 0; i < RG; ++i) {
    float sum = 0.f;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const u32x4 w = q_operand(i, m);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sum += __uint_as_float(w[e] << 16) + __uint_as_float(w[e] & 0xffff0000u);
      if (RG == 1) qb[m] = w;
    }
    qs[i] = sum_xor32(sum_xor16(sum)) * fq;
  }

  // Row r of score tile 0 is position r of a chunk, of tile 1 position 16 + (r ^ 8): then the eight
  // positions that a lane has, and all that either half wavefront reads at a time, lie in LDS banks of their
  // own (with 16 + r, records 16 apart shared theirs: 101 cycles of conflicts a chunk).
  const int k_off[2] = {kSlot4 * n + 32 * g, kSlot4 * (16 + (n ^ 8)) + 32 * g};
  const int side_off[2] = {kSlot4 * 4 * g + kSide4, kSlot4 * (16 + (4 * g ^ 8)) + kSide4};
  // Transposed reads: lane i of 16 names the row of position i % 4 of its four in tile i / 4 % 2, the one of
  // two neighbouring groups of 16 dims for i < 8 and the other above, so that a lane gets one dim of its own
  // eight positions in either.
  const int v_off = kSlot4 * ((n >> 2 & 1 ? 16 + (4 * g ^ 8) : 4 * g) + (n & 3)) + kCodes4 + 8 * (n >> 3);

  // A chunk in stage s: the products of its K codes and the rows, and its scales and zeros.
  struct Chunk {
    f32x4 acc[RG][2];
    uint2 side[8];  // of the lane's positions, row 4 g + e % 4 of tile e / 4: K scale and zero, V scale and zero
    bool whole;
    uint32_t seen;  // bit e, where not whole
  };
  auto read_chunk = [&](int t0, int s, Chunk& c) {
    uint8_t* st = lds.ring[wave][s];
    // A first or last chunk may be partial, or the block unmapped: positions outside get score -inf and,
    // in LDS, a zero V scale and zero (their bytes may be NaN patterns).
    const bool ok_block = mapped >> s & 1u;
    c.whole = ok_block && t0 >= p_lo && t0 + kChunk4 <= p_hi;
    if (!c.whole) {
      // The positions' bits, in a register that the compiler cannot know ahead of the branch.
      const int from = max(p_lo - t0, 0), to = min(p_hi - t0, kChunk4);
      uint32_t bits = ok_block ? (0xffffffffu << from) & (0xffffffffu >> (kChunk4 - to)) : 0u;
      asm volatile("" : "+v"(bits));
      c.seen = (bits >> (4 * g) & 0xfu) | (bits >> (12 + (4 * g ^ 8)) & 0xf0u);
      if (lane < kChunk4 && !(bits >> lane & 1u))
        *reinterpret_cast<uint32_t*>(st + kSlot4 * lane + kSide4 + 4) = 0u;
    }
#pragma unroll
    for (int i = 0; i < RG; ++i) c.acc[i][0] = c.acc[i][1] = splat(0.f);
    u32x4 kw[2][2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        kw[tt][h] = *reinterpret_cast<const u32x4*>(st + k_off[tt] + 16 * h);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const u32x4 k0 = codes_bf16(kw[0][m >> 2][m & 3]), k1 = codes_bf16(kw[1][m >> 2][m & 3]);
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        const u32x4 q = RG == 1 ? qb[m] : q_operand(i, m);
        c.acc[i][0] = mfma16x16x32(k0, q, c.acc[i][0]);
        c.acc[i][1] = mfma16x16x32(k1, q, c.acc[i][1]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      c.side[e] = *reinterpret_cast<const uint2*>(st + side_off[e >> 2] + kSlot4 * (e & 3));
  };
  // Scores of row group i in log2 units, less m.
  auto row_scores = [&](Chunk& c, const float (&ks)[8], int i, float m, float (&r)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r[e] = fmaf(ks[e], c.acc[i][e >> 2][e & 3], fmaf(half_hi_to_float(c.side[e].x), qs[i], -m));
    if (!c.whole) {
      asm volatile("" : "+v"(c.seen));
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = c.seen >> e & 1u ? r[e] : -INFINITY;
    }
  };
  auto largest = [](const float (&r)[8], float m) {
    return max3(max3(max3(max3(m, r[0], r[1]), r[2], r[3]), r[4], r[5]), r[6], r[7]);
  };
  auto largest_abs = [](const float (&r)[8], float m) {
    return max3_abs(max3_abs(max3_abs(max3_abs(m, r[0], r[1]), r[2], r[3]), r[4], r[5]), r[6], r[7]);
  };
  // This wavefront's chunks in turn through its ring (the first S - 1 are on their way).
  auto stream = [&](auto use) {
    for (int j = 0, s = 0; j < nmine; ++j) {
      // The stage that chunk j - 1 was read from (its reads have completed) takes chunk j + S - 1.
      if (j + S - 1 < nmine) {
        OSCAR_WAIT_LGKM();
        issue(j + S - 1, s == 0 ? S - 1 : s - 1);
      }
      wait_chunks(min(nmine - 1 - j, S - 1));  // chunk j has landed
      use((first + wave + W * j) * kChunk4, s);
      s = s == S - 1 ? 0 : s + 1;
    }
  };

  // Weights are taken against a row's reference m_ref: the largest score of its first chunk here, with room
  // for 2^kRoom4 above it, and V scales times v_by, with room for four times the first chunk's largest:
  // then no sum is ever scaled again, and the accumulators stay where the matrix instructions want them
  // (rescaling them as a running maximum grows made the compiler move them about: two row groups spilled
  // registers). Should a later score or scale have needed more room, the wavefront goes through its chunks
  // again, with the largest ones, which it knows by then (32 requests of 32636 positions, one late position of
  // each with scores 15 nats above the mean: 63 us instead of 52).
  float m_ref[RG], m_less[RG], psum[RG], zsum[RG];
  float v_by = 1.f;
  f32x4 o[RG][16];  // o[c]: rows 4 g + v, dim 16 c + n
  auto set_scale = [&](float top) {
    // From fp16's least value, 2^-24, on: with a first chunk of zeros the scaled V scales stay finite.
    const uint32_t eb = min(max(__float_as_uint(top) >> 23, 127u - 24u), 250u);
    v_by = __uint_as_float((127 + 126 - eb) << 23);  // the largest lies in [0.5, 1)
  };
#pragma unroll
  for (int i = 0; i < RG; ++i) {
    m_ref[i] = -INFINITY;
    m_less[i] = 0.f;
  }
  bool placed = false, again = false;
  do {
    // The largest so far of the lane's positions, scores less their reference and scaled V scales.
    float m_top[RG], v_top = 0.f;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
      psum[i] = zsum[i] = 0.f;
      m_top[i] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 16; ++c) o[i][c] = splat(0.f);
    }
    stream([&](int t0, int s) {
      Chunk c;
      read_chunk(t0, s, c);
      // From here to most of the second products this wavefront goes ahead of its SIMD's other one, so that
      // one's vector instructions run beside the other's matrix instructions (2048 tokens against 30400
      // positions 493 -> 453 us; to the end of the products 458, from the products on 481).
      __builtin_amdgcn_s_setprio(1);
      float ks[8], vs[8];  // products with zero added: one instruction with the conversion
#pragma unroll
      for (int e = 0; e < 8; ++e) ks[e] = fmaf(half_lo_to_float(c.side[e].x), fq, 0.f);
      if (!placed && (mapped >> s & 1u)) {
        placed = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) vs[e] = half_lo_to_float(c.side[e].y);
        set_scale(max_xor32(max_xor16(largest_abs(vs, 0.f))));  // the same in every lane
#pragma unroll
        for (int i = 0; i < RG; ++i) {
          float r[8];
          row_scores(c, ks, i, 0.f, r);
          m_ref[i] = max_xor32(max_xor16(largest(r, -INFINITY)));
          m_less[i] = m_ref[i] == -INFINITY ? 0.f : m_ref[i];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) vs[e] = fmaf(half_lo_to_float(c.side[e].y), v_by, 0.f);
      v_top = largest_abs(vs, v_top);
      u32x4 pa[RG];
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        float r[8], pv[8];
        row_scores(c, ks, i, m_less[i], r);
        m_top[i] = largest(r, m_top[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __builtin_amdgcn_exp2f(r[e]);
          psum[i] += p;
          zsum[i] = fmaf(p, half_hi_to_float(c.side[e].y), zsum[i]);
          pv[e] = p * vs[e];
        }
        // Position e of the lane is nibble e of its transposed reads: the order of codes_f16.
        pa[i] = u32x4{pack_f16x2(pv[0], pv[2]), pack_f16x2(pv[4], pv[6]), pack_f16x2(pv[1], pv[3]),
                      pack_f16x2(pv[5], pv[7])};
      }
      const uint8_t* st = lds.ring[wave][s];
#pragma unroll
      for (int c8 = 0; c8 < 8; ++c8) {
        const i32x2 w =
            __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2_ptr_t)(st + v_off + 16 * c8));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (c8 == 6 && h == 0) __builtin_amdgcn_s_setprio(0);
          const u32x4 vf = codes_f16(static_cast<uint32_t>(w[h]));
#pragma unroll
          for (int i = 0; i < RG; ++i) o[i][2 * c8 + h] = mfma16x16x32_f16(pa[i], vf, o[i][2 * c8 + h]);
        }
      }
    });
    if (again) break;
    v_top = max_xor32(max_xor16(v_top));
    again = __any(v_top > kScaleRoom4) != 0;  // else p s v_by < 2^(13 + 2)
#pragma unroll
    for (int i = 0; i < RG; ++i) {
      const float above = max_xor32(max_xor16(m_top[i]));
      // A first chunk of nothing but -inf has no reference, and later scores are as they are.
      again |= __any(above > (m_ref[i] == -INFINITY ? -INFINITY : kRoom4)) != 0;
      m_top[i] = m_ref[i] == -INFINITY ? above : fmaxf(m_ref[i], m_ref[i] + above);
    }
    if (again) {
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        m_ref[i] = m_top[i];
        m_less[i] = m_ref[i] == -INFINITY ? 0.f : m_ref[i];
      }
      set_scale(v_top / v_by);
      OSCAR_WAIT_LGKM();
      start();
    }
  } while (again);

  // ---- the wavefronts' states joined, normalized rows and LSEs written.
  const float v_back = 1.0f / v_by;  // both powers of two
#pragma unroll
  for (int i = 0; i < RG; ++i) {
    const float ps = sum_xor32(sum_xor16(psum[i])), zs = sum_xor32(sum_xor16(zsum[i]));
    if (g == 0) {
      lds.red[0][wave][16 * i + n] = m_ref[i];
      lds.red[1][wave][16 * i + n] = ps;
      lds.red[2][wave][16 * i + n] = zs;
    }
  }
  float* s_o = reinterpret_cast<float*>(&lds.ring[0][0][0]);  // [wavefront][16 rows][256]
#pragma unroll
  for (int i = 0; i < RG; ++i) {
    __syncthreads();  // the ring (or the last rows' sums) has been read
    const int live = min(rows.end - rows.base - 16 * i, 16);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (4 * g + v >= live) continue;
      const int row = 16 * i + 4 * g + v;
      float mx = lds.red[0][0][row];
#pragma unroll
      for (int w = 1; w < W; ++w) mx = fmaxf(mx, lds.red[0][w][row]);
      const float mw = lds.red[0][wave][row];
      const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mx) * v_back;
      float* dst = s_o + (wave * 16 + 4 * g + v) * kHeadDim + n;
#pragma unroll
      for (int c = 0; c < 16; ++c) dst[16 * c] = o[i][c][v] * f;
    }
    __syncthreads();
    // A wavefront takes a row, a lane four dims of it.
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += W) {
      const int row16 = r0 + wave, row = 16 * i + row16, d0 = 4 * lane;
      const RowInfo ri = row_of(a, rows, head, row);
      if (!ri.valid) continue;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mx = fmaxf(mx, lds.red[0][w][row]);
      float den = 0.f, zs = 0.f;
      f32x4 sum = {};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float mw = lds.red[0][w][row];
        const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mx);
        den = fmaf(f, lds.red[1][w][row], den);
        zs = fmaf(f, lds.red[2][w][row], zs);
        sum += *reinterpret_cast<const f32x4*>(s_o + (w * 16 + row16) * kHeadDim + d0);
      }
      const float inv = 1.0f / fmaxf(den, 1.0e-30f);
      const int64_t out_row = (ri.token * a.hq + ri.qhead) * a.splits + split;
      f32x4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (sum[e] + zs) * inv;
      *reinterpret_cast<f32x4*>(a.partials + out_row * kHeadDim + d0) = r;
      if (lane == 0) a.lse[out_row] = den == 0.f ? -INFINITY : (mx + log2f(den)) * kLn2;
    }
  }
}

template <class F>
__global__ __launch_bounds__(F::kThreads) void history4_kernel(const AttnArgs a, int programs) {
  __shared__ typename F::Lds lds;
  const int head = blockIdx.y;
  Task t;
  int split, nsplit, split_tokens;
  if (a.split_tokens < 0) {
    Unit4 unit;
    const int u = static_cast<int>(blockIdx.z) * programs + static_cast<int>(blockIdx.x);
    if (!unit_of_slot<F::W>(a, programs, u, reinterpret_cast<int*>(&lds), unit)) return;
    t = unit.t;
    split = unit.split;
    nsplit = unit.nsplit;
    split_tokens = unit.split_tokens;
    __syncthreads();  // the lengths have been read
  } else {
    if (!read_task(a, t, static_cast<int>(blockIdx.x))) return;
    split = blockIdx.z;
    split_tokens = a.split_tokens;
    nsplit = history_splits(a, t.recent_begin - t.sink_len, split_tokens);
    if (split >= nsplit) {
      write_unused_split(a, t, head, split);
      return;
    }
  }
  int p_lo, p_hi;
  history_positions(a, t, t.recent_begin - t.sink_len, nsplit, split, split_tokens, p_lo, p_hi);
  const Rows4 rows{t.qstart + t.qoff, 0, min(a.qt, t.qlen - t.qoff) * a.g};
  history_rows4<F>(a, t, rows, head, p_lo, p_hi, split, lds);
  // Last, as the other rows' copies would wait for these stores.
  if (a.split_tokens < 0 && split == 0) write_unused_splits<F::kThreads>(a, t, head, nsplit, a.splits);
}

// ---- steps with many query tokens in a request: tiles of 16 RG of its rows instead of tasks, so that a
// tile's unpacked codes meet as many rows as a wavefront's registers hold sums of. The rows past a
// request's last cost matrix products but hardly time where a tile has few: the records' copies
// take as long.

// Request and tile of tile slot x, the requests' tiles in order; false past the last. Every thread of the
// workgroup calls it.
template <class F>
__device__ __forceinline__ bool find_tile4(const AttnArgs& a, int max_reqs, int x, int& req, int& tile) {
  __shared__ int s_carry[F::W], s_found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int reqs = max(min(a.counts[0], max_reqs), 0), active = a.counts[1];
  if (tid == 0) s_found[0] = -1;
  int carry = 0;
  for (int c0 = 0; c0 < reqs && carry <= x; c0 += F::kThreads) {
    const int r = c0 + tid;
    int tiles = 0;
    if (r < reqs) {
      const int q0 = a.qstarts[r], rows = (min(a.qstarts[r + 1], active) - q0) * a.g;
      tiles = rows > 0 ? (rows + 16 * F::RG - 1) / (16 * F::RG) : 0;
    }
    const int incl = wave_scan(tiles);
    if (lane == kWave - 1) s_carry[wave] = incl;
    __syncthreads();
    int before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < F::W; ++w) {
      before += w < wave ? s_carry[w] : 0;
      all += s_carry[w];
    }
    const int base = before + incl - tiles;
    if (x >= base && x < base + tiles) {
      s_found[0] = r;
      s_found[1] = x - base;
    }
    carry += all;
    __syncthreads();  // s_carry is read before the next round writes it
  }
  if (reqs <= 0) return false;
  req = uniform(s_found[0]);
  tile = uniform(s_found[1]);
  return req >= 0;
}

template <class F>
__global__ __launch_bounds__(F::kThreads) void history4_tiles_kernel(const AttnArgs a, int max_reqs) {
  __shared__ typename F::Lds lds;
  // Workgroup ((tile, KV head), split): the tiles that exist dispatch first.
  const int unit = static_cast<int>(blockIdx.x) / a.splits, h = a.L.kv_heads;
  const int split = static_cast<int>(blockIdx.x) - unit * a.splits, head = unit % h;
  Task t{};
  int tile;
  if (!find_tile4<F>(a, max_reqs, unit / h, t.req, tile)) return;
  t.qstart = a.qstarts[t.req];
  t.qlen = min(a.qstarts[t.req + 1], a.counts[1]) - t.qstart;
  t.prefix = a.seq_lens[t.req] - t.qlen;
  t.sink_len = min(a.L.sink, t.prefix);
  t.recent_begin = max(t.sink_len, t.prefix - a.L.recent);
  // Equal numbers of chunks for the splits (split_range's tiles of block_n positions, kernels.py:368-370,
  // at whole chunks of absolute positions).
  const int lo = max(t.sink_len, 0), hi = t.recent_begin;
  const int c0 = lo / kChunk4, chunks = lo < hi ? (hi - 1) / kChunk4 - c0 + 1 : 0;
  const int from = static_cast<int>(static_cast<int64_t>(chunks) * split / a.splits);
  const int to = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / a.splits);
  const int p_lo = max(lo, (c0 + from) * kChunk4), p_hi = min(hi, (c0 + to) * kChunk4);
  const Rows4 rows{t.qstart, tile * 16 * F::RG, t.qlen * a.g};
  history_rows4<F>(a, t, rows, head, p_lo, p_hi, split, lds);
}

// Eight wavefronts, two a SIMD, with two stages each.
using OneGroup = Form4<1, 8, 2>;
using TwoGroups = Form4<2, 8, 2>;
using RowTiles = TwoGroups;

}  // namespace
}  // namespace oscar

extern "C" int oscar_history_int4(const void* query, int64_t q_s0, int64_t q_s1, int64_t q_s2,
                                  const void* history, int64_t history_bytes, const int32_t* qstarts,
                                  const int32_t* seq_lens, const int32_t* block_tables,
                                  int64_t table_stride, int64_t table_columns, const int32_t* counts,
                                  const int32_t* tasks, const int32_t* task_count, int64_t n,
                                  int64_t hq, int64_t programs, int32_t splits, int32_t block_n,
                                  int32_t query_tile, int32_t max_query_len, float scale,
                                  int32_t split_tokens, int32_t row_tiles, int64_t max_reqs,
                                  const oscar_layout* layout, float* partials, float* lse,
                                  void* stream) {
  using namespace oscar;
  AttnArgs a;
  int64_t rows = 0;
  const int st = make_attn_args(query, q_s0, q_s1, q_s2, nullptr, 0, 0, 1, nullptr, 0, 0, 1, history,
                                history_bytes, nullptr, 0, qstarts, seq_lens, block_tables,
                                table_stride, table_columns, counts, tasks, task_count, n, hq, programs,
                                splits, block_n, query_tile, max_query_len, scale, 0, split_tokens,
                                layout, partials, lse, &a, &rows, 4);
  if (st != OSCAR_OK) return st;
  if (history_bytes > 16ll * kNoBlock4) return OSCAR_E_UNSUPPORTED;  // block offsets are 32 bits of 16 bytes
  if (n == 0) return OSCAR_OK;
  hipStream_t s = as_stream(stream);
  if (row_tiles) {
    if (split_tokens) return OSCAR_E_UNSUPPORTED;
    if (max_reqs < 1 || max_reqs > 0x7fffffffll) return OSCAR_E_SHAPE;
    // A request of q tokens has at most q g / R + 1 tiles of R rows.
    constexpr int64_t kRows = 16 * RowTiles::RG;
    const int64_t reqs = n < max_reqs ? n : max_reqs;
    if (n > 0x7fffffffll / hq) return OSCAR_E_SHAPE;
    const int64_t tiles = n * a.g / kRows + reqs;
    if (tiles > 0xffffffffll / RowTiles::kThreads / a.L.kv_heads / splits) return OSCAR_E_SHAPE;
    hipLaunchKernelGGL(history4_tiles_kernel<RowTiles>,
                       dim3(static_cast<unsigned>(tiles * a.L.kv_heads * splits)),
                       dim3(RowTiles::kThreads), 0, s, a, static_cast<int>(max_reqs));
    return static_cast<int>(hipGetLastError());
  }
  const int64_t z = split_tokens < 0 ? device_unit_slices(programs, a.L.kv_heads, split_tokens) : splits;
  if (z > 65535 || a.L.kv_heads > 65535) return OSCAR_E_SHAPE;
  // The lengths of the device rule's task rows lie in the ring.
  if (split_tokens < 0 && programs > kMaxTasks4) return OSCAR_E_UNSUPPORTED;
  if (programs * z > 0xffffffffll / OneGroup::kThreads / a.L.kv_heads) return OSCAR_E_SHAPE;
  const dim3 grid(static_cast<unsigned>(programs), static_cast<unsigned>(a.L.kv_heads),
                  static_cast<unsigned>(z));
  if (rows <= 16)
    hipLaunchKernelGGL(history4_kernel<OneGroup>, grid, dim3(OneGroup::kThreads), 0, s, a,
                       static_cast<int>(programs));
  else
    hipLaunchKernelGGL(history4_kernel<TwoGroups>, grid, dim3(TwoGroups::kThreads), 0, s, a,
                       static_cast<int>(programs));
  return static_cast<int>(hipGetLastError());
}
