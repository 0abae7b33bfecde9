// Up to 16 (query, head) rows against a range of INT2 history positions, by eight wavefronts that
// each stream 64-token chunks of their own: a workgroup's share of shared.hip where few rows see
// the positions (a request's own part behind a shared prefix, a small group).
//
// Wavefront w takes chunks w, w + 8, ... through a private two-stage LDS ring, keeps its own
// online-softmax state, and the eight states are merged once at the end, so the token loop has no
// barrier. In chunk_tile.h such a tile would leave seven wavefronts waiting for one. Operand layouts
// and arithmetic per chunk are those of history.hip's one-tile kernel (four wavefronts there), but
// for the values being centred as in chunk_tile.h, here by P's own sum: one more MFMA against ones
// gives the sum of the rounded P, and sum P c - 1.5 sum P + sum p (z + 1.5 s) is the row.
#pragma once

#include <type_traits>

#include "chunk_tile.h"

namespace oscar {
namespace {

constexpr int kRowTileTable = 512;  // kernel blocks whose offsets live in LDS

struct RowTileLds {
  uint8_t ring[kWavesC][2][kStageBytes] __attribute__((aligned(16)));
  uint32_t off[kRowTileTable];
  float red[4][kWavesC][16];  // per wavefront: row max, sum p, sum p (z_v + 1.5 s_v), P's sum
};
static_assert(kWavesC * 16 * kHeadDim * 4 <= sizeof(RowTileLds::ring), "the merge fits the ring");

// max(a, |b|, |c|) without the quieting of NaN operands (a row with one is NaN by its sum).
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Rows [row_base, rows) (at most 16); everything else as chunk_tile.
__device__ __forceinline__ void row_tile(const AttnArgs& a, const Task& t, int head, int rows,
                                         int row_base, int p_lo, int p_hi, int slot,
                                         RowTileLds& lds) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int first = p_lo >> 6;
  const int nchunk = p_lo < p_hi ? ((p_hi - 1) >> 6) - first + 1 : 0;
  const int nmine = nchunk > wave ? (nchunk - wave + kWavesC - 1) / kWavesC : 0;
  const int kb_first = p_lo >> a.L.bk_shift;
  if (nchunk > 0) {
    const int nkb = min(((p_hi - 1) >> a.L.bk_shift) - kb_first + 1, kRowTileTable);
    for (int j = threadIdx.x; j < nkb; j += kThreadsC)
      lds.off[j] = kernel_block_offset(a, t, head, kb_first + j);
  }
  __syncthreads();

  // ---- copies: 16-byte piece c = 64 i + lane of a chunk is record c / 9, bytes 16 (c % 9).
  const uint32_t tok_bytes = static_cast<uint32_t>(a.L.kv_heads) * kSlot;
  uint32_t voff[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int c = 64 * i + lane;
    voff[i] = static_cast<uint32_t>(c / kPieces) * tok_bytes + 16 * (c % kPieces);
  }
  const uint32_t my_ring = lds_addr(lds.ring[wave][0]);
  const uint32_t in_kb_mask = static_cast<uint32_t>(a.L.bk - 1);
  uint32_t valid_bits = 0;
  auto issue = [&](int j, int s) {  // this wavefront's chunk j -> its stage s
    const int t0 = (first + wave + kWavesC * j) << 6;
    const int local = (t0 >> a.L.bk_shift) - kb_first;
    uint32_t off32 = lds.off[min(local, kRowTileTable - 1)];
    if (local >= kRowTileTable) off32 = kernel_block_offset(a, t, head, t0 >> a.L.bk_shift);
    off32 = uniform(off32);
    const bool ok = off32 != kNoBlock;  // an unmapped block copies the buffer's first records
    const uint8_t* base = a.history;
    if (ok)
      base += (static_cast<uint64_t>(off32) << 5) +
              (static_cast<uint32_t>(t0) & in_kb_mask) * tok_bytes;
    valid_bits = ok ? (valid_bits | (1u << s)) : (valid_bits & ~(1u << s));
    const uint32_t at = my_ring + s * kStageBytes + kSkew;
#pragma unroll
    for (int i = 0; i < kDma; ++i) dma_x4_stream(base, voff[i], at + 1024 * i);
  };
  if (nmine > 0) issue(0, 0);

  // ---- the query rows as FP8 B operands, built by every wavefront for itself (chunk_tile.h; the
  // first term at 2^kQShift times the scale).
  const int my_row = row_base + n;
  const int qi = static_cast<int>(fastdiv(static_cast<uint32_t>(my_row), a.g_div));
  const int64_t my_token = static_cast<int64_t>(t.qstart) + qi;
  const bool valid = my_row < rows && my_token >= 0 && my_token < a.n;
  i32x8 qb[2][kQTerms];
  float qs;
  const float fq = 2.0f * a.scale_log2;  // FP4 holds code / 2
  int sb;
  {
    const uint16_t* src = a.query + (valid ? my_token * a.qs0 +
                                                 (head * a.g + (my_row - qi * a.g)) * a.qs1
                                           : 0);
    float x[2][2][16];
    float mx = 0.f, sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(src + 128 * h + 64 * b + 16 * g + 8 * q);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t pair = valid ? w[i] : 0u;
            const float x0 = __uint_as_float(pair << 16), x1 = __uint_as_float(pair & 0xffff0000u);
            sum += x0 + x1;
            x[h][b][8 * q + 2 * i] = x0;
            x[h][b][8 * q + 2 * i + 1] = x1;
            mx = max3_abs(mx, x0, x1);
          }
        }
    mx = max_xor32(max_xor16(mx));
    qs = 0.5f * sum_xor32(sum_xor16(sum));
    const uint32_t eb = max((__float_as_uint(mx) >> 23) & 0xffu, 8u);
    const float scale = __uint_as_float((eb - 7) << 23);  // row max / scale in [128, 256)
    sb = static_cast<int>(eb) - 7;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = x[h][b][2 * ((4 * d + e) & 7) + ((4 * d + e) >> 3)];
#pragma unroll
          for (int term = 0; term < kQTerms; ++term)
            qb[h][term][4 * b + d] = static_cast<int>(
                fp8x4_scaled_take(v, term == 0 ? scale * (1 << kQShift) : scale));
        }
    sb |= (sb + kQShift) << 8;
  }

  if (nmine > 1) issue(1, 1);

  // Offsets inside a stage (record r at kSkew + 144 r): QK operand of token 16 tt + n; scale | zero
  // of the lane's tokens 16 (e / 4) + 4 g + e % 4; transposed V reads of the rows that hold them.
  const int k_off = kSkew + kRec * n + 8 * g;
  const int sz_off = kSkew + kRec * 4 * g + 64;
  const int v_off = kSkew + kRec * (16 * (n >> 2) + (n & 3)) + kRec * 8 * (g & 1) + kVector;

  float m = -INFINITY, psum = 0.f, zsum = 0.f;
  f32x4 o[16];  // o[2 c + par]: rows 4 g + v, dim 32 c + 2 n + par (units of code / 2)
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 ones_o = {0.f, 0.f, 0.f, 0.f};  // P's sums of rows 4 g + v

  auto process = [&](int j, auto stage_tag) {
    constexpr int S = decltype(stage_tag)::value;
    const uint8_t* st = lds.ring[wave][S];
    f32x4 acc[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 kf[4];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const uint32_t* kp = reinterpret_cast<const uint32_t*>(st + k_off + 16 * kRec * tt + 32 * h);
        const uint32_t w0 = kp[0], w1 = kp[1];
        kf[tt] = u32x4{(uint32_t)even_codes(w0), (uint32_t)odd_codes(w0), (uint32_t)even_codes(w1),
                       (uint32_t)odd_codes(w1)};
      }
#pragma unroll
      for (int term = 0; term < kQTerms; ++term)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) acc[tt] = mfma_q_term(kf[tt], qb[h], term, acc[tt], sb);
    }
    uint32_t ksz[16], vsz[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int off = sz_off + kRec * (16 * (e >> 2) + (e & 3));
      ksz[e] = *reinterpret_cast<const uint32_t*>(st + off);
      vsz[e] = *reinterpret_cast<const uint32_t*>(st + off + kVector);
    }
    float r2[16];  // scores in units of fq (-inf: masked)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      r2[e] = fmaf(h16lo(ksz[e]), acc[e >> 2][e & 3], h16hi(ksz[e]) * qs);
    // Only a first or last chunk is partial (or an unmapped block's): tokens outside get score -inf
    // and a zero V scale and zero (their slots may hold NaN patterns).
    const int t0 = (first + wave + kWavesC * j) << 6;
    const bool ok_block = (valid_bits >> S) & 1u;
    if (!(ok_block && t0 >= p_lo && t0 + kChunk <= p_hi)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool ok = ok_block && static_cast<uint32_t>(t0 + 16 * (e >> 2) + 4 * g + (e & 3) - p_lo) <
                                        static_cast<uint32_t>(p_hi - p_lo);
        vsz[e] = ok ? vsz[e] : 0u;
        r2[e] = ok ? r2[e] : -INFINITY;
      }
    }
    float lm = max3(r2[0], r2[1], r2[2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) lm = max3(lm, r2[e], r2[e + 1]);
    lm = fmaxf(lm, r2[15]) * fq;
    if (__any(lm > m + kTheta)) {  // lazy running max (history.hip)
      const float mn = fmaxf(m, max_xor32(max_xor16(lm)));
      const float alpha = mn == -INFINITY ? 1.0f : exp2f(m - mn);
      m = mn;
      psum *= alpha;
      zsum *= alpha;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float av = __shfl(alpha, 4 * g + v, kWave);
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c][v] *= av;
        ones_o[v] *= av;
      }
    }
    const float nm = m == -INFINITY ? 0.f : -m;
    float av[4][4];
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p = __builtin_amdgcn_exp2f(fmaf(r2[e], fq, nm));
      psum += p;
      zsum = fmaf(p, fmaf(1.5f, h16lo(vsz[e]), h16hi(vsz[e])), zsum);
      av[e >> 2][e & 3] = fmaf(p, h16lo(vsz[e]), 0.0f);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      amax = max3(amax, av[f][0], av[f][1]);
      amax = max3(amax, av[f][2], av[f][3]);
    }
    amax = max_xor32(max_xor16(amax));
    const uint32_t eb = max(__float_as_uint(amax) >> 23, 7u);
    const float scale = __uint_as_float((eb - 6) << 23);  // row max / scale in [64, 128)
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      hi[f] = fp8x4_scaled_take(av[f], scale);
      lo[f] = fp8x4_scaled_last(av[f], scale);
    }
    const i32x8 pa = {(int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3],
                      (int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3]};
    const int sa = static_cast<int>(eb) - 6;
    constexpr int kOnes = 0x22222222;  // FP4 1.0
    ones_o = mfma_pv(pa, i32x8{kOnes, kOnes, kOnes, kOnes, 0, 0, 0, 0}, ones_o, sa);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const i32x2 r0 = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2_ptr_t)(st + v_off + 8 * c));
      const i32x2 r1 =
          __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2_ptr_t)(st + v_off + 4 * kRec + 8 * c));
      const i32x8 be = i32x8{even_codes(r0[0]), even_codes(r0[1]), even_codes(r1[0]),
                             even_codes(r1[1]), 0, 0, 0, 0};
      const i32x8 bo = i32x8{odd_codes(r0[0]), odd_codes(r0[1]), odd_codes(r1[0]),
                             odd_codes(r1[1]), 0, 0, 0, 0};
      o[2 * c] = mfma_pv(pa, be, o[2 * c], sa);
      o[2 * c + 1] = mfma_pv(pa, bo, o[2 * c + 1], sa);
    }
  };

  for (int j = 0; j < nmine; ++j) {
    if (j + 1 < nmine)
      OSCAR_WAIT_VM(kDma);  // chunk j landed; chunk j + 1 may still be in flight
    else
      OSCAR_WAIT_VM(0);
    if (j & 1)
      process(j, std::integral_constant<int, 1>());
    else
      process(j, std::integral_constant<int, 0>());
    if (j + 2 < nmine) {
      OSCAR_WAIT_LGKM();  // every read of this stage has completed
      issue(j + 2, j & 1);
    }
  }

  // ---- the eight states merged, normalized rows and LSE written.
  psum = sum_xor32(sum_xor16(psum));
  zsum = sum_xor32(sum_xor16(zsum));
  if (g == 0) {
    lds.red[0][wave][n] = m;
    lds.red[1][wave][n] = psum;
    lds.red[2][wave][n] = zsum;
  }
  if (n == 0) *reinterpret_cast<f32x4*>(&lds.red[3][wave][4 * g]) = ones_o;
  __syncthreads();  // every chunk consumed; the ring is free for the merge
  float* s_o = reinterpret_cast<float*>(&lds.ring[0][0][0]);  // [wavefront][row][256]
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int row = 4 * g + v;
    if (row_base + row >= rows) break;  // no row: nothing reads its part of the area
    float mx = lds.red[0][0][row];
#pragma unroll
    for (int w = 1; w < kWavesC; ++w) mx = fmaxf(mx, lds.red[0][w][row]);
    const float mw = lds.red[0][wave][row];
    const float f = mw == -INFINITY ? 0.f : exp2f(mw - mx);
    float* dst = s_o + (wave * 16 + row) * kHeadDim + 2 * n;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<float2*>(dst + 32 * c) = make_float2(o[2 * c][v] * f, o[2 * c + 1][v] * f);
  }
  __syncthreads();
  // Thread -> row tid / 32, dims 4 (tid % 32) and 128 further on.
  const int row16 = threadIdx.x >> 5, d0 = 4 * (threadIdx.x & 31);
  const int row = row_base + row16;
  const int rq = static_cast<int>(fastdiv(static_cast<uint32_t>(row), a.g_div));
  const int64_t token = static_cast<int64_t>(t.qstart) + rq;
  if (row >= rows || token < 0 || token >= a.n) return;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWavesC; ++w) mx = fmaxf(mx, lds.red[0][w][row16]);
  float den = 0.f, zs = 0.f;
  f32x4 sum[2] = {};
#pragma unroll
  for (int w = 0; w < kWavesC; ++w) {
    const float mw = lds.red[0][w][row16];
    const float f = mw == -INFINITY ? 0.f : exp2f(mw - mx);
    den = fmaf(f, lds.red[1][w][row16], den);
    zs = fmaf(f, fmaf(-1.5f, lds.red[3][w][row16], lds.red[2][w][row16]), zs);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      sum[h] += *reinterpret_cast<const f32x4*>(s_o + (w * 16 + row16) * kHeadDim + d0 + 128 * h);
  }
  const float inv = 1.0f / fmaxf(den, 1.0e-30f);
  const int64_t out_row = (token * a.hq + head * a.g + (row - rq * a.g)) * a.splits + slot;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = fmaf(2.0f, sum[h][e], zs) * inv;
    *reinterpret_cast<f32x4*>(a.partials + out_row * kHeadDim + d0 + 128 * h) = r;
  }
  if (d0 == 0) a.lse[out_row] = den == 0.f ? -INFINITY : (mx + log2f(den)) * kLn2;
}

}  // namespace
}  // namespace oscar
