// The attention weight that each cached row received, summed over query rows and the query heads of its KV head:
//   out[hk, j] = prior[hk, j] + sum over i, h in group hk of softmax_j(scale * q[h, i] . K[hk, j]),  j <= pos[i],
// what a cache's rows are ranked by before the light ones are dropped (evict.hip). Neither the scores nor the
// weights go to memory (but for one token's scores, below). Short caches have a kernel of their own (weights_short_kernel).
//
// Design: the n x group (token, query head) pairs of a KV head are its rows. A weight needs its row's maximum
// and sum before it can be formed, so the product with K^T runs twice:
//  1. weights_lse_kernel: 128 rows a workgroup (64 in small launches, as in the second pass) walk the cache in 64-row tiles (attention.hip's first half, with the
//     maximum and the sum kept per lane); with few row blocks, in splits of the cache. Leaves L = max + log2(sum) and the
//     position of each row (weights_join_kernel joins the splits, or, of few, each workgroup of the second pass for its rows).
//  2. weights_sum_kernel: 128 cache rows a workgroup hold their operands in registers while the query rows (packed by the
//     first pass: a tile's loads then need no addresses) pass through LDS: S = K Q^T gives a lane four cache rows of one query row, and 2^(s scale - L) adds up in
//     registers over all query rows; the 16 lanes of a cache row meet once, at the end. With few cache blocks the
//     query rows are split, and weights_reduce_kernel adds the parts in order (no atomics: the same sums every time).
// Scores and sums are fp32 throughout, products bf16 x bf16 (exact) accumulated in fp32 on the matrix cores.
//
// Bound: the issue of a SIMD. A wavefront's score a lane costs one matrix instruction at head_dim 128 (four make four) and, to stay in
// fp32, a product, an exponential and an addition (the first pass: half a maximum too); alone these take 16.3 and 17.0 cycles for one
// score a lane, both together 28.3, whichever way the two are interleaved (within a wavefront, across wavefronts, by priority), so they
// hardly overlap. Measured (us, kernels traced, 28 / 4 heads of 128): 8256 causal rows 251 + 258 + 4, of which 175 each is that
// issue at 2.4 GHz and the clock was near 2.0; 64 rows, spread over 32832, 21 + 20 and 4 for the join
// (the last 64 rows, twice the work, 25 + 27 and 4); one row over 8257 4.6 + 4.4.
// Slower: 64 rows a wavefront (275 and 320 us: two wavefronts a SIMD), exponentials one step behind the products (266, 283).
#include <algorithm>

#include "attention_common.hpp"
#include "attention_weights_plan.hpp"

namespace ckv {

constexpr int kWtWholeWaves = 8;
constexpr int kWtShortWaves = 8;

typedef __attribute__((address_space(1))) void wt_gvoid;
typedef __attribute__((address_space(3))) void wt_lvoid;

// SPLIT: split z of the cache's tiles; (max, sum) of a row's split to part[z].
template <int D, int QG, bool SPLIT>
__global__ __launch_bounds__(kWtThreads) void weights_lse_kernel(
    int nqb, int map_group, int xpk_log, int items, uint32_t inv_group, uint32_t inv_nqb,
    const int64_t* __restrict__ pos, int N, int rows, int group, uint32_t inv_gqa, const char* __restrict__ kc,
    int64_t k_hs_b, const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b, float scale_log2,
    RowStat* __restrict__ stat, char* __restrict__ packed, int stat_rows, float2* __restrict__ part, int64_t part_stride, int split_tiles,
    int32_t* __restrict__ err) {
  constexpr int DS = D / 32, CPR = D / 8, ROWB = D * 2, KI = kWtTile * CPR / kWtThreads, BR = 64 * QG;
  __shared__ __attribute__((aligned(1024))) char lds0[kWtTile * ROWB];
  __shared__ __attribute__((aligned(1024))) char lds1[kWtTile * ROWB];
  __shared__ int blk_max_s[kWtThreads / 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  int rb, hk, z;
  if (!attn_work_item(nqb, map_group, xpk_log, items, inv_group, inv_nqb, rb, hk, z)) return;
  const char* kh = kc + (int64_t)hk * k_hs_b;
  int off[KI];
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int P = (wave * KI + i) * 64 + lane, slot = P / CPR;
    off[i] = slot * ROWB + ((P % CPR) ^ swz_k<CPR>(slot)) * 16;
  }
  auto issue = [&](int n0, char* kb) {
    const char* kt = kh + (int64_t)n0 * ROWB;
    const int last = N - 1 - n0;
    auto load = [&](int i, int o) {
      __builtin_amdgcn_global_load_lds((wt_gvoid*)(kt + (uint32_t)o), (wt_lvoid*)(kb + (wave * KI + i) * 1024), 16, 0, 0);
    };
    if (last >= kWtTile - 1) {  // uniform: a whole tile
#pragma unroll
      for (int i = 0; i < KI; ++i) load(i, off[i]);
    } else {  // rows past the cache load its last one; those past every position are masked
#pragma unroll
      for (int i = 0; i < KI; ++i) load(i, min(off[i] / ROWB, last) * ROWB + off[i] % ROWB);
    }
  };
  const int tile_begin = SPLIT ? z * split_tiles : 0;
  issue(tile_begin * kWtTile, lds0);  // known before the positions are
  int my_pos[QG];
  int wmax = -1, wmin = N;
  bf16x8 qf[QG][DS];
#pragma unroll
  for (int qg = 0; qg < QG; ++qg) {
    const int r = rb * BR + (wave * QG + qg) * 16 + lm;
    const int rc = min(r, rows - 1), t = div_by(rc, group, inv_gqa), gh = rc - t * group;
    const int64_t p64 = pos[t];
    int p = p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64;
    if (r < rows) {
      if (p != p64) flag_error(err, CKV_DEVICE_ERR_RANGE);
      wmin = min(wmin, p);
    } else {
      p = -1;
    }
    my_pos[qg] = p;
    wmax = max(wmax, p);
    const char* qr = q + (int64_t)(hk * group + gh) * q_hs_b + (int64_t)t * q_ts_b;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[qg][s] = __builtin_bit_cast(bf16x8, ld16(qr + (32 * s + 8 * g) * 2));
  }
  wmax = __builtin_amdgcn_readfirstlane(row16_reduce(wmax, [](int a, int b) { return max(a, b); }));
  wmin = __builtin_amdgcn_readfirstlane(row16_reduce(wmin, [](int a, int b) { return min(a, b); }));
  if (!SPLIT || z == 0) {  // the rows packed, for the second pass
#pragma unroll
    for (int qg = 0; qg < QG; ++qg) {
      const int r = rb * BR + (wave * QG + qg) * 16 + lm;
#pragma unroll
      for (int s = 0; s < DS; ++s)
        if (r < stat_rows) st16(packed + ((int64_t)hk * stat_rows + r) * ROWB + (32 * s + 8 * g) * 2, __builtin_bit_cast(vec16, qf[qg][s]));
    }
  }
  if (lane == 0) blk_max_s[wave] = wmax;
  __syncthreads();
  int bmax = blk_max_s[0];
#pragma unroll
  for (int w = 1; w < kWtThreads / 64; ++w) bmax = max(bmax, blk_max_s[w]);
  bmax = __builtin_amdgcn_readfirstlane(bmax);
  int n_tiles = bmax / kWtTile + 1;  // a block has a row: bmax >= 0
  if (SPLIT) n_tiles = min(n_tiles, tile_begin + split_tiles);
  // a split past every position: its loads into LDS land before the workgroup ends
  if (tile_begin >= n_tiles) __builtin_amdgcn_s_waitcnt(0x0F70);

  // A lane's own maximum and sum over the cache rows that it gets.
  float m_run[QG], m_sub[QG], l_run[QG];
#pragma unroll
  for (int qg = 0; qg < QG; ++qg) {
    m_run[qg] = -INFINITY;
    m_sub[qg] = 0.f;
    l_run[qg] = 0.f;
  }
  int k_rd[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) k_rd[ds] = lm * ROWB + (((4 * ds + g) ^ swz_k<CPR>(lm)) * 16);
  auto body = [&](int tile, const char* cur, char* nxt) {
    const int n0 = tile * kWtTile;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's loads of the tile landed
    __syncthreads();
    if (tile + 1 < n_tiles) issue(n0 + kWtTile, nxt);
    if (n0 > wmax) return;  // uniform per wavefront
    const bool need_mask = n0 + kWtTile - 1 > wmin;
    constexpr int T = 2;  // 32 cache rows at a time
#pragma unroll
    for (int half = 0; half < kWtTile / (16 * T); ++half) {
      f32x4 s[QG][T];  // lane (g, lm): query lm, cache rows n0 + 32 half + 16 t + 4 g + e
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)  // dependent products four apart
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const bf16x8 a = *(const bf16x8*)(cur + (half * T + t) * 16 * ROWB + k_rd[ds]);
#pragma unroll
          for (int qg = 0; qg < QG; ++qg)
            s[qg][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[qg][ds], ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[qg][t], 0, 0, 0);
        }
      if (need_mask) {
#pragma unroll
        for (int qg = 0; qg < QG; ++qg) {
          const int lim = my_pos[qg] - n0 - 16 * T * half - 4 * g;
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * t + e > lim) s[qg][t][e] = -INFINITY;
        }
      }
      float bm[QG];
      bool raise = false;
#pragma unroll
      for (int qg = 0; qg < QG; ++qg) {
        bm[qg] = s[qg][0][0];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) bm[qg] = fmaxf(bm[qg], s[qg][t][e]);
        bm[qg] *= scale_log2;  // > 0: max commutes
        raise = raise || bm[qg] > m_run[qg] + 8.f;  // a sum's fp32 range takes weights up to 2^8
      }
      if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
        for (int qg = 0; qg < QG; ++qg) {
          const float m_new = bm[qg] > m_run[qg] + 8.f ? bm[qg] : m_run[qg];
          l_run[qg] *= m_run[qg] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[qg] - m_new);
          m_run[qg] = m_new;
          m_sub[qg] = m_new == -INFINITY ? 0.f : m_new;
        }
      }
#pragma unroll
      for (int qg = 0; qg < QG; ++qg)
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            l_run[qg] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[qg][t][e], scale_log2, -m_sub[qg]));
    }
  };
  for (int tile = tile_begin; tile < n_tiles; tile += 2) {
    body(tile, lds0, lds1);
    if (tile + 1 < n_tiles) body(tile + 1, lds1, lds0);
  }
#pragma unroll
  for (int qg = 0; qg < QG; ++qg) {
    // the four lanes of a query
    const float m = group_max(m_run[qg]);
    float l = m_run[qg] == -INFINITY ? 0.f : l_run[qg] * __builtin_amdgcn_exp2f(m_run[qg] - m);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = rb * BR + (wave * QG + qg) * 16 + lm;
    if (r >= stat_rows || g != 0) continue;
    const int64_t at = (int64_t)hk * stat_rows + r;
    if (SPLIT) part[z * part_stride + at] = make_float2(m, l);
    else stat[at] = r < rows ? RowStat{m + __builtin_amdgcn_logf(l), my_pos[qg]} : RowStat{INFINITY, -1};
  }
}

// Joins the splits (at most 64) of the first pass: a row a wavefront, a split a lane.
__global__ __launch_bounds__(256) void weights_join_kernel(const float2* __restrict__ part, int64_t stride, int splits,
                                                           const int64_t* __restrict__ pos, int N, int rows, int group,
                                                           RowStat* __restrict__ stat, int stat_rows, int64_t total) {
  const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x % 64;
  if (at >= total) return;
  const float2 p = part[min(lane, splits - 1) * stride + at];
  const int row = (int)(at % stat_rows);
  const int64_t p64 = pos[min(row, rows - 1) / group];
  float m = lane < splits ? p.x : -INFINITY;
  const float mine = m;
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float l = wave_butterfly_sum(mine == -INFINITY ? 0.f : p.y * __builtin_amdgcn_exp2f(mine - m));
  if (lane == 0)
    stat[at] = row < rows ? RowStat{m + __builtin_amdgcn_logf(l), p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64} : RowStat{INFINITY, -1};
}

// What a second pass that joins the first's splits itself reads (as weights_join_kernel does).
struct WeightsJoin {
  const float2* part;
  int64_t stride;
  int splits;
  const int64_t* pos;
  int rows, group;
};

// PARTS: part z of the query rows; sums to ws[z], else prior + sum to out. JOIN: at most kWtJoinRows rows a part, whose normalisers
// every workgroup makes for itself.
template <int D, int KG, bool PARTS, bool JOIN>
__global__ __launch_bounds__(kWtThreads, 4) void weights_sum_kernel(
    int nkb, int map_group, int xpk_log, int items, uint32_t inv_group, uint32_t inv_nkb, int N, int stat_rows,
    const char* __restrict__ kc, int64_t k_hs_b, const char* __restrict__ packed, float scale_log2,
    const RowStat* __restrict__ stat, const float* prior, float* out, int64_t part_stride, int part_tiles, WeightsJoin join) {
  constexpr int DS = D / 32, CPR = D / 8, ROWB = D * 2, KI = kWtTile * CPR / kWtThreads, QT = kWtTile / 16;
  __shared__ __attribute__((aligned(1024))) char lds0[kWtTile * ROWB];
  __shared__ __attribute__((aligned(1024))) char lds1[kWtTile * ROWB];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  int kb, hk, z;
  if (!attn_work_item(nkb, map_group, xpk_log, items, inv_group, inv_nkb, kb, hk, z)) return;
  kb = nkb - 1 - kb;  // the first cache rows, which the most queries see, first
  const RowStat* st = stat + (int64_t)hk * stat_rows;
  const int tile_begin = PARTS ? z * part_tiles : 0, tiles = stat_rows / kWtTile;
  const int tile_end = PARTS ? min(tiles, tile_begin + part_tiles) : tiles;
  const int k0 = (kb * (kWtThreads / 64) + wave) * (16 * KG);  // this wavefront's cache rows

  __shared__ RowStat s_stat[JOIN ? kWtJoinRows : 1];
  // does any query row of the part see these cache rows?
  bool any = true;
  if constexpr (PARTS || JOIN) {
    int seen = -1;
    for (int r = tile_begin * kWtTile + (int)threadIdx.x; r < tile_end * kWtTile; r += kWtThreads) {
      if constexpr (JOIN) {
        const float2* pr = join.part + (int64_t)hk * stat_rows + r;
        const int64_t p64 = join.pos[min(r, join.rows - 1) / join.group];
        float2 p[kWtJoinSplits];
#pragma unroll
        for (int z = 0; z < kWtJoinSplits; ++z) {
          p[z] = make_float2(-INFINITY, 0.f);
          if (z < kWtJoinSplits / 2 || join.splits > kWtJoinSplits / 2)  // uniform
            p[z] = pr[min(z, join.splits - 1) * join.stride];
        }
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int z = 0; z < kWtJoinSplits; ++z) m = fmaxf(m, p[z].x);
#pragma unroll
        for (int z = 0; z < kWtJoinSplits; ++z)
          l += z < join.splits && p[z].x != -INFINITY ? p[z].y * __builtin_amdgcn_exp2f(p[z].x - m) : 0.f;
        const RowStat own = r < join.rows ? RowStat{m + __builtin_amdgcn_logf(l), p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64}
                                          : RowStat{INFINITY, -1};
        s_stat[r - tile_begin * kWtTile] = own;
        seen = max(seen, own.pos);
      } else {
        seen = max(seen, st[r].pos);
      }
    }
    any = __syncthreads_or(seen >= kb * (kWtThreads / 64) * 16 * KG);
  }

  f32x4 acc[KG];
#pragma unroll
  for (int kg = 0; kg < KG; ++kg) acc[kg] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (any) {
    const char* kh = kc + (int64_t)hk * k_hs_b;
    const char* qh = packed + (int64_t)hk * stat_rows * ROWB;
    int off[KI];
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int P = (wave * KI + i) * 64 + lane, slot = P / CPR;
      off[i] = slot * ROWB + ((P % CPR) ^ swz_k<CPR>(slot)) * 16;
    }
    auto issue = [&](int tile, char* qb, RowStat(&s)[QT]) {
      const char* qt = qh + (int64_t)tile * (kWtTile * ROWB);
#pragma unroll
      for (int i = 0; i < KI; ++i)
        __builtin_amdgcn_global_load_lds((wt_gvoid*)(qt + (uint32_t)off[i]), (wt_lvoid*)(qb + (wave * KI + i) * 1024), 16, 0, 0);
      const RowStat* sr = JOIN ? s_stat + (tile - tile_begin) * kWtTile : st + (int64_t)tile * kWtTile;
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t] = sr[(uint32_t)(t * 16 + lm)];
    };
    int q_rd[DS];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) q_rd[ds] = lm * ROWB + (((4 * ds + g) ^ swz_k<CPR>(lm)) * 16);
    RowStat st0[QT], st1[QT];
    issue(tile_begin, lds0, st0);
    bf16x8 kf[KG][DS];
#pragma unroll
    for (int kg = 0; kg < KG; ++kg)
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
        kf[kg][ds] = __builtin_bit_cast(bf16x8, ld16(kh + (int64_t)min(k0 + 16 * kg + lm, N - 1) * ROWB + (32 * ds + 8 * g) * 2));
    auto body = [&](int tile, const char* cur, char* nxt, const RowStat(&now)[QT], RowStat(&next)[QT]) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
      if (tile + 1 < tile_end) issue(tile + 1, nxt, next);
      int top = now[0].pos, low = now[0].pos;
#pragma unroll
      for (int t = 1; t < QT; ++t) {
        top = max(top, now[t].pos);
        low = min(low, now[t].pos);
      }
      if (!__builtin_amdgcn_ballot_w64(top >= k0)) return;  // uniform per wavefront
      const bool need_mask = __builtin_amdgcn_ballot_w64(low < k0 + 16 * KG - 1);
      constexpr int U = 4 / KG;  // query groups at a time: dependent products four apart
#pragma unroll
      for (int t0 = 0; t0 < QT; t0 += U) {
        f32x4 s[U][KG];
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bf16x8 b = *(const bf16x8*)(cur + (t0 + u) * 16 * ROWB + q_rd[ds]);
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
              s[u][kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kg][ds], b, ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[u][kg], 0, 0, 0);
          }
        if (need_mask) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int lim = now[t0 + u].pos - k0 - 4 * g;
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (16 * kg + e > lim) s[u][kg][e] = -INFINITY;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[kg][e] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][kg][e], scale_log2, -now[t0 + u].lse));
      }
    };
    for (int tile = tile_begin; tile < tile_end; tile += 2) {
      body(tile, lds0, lds1, st0, st1);
      if (tile + 1 < tile_end) body(tile + 1, lds1, lds0, st1, st0);
    }
  }
#pragma unroll
  for (int kg = 0; kg < KG; ++kg)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float sum = row16_reduce(acc[kg][e], [](float a, float b) { return a + b; });
      const int j = k0 + 16 * kg + 4 * g + e;
      if (lm != 0 || j >= N) continue;
      const int64_t at = (int64_t)hk * N + j;
      if (PARTS) out[z * part_stride + at] = sum;
      else out[at] = prior != nullptr ? prior[at] + sum : sum;
    }
}

__global__ __launch_bounds__(256) void weights_reduce_kernel(const float* __restrict__ part, int64_t stride, int parts,
                                                             const float* prior, float* out, int64_t total) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;
  float sum = 0.f;
  for (int z = 0; z < parts; z += 8) {  // eight loads in flight
    float p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u] = part[min(z + u, parts - 1) * stride + at];
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += z + u < parts ? p[u] : 0.f;
  }
  out[at] = prior != nullptr ? prior[at] + sum : sum;
}

// ---- few rows (one token's heads) ----------------------------------------------------------------------
// Up to 16 query rows of a KV head are one matrix tile: weights_scores_kernel streams K once, a wavefront its own 32-row
// chunks (whole-row loads into its part of LDS, the next chunk's in flight), leaves the scores in the workspace, a
// fraction of K's bytes, and each split's maxima and sums; weights_from_scores_kernel joins those and adds up. One row of 28 / 4
// heads of 128 over 8257: 8.4 us in the place of 28 by the passes above. Up to 1024 cache rows one workgroup a head keeps its
// scores in LDS and is the whole call (eager calls, which the host's launches bound: 9.3 -> 4.9 us, 7.9 at 1000 rows).
// WHOLE: one workgroup of W wavefronts takes a head's whole cache, of at most kWtWholeRows rows: the scores stay in LDS and it
// adds them up itself.
template <int D, int W, bool WHOLE>
__global__ __launch_bounds__(W * 64) void weights_scores_kernel(
    const int64_t* __restrict__ pos, int N, int rows, int group, const char* __restrict__ kc, int64_t k_hs_b,
    const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b, float scale_log2, int split_chunks, int splits,
    float* __restrict__ scores, int64_t score_stride, float2* __restrict__ part, const float* prior, float* out,
    int32_t* __restrict__ err) {
  constexpr int DS = D / 32, CPR = D / 8, ROWB = D * 2, CH = 32, LI = CH * CPR / 64;
  constexpr int PITCH = kWtWholeRows + 4;  // of a row's scores in LDS
  __shared__ __attribute__((aligned(1024))) char lds[W * CH * ROWB];
  __shared__ __attribute__((aligned(16))) float s_scores[WHOLE ? kWtFewRows * PITCH : 4];
  __shared__ float s_lse[kWtFewRows];
  __shared__ int s_pos[kWtFewRows];
  __shared__ float2 s_ml[W][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  const int z = blockIdx.x, hk = blockIdx.y;
  const char* kh = kc + (int64_t)hk * k_hs_b;
  vec16 kr[LI];
  auto load = [&](int c) {  // rows past the cache load its last one
    c = min(c, (N - 1) / CH);
    const char* base = kh + (int64_t)c * (CH * ROWB);
    const int last = N - 1 - c * CH;
#pragma unroll
    for (int i = 0; i < LI; ++i) kr[i] = ld16(base + min((i * 64 + lane) / CPR, last) * ROWB + (lane % CPR) * 16);
  };
  const int begin = z * split_chunks;
  int c = begin + wave;
  load(c);
  const int r = min(lm, rows - 1), t = r / group;
  const char* qr = q + (int64_t)(hk * group + r - t * group) * q_hs_b + (int64_t)t * q_ts_b;
  bf16x8 qf[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) qf[ds] = __builtin_bit_cast(bf16x8, ld16(qr + (32 * ds + 8 * g) * 2));
  const int64_t p64 = pos[t];
  const int p = p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64;
  if (p != p64 && lm < rows) flag_error(err, CKV_DEVICE_ERR_RANGE);
  const int wmax = __builtin_amdgcn_readfirstlane(row16_reduce(p, [](int a, int b) { return max(a, b); }));
  const int wmin = __builtin_amdgcn_readfirstlane(row16_reduce(p, [](int a, int b) { return min(a, b); }));
  const int c_end = min(wmax / CH + 1, begin + split_chunks);
  char* wl = lds + wave * CH * ROWB;
  float m_run = -INFINITY, l_run = 0.f;
  float* srow = WHOLE ? s_scores + lm * PITCH : scores + (int64_t)(hk * rows + r) * score_stride;
  for (; c < c_end; c += W) {
    wave_lds_stage();
#pragma unroll
    for (int i = 0; i < LI; ++i) {
      const int slot = (i * 64 + lane) / CPR;
      *(vec16*)(wl + slot * ROWB + (((lane % CPR) ^ swz_k<CPR>(slot)) * 16)) = kr[i];
    }
    if (c + W < c_end) load(c + W);  // lands while this chunk is worked on
    wave_lds_stage();
    const int n0 = c * CH;
    f32x4 s[2];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int slot = 16 * h + lm;
        const bf16x8 a = *(const bf16x8*)(wl + slot * ROWB + (((4 * ds + g) ^ swz_k<CPR>(slot)) * 16));
        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[ds], ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[h], 0, 0, 0);
      }
    // lane (g, lm): row lm, cache rows n0 + 16 h + 4 g + e
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] *= scale_log2;
      if (lm < rows) *(f32x4*)(srow + n0 + 16 * h + 4 * g) = s[h];
    }
    if (n0 + CH - 1 > wmin) {
      const int lim = p - n0 - 4 * g;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * h + e > lim) s[h][e] = -INFINITY;
    }
    float bm = s[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) bm = fmaxf(bm, s[j / 4][j % 4]);
    const float m_new = fmaxf(m_run, bm), sub = m_new == -INFINITY ? 0.f : m_new;
    l_run *= __builtin_amdgcn_exp2f(m_run - sub);  // 0 while m_run is -inf
#pragma unroll
    for (int j = 0; j < 8; ++j) l_run += __builtin_amdgcn_exp2f(s[j / 4][j % 4] - sub);
    m_run = m_new;
  }
  // a row's four lanes, then the wavefronts
  const float m = group_max(m_run);
  float l = m_run == -INFINITY ? 0.f : l_run * __builtin_amdgcn_exp2f(m_run - m);
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) s_ml[wave][lm] = make_float2(m, l);
  __syncthreads();
  if ((int)threadIdx.x < rows) {
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_ml[w][lm].x);
#pragma unroll
    for (int w = 0; w < W; ++w) sum += s_ml[w][lm].x == -INFINITY ? 0.f : s_ml[w][lm].y * __builtin_amdgcn_exp2f(s_ml[w][lm].x - mx);
    if constexpr (WHOLE) {
      s_lse[lm] = mx + __builtin_amdgcn_logf(sum);
      s_pos[lm] = p;
    } else {
      part[(int64_t)(hk * rows + lm) * splits + z] = make_float2(mx, sum);
    }
  }
  if constexpr (WHOLE) {
    __syncthreads();
    for (int j = threadIdx.x; j < N; j += W * 64) {
      const int64_t at = (int64_t)hk * N + j;
      float total = 0.f;
      for (int r = 0; r < rows; ++r) total += j <= s_pos[r] ? __builtin_amdgcn_exp2f(s_scores[r * PITCH + j] - s_lse[r]) : 0.f;
      out[at] = prior != nullptr ? prior[at] + total : total;
    }
  }
}


__global__ __launch_bounds__(kWtThreads) void weights_from_scores_kernel(
    const int64_t* __restrict__ pos, int N, int rows, int group, const float* __restrict__ scores, int64_t score_stride,
    const float2* __restrict__ part, int splits, const float* prior, float* out) {
  __shared__ float s_lse[kWtFewRows];
  __shared__ int s_pos[kWtFewRows];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, hk = blockIdx.y;
  const int j = blockIdx.x * kWtThreads + threadIdx.x;
  float s[kWtFewRows];
  const float* sc = scores + (int64_t)hk * rows * score_stride + min(j, N - 1);
#pragma unroll
  for (int r = 0; r < kWtFewRows; ++r)
    if (r < rows) s[r] = sc[r * score_stride];
  const float before = prior != nullptr && j < N ? prior[(int64_t)hk * N + j] : 0.f;
  for (int r = wave; r < rows; r += kWtThreads / 64) {
    const float2* pr = part + (int64_t)(hk * rows + r) * splits;
    static_assert(kWtMostParts == 128, "two splits a lane");
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 a = lane < splits ? pr[lane] : none, b = lane + 64 < splits ? pr[lane + 64] : none;
    float m = fmaxf(a.x, b.x);
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float l = wave_butterfly_sum((a.x == -INFINITY ? 0.f : a.y * __builtin_amdgcn_exp2f(a.x - m)) +
                                       (b.x == -INFINITY ? 0.f : b.y * __builtin_amdgcn_exp2f(b.x - m)));
    if (lane == 0) {
      const int64_t p64 = pos[r / group];
      s_lse[r] = m + __builtin_amdgcn_logf(l);
      s_pos[r] = p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64;
    }
  }
  __syncthreads();
  if (j >= N) return;
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < kWtFewRows; ++r)
    if (r < rows) sum += j <= s_pos[r] ? __builtin_amdgcn_exp2f(s[r] - s_lse[r]) : 0.f;
  out[(int64_t)hk * N + j] = before + sum;
}

// ---- short caches -----------------------------------------------------------------------------------------
// Up to 16 T cache rows one workgroup a KV head is the whole call: K in LDS, a wavefront 16 query rows at a time with all their
// scores in registers (lane (g, lm): row lm, cache rows 16 t + 4 g + e), so a weight is formed from the exponential that its row's sum
// took, and adds up in place over the wavefront's rows; lanes and wavefronts meet once, at the end.
template <int D, int T>
__global__ __launch_bounds__(kWtShortWaves * 64) void weights_short_kernel(
    const int64_t* __restrict__ pos, int N, int rows, int group, uint32_t inv_gqa, const char* __restrict__ kc, int64_t k_hs_b,
    const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b, float scale_log2, const float* prior, float* out,
    int32_t* __restrict__ err) {
  constexpr int W = kWtShortWaves, DS = D / 32, CPR = D / 8, ROWB = D * 2, LI = T * 16 * CPR / (W * 64);
  static_assert(LI >= 1 && T * 16 * CPR % (W * 64) == 0 && T % 4 == 0, "whole loads");
  __shared__ __attribute__((aligned(1024))) char lds[T * 16 * ROWB];
  __shared__ float s_part[W][T * 16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16, hk = blockIdx.x;
  const char* kh = kc + (int64_t)hk * k_hs_b;
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int P = (wave * LI + i) * 64 + lane, slot = P / CPR;
    const uint32_t off = (uint32_t)(min(slot, N - 1) * ROWB + ((P % CPR) ^ swz_k<CPR>(slot)) * 16);
    __builtin_amdgcn_global_load_lds((wt_gvoid*)(kh + off), (wt_lvoid*)(lds + (wave * LI + i) * 1024), 16, 0, 0);
  }
  bf16x8 qf[DS];
  int my_pos;
  auto load_rows = [&](int r0) {
    const int r = r0 + lm, rc = min(r, rows - 1), t = div_by(rc, group, inv_gqa), gh = rc - t * group;
    const char* qr = q + (int64_t)(hk * group + gh) * q_hs_b + (int64_t)t * q_ts_b;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[ds] = __builtin_bit_cast(bf16x8, ld16(qr + (32 * ds + 8 * g) * 2));
    const int64_t p64 = pos[t];
    const int p = p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64;
    if (r < rows && p != p64) flag_error(err, CKV_DEVICE_ERR_RANGE);
    my_pos = r < rows ? p : -1;
  };
  load_rows(wave * 16);
  int k_rd[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) k_rd[ds] = lm * ROWB + (((4 * ds + g) ^ swz_k<CPR>(lm)) * 16);
  f32x4 acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's part of K landed
  __syncthreads();
  for (int r0 = wave * 16; r0 < rows; r0 += W * 16) {
    f32x4 s[T];
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < T; u += 4) {
      if (16 * u >= N) continue;  // uniform
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)  // dependent products four apart
#pragma unroll
        for (int t = u; t < u + 4; ++t)
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)(lds + t * 16 * ROWB + k_rd[ds]), qf[ds],
                                                         ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[t], 0, 0, 0);
#pragma unroll
      for (int t = u; t < u + 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (16 * t + 4 * g + e > my_pos) s[t][e] = -INFINITY;
          m = fmaxf(m, s[t][e]);
        }
    }
    if (r0 + W * 16 < rows) load_rows(r0 + W * 16);
    m = group_max(m) * scale_log2;  // > 0: max commutes
    const float sub = m == -INFINITY ? 0.f : m;  // no such row
    float l = 0.f;
#pragma unroll
    for (int u = 0; u < T; u += 4) {
      if (16 * u >= N) continue;
#pragma unroll
      for (int t = u; t < u + 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], scale_log2, -sub));
          l += s[t][e];
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int u = 0; u < T; u += 4) {
      if (16 * u >= N) continue;
#pragma unroll
      for (int t = u; t < u + 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(s[t][e], inv, acc[t][e]);
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    if (16 * t >= N) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float sum = row16_reduce(acc[t][e], [](float a, float b) { return a + b; });
      if (lm == 0) s_part[wave][16 * t + 4 * g + e] = sum;
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < N; j += W * 64) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) total += s_part[w][j];
    const int64_t at = (int64_t)hk * N + j;
    out[at] = prior != nullptr ? prior[at] + total : total;
  }
}

template <int I>
using Int = std::integral_constant<int, I>;

}  // namespace ckv

extern "C" int64_t ckv_attention_weights_workspace_bytes(int32_t n_queries, int32_t n_tokens, int32_t n_q_heads,
                                                         int32_t n_kv_heads, int32_t head_dim) {
  using namespace ckv;
  if (n_queries <= 0 || n_tokens <= 0 || n_kv_heads <= 0 || n_q_heads <= 0 || head_dim <= 0 || n_q_heads % n_kv_heads ||
      (int64_t)n_queries * (n_q_heads / n_kv_heads) > INT32_MAX / 2)
    return 0;
  if (n_queries * (n_q_heads / n_kv_heads) <= kWtFewRows && n_tokens <= kWtWholeRows) return 0;
  if (n_queries * (n_q_heads / n_kv_heads) <= kWtFewRows) return few_plan(n_queries * (n_q_heads / n_kv_heads), n_tokens, n_kv_heads).bytes;
  if (short_cache(n_queries * (n_q_heads / n_kv_heads), n_tokens)) return 0;
  const WeightsPlan p = weights_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim);
  return p.stat_bytes + (int64_t)n_kv_heads * p.stat_rows * head_dim * 2 +
         (p.join ? p.part_bytes + p.sum_bytes : std::max(p.part_bytes, p.sum_bytes));
}

extern "C" int32_t ckv_attention_weights(float* out, const float* prior, const void* q, int64_t q_head_stride,
                                         int64_t q_token_stride, const void* k_cache, int64_t k_head_stride,
                                         const int64_t* positions, int32_t n_queries, int32_t n_tokens,
                                         int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                                         double scale, void* workspace, int64_t workspace_bytes, int32_t* err,
                                         void* stream) {
  using namespace ckv;
  if (out == nullptr) return CKV_ERR_INVALID_ARGUMENT;
  if (dtype != CKV_DTYPE_BF16 || (head_dim != 64 && head_dim != 128)) return CKV_ERR_INVALID_ARGUMENT;
  if (n_queries < 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || log2_scale(scale) == 0.f)
    return CKV_ERR_INVALID_ARGUMENT;
  const int group = n_q_heads / n_kv_heads;
  hipStream_t s = (hipStream_t)stream;
  const int64_t total = (int64_t)n_kv_heads * n_tokens;
  const unsigned total_blocks = (unsigned)((total + 255) / 256);
  if (prior != nullptr && prior != out) {  // one buffer or two: a workgroup's sums would meet another's prior
    const intptr_t apart = (intptr_t)prior - (intptr_t)out;
    if ((apart < 0 ? -apart : apart) < total * 4) return CKV_ERR_INVALID_ARGUMENT;
  }
  if (n_queries == 0) {  // no query: prior, or zeros
    if (prior == out) return CKV_OK;
    hipLaunchKernelGGL(weights_reduce_kernel, dim3(total_blocks), dim3(256), 0, s, (const float*)nullptr, (int64_t)0, 0, prior, out, total);
    CKV_RETURN_IF_LAUNCH_FAILED();
    return CKV_OK;
  }
  if (q == nullptr || k_cache == nullptr || positions == nullptr) return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride % 8 || q_head_stride % 8 || k_head_stride % 8) return CKV_ERR_INVALID_ARGUMENT;  // 16-byte rows
  if (((uintptr_t)q | (uintptr_t)k_cache) % 16) return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride < head_dim || k_head_stride < (int64_t)n_tokens * head_dim) return CKV_ERR_OUT_OF_RANGE;
  if ((int64_t)n_queries * group > INT32_MAX / 2 || n_kv_heads > 65535) return CKV_ERR_TOO_LARGE;
  const int64_t need = ckv_attention_weights_workspace_bytes(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim);
  if (need > 0 && (workspace == nullptr || (uintptr_t)workspace % 16 || workspace_bytes < need)) return CKV_ERR_INVALID_ARGUMENT;
  const float scale_log2 = log2_scale(scale);
  if (n_queries * group <= kWtFewRows) {
    const bool whole = n_tokens <= kWtWholeRows;
    const FewPlan p = few_plan(n_queries * group, n_tokens, n_kv_heads);
    float* scores = (float*)workspace;
    float2* part = (float2*)((char*)workspace + p.score_bytes);
    auto launch = [&](auto kernel, int splits, int waves) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)splits, (unsigned)n_kv_heads), dim3(waves * 64), 0, s, positions, n_tokens, p.rows,
                         group, (const char*)k_cache, k_head_stride * 2, (const char*)q, q_head_stride * 2, q_token_stride * 2,
                         scale_log2, whole ? p.chunks : p.split_chunks, p.splits, scores, p.score_stride, part, prior, out, err);
    };
    if (whole) {
      if (head_dim == 128) launch(weights_scores_kernel<128, kWtWholeWaves, true>, 1, kWtWholeWaves);
      else launch(weights_scores_kernel<64, kWtWholeWaves, true>, 1, kWtWholeWaves);
      CKV_RETURN_IF_LAUNCH_FAILED();
      return CKV_OK;
    }
    if (head_dim == 128) launch(weights_scores_kernel<128, 4, false>, p.splits, 4);
    else launch(weights_scores_kernel<64, 4, false>, p.splits, 4);
    CKV_RETURN_IF_LAUNCH_FAILED();
    hipLaunchKernelGGL(weights_from_scores_kernel, dim3((unsigned)((n_tokens + kWtThreads - 1) / kWtThreads), (unsigned)n_kv_heads),
                       dim3(kWtThreads), 0, s, positions, n_tokens, p.rows, group, (const float*)scores, p.score_stride,
                       (const float2*)part, p.splits, prior, out);
    CKV_RETURN_IF_LAUNCH_FAILED();
    return CKV_OK;
  }
  if (short_cache(n_queries * group, n_tokens)) {
    const int rows = n_queries * group;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)n_kv_heads), dim3(kWtShortWaves * 64), 0, s, positions, n_tokens, rows, group,
                         inverse_of(rows, group), (const char*)k_cache, k_head_stride * 2, (const char*)q, q_head_stride * 2,
                         q_token_stride * 2, scale_log2, prior, out, err);
    };
    if (head_dim == 128) n_tokens <= 64 ? launch(weights_short_kernel<128, 4>) : launch(weights_short_kernel<128, 16>);
    else n_tokens <= 64 ? launch(weights_short_kernel<64, 4>) : launch(weights_short_kernel<64, 16>);
    CKV_RETURN_IF_LAUNCH_FAILED();
    return CKV_OK;
  }
  const WeightsPlan p = weights_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim);
  const uint32_t inv_gqa = inverse_of(p.rows, group);
  RowStat* stat = (RowStat*)workspace;
  char* packed = (char*)workspace + p.stat_bytes;
  float* scratch = (float*)(packed + (int64_t)n_kv_heads * p.stat_rows * head_dim * 2);  // the splits' rows, then the parts' sums
  float* sums = scratch + (p.join ? p.part_bytes / 4 : 0);  // the joined splits are read while the sums are written
  const int64_t rows_total = (int64_t)n_kv_heads * p.stat_rows;
  {
    const AttnMap m = attn_map(p.row_blocks, n_kv_heads, 1, p.splits);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(m.blocks), dim3(kWtThreads), 0, s, m.nqb, m.group, m.xpk_log, m.items, m.inv_group,
                         m.inv_nqb, positions, n_tokens, p.rows, group, inv_gqa, (const char*)k_cache, k_head_stride * 2,
                         (const char*)q, q_head_stride * 2, q_token_stride * 2, scale_log2, stat, packed, p.stat_rows, (float2*)scratch,
                         rows_total, p.split_tiles, err);
    };
    auto form = [&](auto dim, auto qg) {
      constexpr int D = decltype(dim)::value, QG = decltype(qg)::value;
      p.splits > 1 ? launch(weights_lse_kernel<D, QG, true>) : launch(weights_lse_kernel<D, QG, false>);
    };
    if (head_dim == 128) p.qg == 1 ? form(Int<128>{}, Int<1>{}) : form(Int<128>{}, Int<2>{});
    else p.qg == 1 ? form(Int<64>{}, Int<1>{}) : form(Int<64>{}, Int<2>{});
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  if (p.splits > 1 && !p.join) {
    hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)((rows_total + 3) / 4)), dim3(256), 0, s, (const float2*)scratch,
                       rows_total, p.splits, positions, n_tokens, p.rows, group, stat, p.stat_rows, rows_total);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  {
    const AttnMap m = attn_map(p.key_blocks, n_kv_heads, 1, p.parts);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(m.blocks), dim3(kWtThreads), 0, s, m.nqb, m.group, m.xpk_log, m.items, m.inv_group,
                         m.inv_nqb, n_tokens, p.stat_rows, (const char*)k_cache, k_head_stride * 2, (const char*)packed, scale_log2,
                         (const RowStat*)stat, prior,
                         p.parts > 1 ? sums : out, total, p.part_tiles,
                         WeightsJoin{(const float2*)scratch, rows_total, p.splits, positions, p.rows, group});
    };
    auto form = [&](auto dim, auto kg) {
      constexpr int D = decltype(dim)::value, KG = decltype(kg)::value;
      if (p.join) p.parts > 1 ? launch(weights_sum_kernel<D, KG, true, true>) : launch(weights_sum_kernel<D, KG, false, true>);
      else p.parts > 1 ? launch(weights_sum_kernel<D, KG, true, false>) : launch(weights_sum_kernel<D, KG, false, false>);
    };
    if (head_dim == 128) p.kg == 1 ? form(Int<128>{}, Int<1>{}) : form(Int<128>{}, Int<2>{});
    else p.kg == 1 ? form(Int<64>{}, Int<1>{}) : form(Int<64>{}, Int<2>{});
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  if (p.parts > 1) {
    hipLaunchKernelGGL(weights_reduce_kernel, dim3(total_blocks), dim3(256), 0, s, sums, total, p.parts, prior, out, total);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  return CKV_OK;
}
