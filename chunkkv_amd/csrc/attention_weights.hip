// The attention weight that each cached row received, summed over query rows and the query heads of its KV head:
//   out[hk, j] = prior[hk, j] + sum over i, h in group hk of softmax_j(scale * q[h, i] . K[hk, j]),  j <= pos[i],
// what a cache's rows are ranked by before the light ones are dropped (evict.hip). Neither the scores nor the
// weights go to memory.
//
// Design: the n x group (token, query head) pairs of a KV head are its rows. A weight needs its row's maximum
// and sum before it can be formed, so the product with K^T runs twice:
//  1. weights_lse_kernel: 128 rows a workgroup walk the cache in 64-row tiles (attention.hip's first half, with the
//     maximum and the sum kept per lane); with few row blocks, in splits of the cache. Leaves L = max + log2(sum) and the
//     position of each row (weights_join_kernel joins the splits).
//  2. weights_sum_kernel: 128 cache rows a workgroup hold their operands in registers while the query rows pass
//     through LDS: S = K Q^T gives a lane four cache rows of one query row, and 2^(s scale - L) adds up in
//     registers over all query rows; the 16 lanes of a cache row meet once, at the end. With few cache blocks the
//     query rows are split, and weights_reduce_kernel adds the parts in order (no atomics: the same sums every time).
// Scores and sums are fp32 throughout, products bf16 x bf16 (exact) accumulated in fp32 on the matrix cores.
#include <algorithm>

#include "attention_common.hpp"

namespace ckv {

constexpr int kWtThreads = 256;
constexpr int kWtRows = 128;   // query rows of a workgroup of the first pass, cache rows of one of the second
constexpr int kWtTile = 64;    // cache rows of a tile of the first pass, query rows of one of the second

// A query row's normaliser and position, as the second pass reads it.
struct RowStat {
  float lse;  // log2 domain
  int pos;
};

typedef __attribute__((address_space(1))) void wt_gvoid;
typedef __attribute__((address_space(3))) void wt_lvoid;

// SPLIT: split z of the cache's tiles; (max, sum) of a row's split to part[z].
template <int D, bool SPLIT>
__global__ __launch_bounds__(kWtThreads) void weights_lse_kernel(
    int nqb, int map_group, int xpk_log, int items, uint32_t inv_group, uint32_t inv_nqb,
    const int64_t* __restrict__ pos, int N, int rows, int group, uint32_t inv_gqa, const char* __restrict__ kc,
    int64_t k_hs_b, const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b, float scale_log2,
    RowStat* __restrict__ stat, float2* __restrict__ part, int64_t part_stride, int split_tiles,
    int32_t* __restrict__ err) {
  constexpr int DS = D / 32, CPR = D / 8, ROWB = D * 2, QG = 2, KI = kWtTile * CPR / kWtThreads;
  __shared__ __attribute__((aligned(1024))) char lds0[kWtTile * ROWB];
  __shared__ __attribute__((aligned(1024))) char lds1[kWtTile * ROWB];
  __shared__ int blk_max_s[kWtThreads / 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  int rb, hk, z;
  if (!attn_work_item(nqb, map_group, xpk_log, items, inv_group, inv_nqb, rb, hk, z)) return;
  int my_pos[QG];
  int wmax = -1, wmin = N;
  bf16x8 qf[QG][DS];
#pragma unroll
  for (int qg = 0; qg < QG; ++qg) {
    const int r = rb * kWtRows + wave * 32 + qg * 16 + lm;
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
  if (lane == 0) blk_max_s[wave] = wmax;
  __syncthreads();
  int bmax = blk_max_s[0];
#pragma unroll
  for (int w = 1; w < kWtThreads / 64; ++w) bmax = max(bmax, blk_max_s[w]);
  bmax = __builtin_amdgcn_readfirstlane(bmax);
  int n_tiles = bmax / kWtTile + 1;  // a block has a row: bmax >= 0
  const int tile_begin = SPLIT ? z * split_tiles : 0;
  if (SPLIT) n_tiles = min(n_tiles, tile_begin + split_tiles);

  // A lane's own maximum and sum over the cache rows that it gets.
  float m_run[QG], l_run[QG];
#pragma unroll
  for (int qg = 0; qg < QG; ++qg) {
    m_run[qg] = -INFINITY;
    l_run[qg] = 0.f;
  }
  const char* kh = kc + (int64_t)hk * k_hs_b;
  int off[KI];
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int P = (wave * KI + i) * 64 + lane, slot = P / CPR;
    off[i] = slot * ROWB + ((P % CPR) ^ swz_k<CPR>(slot)) * 16;
  }
  auto issue = [&](int n0, char* kb) {
    const char* kt = kh + (int64_t)n0 * ROWB;
    const int last = bmax - n0;  // rows past every position load the last one's
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int o = min(off[i] / ROWB, last) * ROWB + off[i] % ROWB;
      __builtin_amdgcn_global_load_lds((wt_gvoid*)(kt + (uint32_t)o), (wt_lvoid*)(kb + (wave * KI + i) * 1024), 16, 0, 0);
    }
  };
  int k_rd[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) k_rd[ds] = lm * ROWB + (((4 * ds + g) ^ swz_k<CPR>(lm)) * 16);
  if (tile_begin < n_tiles) issue(tile_begin * kWtTile, lds0);
  auto body = [&](int tile, const char* cur, char* nxt) {
    const int n0 = tile * kWtTile;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's loads of the tile landed
    __syncthreads();
    if (tile + 1 < n_tiles) issue(n0 + kWtTile, nxt);
    if (n0 > wmax) return;  // uniform per wavefront
    const bool need_mask = n0 + kWtTile - 1 > wmin;
    constexpr int T = kWtTile / 16;
    f32x4 s[QG][T];  // lane (g, lm): query lm, cache rows n0 + 16 t + 4 g + e
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const bf16x8 a = *(const bf16x8*)(cur + t * 16 * ROWB + k_rd[ds]);
#pragma unroll
        for (int qg = 0; qg < QG; ++qg)
          s[qg][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[qg][ds], ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[qg][t], 0, 0, 0);
      }
#pragma unroll
    for (int qg = 0; qg < QG; ++qg) {
      if (need_mask) {
        const int lim = my_pos[qg] - n0 - 4 * g;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * t + e > lim) s[qg][t][e] = -INFINITY;
      }
      float bm = -INFINITY;
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) bm = fmaxf(bm, s[qg][t][e]);
      bm *= scale_log2;  // > 0: max commutes
      // raised only by more than 2^8, which the sum's fp32 range takes
      if (__builtin_amdgcn_ballot_w64(bm > m_run[qg] + 8.f)) {
        const float m_new = bm > m_run[qg] + 8.f ? bm : m_run[qg];
        l_run[qg] *= m_run[qg] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[qg] - m_new);
        m_run[qg] = m_new;
      }
      const float sub = m_run[qg] == -INFINITY ? 0.f : m_run[qg];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          l_run[qg] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[qg][t][e], scale_log2, -sub));
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
    const int r = rb * kWtRows + wave * 32 + qg * 16 + lm;
    if (r >= rows || g != 0) continue;
    const int64_t at = (int64_t)hk * rows + r;
    if (SPLIT) part[z * part_stride + at] = make_float2(m, l);
    else stat[at] = RowStat{m + __builtin_amdgcn_logf(l), my_pos[qg]};
  }
}

// Joins the splits of the first pass, a row a thread.
__global__ __launch_bounds__(256) void weights_join_kernel(const float2* __restrict__ part, int64_t stride, int splits,
                                                           const int64_t* __restrict__ pos, int N, int rows, int group,
                                                           RowStat* __restrict__ stat, int64_t total) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;
  float m = -INFINITY, l = 0.f;
  for (int z = 0; z < splits; ++z) {
    const float2 p = part[z * stride + at];
    if (p.x == -INFINITY) continue;
    const float mn = fmaxf(m, p.x);
    l = l * __builtin_amdgcn_exp2f(m - mn) + p.y * __builtin_amdgcn_exp2f(p.x - mn);
    m = mn;
  }
  const int64_t p64 = pos[(int)(at % rows) / group];
  stat[at] = RowStat{m + __builtin_amdgcn_logf(l), p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64};
}

// PARTS: part z of the query rows; sums to ws[z], else prior + sum to out.
template <int D, bool PARTS>
__global__ __launch_bounds__(kWtThreads) void weights_sum_kernel(
    int nkb, int map_group, int xpk_log, int items, uint32_t inv_group, uint32_t inv_nkb, int N, int rows, int group,
    uint32_t inv_gqa, const char* __restrict__ kc, int64_t k_hs_b, const char* __restrict__ q, int64_t q_hs_b,
    int64_t q_ts_b, float scale_log2, const RowStat* __restrict__ stat, const float* prior, float* out,
    int64_t part_stride, int part_tiles) {
  constexpr int DS = D / 32, CPR = D / 8, ROWB = D * 2, KG = 2, KI = kWtTile * CPR / kWtThreads, QT = kWtTile / 16;
  __shared__ __attribute__((aligned(1024))) char lds0[kWtTile * ROWB];
  __shared__ __attribute__((aligned(1024))) char lds1[kWtTile * ROWB];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  int kb, hk, z;
  if (!attn_work_item(nkb, map_group, xpk_log, items, inv_group, inv_nkb, kb, hk, z)) return;
  kb = nkb - 1 - kb;  // the first cache rows, which the most queries see, first
  const RowStat* st = stat + (int64_t)hk * rows;
  const int tile_begin = PARTS ? z * part_tiles : 0;
  const int tiles = (rows + kWtTile - 1) / kWtTile;
  const int tile_end = PARTS ? min(tiles, tile_begin + part_tiles) : tiles;
  const int k0 = kb * kWtRows + wave * 32;  // this wavefront's cache rows

  // does any query row of the part see these cache rows?
  int seen = -1;
  for (int r = tile_begin * kWtTile + (int)threadIdx.x; r < min(tile_end * kWtTile, rows); r += kWtThreads) seen = max(seen, st[r].pos);
  const bool any = __syncthreads_or(seen >= kb * kWtRows);

  f32x4 acc[KG];
#pragma unroll
  for (int kg = 0; kg < KG; ++kg) acc[kg] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (any) {
    const char* kh = kc + (int64_t)hk * k_hs_b;
    bf16x8 kf[KG][DS];
#pragma unroll
    for (int kg = 0; kg < KG; ++kg)
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
        kf[kg][ds] = __builtin_bit_cast(bf16x8, ld16(kh + (int64_t)min(k0 + 16 * kg + lm, N - 1) * ROWB + (32 * ds + 8 * g) * 2));
    const char* qh = q + (int64_t)hk * group * q_hs_b;
    RowStat nx[QT];
    auto issue = [&](int tile, char* qb) {
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int P = (wave * KI + i) * 64 + lane, slot = P / CPR;
        const int r = min(tile * kWtTile + slot, rows - 1), t = div_by(r, group, inv_gqa);
        const char* src = qh + (int64_t)(r - t * group) * q_hs_b + (int64_t)t * q_ts_b + ((P % CPR) ^ swz_k<CPR>(slot)) * 16;
        __builtin_amdgcn_global_load_lds((wt_gvoid*)src, (wt_lvoid*)(qb + (wave * KI + i) * 1024), 16, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int r = tile * kWtTile + t * 16 + lm;
        nx[t] = st[min(r, rows - 1)];
        if (r >= rows) nx[t].pos = -1;
      }
    };
    int q_rd[DS];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) q_rd[ds] = lm * ROWB + (((4 * ds + g) ^ swz_k<CPR>(lm)) * 16);
    issue(tile_begin, lds0);
    auto body = [&](int tile, const char* cur, char* nxt) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
      RowStat now[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) now[t] = nx[t];
      if (tile + 1 < tile_end) issue(tile + 1, nxt);
      int top = now[0].pos, low = now[0].pos;
#pragma unroll
      for (int t = 1; t < QT; ++t) {
        top = max(top, now[t].pos);
        low = min(low, now[t].pos);
      }
      if (!__builtin_amdgcn_ballot_w64(top >= k0)) return;  // uniform per wavefront
      const bool need_mask = __builtin_amdgcn_ballot_w64(low < k0 + 31);
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        f32x4 s[KG];
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
          const bf16x8 b = *(const bf16x8*)(cur + t * 16 * ROWB + q_rd[ds]);
#pragma unroll
          for (int kg = 0; kg < KG; ++kg)
            s[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kg][ds], b, ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[kg], 0, 0, 0);
        }
        if (need_mask) {
          const int lim = now[t].pos - k0 - 4 * g;
#pragma unroll
          for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * kg + e > lim) s[kg][e] = -INFINITY;
        }
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[kg][e] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[kg][e], scale_log2, -now[t].lse));
      }
    };
    for (int tile = tile_begin; tile < tile_end; tile += 2) {
      body(tile, lds0, lds1);
      if (tile + 1 < tile_end) body(tile + 1, lds1, lds0);
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
  for (int z = 0; z < parts; ++z) sum += part[z * stride + at];
  out[at] = prior != nullptr ? prior[at] + sum : sum;
}

struct WeightsPlan {
  int rows = 0, row_blocks = 0, splits = 1, split_tiles = 0, key_blocks = 0, parts = 1, part_tiles = 0;
  int64_t stat_bytes = 0, part_bytes = 0, sum_bytes = 0;
};

static WeightsPlan weights_plan(int n, int N, int Hq, int Hkv) {
  WeightsPlan p;
  p.rows = n * (Hq / Hkv);
  p.row_blocks = (p.rows + kWtRows - 1) / kWtRows;
  const int tiles = (N + kWtTile - 1) / kWtTile, row_tiles = (p.rows + kWtTile - 1) / kWtTile;
  p.key_blocks = (N + kWtRows - 1) / kWtRows;
  const int64_t lse_blocks = (int64_t)p.row_blocks * Hkv, sum_blocks = (int64_t)p.key_blocks * Hkv;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({512 / lse_blocks, tiles / 2, 64}));
  p.split_tiles = (int)((tiles + splits - 1) / splits);
  p.splits = (tiles + p.split_tiles - 1) / p.split_tiles;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(2048 / sum_blocks, row_tiles / 4));
  p.part_tiles = (int)((row_tiles + parts - 1) / parts);
  p.parts = (row_tiles + p.part_tiles - 1) / p.part_tiles;
  const int64_t total = (int64_t)Hkv * p.rows;
  p.stat_bytes = (total * (int64_t)sizeof(RowStat) + 15) / 16 * 16;
  p.part_bytes = p.splits > 1 ? (total * 8 * p.splits + 15) / 16 * 16 : 0;
  p.sum_bytes = p.parts > 1 ? (int64_t)Hkv * N * 4 * p.parts : 0;
  return p;
}

}  // namespace ckv

extern "C" int64_t ckv_attention_weights_workspace_bytes(int32_t n_queries, int32_t n_tokens, int32_t n_q_heads,
                                                         int32_t n_kv_heads) {
  using namespace ckv;
  if (n_queries <= 0 || n_tokens <= 0 || n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads ||
      (int64_t)n_queries * (n_q_heads / n_kv_heads) > INT32_MAX / 2)
    return 0;
  const WeightsPlan p = weights_plan(n_queries, n_tokens, n_q_heads, n_kv_heads);
  return p.stat_bytes + std::max(p.part_bytes, p.sum_bytes);
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
  if (n_queries < 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || !(scale > 0.0))
    return CKV_ERR_INVALID_ARGUMENT;
  const int group = n_q_heads / n_kv_heads;
  hipStream_t s = (hipStream_t)stream;
  const int64_t total = (int64_t)n_kv_heads * n_tokens;
  const unsigned total_blocks = (unsigned)((total + 255) / 256);
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
  if ((int64_t)n_queries * group > INT32_MAX / 2) return CKV_ERR_TOO_LARGE;
  if (workspace == nullptr || (uintptr_t)workspace % 16 ||
      workspace_bytes < ckv_attention_weights_workspace_bytes(n_queries, n_tokens, n_q_heads, n_kv_heads))
    return CKV_ERR_INVALID_ARGUMENT;
  const WeightsPlan p = weights_plan(n_queries, n_tokens, n_q_heads, n_kv_heads);
  const float scale_log2 = (float)(scale * 1.4426950408889634);  // exp(x) = exp2(x log2 e)
  const uint32_t inv_gqa = inverse_of(p.rows, group);
  RowStat* stat = (RowStat*)workspace;
  float* scratch = (float*)((char*)workspace + p.stat_bytes);  // the splits' rows, then the parts' sums
  const int64_t rows_total = (int64_t)n_kv_heads * p.rows;
  {
    const AttnMap m = attn_map(p.row_blocks, n_kv_heads, 1, p.splits);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(m.blocks), dim3(kWtThreads), 0, s, m.nqb, m.group, m.xpk_log, m.items, m.inv_group,
                         m.inv_nqb, positions, n_tokens, p.rows, group, inv_gqa, (const char*)k_cache, k_head_stride * 2,
                         (const char*)q, q_head_stride * 2, q_token_stride * 2, scale_log2, stat, (float2*)scratch,
                         rows_total, p.split_tiles, err);
    };
    if (head_dim == 128) p.splits > 1 ? launch(weights_lse_kernel<128, true>) : launch(weights_lse_kernel<128, false>);
    else p.splits > 1 ? launch(weights_lse_kernel<64, true>) : launch(weights_lse_kernel<64, false>);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  if (p.splits > 1) {
    hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)((rows_total + 255) / 256)), dim3(256), 0, s, (const float2*)scratch,
                       rows_total, p.splits, positions, n_tokens, p.rows, group, stat, rows_total);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  {
    const AttnMap m = attn_map(p.key_blocks, n_kv_heads, 1, p.parts);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(m.blocks), dim3(kWtThreads), 0, s, m.nqb, m.group, m.xpk_log, m.items, m.inv_group,
                         m.inv_nqb, n_tokens, p.rows, group, inv_gqa, (const char*)k_cache, k_head_stride * 2, (const char*)q,
                         q_head_stride * 2, q_token_stride * 2, scale_log2, (const RowStat*)stat, prior,
                         p.parts > 1 ? scratch : out, total, p.part_tiles);
    };
    if (head_dim == 128) p.parts > 1 ? launch(weights_sum_kernel<128, true>) : launch(weights_sum_kernel<128, false>);
    else p.parts > 1 ? launch(weights_sum_kernel<64, true>) : launch(weights_sum_kernel<64, false>);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  if (p.parts > 1) {
    hipLaunchKernelGGL(weights_reduce_kernel, dim3(total_blocks), dim3(256), 0, s, (const float*)scratch, total, p.parts, prior, out, total);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  return CKV_OK;
}
