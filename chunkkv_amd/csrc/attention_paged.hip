// Attention of new tokens, one or a chunk a sequence, over a paged cache (pages.hip): query i of a sequence's c new
// tokens, of its `rows` cached ones the last c, sees its rows j <= p = rows - c + i:
//   out = sum_j w_j V[row(j)] / sum_j w_j,  w_j = exp(scale q . K[row(j)]),  row(j) = table[j / T] T + j % T
// in attention.hip's manner (scores, softmax and sums in fp32, weights rounded to bf16 for the second product).
//
//  - Tiles of 16 or 32 (token, query head) rows of a sequence's KV head, decode among them: attn_paged_kernel below.
//  - Of 128, where many tokens fill the card: attention_large.hpp's workgroups, with splits of the cache where they are
//    few. 4096 tokens over 32832 rows, 28 / 4 heads of 128, 1.67 ms: 1.08 PFLOP/s, as fast as that kernel over one
//    contiguous cache (1.83 on the card where this took 1.78).
// attention_paged.hpp says how the work is shared out, attention_paged_plan.hpp by which rule.
#include <algorithm>

#include "attention_large.hpp"

namespace ckv {

// ---- few rows of a sequence ------------------------------------------------------------------------------------
// A workgroup streams its share of the units, a unit of 128 cached rows a step of its four wavefronts, for one tile of
// 16 QG (token, query head) rows after the other: mostly a part of one sequence, or the end of one and the beginning of
// the next. Each wavefront takes every fourth chunk of 32 rows with a softmax of its own (no barrier in the loop),
// loads it straight into LDS, two stages, and the four results meet in LDS behind a tile's last chunk. A chunk lies
// within a page; the pages of a wavefront's next 64 chunks are held a chunk a lane. Bound: the cache's bytes; for one
// short sequence the chain of its loads. Traced, 28 / 4 heads of 128: one token over 8302 rows 7.1 us (17 MB; the join
// 3.9), 28 sequences' over 97000 rows together 33.0 (199 MB, 6.0 TB/s, part of them in the memory-side cache; the join
// 4.7).
template <int D, int QG, bool MANY>
__global__ __launch_bounds__(kPagedWaves * 64) void attn_paged_kernel(AttnMap map, PagedRows b, int n, const char* __restrict__ kc,
                                                                      const char* __restrict__ vc, int64_t kv_hs_b,
                                                                      const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b,
                                                                      int Hq, int group, float scale_log2, char* __restrict__ out,
                                                                      float* __restrict__ ws) {
  constexpr int W = kPagedWaves, CH = kWaveChunk, DS = D / 32, DT = D / 16, CPR = D / 8, ROWB = D * 2, ROWS = 16 * QG;
  constexpr int LI = CH * CPR / 64;  // 1 KB loads of K, and of V, a chunk
  constexpr int STAGE = 2 * CH * ROWB;  // of a wavefront: K rows, then V rows
  __shared__ __attribute__((aligned(1024))) char lds0[W * STAGE];
  __shared__ __attribute__((aligned(1024))) char lds1[W * STAGE];
  __shared__ float s_m[W][ROWS], s_l[W][ROWS];
  static_assert(W * STAGE >= W * ROWS * D * 4, "partial rows take a stage's place");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  typedef __attribute__((address_space(1))) void gvoid;
  typedef __attribute__((address_space(3))) void lvoid;
  int g_share, hk, unused;
  if (!attn_work_item(map.nqb, map.group, map.xpk_log, map.items, map.inv_group, map.inv_nqb, g_share, hk, unused)) return;
  g_share = map.nqb - 1 - g_share;
  const PagedShare<ROWS, kPagedUnit, MANY> shares(b, n, group);
  const uint32_t share = shares.share, begin_at = shares.apart ? (uint32_t)g_share : (uint32_t)g_share * share;
  const uint32_t end_at = begin_at + (shares.apart ? 1 : share);
  const char* kh = kc + (int64_t)hk * kv_hs_b;
  const char* vh = vc + (int64_t)hk * kv_hs_b;
  int off_k[LI], off_v[LI];
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int P = i * 64 + lane, slot = P / CPR, pc = P % CPR;
    off_k[i] = kslot_row(slot) * ROWB + (pc ^ swz_k<CPR>(slot)) * 16;
    off_v[i] = slot * ROWB + (pc ^ swz_v<CPR>(slot)) * 16;
  }
  PagedSeq it;
  for (uint32_t at = begin_at; at < end_at && shares.part(at, it);) {  // uniform
    const uint32_t parts = shares.parts_of(it), local = at - it.before;
    const uint32_t tile = parts == 1 ? local : it.tiles == 1 ? 0 : local / parts, from = local - tile * parts;
    // units [u0, u1) of the tile
    const uint32_t u0 = shares.apart ? from * share : from;
    const uint32_t u1 = min((uint32_t)it.units, shares.apart ? u0 + share : u0 + (end_at - at));
    const bool whole = u0 == 0 && u1 == (uint32_t)it.units;
    const int slot = 2 * g_share + (at != begin_at);
    at += shares.apart ? 1 : u1 - u0;
    const int rows = it.count * group, r0 = (int)tile * ROWS;

    // Positions of this lane's rows; -1: no row, or none that it sees.
    int my_pos[QG], wmax = -1, wmin = it.rows;
#pragma unroll
    for (int qg = 0; qg < QG; ++qg) {
      const int m = r0 + qg * 16 + lm;
      my_pos[qg] = -1;
      if (m < rows) {
        my_pos[qg] = max(it.rows - it.count + div_by(m, group, b.inv_gqa), -1);
        wmin = min(wmin, my_pos[qg]);
      }
      wmax = max(wmax, my_pos[qg]);
    }
    wmax = __builtin_amdgcn_readfirstlane(row16_reduce(wmax, [](int x, int y) { return max(x, y); }));
    wmin = __builtin_amdgcn_readfirstlane(row16_reduce(wmin, [](int x, int y) { return min(x, y); }));
    int c_end = wmax < 0 ? 0 : wmax / CH + 1;
    if (!whole) c_end = min(c_end, (int)u1 * W);

    const int32_t* table = b.table + (int64_t)it.seq * b.M;
    int c = (int)u0 * W + wave;
    int pages = 0, step = 0;
    auto load_pages = [&](int c) {
      pages = paged_page(b, table, (int)min(((int64_t)c + lane * W) * CH, (int64_t)wmax) >> b.T_log);
      asm volatile("" : "+v"(pages));  // waited for here, not at every use
    };
    // Q operands: row lm of group qg, head-dim 32 ds + 8 g .. + 8.
    bf16x8 qf[QG][DS];
#pragma unroll
    for (int qg = 0; qg < QG; ++qg) {
      const int m = min(r0 + qg * 16 + lm, rows - 1), t = div_by(m, group, b.inv_gqa);
      const char* qr = q + (int64_t)(hk * group + m - t * group) * q_hs_b + (int64_t)(it.first + t) * q_ts_b;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) qf[qg][ds] = __builtin_bit_cast(bf16x8, ld16(qr + (32 * ds + 8 * g) * 2));
    }
    if (c < c_end) load_pages(c);
    auto issue = [&](int c, int step, char* to) {
      const int64_t row = ((int64_t)__builtin_amdgcn_readlane(pages, step) << b.T_log) + ((c * CH) & ((1 << b.T_log) - 1));
      const char* kt = kh + row * ROWB;
      const char* vt = vh + row * ROWB;
      char* wl = to + wave * STAGE;
      const int last = wmax - c * CH;  // >= 0; rows behind it load it: they are masked, but their zero weights meet the values
      auto load = [&](const char* t, int off, char* to) {
        __builtin_amdgcn_global_load_lds((gvoid*)(t + (uint32_t)off), (lvoid*)to, 16, 0, 0);
      };
      if (last >= CH - 1) {
#pragma unroll
        for (int i = 0; i < LI; ++i) load(kt, off_k[i], wl + i * 1024);
#pragma unroll
        for (int i = 0; i < LI; ++i) load(vt, off_v[i], wl + CH * ROWB + i * 1024);
      } else {
        auto clamp = [&](int off) { return min(off / ROWB, last) * ROWB + off % ROWB; };
#pragma unroll
        for (int i = 0; i < LI; ++i) load(kt, clamp(off_k[i]), wl + i * 1024);
#pragma unroll
        for (int i = 0; i < LI; ++i) load(vt, clamp(off_v[i]), wl + CH * ROWB + i * 1024);
      }
    };
    if (c < c_end) issue(c, 0, lds0);

    f32x4 o[QG][DT], l_acc[QG];
    float m_run[QG];
    const bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f,
                         (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int qg = 0; qg < QG; ++qg) {
      m_run[qg] = -INFINITY;
      l_acc[qg] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[qg][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto body = [&](const char* cur, char* nxt) {
      const char* kl = cur + wave * STAGE;
      const char* vl = kl + CH * ROWB;
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this chunk's rows landed
      wave_lds_stage();
      if (c + W < c_end) {
        if (++step == 64) {
          step = 0;
          load_pages(c + W);
        }
        issue(c + W, step, nxt);  // lands while this chunk is worked on
      }
      const int n0 = c * CH;
      f32x4 s[QG][2];
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int slot = 16 * t + lm;
          const bf16x8 a = *(const bf16x8*)(kl + slot * ROWB + (((4 * ds + g) ^ swz_k<CPR>(slot)) * 16));
#pragma unroll
          for (int qg = 0; qg < QG; ++qg)
            s[qg][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[qg][ds], ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[qg][t], 0, 0, 0);
        }
      const bool need_mask = n0 + CH - 1 > wmin;
      bf16x8 pb[QG];
#pragma unroll
      for (int qg = 0; qg < QG; ++qg) {
        float x[8];  // rows n0 + 8 g + j
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[qg][j / 4][j % 4];
        if (need_mask) {
          const int lim = my_pos[qg] - n0 - 8 * g;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j > lim) x[j] = -INFINITY;
        }
        float bm = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) bm = fmaxf(bm, x[j]);
        bm *= scale_log2;  // > 0: max commutes
        if (__builtin_amdgcn_ballot_w64(bm > m_run[qg] + 8.f)) {  // weights up to 2^8 need no new maximum
          bm = group_max(bm);
          const bool raise = bm > m_run[qg] + 8.f;
          const float m_new = raise ? bm : m_run[qg];
          const float alpha = m_run[qg] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[qg] - m_new);
          l_acc[qg] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[qg][dt] *= alpha;
          m_run[qg] = m_new;
        }
        const float sub = m_run[qg] == -INFINITY ? 0.f : m_run[qg];
#pragma unroll
        for (int j = 0; j < 8; ++j) pb[qg][j] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[j], scale_log2, -sub));
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 a = v_operand<CPR>(vl, dt, g, lm);
#pragma unroll
        for (int qg = 0; qg < QG; ++qg) o[qg][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[qg], o[qg][dt], 0, 0, 0);
      }
#pragma unroll
      for (int qg = 0; qg < QG; ++qg) l_acc[qg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[qg], l_acc[qg], 0, 0, 0);
      c += W;
      wave_lds_stage();
    };
    while (c < c_end) {
      body(lds0, lds1);
      if (c < c_end) body(lds1, lds0);
    }

    // Join the wavefronts: each scales its rows to the common maximum and leaves them in the first stage's place,
    // column group j of row r at j ^ r % 8 of its eighths.
#pragma unroll
    for (int qg = 0; qg < QG; ++qg)
      if (g == 0) s_m[wave][qg * 16 + lm] = m_run[qg];
    __syncthreads();  // every wavefront is past its last chunk
    float* so = reinterpret_cast<float*>(lds0);
    auto place = [](int w, int row, int col) { return (w * ROWS + row) * D + (col ^ ((row % 8) * (D / 8))); };
#pragma unroll
    for (int qg = 0; qg < QG; ++qg) {
      const int r = qg * 16 + lm;
      float mx = s_m[0][r];
#pragma unroll
      for (int w = 1; w < W; ++w) mx = fmaxf(mx, s_m[w][r]);
      const float sc = m_run[qg] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[qg] - mx);
      if (g == 0) s_l[wave][r] = l_acc[qg][0] * sc;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *(f32x4*)(so + place(wave, r, dt * 16 + 4 * g)) = o[qg][dt] * sc;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * (D / 8); i += W * 64) {
      const int r = i / (D / 8), col = (i % (D / 8)) * 8, m = r0 + r;
      if (m >= rows) break;  // later ones are later rows
      f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
      float l = 0.f, mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        x += *(const f32x4*)(so + place(w, r, col));
        y += *(const f32x4*)(so + place(w, r, col + 4));
        l += s_l[w][r];
        mx = fmaxf(mx, s_m[w][r]);
      }
      if (!whole) {
        float* prow = ws + (((int64_t)hk * 2 * b.cap + slot) * ROWS + r) * (D + 4);  // 16-byte aligned rows
        *(f32x4*)(prow + col) = x;
        *(f32x4*)(prow + col + 4) = y;
        if (col == 0) {
          prow[D] = mx;
          prow[D + 1] = l;
        }
      } else {
        const int t = div_by(m, group, b.inv_gqa);
        const float inv = it.rows - it.count + t < 0 ? 0.f : 1.f / l;  // a row that sees nothing; scores of -inf alone give NaN
        x *= inv;
        y *= inv;
        *(vec16*)(out + ((int64_t)(it.first + t) * Hq + hk * group + m - t * group) * ROWB + col * 2) =
            vec16{f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3]), f32x2_to_bf16x2_bits(y[0], y[1]),
                  f32x2_to_bf16x2_bits(y[2], y[3])};
      }
    }
    __syncthreads();  // the next tile's loads go where these results were
  }
}

// ---- the partial rows joined -----------------------------------------------------------------------------------
// D / 4 lanes have a (token, query head) row's columns, so a wavefront has JH = 64 / (D / 4) heads of a token side by
// side and nothing crosses its lanes; it goes through their partial rows, some in flight. Finding the token's items
// costs as many instructions as a few rows, and instructions are what a launch of many rows waits for, so such launches
// (WPR = 1) give a wavefront kJoinTurns times JH heads; those of few rows and more splits (WPR = 4) spread a row's
// partials over four wavefronts. Partials past the row's position are not read. Rows of tiles that were whole are
// written already. kJoinSpread: 40 partials at once. 32 in its place take a round more of 33 to 40 of them: one token
// over 8302 rows, 28 / 4 heads of 128, 11.95 us for 11.45, over 10000 12.6 for 11.9 (14 / 2 of 64 9.7 for 9.2, 9.9 for
// 9.3); with fewer or more of them they take 0.0-0.15 less (2000 rows 9.7 and 9.75, 5000 10.75 and 10.85, 12000 12.9
// and 13.05, 32000 20.1 and 20.2).
constexpr int kJoinTurns = 2, kJoinInFlight = 8, kJoinSpread = 10;
template <int D>
constexpr int kJoinHeads = 256 / D;

template <int D, int ROWS, int UNIT, int WPR, bool MANY>
__global__ __launch_bounds__(256) void join_paged_kernel(char* __restrict__ out, const float* __restrict__ ws, PagedRows b, int n,
                                                         int Hq, int group) {
  constexpr int LR = D / 4, JH = kJoinHeads<D>, U = WPR == 4 ? kJoinSpread : kJoinInFlight, TURNS = WPR == 4 ? 1 : kJoinTurns;
  constexpr bool SHARES = ROWS < kAttnBM;
  static_assert(WPR == 1 || WPR == 4, "a wavefront or a workgroup a row");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, sub = lane / LR, col = lane % LR * 4;
  const int t = WPR == 4 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
  if (t >= n) return;
  PagedItem it;
  uint32_t share = 1, splits = 0;  // splits 0: shares are not apart
  if constexpr (SHARES) {
    const PagedShare<ROWS, UNIT, MANY> shares(b, n, group);
    share = shares.share;
    if (!shares.token(t, it)) return;
    splits = shares.apart ? shares.splits_of(it) : 0;
    if (splits == 1) return;
  } else {
    const auto mine = [&](const PagedSeq& q, uint32_t, uint32_t) { return t >= q.first && t - q.first < q.count; };
    if (!paged_find<ROWS, UNIT>(b, n, group, mine, it)) return;
    if (it.splits == 1) return;
  }
  const int p = it.rows - it.count + t - it.first;  // the row's position
  __shared__ f32x4 s_o[WPR][64];
  __shared__ float s_m[WPR][JH], s_l[WPR][JH];
#pragma unroll
  for (int turn = 0; turn < TURNS; ++turn) {
    const int h = ((int)blockIdx.y * TURNS + turn) * JH + sub, hc = min(h, Hq - 1), hk = div_by(hc, group, b.inv_gqa);
    const int m = (t - it.first) * group + hc - hk * group, tile = m / ROWS;
    // Partial z of the row is at slot + (z > 0 ? later + z * step : 0), for z < parts; done: the row is written
    // already.
    int64_t slot, later = 0, step;
    int parts, most;  // most: of the wavefront's rows
    bool done = h >= Hq;
    if constexpr (SHARES) {
      step = 2;
      if (splits > 0) {  // uniform
        parts = p < 0 ? 0 : min((int)splits, (int)((uint32_t)p / (share * UNIT)) + 1);
        slot = 2 * (it.before + (int64_t)tile * splits);
      } else {
        const uint32_t at = it.before + (uint32_t)tile * (uint32_t)it.units, g = at / share;
        done = done || (at + (uint32_t)it.units - 1) / share == g;
        parts = p < 0 || done ? 0 : (int)((at + (uint32_t)p / UNIT) / share - g) + 1;
        slot = 2 * (int64_t)g + (at != g * share);  // a share's first tile or another; the shares behind begin with this one
        later = 2 * (int64_t)g - slot;
      }
      if (slot / 2 + parts > b.cap) parts = 0;  // starts that descend: no such shares were run
      slot += (int64_t)hk * 2 * b.cap;
      most = parts;
#pragma unroll
      for (int d = LR; d < 64; d *= 2) most = max(most, __shfl_xor(most, d));
      most = __builtin_amdgcn_readfirstlane(most);
    } else {
      most = __builtin_amdgcn_readfirstlane(p < 0 ? 0 : min(it.splits, (int)((uint32_t)p / (uint32_t)(it.split_units * UNIT)) + 1));
      slot = it.before + it.tiles - 1 - tile;
      step = it.tiles;
      parts = slot + (most - 1) * step < b.cap ? most : 0;  // as above
      slot += (int64_t)hk * b.cap;
    }
    const float* first = ws + (slot * ROWS + m % ROWS) * (D + 4);
    const float* rest = first + later * (ROWS * (D + 4));  // z = 0 in the place that later ones count from
    const int64_t stride = step * (ROWS * (D + 4));
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int z0 = WPR == 4 ? wave * U : 0; z0 < parts; z0 += WPR * U) {
      f32x4 o[U];
      float2 ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        ml[u] = make_float2(-INFINITY, 0.f);
        if (z0 + u >= most) continue;  // uniform
        const int z = min(z0 + u, parts - 1);  // past this row's own: its last one again, weighing nothing
        const float* pz = z == 0 ? first : rest + z * stride;
        o[u] = *(const f32x4*)(pz + col);
        ml[u] = *(const float2*)(pz + D);
      }
      float mn = M;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (SHARES && z0 + u >= parts) ml[u].x = -INFINITY;
        mn = fmaxf(mn, ml[u].x);
      }
      const float ref = mn == -INFINITY ? 0.f : mn, a = __builtin_amdgcn_exp2f(M - ref);  // 0 of -inf
      L *= a;
      acc *= a;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = __builtin_amdgcn_exp2f(ml[u].x - ref);
        L += ml[u].y * e;
        acc += o[u] * e;
      }
      M = mn;
    }
    if constexpr (WPR == 4) {
      s_o[wave][lane] = acc;
      if (col == 0) {
        s_m[wave][sub] = M;
        s_l[wave][sub] = L;
      }
      __syncthreads();
      if (wave != 0) return;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, s_m[w][sub]);
      L = 0.f;
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float e = s_m[w][sub] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][sub] - mx);
        L += s_l[w][sub] * e;
        acc += s_o[w][lane] * e;
      }
    }
    const float inv = parts <= 0 ? 0.f : 1.f / L;  // sees nothing
    if (!done)
      *(uint2*)(out + ((int64_t)t * Hq + h) * (D * 2) + col * 2) =
          uint2{f32x2_to_bf16x2_bits(acc[0] * inv, acc[1] * inv), f32x2_to_bf16x2_bits(acc[2] * inv, acc[3] * inv)};
  }
}

}  // namespace ckv

extern "C" int64_t ckv_attention_paged_workspace_bytes(int32_t n_tokens, int32_t n_sequences, int32_t most_tokens,
                                                       int32_t most_rows, int64_t total_rows, int32_t n_entries,
                                                       int32_t page_tokens, int32_t n_q_heads, int32_t n_kv_heads,
                                                       int32_t head_dim) {
  if (n_tokens <= 0 || n_sequences <= 0 || most_tokens < 0 || most_rows < 0 || total_rows < 0 || n_entries <= 0 ||
      page_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_q_heads % n_kv_heads)
    return 0;
  const int64_t rows = (int64_t)n_entries * page_tokens;
  return ckv::paged_plan(n_tokens, n_sequences, most_tokens == 0 ? n_tokens : most_tokens, most_rows == 0 ? rows : most_rows,
                         total_rows, rows, n_q_heads, n_kv_heads, head_dim, INT64_MAX).ws_bytes;
}

extern "C" int32_t ckv_attention_paged(void* out, const void* q, int64_t q_head_stride, int64_t q_token_stride, const void* k_pool,
                                       const void* v_pool, int64_t kv_head_stride, const int32_t* table, const int32_t* lengths,
                                       const int32_t* starts, int32_t n_tokens, int32_t most_tokens, int32_t most_rows,
                                       int64_t total_rows, int32_t n_sequences, int32_t n_entries, int32_t n_pages,
                                       int32_t page_tokens, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                       int32_t dtype, double scale, void* workspace, int64_t workspace_bytes, int32_t* err, void* stream) {
  using namespace ckv;
  if (dtype != CKV_DTYPE_BF16 || (head_dim != 64 && head_dim != 128)) return CKV_ERR_INVALID_ARGUMENT;
  if (page_tokens != 32 && page_tokens != 64 && page_tokens != 128) return CKV_ERR_INVALID_ARGUMENT;
  if (n_tokens < 0 || most_tokens < 0 || most_rows < 0 || total_rows < 0 || n_sequences <= 0 || n_entries <= 0 || n_pages <= 0 ||
      n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || log2_scale(scale) == 0.f)
    return CKV_ERR_INVALID_ARGUMENT;
  if (n_tokens == 0) return CKV_OK;
  if (out == nullptr || q == nullptr || k_pool == nullptr || v_pool == nullptr || table == nullptr || lengths == nullptr ||
      starts == nullptr)
    return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride % 8 || q_head_stride % 8 || kv_head_stride % 8) return CKV_ERR_INVALID_ARGUMENT;  // 16-byte rows
  if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16) return CKV_ERR_INVALID_ARGUMENT;
  const int64_t group = n_q_heads / n_kv_heads, pool_rows = (int64_t)n_pages * page_tokens;
  if (q_token_stride < head_dim || (n_kv_heads > 1 && kv_head_stride < pool_rows * head_dim)) return CKV_ERR_OUT_OF_RANGE;
  if (n_sequences > 4096 || n_q_heads > 65535 || (int64_t)n_entries * page_tokens > INT32_MAX - 128 || pool_rows > INT32_MAX ||
      n_tokens * group > (1 << 30))
    return CKV_ERR_TOO_LARGE;
  if (workspace == nullptr || (uintptr_t)workspace % 16) workspace_bytes = 0;
  const int64_t rows = (int64_t)n_entries * page_tokens;
  const PagedPlan plan = paged_plan(n_tokens, n_sequences, most_tokens == 0 ? n_tokens : most_tokens,
                                    most_rows == 0 ? rows : most_rows, total_rows, rows, n_q_heads, n_kv_heads, head_dim,
                                    workspace_bytes);
  if (plan.map.blocks == 0) return CKV_ERR_TOO_LARGE;
  float* ws = plan.target > 0 ? (float*)workspace : nullptr;
  const bool many = n_sequences > 64;
  const PagedRows b = {table, lengths, starts, n_sequences, n_entries, n_pages, page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7,
                       (int)plan.items, plan.target, plan.target > 0 ? 1.f / (float)plan.target : 0.f, plan.min_units,
                       inverse_of(std::max((int64_t)n_tokens * group + kAttnBM, (int64_t)n_q_heads), group), err};
  const AttnMap& map = plan.map;
  const float scale_log2 = log2_scale(scale);
  hipStream_t st = (hipStream_t)stream;
  if (plan.rows < kAttnBM) {
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(kPagedWaves * 64), 0, st, map, b, n_tokens, (const char*)k_pool,
                         (const char*)v_pool, kv_head_stride * 2, (const char*)q, q_head_stride * 2, q_token_stride * 2, n_q_heads,
                         (int)group, scale_log2, (char*)out, ws);
    };
#define CKV_ROWS(D, QG) many ? launch(attn_paged_kernel<D, QG, true>) : launch(attn_paged_kernel<D, QG, false>)
    if (head_dim == 128) {
      if (plan.rows == 16) CKV_ROWS(128, 1);
      else CKV_ROWS(128, 2);
    } else {
      if (plan.rows == 16) CKV_ROWS(64, 1);
      else CKV_ROWS(64, 2);
    }
#undef CKV_ROWS
  } else {
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(kAttnWaves * 64), 0, st, map.nqb, map.group, map.xpk_log, map.items,
                         map.inv_group, map.inv_nqb, (const int64_t*)nullptr, n_tokens, 0, (const char*)k_pool,
                         (const char*)v_pool, kv_head_stride * 2, (const char*)q, q_head_stride * 2, q_token_stride * 2, n_q_heads,
                         (int)group, scale_log2, (char*)out, err, ws, 0, b);
    };
#define CKV_LARGE(D) \
  ws != nullptr ? launch(attn_active_kernel<D, true, PagedRows>) : launch(attn_active_kernel<D, false, PagedRows>)
    if (head_dim == 128) CKV_LARGE(128);
    else CKV_LARGE(64);
#undef CKV_LARGE
  }
  CKV_RETURN_IF_LAUNCH_FAILED();
  if (ws != nullptr) {
    auto join = [&](auto kernel, int tokens, int heads) {
      const dim3 grid((unsigned)((n_tokens + tokens - 1) / tokens), (unsigned)((n_q_heads + heads - 1) / heads));
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, (char*)out, (const float*)ws, b, n_tokens, n_q_heads, (int)group);
    };
#define CKV_JOIN(D, ROWS, UNIT, MANY)                                                       \
  plan.spread_join ? join(join_paged_kernel<D, ROWS, UNIT, 4, MANY>, 1, kJoinHeads<D>)     \
                   : join(join_paged_kernel<D, ROWS, UNIT, 1, MANY>, 4, kJoinTurns * kJoinHeads<D>)
#define CKV_JOIN_ROWS(D)                                                                    \
  if (plan.rows == kAttnBM) CKV_JOIN(D, kAttnBM, kAttnBN, true);                            \
  else if (plan.rows == 16) many ? CKV_JOIN(D, 16, kPagedUnit, true) : CKV_JOIN(D, 16, kPagedUnit, false); \
  else many ? CKV_JOIN(D, 32, kPagedUnit, true) : CKV_JOIN(D, 32, kPagedUnit, false)
    if (head_dim == 128) {
      CKV_JOIN_ROWS(128);
    } else {
      CKV_JOIN_ROWS(64);
    }
#undef CKV_JOIN_ROWS
#undef CKV_JOIN
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  return CKV_OK;
}
