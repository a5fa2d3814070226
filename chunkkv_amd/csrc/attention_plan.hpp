// How an attention launch runs (attention.hip): which kernel and form, over which work items. Host
// arithmetic only, without HIP, so that it can be walked on a machine without a GPU.
#pragma once

#include <algorithm>
#include <cstdint>

namespace ckv {

#ifndef CKV_ATTN_QG
#define CKV_ATTN_QG 2
#endif
constexpr int kAttnWaves = 4;
constexpr int kAttnQG = CKV_ATTN_QG;                // 16-query groups per wavefront
constexpr int kAttnBM = kAttnWaves * kAttnQG * 16;  // queries per workgroup
constexpr int kAttnBN = 64;                         // cache rows per tile
constexpr int kWaveChunk = 32;                      // cache rows per step of attn_wave_kernel's wavefronts

// scale * log2(e), with which the kernels form exp(scale x) = exp2(x scale log2 e); 0 (no scale) where that is no normal fp32
// number: a masked score, -infinity, times 0 is a NaN, and so is a score of 0 times infinity.
static inline float log2_scale(double scale) {
  const double s = scale * 1.4426950408889634;
  return s >= 0x1p-126 && s < 0x1p128 * (1 - 0x1p-25) ? (float)s : 0.f;
}

constexpr int kXcds = 8;  // MI355X: workgroups go round-robin to 8 XCDs, each with its own L2

// Which work item (query block qb, head h, cache split z) a workgroup takes. The hardware hands
// workgroup L of a 1-D grid to XCD L % 8, so items are assigned through L: the XCDs split evenly
// over the KV heads (8 / Hkv XCDs each), every item of one KV head lands on that head's XCDs (its
// K/V stay in their L2s and are read there by all `group` query heads together), consecutive items
// of an XCD cycle through the group's query heads on one query block and split, and query blocks
// go latest position first, alternating between the head's XCDs so their work stays balanced. The
// grid is padded to whole rounds of 8; a workgroup past a head's last item returns. With a KV-head
// count that does not divide 8, all heads are one group over all XCDs. The two divisions are
// multiplications by the host's reciprocals: hardware has no integer division, and four or five
// emulated ones were half a microsecond of every workgroup's start.
struct AttnMap {
  int nqb = 0, group = 0, xpk_log = 0, items = 0;  // items: of one KV head
  uint32_t inv_group = 0, inv_nqb = 0;
  uint32_t blocks = 0;  // the grid
};

// For x / d as a multiplication (div_by): ceil(2^32 / d) where that is exact for every x <= most
// (most d < 2^32), 0 elsewhere.
static inline uint32_t inverse_of(int64_t most, int64_t d) {
  return d > 1 && most * d < (1ll << 32) ? (uint32_t)(((1ll << 32) + d - 1) / d) : 0;
}

static inline AttnMap attn_map(int64_t nqb, int Hkv, int group, int64_t splits) {
  AttnMap m;
  if (kXcds % Hkv != 0) {
    group *= Hkv;
    Hkv = 1;
  }
  while ((Hkv << m.xpk_log) < kXcds) ++m.xpk_log;
  m.nqb = (int)nqb;
  m.group = group;
  m.items = (int)(group * nqb * splits);
  m.inv_group = inverse_of(m.items, group);
  m.inv_nqb = inverse_of(nqb * splits, nqb);
  m.blocks = (uint32_t)((((int64_t)m.items + (1 << m.xpk_log) - 1) >> m.xpk_log) * kXcds);
  return m;
}

// How a launch runs.
struct AttnPlan {
  bool wave = false;     // attn_wave_kernel, else attn_active_kernel (its splits are whole tiles)
  bool grouped = false;  // rows are the (token, query head) pairs of a KV head
  int qg = 0, waves = 0;
  int splits = 1, split_chunks = 0;
  AttnMap map;
};

// The (head_dim, QG, W, GROUPED) forms of attn_wave_kernel that attn_plan picks from.
#define CKV_WAVE_FORMS(X)                                                                  \
  X(128, 1, 4, true) X(128, 1, 8, true) X(128, 2, 8, true)                                  \
  X(128, 1, 4, false) X(128, 1, 8, false) X(128, 2, 4, false) X(128, 2, 8, false)           \
  X(64, 1, 4, true) X(64, 1, 8, true)                                                       \
  X(64, 1, 4, false) X(64, 1, 8, false) X(64, 2, 4, false) X(64, 2, 8, false)

// Where the 128-query workgroups are too few: below about one for each of the 256 CUs at head_dim
// 128 (us, 28 heads, this first: 768 causal rows, 168 workgroups, 19.7 against 20.6; 1000 of 8256
// rows, 224, 157 against 164; 1103 causal rows, 252, 27.8 against 27.1; 1500, 336, 41.1 against
// 36.5), below two at head_dim 64, where they also hold less work each (14 heads: 3000 causal rows,
// 336 workgroups, 37.6 against 46.5; 4000, 448, 58.9 against 61.8; 4500, 504, 72.4 against 69.8).
static inline bool wave_launch(int n, int Hq, int head_dim) {
  const int64_t blocks = (int64_t)((n + kAttnBM - 1) / kAttnBM) * Hq;
  return blocks < (head_dim == 128 ? 256 : 450);
}

constexpr int kWaveFill = 256;  // workgroups that a split launch aims at: one for each CU

// The most splits a launch takes: a workgroup has at most 32 (token, query head) rows, a split's
// four wavefronts a chunk each.
static inline int64_t most_splits(int n, int N, int Hq, int head_dim) {
  const int64_t chunks = (N + kWaveChunk - 1) / kWaveChunk;
  if (!wave_launch(n, Hq, head_dim) || chunks <= 16) return 1;
  return std::max<int64_t>(1, std::min<int64_t>(kWaveFill * 32 / ((int64_t)n * Hq), (chunks + 3) / 4));
}

// The plan of attn_wave_kernel.
static inline AttnPlan attn_wave_plan(int n, int N, int Hq, int Hkv, int head_dim, int64_t workspace_bytes) {
  AttnPlan p;
  const int group = Hq / Hkv;
  p.wave = true;
  p.grouped = group > 1 && (int64_t)n * group <= kAttnBM;
  const int rows = p.grouped ? n * group : n, heads = p.grouped ? Hkv : Hq;
  const int chunks = (N + kWaveChunk - 1) / kWaveChunk;
  const int b16 = (rows + 15) / 16 * heads, b32 = (rows + 31) / 32 * heads;
  // 16 rows a workgroup while those workgroups are all resident at once (two or four of four
  // wavefronts on a CU, by registers), else 32, which read each cache row half as often: 28 heads
  // of 128, 192 causal rows 5.9 against 7.2 us, 320 rows (560 workgroups) 9.8 against 9.0. A long
  // cache is read often enough to prefer 32 earlier at head_dim 128 (251 of 1103 rows 13.7 against
  // 14.1, 300 of 4000 34 against 43).
  const bool lng = chunks >= 24;
  if (rows <= 16) p.qg = 1;
  else if (lng) p.qg = head_dim == 64 && b16 <= 512 ? 1 : 2;
  else p.qg = b16 <= (head_dim == 64 ? 800 : 512) ? 1 : 2;
  // Grouped launches have forms of 16 rows, and at head_dim 128 of 32 rows by eight wavefronts. Up to
  // 64 KV heads the rules ask for no other; with more, the nearest of these.
  if (p.grouped && head_dim == 64) p.qg = 1;
  // 17 to 128 rows over 24 to 63 chunks at head_dim 128: a workgroup's own chain of them is the time
  // (5 queries of 28 heads over 1103 rows 13.9 us, over 1600 17.9), so 16 rows by four wavefronts,
  // split (8.8, 8.9); the three microseconds of the merge are not worth it at head_dim 64 (7.1 whole).
  const int64_t row_b = (int64_t)Hq * n * (head_dim + 4) * 4;
  const int64_t can = std::min<int64_t>(most_splits(n, N, Hq, head_dim), workspace_bytes / row_b);
  if (head_dim == 128 && rows > 16 && lng && chunks < 64) {
    const int64_t splits = std::min<int64_t>(std::min<int64_t>(can, kWaveFill / b16), chunks / 4);
    if (splits > 1) {
      p.qg = 1;
      p.waves = 4;
      p.split_chunks = (int)((chunks + splits - 1) / splits);
      p.splits = (chunks + p.split_chunks - 1) / p.split_chunks;
      p.map = attn_map(b16 / heads, Hkv, p.grouped ? 1 : group, p.splits);
      return p;
    }
  }
  const int blocks = p.qg == 1 ? b16 : b32;
  // Eight wavefronts halve a workgroup's chain where it is long, if the workgroups still fit (one
  // or two on a CU): 300 of 4000 rows 34 against 45 us with four, 768 causal rows 24.5 against 19.1.
  p.waves = (lng && (blocks <= 288 || (blocks <= 450 && chunks >= 128))) || (p.grouped && p.qg == 2) ? 8 : 4;
  // Splits cost the merge launch, about 3 us: taken for one token's rows from 17 chunks on (28
  // heads, 700 rows 7.1 against 8.5 us, 8288 rows 8.7 against 45), else where eight wavefronts
  // would have eight chunks each (150 of 1500 rows, 47 chunks, 8.5 us whole and 9.5 in two).
  int64_t splits = std::min<int64_t>(can, kWaveFill / std::max(blocks, 1));
  if (rows > 16 && chunks < 64) splits = 1;
  if (rows <= 16) p.waves = splits > 1 ? 4 : 8;
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, (chunks + p.waves - 1) / p.waves));
  p.split_chunks = (int)((chunks + splits - 1) / splits);
  p.splits = (chunks + p.split_chunks - 1) / p.split_chunks;
  p.map = attn_map(blocks / heads, Hkv, p.grouped ? 1 : group, p.splits);
  return p;
}

// The plan without split 128-query workgroups.
static inline AttnPlan attn_base_plan(int n, int N, int Hq, int Hkv, int head_dim, int64_t workspace_bytes) {
  AttnPlan p;
  const int group = Hq / Hkv;
  if (!wave_launch(n, Hq, head_dim)) {
    p.map = attn_map((n + kAttnBM - 1) / kAttnBM, Hkv, group, 1);
    return p;
  }
  return attn_wave_plan(n, N, Hq, Hkv, head_dim, workspace_bytes);
}

// 128-query workgroups over splits of a long cache. Where a launch has few query blocks the small
// launches' form reads the cache once for every 16 or 32 rows, at half the large kernel's rate, and
// the large kernel unsplit is a chain of every tile on a part of the CUs. The splits that fill the
// card once: of q = n / 128 query blocks (a last block of few rows is little work) with positions
// spread over the cache, split z of s concerns those that reach it, about s (q + 1) / 2 + (q - 1) / 2 of
// a head's q s workgroups, and 512 (head_dim 64: 768) are resident at once.
static inline int64_t large_splits(int n, int N, int Hq, int head_dim) {
  const int64_t tiles = (N + kAttnBN - 1) / kAttnBN;
  if (tiles < 80) return 1;  // shorter caches: no form gained enough
  const double q = std::max(1.0, (double)n / kAttnBM), per_head = (head_dim == 128 ? 1024.0 : 1536.0) / Hq;
  const double s = (per_head - (q - 1)) / (q + 1) + 0.1;
  return s < 2.0 ? 1 : std::min<int64_t>({(int64_t)s, tiles / 4, 32});
}

// Estimates (us) of a base plan and of the large kernel in `splits`, fitted to 13,000 launches of
// seven head layouts (28 / 4, 32 / 8, 64 / 8, 32 / 32 and 8 / 2 heads of 128, 14 / 2, 32 / 8 and 16 / 16
// of 64; 3-3000 queries over 1103-32832 rows), within about 10 %: a workgroup's chain of chunks or
// tiles, or all chunks at the rate of the card, and the partial rows written and read.
static inline double base_plan_us(const AttnPlan& p, int n, int N, int Hq, int Hkv, int head_dim) {
  const bool d128 = head_dim == 128;
  if (!p.wave) return 4.0 + (d128 ? 1.35 : 0.95) * ((N + kAttnBN - 1) / kAttnBN);
  const int rows = p.grouped ? n * (Hq / Hkv) : n, heads = p.grouped ? Hkv : Hq;
  const double chunks = (N + kWaveChunk - 1) / kWaveChunk, blocks = (double)((rows + 16 * p.qg - 1) / (16 * p.qg)) * heads;
  const double chain = (int64_t)(chunks + p.splits * p.waves - 1) / (p.splits * p.waves);
  const double step = p.waves == 8 ? (d128 ? 1.9 : 1.05) : (d128 ? 1.4 : 0.9);
  const double work = p.qg == 1 ? (d128 ? 0.27 : 0.12) : (d128 ? 0.34 : 0.185);  // of a CU
  const double seen = p.grouped ? 1.0 : 0.5;  // half the cache, on average
  return 4.0 + std::max(chain * step, blocks * chunks * seen * work / 256) + (p.splits > 1 ? 4.0 : 0.0);
}
static inline double large_split_us(int n, int N, int Hq, int head_dim, int64_t splits) {
  const int64_t tiles = (N + kAttnBN - 1) / kAttnBN, chain = (tiles + splits - 1) / splits;
  const double partial_mb = (double)splits * n * Hq * (head_dim + 4) * 4e-6;
  return head_dim == 128 ? 10.0 + 2.1 * chain + 0.31 * partial_mb : 7.0 + 1.6 * chain + 0.45 * partial_mb;
}

// Bytes of partial rows at the most splits that a launch of this shape may take; 0: it never splits.
static inline int64_t attn_most_splits(int n, int N, int Hq, int head_dim) {
  return std::max(most_splits(n, N, Hq, head_dim), large_splits(n, N, Hq, head_dim));
}
static inline int64_t attn_workspace_bytes(int n, int N, int Hq, int head_dim) {
  const int64_t splits = attn_most_splits(n, N, Hq, head_dim);
  return splits > 1 ? splits * Hq * n * (head_dim + 4) * 4 : 0;
}

// The base plan, or the large kernel in splits where that is estimated to be clearly faster (the
// estimate of an unsplit small launch is the least certain): 28 heads of 128 (us, the base plan first),
// 130 of 8256 rows 63.7 and 45.0, 251 of 32832 232 and 135, 1153 of 8256 168 and 132; 14 heads of 64, 251
// of 32832 116 and 44.8, 1153 of 16400 127 and 76.7. Below 64 rows of a KV head the small launches' form
// stays ahead. Over 1651 shapes of the layouts above 0.90 of the base plan's time in the mean; 11 are
// more than 3 % slower than it, the worst 1.19 (64 / 8 heads of 128, 180 of 32832 rows, 235 and 279).
static inline AttnPlan attn_plan(int n, int N, int Hq, int Hkv, int head_dim, int64_t workspace_bytes) {
  AttnPlan p = attn_base_plan(n, N, Hq, Hkv, head_dim, workspace_bytes);
  const int group = Hq / Hkv;
  const int64_t splits = large_splits(n, N, Hq, head_dim);
  if (splits < 2 || (int64_t)n * group < 64 || workspace_bytes / ((int64_t)Hq * n * (head_dim + 4) * 4) < splits ||
      large_split_us(n, N, Hq, head_dim, splits) >
          (p.wave && p.splits == 1 ? 0.8 : 0.92) * base_plan_us(p, n, N, Hq, Hkv, head_dim))
    return p;
  const int tiles = (N + kAttnBN - 1) / kAttnBN;
  const int split_tiles = (int)((tiles + splits - 1) / splits);
  p = AttnPlan{};
  p.split_chunks = split_tiles * (kAttnBN / kWaveChunk);
  p.splits = (tiles + split_tiles - 1) / split_tiles;
  p.map = attn_map((n + kAttnBM - 1) / kAttnBM, Hkv, group, p.splits);
  return p;
}

// 128-query workgroups of an 8-bit cache whose rows are the (token, query head) pairs of a KV head, over splits of the cache
// (splits >= 2, else the launch takes attn_plan's form). A block then holds the heads of few neighbouring tokens: full where there are
// few tokens, and near in position, so that it stops early; every row it loads and converts serves all of them.
// us, attn_plan's form and this: 28 / 4 heads of 128 over 28787 rows, 33 queries 64.9 and 32, 84 64.1 and 43, 160 117 and 62, 300 177 and
// 100, 800 295 and 222, 1100 294 and 316; over 8302, 25 queries 18.2 and 18.9, 33 25.3 and 21, 251 51.9 and 39; over 4100, 33 18.2 and 17.0, 128
// 25.6 and 27.4, 160 35.3 and 28.2; over 3000, 251 28.3 and 28.1; 32 / 8 heads of 128 over
// 28787, 160 132 and 68, 500 192 and 166; 14 / 2 heads of 64 over 28787, 25 20.6 and 17.5, 500 72 and 53, 1500 128 and 127, 2000 164 and
// 169; over 4100, 160 19.2 and 14.3, 800 24.0 and 30.4; 16 / 16 heads of 64 over 41741, 288 51.9 and 41, 1000 100 and 80, 4000 270 and 241; 32 / 32
// of 128, 130 171 and 179, 1000 671 and 460.
// Those are of positions spread over the cache, which the splits below are counted for. Of query rows at its end, as a follow-up question
// has them, every block has work in every split, 700 to 880 workgroups for the 512 places; the same, in graph replays: 28 / 4 heads of 128 over
// 28787, 33 queries 65 and 36, 84 62 and 64, 160 126 and 92, 251 139 and 136, 500 254 and 256, 800 390 and 368; over 8302, 33 25.6 and 26.6, 84 31.7
// and 37.9, 160 52.8 and 47.8, 251 57.7 and 56.6, 500 123 and 89; over 4100, 160 35.3 and 32.0, 500 65.8 and 58.1; 32 / 8 of 128 over 28787, 160 131 and 98, 500
// 258 and 257; 14 / 2 of 64 over 28787, 40 27.0 and 23.9, 160 47.8 and 41.1, 500 84.2 and 79.7; 32 / 32 of 128 over 41741, 130 180 and 185, 1000 676 and 705.
struct GroupedPlan {
  int splits = 0, split_tiles = 0;
  AttnMap map;
};
static inline GroupedPlan attn_grouped_plan(int n, int N, int Hq, int Hkv, int head_dim, int64_t workspace_bytes) {
  GroupedPlan p;
  const bool d128 = head_dim == 128;
  const int64_t group = Hq / Hkv, rows = n * group;
  if (rows <= kAttnBM || rows > (d128 ? 6400 : 11000) || N < 4000 || rows * N < (d128 ? 1300000 : 2400000)) return p;
  if (!d128 && N < 7000 && rows > N / 2) return p;
  const int64_t tiles = (N + kAttnBN - 1) / kAttnBN, q = (rows + kAttnBM - 1) / kAttnBM;
  // Of positions spread over the cache a head's q blocks have s (q + 1) / 2 + (q - 1) / 2 splits with work. As many splits as
  // keep those somewhat below the head's share of the 512 (head_dim 64: 768) workgroups that are resident at once: where a part of
  // them waits, most of what shorter splits save is lost (28 / 4 heads of 128, 128 places a head, 84 queries over 28787: 110
  // workgroups with work 48.6 us, 122 58.3; 500 queries, 115 152 us, 130 185). Of four or five splits or fewer one more saves
  // more than that (32 / 8 heads, 64 places, 800 queries: three splits and 51 workgroups 315 us, four and 64 251).
  // Of eight heads or more at head_dim 128, each on one XCD or all over all of them, less room serves for what is uneven (32 / 8, 400
  // queries 147 and 132 us). A second block of a few rows is little work (32 / 32 heads, 130 queries over 41741 232 and 179).
  const bool even = d128 && Hkv >= 8;
  const double places = (d128 ? 512.0 : 768.0) / Hkv, b = rows <= kAttnBM + 24 ? (double)rows / kAttnBM : (double)q;
  int64_t fill = std::max<int64_t>(0, (int64_t)((2 * (even ? 0.93 : 0.87) * places - (b - 1)) / (b + 1) + 0.4));
  if (fill <= (even ? 3 : 4) && (double)(fill + 1) * (b + 1) + (b - 1) <= 2.5 * places) ++fill;
  // and no more than the partial rows cost: a split's chain falls by as much as writing and reading its rows takes
  const double chain_us = (double)tiles * (d128 ? 1.5 : 0.9), part_us = (double)n * Hq * (head_dim + 4) * 4e-6 * (d128 ? 0.18 : 0.25);
  const int64_t row_b = (int64_t)Hq * n * (head_dim + 4) * 4;
  int64_t splits = std::min<int64_t>({fill, tiles / 4, 64, workspace_bytes / row_b});
  while (splits > 2 && (double)splits * splits * part_us > chain_us) --splits;
  if (splits < 2) return p;
  p.split_tiles = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.split_tiles - 1) / p.split_tiles);
  // An odd count of blocks, with one of no rows if need be: workgroups go round-robin to the 32 CUs of an XCD, and with an even
  // one the latest blocks, which every split concerns, would always meet the same CUs (32 / 8 heads of 128 over 28787, 128 queries 92
  // and 67 us, 251 147 and 102). Of two or three blocks of head_dim 64 there are too few for that (25 queries of 14 / 2 heads 17.4 and 20.4).
  p.map = attn_map(d128 || q > 3 ? q | 1 : q, Hkv, 1, p.splits);
  return p;
}

}  // namespace ckv
