// How a launch of attention over a paged cache runs (attention_paged.hip). Host arithmetic only, without HIP, so that
// it can be walked on a machine without a GPU.
#pragma once

#include <cmath>

#include "attention_plan.hpp"

#ifdef __HIPCC__
#define CKV_HOST_DEVICE __host__ __device__
#else
#define CKV_HOST_DEVICE
#endif

namespace ckv {

constexpr int kPagedWaves = 4;                           // wavefronts of attn_paged_kernel
constexpr int kPagedUnit = kPagedWaves * kWaveChunk;     // cache rows that a split is a multiple of there

// Units of all tiles up to which a split is one unit, else two at least. Measured in graph replays, 28 / 4 heads of 128
// where none are named: 16 in its place costs one token over 3000 rows 0.6 us (9.85 and 10.5). 40, the partial rows
// that a spread join has in flight, saves 0.5-0.6 where there are 33 to 40 units (one token over 5000 rows 10.85 and
// 10.2, four sequences of 1100 10.45 and 9.9; 14 / 2 heads of 64 0.1-0.3) and costs 8 / 8 heads of 64 0.2-0.3 (one
// token over 4600 rows 9.05 and 9.35) and 20 short sequences whose longest is not told 1.2 (8.8 and 9.95).
constexpr float kPagedShort = 32.f;

// Units of a split or share, from a launch's work (tiles x units, summed in fp32) and 1 / target. The sum is off by
// less than 2^-17 of itself (64 additions in a lane, 6 across, roundings of 2^-24), so this, rounded up from more than
// that above it, is no less than work / target: splits add no more than target items, and target shares are all of the
// work.
CKV_HOST_DEVICE static inline int paged_split_units(float work, float inv_target, int min_units) {
  const int each = (int)fminf(work * inv_target * (1.f + 0x1p-16f), 0x1p29f) + 1;
  const int least = work <= kPagedShort ? 1 : min_units;
  return each > least ? each : least;
}
// ceil(units / split_units), at least 1; inv = 1.f / split_units, within 2^-22. The product is at most one off: of a
// tile there are no more than about target splits.
CKV_HOST_DEVICE static inline int paged_splits(int units, int split_units, float inv) {
  const int s = (int)((float)units * inv), some = s > 1 ? s : 1;
  return (int64_t)some * split_units < units ? some + 1 : some;
}

struct PagedPlan {
  int rows = 0;    // (token, query head) rows of a tile: 16 or 32 (attn_paged_kernel), 128 (attn_active_kernel)
  int target = 0;  // shares of the units of a KV head, or items that splits aim at, beside the tiles; 0: tiles are whole
  int min_units = 0;
  bool spread_join = false;  // a row's partials are spread over four wavefronts
  int64_t items = 0;  // of a KV head, at most; or shares
  int64_t ws_bytes = 0;
  AttnMap map;
};

// A kernel form's time in a graph replay, us at one load: `start` and a `step` for each 128 rows that its workgroups
// read one after the other, of head sizes 64 and 128; `places`: workgroups that the card holds of it; `tile`: steps
// that a tile's beginning and end cost where a place has several. From 357 shapes (28 / 4, 32 / 8, 8 / 2 and 16 / 16
// heads of 128, 14 / 2, 8 / 8 and 32 / 1 of 64; 1 to 100 sequences of 200 to 8302 rows, equal, ragged and one long
// among short ones, 1 to 500 new tokens each), every form timed: the one with the least estimate takes 1.1 % more than
// the fastest on average and 29 % at most, where the rows of all are not told 1.7 and 124 % (40 sequences, one of 2992
// rows, the others 187: 66.9 for 29.8; profiles/paged_attention_forms.csv has all of them); tiles by a launch's load
// alone and splits from 512 or 1024 rows on 4.1 and 79 %.
struct PagedForm {
  int rows;
  double start, step[2], tile;
  int places[2];
};
constexpr PagedForm kPagedForms[] = {{16, 5.5, {0.5, 0.8}, 1.5, {512, 256}},
                                     {32, 6.0, {0.55, 1.1}, 1.5, {512, 256}},
                                     {kAttnBM, 5.0, {1.5, 2.4}, 0.5, {768, 512}}};
// us that splitting adds, and for each byte in fp32 of the results that are split
constexpr double kPagedJoin = 4.5, kPagedJoinByte = 1.5e-6;
constexpr double kPagedMean = 0.5;  // of the longest sequence's rows, where the sum is not known

// n new tokens of S sequences; `most` of one, `longest` cached rows of one and `total` of all that have tokens (0: not
// known) are estimates, `rows` is the most that a sequence can have. Lengths are the device's: the items are bounded by
// tiles (a sequence's last one may be partial) and by what splits add. Of a sequence whose (token, query head) rows fit
// 16 or 32 larger tiles read the cache as often for nothing. us, whole and split, and other tiles:
//   28 / 4 heads of 128, one token over 512 rows 8.5 and 9.3, 768 9.8 and 9.4, 31 sequences of 683 12.6 and 15.9, 69 of
//     up to 576, 1 to 3 tokens, 13.7 and 24.4
//   4 sequences of 500 rows and tokens 17.7 (128), 19.8 split; 2 of 832 rows, 57 tokens, 11.1 (16), 18.5 split
//   14 / 2 of 64, 9 sequences of up to 2000 rows, 1280 tokens, 16.5 (32), 18.1 (16), 21.8 (128, split), 32.9 (128)
//   8 / 8 of 64, 22 of up to 1976 rows, 1314 tokens, 15.8 (16), 16.6 (32), 19.4 (128, split), 26.8 (16, split)
static inline PagedPlan paged_plan(int64_t n, int64_t S, int64_t most, int64_t longest, int64_t total, int64_t rows, int Hq,
                                   int Hkv, int head_dim, int64_t workspace_bytes) {
  PagedPlan p;
  const int64_t group = Hq / Hkv, used = std::min(S, n), one = std::min(most, n) * group;
  const int d128 = head_dim == 128;
  const double longer = (double)std::min(longest, rows);
  const double mean = total > 0 ? std::min((double)total / (double)used, longer) : kPagedMean * longer;
  double least = INFINITY;
  for (const PagedForm& f : kPagedForms) {
    if ((f.rows > 16 && one <= 16) || (f.rows > 32 && one <= 32)) continue;
    const bool large = f.rows == kAttnBM;
    const int64_t unit = large ? kAttnBN : kPagedUnit, tiles = n * group / f.rows + used;
    const double least_units = (double)unit / 128.0, units = std::ceil(longer / (double)unit) * least_units;
    const double mean_units = std::min(std::max(mean / 128.0 + least_units / 2.0, least_units), units);
    const double likely = (double)std::min(tiles, used * ((one + f.rows - 1) / f.rows));
    const double load = 1.3 * (mean_units + f.tile) * likely * Hkv / f.places[d128];  // of a workgroup, if three of four are busy
    const double whole = f.start + f.step[d128] * std::max(units, load);
    if (whole < least) {
      least = whole;
      p = {};
      p.rows = f.rows;
      p.items = tiles;
    }
    PagedPlan s;
    s.rows = f.rows;
    s.min_units = large ? 4 : 2;
    const int64_t row_b = (int64_t)Hkv * f.rows * (head_dim + 4) * 4;
    if (large) {
      s.target = std::max(1, 512 / Hkv);
      s.items = tiles + s.target;
      s.ws_bytes = s.items * row_b;
      if (n * group / f.rows >= s.target) continue;  // enough tiles
    } else {
      s.target = std::max(1, f.places[d128] / Hkv);
      s.items = s.target;
      s.ws_bytes = 2 * s.items * row_b;  // of a share, its first and its last tile may be partial
      if (tiles * ((rows + unit - 1) / unit) > INT32_MAX / 2) continue;  // units are counted in 32 bits
    }
    // tiles of short sequences are mostly whole
    const double joined = 4.0 * (double)(n * Hq * head_dim) * (total > 0 ? mean_units / units : 1.0);
    const double split = f.start + kPagedJoin + kPagedJoinByte * joined + f.step[d128] * std::max(2.0, load);
    if (split < least && s.ws_bytes <= workspace_bytes) {
      least = split;
      s.spread_join = s.target >= 8 * tiles || n * Hq <= 2048;
      p = s;
    }
  }
  if (p.items * Hkv < (1 << 30)) p.map = attn_map(p.items, Hkv, 1, 1);
  return p;
}

}  // namespace ckv
