// How a launch of attention over a paged cache runs (attention_paged.hip). Host arithmetic only, without HIP, so that it
// can be walked on a machine without a GPU.
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

// Units of all tiles up to which a split is one unit: as many partial rows as a join reads at once.
constexpr float kPagedShort = 32.f;

// Units of a split or share, from a launch's work (tiles x units, summed in fp32) and 1 / target. The sum is off by less than 2^-17 of itself
// (64 additions in a lane, 6 across, roundings of 2^-24), so this, rounded up from more than that above it, is no less than work / target: splits
// add no more than target items, and target shares are all of the work.
CKV_HOST_DEVICE static inline int paged_split_units(float work, float inv_target, int min_units) {
  const int each = (int)fminf(work * inv_target * (1.f + 0x1p-16f), 0x1p29f) + 1;
  const int least = work <= kPagedShort ? 1 : min_units;
  return each > least ? each : least;
}
// ceil(units / split_units), at least 1; inv = 1.f / split_units, within 2^-22. The product is at most one off: of a tile there are no more
// than about target splits.
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

// n new tokens of S sequences, at most `most` of one, over at most `rows` cached rows each. Lengths are the device's: the items
// are bounded by tiles (a sequence's last one may be partial) and by what splits add.
static inline PagedPlan paged_plan(int64_t n, int64_t S, int64_t most, int64_t rows, int Hq, int Hkv, int head_dim, int64_t workspace_bytes) {
  PagedPlan p;
  const int64_t group = Hq / Hkv, one = std::min(most, n) * group;
  auto tiles_of = [&](int64_t r) { return n * group / r + std::min(S, n); };
  auto units_of = [&](int64_t unit) { return (rows + unit - 1) / unit; };
  const int64_t places = std::max(1, (head_dim == 128 ? 256 : 512) / Hkv);  // workgroups of attn_paged_kernel that are resident, a KV head
  // Units that each has to read, of tiles of r rows over sequences as long as they may be.
  auto share_of = [&](int64_t r) { return (double)tiles_of(r) * (double)units_of(kPagedUnit) / (double)places; };
  // Few rows of a sequence are read by attn_paged_kernel whatever their number, and more of them where its tiles are few: a step of it is short,
  // though for a row it costs up to three times what the 128-row tiles take, which need splits and a longer start. us, tiles of 16, 32 and 128:
  // 28 / 4 heads of 128 over 8302 rows, 9 tokens (4 units) 15.2, 15.8 and 17.2, 18 (9 and 4) 18.2, 18.7, 20.3, 36 (17 and 8) 26.2, 23.6,
  // 23.0; 8 sequences of 500 rows, 40 tokens each (9 and 5), 17.4, 15.2, 17.2; 16 of up to 4000 rows, 9 each (36 and 24), 23.4, 20.9, 20.6; 14 / 2 heads of 64,
  // 16 of 500, 18 each (2 and 1) 9.3, 10.2, 12.2, 16 of up to 4000, 9 each (10 and 6) 12.5, 11.9, 12.5; 8 / 8 of 64 over 8302, 64 (5) 13.1, 13.2, 15.4.
  const bool d128 = head_dim == 128;
  if (one <= 16 || (one > 32 && share_of(16) <= (d128 ? 8 : 5))) p.rows = 16;
  else if (one <= 32 || share_of(32) <= (d128 ? 5 : 6)) p.rows = 32;
  else p.rows = kAttnBM;
  if (p.rows < kAttnBM && tiles_of(p.rows) * units_of(kPagedUnit) > INT32_MAX / 2) p.rows = kAttnBM;  // units are counted in 32 bits
  const bool large = p.rows == kAttnBM;
  const int64_t tiles = tiles_of(p.rows), row_b = (int64_t)Hkv * p.rows * (head_dim + 4) * 4;
  p.min_units = large ? 4 : 2;
  // Tiles over few rows are whole, without the second launch of a join. us, split and whole: tiles of few rows, one token a sequence, 28 / 4 heads
  // of 128 over 512 rows 9.3 and 8.5, 768 rows 9.4 and 9.8, 64 sequences of 512 14.0 and 9.4; 14 / 2 of 64 over 1024 8.5 and 7.9, 2048 8.6 and
  // 11.2, 32 sequences of 1024 9.0 and 7.9; tiles of 128, 28 / 4 of 128, 4 sequences of 500 rows and tokens 19.8 and 17.7, of 1000 26.5 and 28.0.
  if (rows > (large || d128 ? 512 : 1024)) {
    if (!large) {
      p.target = (int)places;
      p.items = p.target;
      p.ws_bytes = 2 * p.target * row_b;  // of a share, its first and its last tile may be partial
    } else if (n * group / p.rows < 512 / Hkv) {
      p.target = std::max(1, 512 / Hkv);
      p.items = tiles + p.target;
      p.ws_bytes = p.items * row_b;
    }
  }
  if (p.target == 0 || p.ws_bytes > workspace_bytes) {
    p.target = 0;
    p.items = tiles;
    p.ws_bytes = 0;
  }
  p.spread_join = p.target >= 8 * tiles || n * Hq <= 2048;
  if (p.items * Hkv < (1 << 30)) p.map = attn_map(p.items, Hkv, 1, 1);
  return p;
}

}  // namespace ckv
