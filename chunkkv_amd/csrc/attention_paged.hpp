// What the attention kernels need of a paged cache (pages.hip describes it): where a sequence's rows lie, and which
// part of a launch's work a workgroup has.
//
// New tokens are ragged over the sequences and only the device knows the lengths, so a launch is sized by what the host
// knows (tokens, sequences) and shared out on the device. The rows of a KV head are the (token, query head) pairs of a
// sequence, cut into tiles of ROWS. Where a launch has few tiles, a tile's part of the cache is cut further, into splits of
// split_units x UNIT rows: as long as all of a launch's work (tiles x units) over the workgroups it aims at, so long
// sequences get many and short ones one. The (sequence, split, tile) items are numbered in that order, tiles from a sequence's last, and
// each wavefront finds its own by a prefix sum over the sequences. Workgroups without an item come last in the grid: in front they
// held CUs that the others waited for (one token over 8302 rows 12.4 us, last 11.9).
#pragma once

#include "attention_common.hpp"
#include "attention_paged_plan.hpp"

namespace ckv {

struct PagedRows {
  const int32_t* table;    // (S, M) pages of T rows
  const int32_t* lengths;  // (S) rows, the new tokens' among them
  const int32_t* starts;   // (S + 1) new tokens before each sequence's
  int S, M, P, T_log;
  int cap;     // items of a KV head that the launch has room for
  int target;  // items that splits aim at, beside the tiles; 0: no splits
  float inv_target;
  int min_units;
  uint32_t inv_gqa;
  int32_t* err;
};

struct PagedItem {
  int seq, first, count, rows;  // the sequence, its first new token and their number, its rows
  int item0, tiles, splits, split_units;
  int tile, z;  // set by paged_item
};

// The sequence that `mine(first, count, items before it, its items)` names (the first one); false: none. Uniform.
template <int ROWS, int UNIT, typename F>
__device__ __forceinline__ bool paged_find(const PagedRows& b, int n, int group, F mine, PagedItem& it) {
  const int lane = lane_id();
  struct Seq {
    int first, count, rows;
  };
  auto seq = [&](int s) {
    Seq q = {0, 0, 0};
    if (s < b.S) {
      q.first = min(max(b.starts[s], 0), n);
      q.count = min(max(b.starts[s + 1], q.first), n) - q.first;
      q.rows = min(max(b.lengths[s], 0), b.M << b.T_log);
    }
    return q;
  };
  auto tiles_of = [&](const Seq& q) { return (int)(((uint32_t)q.count * (uint32_t)group + ROWS - 1) / ROWS); };
  auto units_of = [&](const Seq& q) { return (int)(((uint32_t)q.rows + UNIT - 1) / UNIT); };
  const Seq head = seq(lane);
  int split_units = 1 << 30;
  if (b.target > 0) {
    float work = 0.f;
    for (int s0 = 0; s0 < b.S; s0 += 64) {
      const Seq q = s0 == 0 ? head : seq(s0 + lane);
      work += (float)tiles_of(q) * (float)units_of(q);
    }
    work = wave_butterfly_sum(work);
    split_units = paged_split_units(work, b.inv_target, b.min_units);  // the same in every wavefront
  }
  const float inv_split = 1.f / (float)split_units;
  int before = 0;
  for (int s0 = 0; s0 < b.S; s0 += 64) {
    const Seq q = s0 == 0 ? head : seq(s0 + lane);
    const int tiles = tiles_of(q), units = units_of(q);
    const int splits = paged_splits(units, split_units, inv_split);
    const int items = tiles * splits;
    const int incl = before + (int)wave_incl_scan((uint32_t)items);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(mine(q.first, q.count, incl - items, items));
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      it.seq = s0 + l;
      it.first = of(q.first);
      it.count = of(q.count);
      it.rows = of(q.rows);
      it.item0 = of(incl - items);
      it.tiles = of(tiles);
      it.splits = of(splits);
      it.split_units = split_units;
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// Item `item` of a KV head; false: the launch has no such item.
template <int ROWS, int UNIT>
__device__ __forceinline__ bool paged_item(const PagedRows& b, int n, int group, int item, PagedItem& it) {
  if (!paged_find<ROWS, UNIT>(b, n, group, [&](int, int, int i0, int items) { return item >= i0 && item - i0 < items; }, it)) return false;
  const int local = item - it.item0;
  it.z = it.splits == 1 ? 0 : (int)((uint32_t)local / (uint32_t)it.tiles);
  it.tile = it.tiles - 1 - (local - it.z * it.tiles);
  return true;
}

// The page of rows j * T .. of a sequence; one that the pool does not have is flagged and read as page 0.
__device__ __forceinline__ int paged_page(const PagedRows& b, const int32_t* row, int j) {
  const int p = row[j];
  if ((uint32_t)p < (uint32_t)b.P) return p;
  flag_error(b.err, CKV_DEVICE_ERR_RANGE);
  return 0;
}

}  // namespace ckv
