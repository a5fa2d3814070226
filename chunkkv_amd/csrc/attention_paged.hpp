// What the attention kernels need of a paged cache (pages.hip describes it): where a sequence's rows lie, and which
// part of a launch's work a workgroup has.
//
// New tokens are ragged over the sequences and only the device knows the lengths, so a launch is sized by what the host
// knows (tokens, sequences) and shared out on the device. The rows of a KV head are the (token, query head) pairs of a
// sequence, cut into tiles of ROWS; a tile's part of the cache is its units of UNIT rows. Two ways of sharing:
//  - Tiles of 16 or 32 rows: all units of all tiles in a row, in equal shares (PagedShare), so that every workgroup
//    reads as much of the cache whatever the lengths are. A tile that lies in several shares has a partial row in each.
//  - Tiles of 128: items of a tile and a split of its units (paged_item), as long as all the work over the workgroups
//    that the launch aims at, numbered by (sequence, split, tile), tiles from a sequence's last. Workgroups without an
//    item come last in the grid: in front they held CUs that the others waited for.
// Each wavefront finds its own part by a prefix sum over the sequences.
#pragma once

#include "attention_common.hpp"
#include "attention_paged_plan.hpp"

namespace ckv {

struct PagedRows {
  const int32_t* table;    // (S, M) pages of T rows
  const int32_t* lengths;  // (S) rows, the new tokens' among them
  const int32_t* starts;   // (S + 1) new tokens before each sequence's
  int S, M, P, T_log;
  int cap;     // items (or shares) of a KV head that the launch has room for
  int target;  // items that splits aim at, beside the tiles, or shares; 0: a tile is whole
  float inv_target;
  int min_units;
  uint32_t inv_gqa;
  int32_t* err;
};

// A sequence of the launch, or none.
struct PagedSeq {
  int seq, first, count, rows;  // its number, its first new token and their number, its rows
  int tiles, units;             // units of each tile
  uint32_t before;              // of what `find` counts, those of the sequences before
};

// MANY: more than 64 sequences, a wavefront's lanes; without it every wavefront's way to its work is 0.2 us shorter.
template <int ROWS, int UNIT, bool MANY>
struct PagedWalk {
  const PagedRows& b;
  const int n, group;
  PagedSeq head;  // of sequence `lane`

  __device__ PagedWalk(const PagedRows& b, int n, int group) : b(b), n(n), group(group), head(seq(lane_id())) {}

  __device__ PagedSeq seq(int s) const {
    PagedSeq q = {s, 0, 0, 0, 0, 0, 0};
    if (s < b.S) {
      q.first = min(max(b.starts[s], 0), n);
      q.count = min(max(b.starts[s + 1], q.first), n) - q.first;
      q.rows = min(max(b.lengths[s], 0), b.M << b.T_log);
    }
    q.tiles = (int)(((uint32_t)q.count * (uint32_t)group + ROWS - 1) / ROWS);
    q.units = max(1, (int)(((uint32_t)q.rows + UNIT - 1) / UNIT));
    return q;
  }
  // f over the lane's sequences.
  template <typename F>
  __device__ void each(F f) const {
    f(head);
    if constexpr (MANY) {
      for (int s0 = 64; s0 < b.S; s0 += 64) f(seq(s0 + lane_id()));
    }
  }
  // The first sequence for which mine(sequence, those before, its own), counting count(sequence); false: none. Uniform.
  template <typename C, typename F>
  __device__ bool find(C count, F mine, PagedSeq& it) const {
    uint32_t before = 0;
    for (int s0 = 0; s0 < (MANY ? b.S : 1); s0 += 64) {
      const PagedSeq q = s0 == 0 ? head : seq(s0 + lane_id());
      const uint32_t own = count(q), incl = before + wave_incl_scan(own);
      const uint64_t hit = __builtin_amdgcn_ballot_w64(mine(q, incl - own, own));
      if (hit != 0) {
        const int l = __builtin_ctzll(hit);
        auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
        it = {s0 + l, of(q.first), of(q.count), of(q.rows), of(q.tiles), of(q.units), (uint32_t)of((int)(incl - own))};
        return true;
      }
      before = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    return false;
  }
};

// ---- equal shares of units -------------------------------------------------------------------------------------
// Where shares that keep tiles apart would be hardly longer (one unit, of which a launch of little work has few), they
// do: ending a tile and beginning the next costs a workgroup more than a microsecond. A launch without splits takes
// whole tiles. Counts fit 32 bits (the plan sees to it).
template <int ROWS, int UNIT, bool MANY>
struct PagedShare {
  const PagedWalk<ROWS, UNIT, MANY> walk;
  uint32_t share;  // units
  bool apart;      // a share has units of one tile

  __device__ PagedShare(const PagedRows& b, int n, int group) : walk(b, n, group), share(1u << 30), apart(true) {
    if (b.target == 0) return;
    uint32_t units = 0, tiles = 0;
    walk.each([&](const PagedSeq& q) {
      units += (uint32_t)q.tiles * (uint32_t)q.units;
      tiles += (uint32_t)q.tiles;
    });
    units = (uint32_t)__builtin_amdgcn_readlane((int)wave_incl_scan(units), 63);
    tiles = (uint32_t)__builtin_amdgcn_readlane((int)wave_incl_scan(tiles), 63);
    share = (uint32_t)paged_split_units((float)units, b.inv_target, b.min_units);
    apart = false;
    if (tiles < (uint32_t)b.target) {  // then no more than units / longer + tiles shares
      const float inv_left = __builtin_amdgcn_rcpf((float)(b.target - (int)tiles));
      const uint32_t longer = (uint32_t)paged_split_units((float)units, inv_left, b.min_units);
      apart = longer <= share + 1;
      if (apart) share = longer;
    }
  }
  // Shares of each of a sequence's tiles, where they are apart.
  __device__ uint32_t splits_of(const PagedSeq& q) const {
    return (uint32_t)paged_splits(q.units, (int)share, __builtin_amdgcn_rcpf((float)(int)share));
  }
  // What shares are counted in: shares, where they are apart, or units.
  __device__ uint32_t parts_of(const PagedSeq& q) const { return apart ? splits_of(q) : (uint32_t)q.units; }
  __device__ auto counter() const {
    return [this](const PagedSeq& q) { return (uint32_t)q.tiles * parts_of(q); };
  }
  // The sequence that has part `at`.
  __device__ bool part(uint32_t at, PagedSeq& it) const {
    const auto mine = [at](const PagedSeq&, uint32_t before, uint32_t own) { return at >= before && at - before < own; };
    return walk.find(counter(), mine, it);
  }
  // The sequence that has token t.
  __device__ bool token(int t, PagedSeq& it) const {
    return walk.find(counter(), [t](const PagedSeq& q, uint32_t, uint32_t) { return t >= q.first && t - q.first < q.count; }, it);
  }
};

// ---- items of a tile and a split -------------------------------------------------------------------------------
struct PagedItem : PagedSeq {
  int splits, split_units;
  int tile, z;  // set by paged_item
};

template <int ROWS, int UNIT, typename F>
__device__ __forceinline__ bool paged_find(const PagedRows& b, int n, int group, F mine, PagedItem& it) {
  const PagedWalk<ROWS, UNIT, true> walk(b, n, group);
  int split_units = 1 << 30;
  if (b.target > 0) {
    float work = 0.f;
    walk.each([&](const PagedSeq& q) { work += (float)q.tiles * (float)q.units; });
    split_units = paged_split_units(wave_butterfly_sum(work), b.inv_target, b.min_units);  // the same in every wavefront
  }
  const float inv_split = __builtin_amdgcn_rcpf((float)split_units);
  const auto items = [&](const PagedSeq& q) { return (uint32_t)(q.tiles * paged_splits(q.units, split_units, inv_split)); };
  if (!walk.find(items, mine, it)) return false;
  it.split_units = split_units;
  it.splits = paged_splits(it.units, split_units, inv_split);
  return true;
}

// Item `item` of a KV head; false: the launch has no such item.
template <int ROWS, int UNIT>
__device__ __forceinline__ bool paged_item(const PagedRows& b, int n, int group, int item, PagedItem& it) {
  const auto mine = [item](const PagedSeq&, uint32_t before, uint32_t own) {
    return (uint32_t)item >= before && (uint32_t)item - before < own;
  };
  if (!paged_find<ROWS, UNIT>(b, n, group, mine, it)) return false;
  const int local = item - (int)it.before;
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
