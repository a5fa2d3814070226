// How a launch of the attention weights runs (attention_weights.hip): which kernels and forms, in how many splits and parts, on
// how much workspace. Host arithmetic only, without HIP, so that it can be walked on a machine without a GPU.
#pragma once

#include <algorithm>
#include <cstdint>

namespace ckv {

constexpr int kWtThreads = 256;
constexpr int kWtTile = 64;    // cache rows of a tile of the first pass, query rows of one of the second
constexpr int kWtFewRows = 16;  // query rows of a KV head up to which scores go through memory
constexpr int kWtMostParts = 128;  // splits of the cache there
constexpr int kWtWholeRows = 1024;  // cache rows up to which one workgroup a head does all of it
constexpr int kWtJoinSplits = 16;   // splits of the first pass, and query rows of a part of the second, that the second joins
constexpr int kWtJoinRows = 512;

// A query row's normaliser and position, as the second pass reads it.
struct RowStat {
  float lse;  // log2 domain
  int pos;
};

// Up to kWtFewRows query rows of a KV head over more than kWtWholeRows cached rows: splits of the cache in chunks of 32 rows, and the
// scores and (maximum, sum) pairs that they leave in the workspace.
struct FewPlan {
  int rows, chunks, splits, split_chunks;
  int64_t score_stride, score_bytes, bytes;
};
static inline FewPlan few_plan(int rows, int N, int Hkv) {
  const int chunks = (N + 31) / 32;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({512 / Hkv, (chunks + 3) / 4, kWtMostParts}));
  FewPlan p;
  p.rows = rows;
  p.chunks = chunks;
  p.split_chunks = (int)((chunks + splits - 1) / splits);
  p.splits = (chunks + p.split_chunks - 1) / p.split_chunks;
  p.score_stride = (int64_t)chunks * 32;
  p.score_bytes = (int64_t)Hkv * rows * p.score_stride * 4;
  p.bytes = p.score_bytes + (int64_t)Hkv * rows * p.splits * 8;
  return p;
}

// Whether a launch of more than kWtFewRows rows takes weights_short_kernel: while its chain, 128 rows at a time over 64 cache rows, is
// shorter than two launches. us (eager, two launches or three and one), 28 / 4 heads of 128: 17 queries over 64 8.4 and 4.8, 64 over 64
// 11.0 and 7.4, 50 over 128 11.0 and 10.1, 91 over 128 12.4 and 14.2, 17 over 256 10.0 and 8.8, 30 over 256 11.2 and 12.1; 14 / 2 of 64,
// 30 over 190 8.6 and 8.3, 50 over 190 9.5 and 10.4.
static inline bool short_cache(int rows, int N) { return N <= 256 && (int64_t)rows * ((N + 63) / 64 * 64) <= 50000; }

struct WeightsPlan {
  int rows = 0, stat_rows = 0, row_blocks = 0,  // stat_rows: rows in whole tiles
      splits = 1, split_tiles = 0, key_blocks = 0, parts = 1, part_tiles = 0,
      qg = 2, kg = 2;  // 16-row groups of a wavefront: query rows of the first pass, cache rows of the second
  bool join = false;  // the second pass joins the first's splits
  int64_t stat_bytes = 0, part_bytes = 0, sum_bytes = 0;
};

// Splits of the first pass until its workgroups are all that the card holds at once (1024; half as many took 28 us where
// these take 24); parts of the second until eight times that (its work is the lower triangle: parts that see nothing return at
// once), of four tiles of query rows or a few more (parts of four, 256 rows: 128 queries of 28 / 4 heads over 1103 15.6 us, in parts of
// five 18.4). Up to 80 tiles no more splits than the second pass joins (30 over 4100 14.3 -> 13.7; over 8302 17.5 -> 18.1).
static inline WeightsPlan weights_plan(int n, int N, int Hq, int Hkv, int head_dim) {
  WeightsPlan p;
  p.rows = n * (Hq / Hkv);
  const int tiles = (N + kWtTile - 1) / kWtTile, row_tiles = (p.rows + kWtTile - 1) / kWtTile;
  // 64 rows a workgroup of the first pass in the place of 128 where there is little work (a wavefront's chain over a tile is half as
  // long, every K row is read twice as often): 28 / 4 heads of 128 (us, 128 rows and 64), 30 queries over 1103 16.0 and 14.1, 128 over
  // 8302 36.4 and 34.2, 128 over 16400 51.6 and 51.1, 251 84.9 and 87.8; over 65536 17 queries 37.8 and 40.2, but 8, which 64 rows
  // hold, 33.8 and 28.9. 14 / 2 heads of 64, 251 over 16400 40.5 and 39.3, 500 over 32832 106 and 109. The sides of the bound, in graph
  // replays: with positions spread over the cache 64 rows lead to work = 14392 and past it (28 / 4 over 16400, 128 queries, work 7196, 42.8 and
  // 40.4, 146, 8224, 50.1 and 49.4, 251, 14392, 64.2 and 63.6; 64 over 32832, 8208, 45.1 and 43.0); with query rows at the end of the
  // cache up to it (128 52.4 and 51.4, 146 57.7 and 57.1, 64 over 32832 55.8 and 53.2) and not behind it (160 queries, 9252, 61.4 and 62.3;
  // 91 over 32832, 10260, 69.2 and 71.2; 251 82.7 and 86.8).
  const int64_t work = (int64_t)((p.rows + 127) / 128) * tiles * Hkv;
  const bool short_rows = work <= 8300 && (int64_t)N * head_dim <= 5 << 20;
  p.qg = p.rows <= 64 || short_rows ? 1 : 2;
  p.row_blocks = (p.rows + 64 * p.qg - 1) / (64 * p.qg);
  const int64_t lse_blocks = (int64_t)p.row_blocks * Hkv;
  // With much work over a long cache two or four times as many even out what the blocks see of it (us, positions spread over it, 1024
  // workgroups and more: 14 / 2 heads of 64, 750 queries over 21000 92 and 78; 28 / 4 of 128, 1750 over 32832 532 and 483, but 1000 over
  // 8302 102 and 106), unless the blocks alone are about as many as the card holds (5000 over 13000 518 and 551).
  const int64_t most = N < 12000 || work < 10000 || lse_blocks > 700 ? 1024 : work < 50000 ? 2048 : 4096;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({most / lse_blocks, tiles / 2, tiles <= 80 ? kWtJoinSplits : 64}));
  p.split_tiles = (int)((tiles + splits - 1) / splits);
  p.splits = (tiles + p.split_tiles - 1) / p.split_tiles;
  auto parts_of = [&](int64_t blocks) { return std::max<int64_t>(1, std::min<int64_t>(8192 / blocks, row_tiles < 8 ? 1 : (row_tiles + 3) / 4)); };
  // The same in the second pass, 64 cache rows a workgroup for 128, while two of these a CU do not fill the card: 28 / 4 heads of 128
  // (us, 128 cache rows and 64), 64 queries over 1103 19.1 and 16.5, over 8302 26.9 and 24.3, 251 over 2048 27.7 and 27.8, 128 over 8302
  // 36.4 and 37.3.
  const int64_t wide = (int64_t)((N + 127) / 128) * Hkv;
  p.kg = wide * parts_of(wide) <= 512 ? 1 : 2;
  p.key_blocks = (N + 64 * p.kg - 1) / (64 * p.kg);
  const int64_t parts = parts_of((int64_t)p.key_blocks * Hkv);
  p.part_tiles = (int)((row_tiles + parts - 1) / parts);
  p.parts = (row_tiles + p.part_tiles - 1) / p.part_tiles;
  p.stat_rows = row_tiles * kWtTile;
  // A launch less where each workgroup of the second pass finds its rows' normalisers as fast itself, 256 rows at a time, from at
  // most 16 splits in all: 28 / 4 heads of 128 (us, eager, joined by a launch and so), 17 queries over 1103 12.6 and 11.1, 251
  // 21.2 and 19.6, 1000 40.1 and 35.1; but 64 over 2048, 448 rows and 16 splits, 15.6 and 17.6.
  p.join = p.splits > 1 && p.part_tiles * kWtTile <= kWtJoinRows &&
           p.splits * ((p.part_tiles * kWtTile + kWtThreads - 1) / kWtThreads) <= kWtJoinSplits;
  const int64_t total = (int64_t)Hkv * p.stat_rows;
  p.stat_bytes = (total * (int64_t)sizeof(RowStat) + 15) / 16 * 16;
  p.part_bytes = p.splits > 1 ? (total * 8 * p.splits + 15) / 16 * 16 : 0;
  p.sum_bytes = p.parts > 1 ? (int64_t)Hkv * N * 4 * p.parts : 0;
  return p;
}

}  // namespace ckv
