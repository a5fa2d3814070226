// How a launch of attention over an 8-bit cache runs (attention_quantized.hip), beside attention_plan.hpp's forms. Host arithmetic only,
// without HIP, so that it can be walked on a machine without a GPU.
#pragma once

#include "attention_plan.hpp"

namespace ckv {

constexpr int kCodeWaves = 4;   // wavefronts of attn_codes_kernel
constexpr int kCodeRows = 16;   // (token, query head) rows of a KV head that it takes

struct CodesPlan {
  int splits, split_chunks;
};
// Splits of a launch of up to kCodeRows rows a KV head: a workgroup for each CU (two were slower to join and no faster
// to read: 28 / 4 heads of 128 over 32832 rows 16.8 us, one 12.4), a chunk at least for each wavefront.
static inline CodesPlan codes_plan(int n, int N, int Hq, int Hkv, int head_dim, int64_t workspace_bytes) {
  const int64_t chunks = (N + kWaveChunk - 1) / kWaveChunk, row_b = (int64_t)Hq * n * (head_dim + 4) * 4;
  // whole up to 1024 rows of 128 and 1536 of 64: the join is a launch (us, eager calls, whole and split: 28 / 4 heads of 128, 1000
  // rows 7.8 and 9.6, 1400 rows 9.2 and 9.5 but 7.2 in a graph; 14 / 2 heads of 64, 1500 rows 7.5 and 9.6)
  int64_t splits = chunks <= (head_dim == 128 ? 32 : 48) ? 1 : std::min<int64_t>(kWaveFill / Hkv, (chunks + kCodeWaves - 1) / kCodeWaves);
  splits = std::max<int64_t>(1, std::min(splits, workspace_bytes / row_b));
  CodesPlan p;
  p.split_chunks = (int)((chunks + splits - 1) / splits);
  p.splits = (int)((chunks + p.split_chunks - 1) / p.split_chunks);
  return p;
}
static inline bool few_rows(int n, int Hq, int Hkv) { return (int64_t)n * (Hq / Hkv) <= kCodeRows; }
// (token, query head) rows of a KV head from which a launch converts the cache first. That pass is the cache's bytes, the
// conversion inside the kernel grows with the rows. Most launches near the bound take grouped rows (attn_grouped_plan); it decides
// over caches of fewer than 4000 rows, and far behind it the launches of more rows than those take. us in graph replays, converting
// inside and first, positions spread over the cache (at its end): 64 / 8 heads of 128 over 3900 rows, 3496 rows of a KV head 88.4 and 91.7 (89.3
// and 92.7), 4800 92.9 and 95.4 (114.0 and 111.5), 16000 154.7 and 147.9 (189.7 and 182.6); 28 / 4 of 128 over 3900, 8400 88.6 and 89.2 (97.5 and
// 93.8), 21000 99.6 and 98.1 (130.5 and 124.2); over 8302, 7000 107.8 and 101.7 (152 and 146); over 28787, 7000 318 and 290 (483 and 453), 20832 682
// and 631 (1319 and 1196); 14 / 2 of 64 over 28787, 11900 148 and 141 (222 and 211). Without shared heads a row of the cache serves
// one head and converting inside stays ahead over such a cache: 32 / 32 of 128, 3900 142.0 and 147.3, 16 / 16 of 64, 3900 60.0 and 70.8.
constexpr int kDecodeRows = 3500;
static inline bool decode_first(int n, int N, int Hq, int Hkv, int head_dim) {
  return (int64_t)n * (Hq / Hkv) > kDecodeRows &&
         !attn_plan(n, N, Hq, Hkv, head_dim, attn_workspace_bytes(n, N, Hq, head_dim)).wave;
}
static inline int64_t decoded_bytes(int N, int Hkv, int head_dim) { return (int64_t)Hkv * N * head_dim * 4; }

}  // namespace ckv
