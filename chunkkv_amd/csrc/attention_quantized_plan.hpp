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
// conversion inside the kernel grows with the rows (us, converting inside and first: 28 / 4 heads of 128 over 28787 rows 128
// queries 67 and 80, 500 175 and 176, 800 311 and 298; 14 / 2 heads of 64 over 65536, 128 57 and 65, 800 199 and 194; 16 / 16 of
// 64 over 28787, 128 25 and 42, 2976 166 and 170). Cache lengths move the crossing little: both costs grow with them.
constexpr int kDecodeRows = 3500;
static inline bool decode_first(int n, int N, int Hq, int Hkv, int head_dim) {
  return (int64_t)n * (Hq / Hkv) > kDecodeRows &&
         !attn_plan(n, N, Hq, Hkv, head_dim, attn_workspace_bytes(n, N, Hq, head_dim)).wave;
}
static inline int64_t decoded_bytes(int N, int Hkv, int head_dim) { return (int64_t)Hkv * N * head_dim * 4; }

}  // namespace ckv
