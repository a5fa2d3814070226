// Attention of the active rows over the whole cache, with the causal mask given by positions:
// query row i (absolute position pos[i]) attends to cache rows j <= pos[i] of its KV head.
//
// Reference semantics (src/chunkkv/engine/torch_engine.py): the mask is materialised as a
// boolean (n_active x N) tensor, mask = active[:, None] >= arange(N)[None, :] (:157), and
// F.scaled_dot_product_attention(q, K, V, attn_mask=mask, enable_gqa=True) (:68-72) runs with
// the default scale 1/sqrt(head_dim); query head h reads KV head h / (Hq / Hkv). This kernel
// computes the same function from the positions alone: no mask tensor, no KV-head expansion.
//
// Design (gfx950, flash-attention forward): one workgroup = 4 wavefronts = 128 queries of one
// query head; it walks the cache in 64-row tiles up to the largest position among its queries
// (tiles past a wavefront's own queries are skipped by that wavefront). Both products run on
// the bf16 matrix cores (v_mfma_f32_16x16x32_bf16) in transposed form:
//   S^T = K Q^T   (A = K rows from LDS, B = the wavefront's Q rows held in registers)
//   O^T = V^T P^T (A = V^T rows from LDS, B = P straight from the S^T accumulators)
// so that every lane owns one query (lane % 16) for the whole computation: the online-softmax
// max/sum and the output rows live in that lane and only two xor-shuffles per tile combine the
// four lane groups. K/V tiles go from global memory straight into double-buffered LDS (no
// register staging, one barrier per tile), in swizzled rows that make the fragment reads
// conflict-free; V^T comes out of row-major V through transposing LDS reads. Scores and the output accumulate in
// fp32; P is rounded to bf16 for the second product (as fused SDPA kernels do). Launches with too
// few 128-query workgroups to fill the chip (decode, short prompts, small blends) run
// attention_wave.hpp's kernel instead, or, over a long cache, this one in splits of the cache whose
// partial rows attn_combine_kernel merges (attention_plan.hpp). Built with the MFMA VGPR form (no accumulator-register
// copies around the online-softmax rescale).
// Bound: issue and power together. The matrix cores run half of the cycles and the vector
// instructions most of the rest, so every vector instruction that is not softmax costs time: tile
// addresses are a kept offset on a uniform base (62 -> 8 instructions a tile), wavefront extremes
// are scalar (branches, not selects), the four lanes of a query agree on its max only where a lane
// asks to raise it. Measured (us, 28 heads of 128): 2976 rows over 8256, 216 -> 196 with the
// rows spread evenly (199 GFLOP: 1010 TFLOP/s) and 234 -> 216 as a blend keeps them, most in the chunks
// that moved (215 GFLOP: 996; 203-226 on other cards); 8256 causal rows 480 -> 449 (1089), 2000 51.2 ->
// 47.4; 14 heads of 64, 8256 causal rows 162 -> 144.
// A square bf16 product of 8192 reaches 1300-1400 on this card; inputs of zeros (no toggling) 10 %
// more than these. Not faster: tiles one ahead so that the matrix cores work beside the exponentials
// (209-214 / 478 before this form, with spills), V operands read ahead of their products (the same),
// eight wavefronts on one tile (233 / 476), 48 or 64 queries a wavefront (275 / 453, 322 / 649).
#include <algorithm>

#include "attention_large.hpp"
#include "attention_wave.hpp"

extern "C" int64_t ckv_attention_workspace_bytes(int32_t n_queries, int32_t n_tokens, int32_t n_q_heads,
                                                 int32_t head_dim, int32_t* splits_out, int32_t* split_tiles_out) {
  using namespace ckv;
  const bool some = n_queries > 0 && n_tokens > 0 && n_q_heads > 0 && head_dim > 0;
  const int64_t splits = some ? attn_most_splits(n_queries, n_tokens, n_q_heads, head_dim) : 1;
  const int tiles = n_tokens > 0 ? (n_tokens + kAttnBN - 1) / kAttnBN : 0;
  if (splits_out != nullptr) *splits_out = (int32_t)splits;
  if (split_tiles_out != nullptr) *split_tiles_out = splits > 1 ? (int32_t)((tiles + splits - 1) / splits) : 0;
  return some ? attn_workspace_bytes(n_queries, n_tokens, n_q_heads, head_dim) : 0;
}

extern "C" int32_t ckv_attention_active(void* out, const void* q, int64_t q_head_stride, int64_t q_token_stride,
                                        const void* k_cache, const void* v_cache, int64_t kv_head_stride,
                                        const int64_t* positions, int32_t n_queries, int32_t n_tokens,
                                        int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                                        double scale, void* workspace, int64_t workspace_bytes, int32_t* err,
                                        void* stream) {
  using namespace ckv;
  if (out == nullptr || q == nullptr || k_cache == nullptr || v_cache == nullptr || positions == nullptr)
    return CKV_ERR_INVALID_ARGUMENT;
  if (dtype != CKV_DTYPE_BF16 || (head_dim != 64 && head_dim != 128)) return CKV_ERR_INVALID_ARGUMENT;
  if (n_queries < 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 ||
      !(scale > 0.0))
    return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride % 8 || q_head_stride % 8 || kv_head_stride % 8) return CKV_ERR_INVALID_ARGUMENT;  // 16-byte rows
  if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16) return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride < head_dim || kv_head_stride < (int64_t)n_tokens * head_dim) return CKV_ERR_OUT_OF_RANGE;
  if (n_queries == 0) return CKV_OK;
  if (n_q_heads > 65535) return CKV_ERR_TOO_LARGE;
  const float scale_log2 = (float)(scale * 1.4426950408889634);  // exp(x) = exp2(x log2 e)
  const int group = n_q_heads / n_kv_heads;
  hipStream_t st = (hipStream_t)stream;
  const AttnPlan plan = attn_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim,
                                  workspace != nullptr && (uintptr_t)workspace % 16 == 0 ? workspace_bytes : 0);
  const AttnMap& map = plan.map;
  float* ws = plan.splits > 1 ? (float*)workspace : nullptr;
  if (plan.wave) {
    const uint32_t inv_gqa = inverse_of((int64_t)n_queries * group, group);
    auto launch = [&](auto kernel, int waves) {
      hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(waves * 64), 0, st, map.nqb, map.group, map.xpk_log, map.items,
                         map.inv_group, map.inv_nqb, positions, n_queries, n_tokens, (const char*)k_cache,
                         (const char*)v_cache, kv_head_stride * 2, (const char*)q, q_head_stride * 2, q_token_stride * 2,
                         n_q_heads, group, inv_gqa, scale_log2, plan.split_chunks, (char*)out, ws, err);
    };
#define CKV_WAVE(HD, QG, W, GR) \
  else if (head_dim == HD && plan.qg == QG && plan.waves == W && plan.grouped == GR) \
    launch(attn_wave_kernel<HD, QG, W, GR>, W);
    if (false) {
    }
    CKV_WAVE_FORMS(CKV_WAVE)
    else return CKV_ERR_INVALID_ARGUMENT;  // a plan outside the list
#undef CKV_WAVE
  } else {
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(kAttnWaves * 64), 0, st, map.nqb, map.group, map.xpk_log, map.items,
                         map.inv_group, map.inv_nqb, positions, n_queries, n_tokens, (const char*)k_cache,
                         (const char*)v_cache, kv_head_stride * 2, (const char*)q, q_head_stride * 2, q_token_stride * 2,
                         n_q_heads, group, scale_log2, (char*)out, err, ws, plan.split_chunks / (kAttnBN / kWaveChunk));
    };
    if (head_dim == 128) ws != nullptr ? launch(attn_active_kernel<128, true>) : launch(attn_active_kernel<128, false>);
    else ws != nullptr ? launch(attn_active_kernel<64, true>) : launch(attn_active_kernel<64, false>);
  }
  CKV_RETURN_IF_LAUNCH_FAILED();
  if (ws != nullptr) {
    const dim3 grid((unsigned)n_queries, (unsigned)n_q_heads);
    const dim3 block(64 * (unsigned)std::min((plan.splits + kCombineParts - 1) / kCombineParts, kCombineMaxWaves));
    auto merge = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, (char*)out, ws, n_queries, n_q_heads, plan.splits); };
    if (head_dim == 128) merge(attn_combine_kernel<128>);
    else merge(attn_combine_kernel<64>);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  return CKV_OK;
}
