// Attention of the active rows over an 8-bit cache (quantize.hip): the function of attention.hip on the rows
// that codes and scales stand for. A code times its power of two is a bf16 value, so both forms here compute
// with exactly the rows a bf16 cache would hold, and scores, softmax and output are attention.hip's.
//
//  - Few query rows (decode, short prompts): attention_wave.hpp's kernel reads the codes and makes them bf16
//    on their way into LDS, a wavefront its own 32 rows. Bound: the cache's bytes, half of a bf16 cache's.
//  - Many: one pass writes the cache as bf16 into the workspace and attention.hip runs on it. There every
//    row is read by many workgroups of 128 queries, and each would convert it again.
#include "attention_common.hpp"
#include "attention_wave.hpp"

namespace ckv {

// One 16-byte piece of codes of K (y = 0) or V (y = 1) a thread.
template <int D>
__global__ __launch_bounds__(256) void decode_rows_kernel(char* __restrict__ k_out, char* __restrict__ v_out,
                                                          const char* __restrict__ k_codes,
                                                          const char* __restrict__ v_codes,
                                                          const uint8_t* __restrict__ k_scales,
                                                          const uint8_t* __restrict__ v_scales, int N, int blocks,
                                                          int block_log) {
  const int64_t piece = (int64_t)blockIdx.x * 256 + threadIdx.x;  // of a head
  const int h = blockIdx.y;
  if (piece >= (int64_t)N * (D / 16)) return;
  const bool is_v = blockIdx.z != 0;
  const int row = (int)(piece / (D / 16));
  const int64_t at = (int64_t)h * N * D + piece * 16;
  const vec16 c = ld16_stream((is_v ? v_codes : k_codes) + at);
  const uint32_t b = (is_v ? v_scales : k_scales)[(int64_t)h * blocks + (row >> block_log)];
  vec16 lo, hi;
  decode16(c, __uint_as_float(b << 23), lo, hi);
  char* out = (is_v ? v_out : k_out) + at * 2;
  st16(out, lo);
  st16(out + 16, hi);
}

// Whether a launch converts the cache first.
static bool decode_first(int n, int N, int Hq, int Hkv, int head_dim) {
  return !attn_plan(n, N, Hq, Hkv, head_dim, attn_workspace_bytes(n, N, Hq, head_dim)).wave;
}
#ifndef FILL
#define FILL 512
#endif
static int wave_fill(int N) { return N >= 4096 ? FILL : kWaveFill; }
static int64_t wave_workspace_bytes(int n, int N, int Hq, int head_dim) {
  const int64_t splits = most_splits(n, N, Hq, head_dim, wave_fill(N));
  return splits > 1 ? splits * Hq * n * (head_dim + 4) * 4 : 0;
}
static int64_t decoded_bytes(int N, int Hkv, int head_dim) { return (int64_t)Hkv * N * head_dim * 4; }

}  // namespace ckv

extern "C" int64_t ckv_attention_quantized_workspace_bytes(int32_t n_queries, int32_t n_tokens, int32_t n_q_heads,
                                                           int32_t n_kv_heads, int32_t head_dim) {
  using namespace ckv;
  if (n_queries <= 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_q_heads % n_kv_heads) return 0;
  return decode_first(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim)
             ? decoded_bytes(n_tokens, n_kv_heads, head_dim) + attn_workspace_bytes(n_queries, n_tokens, n_q_heads, head_dim)
             : wave_workspace_bytes(n_queries, n_tokens, n_q_heads, head_dim);
}

extern "C" int32_t ckv_attention_quantized(void* out, const void* q, int64_t q_head_stride, int64_t q_token_stride,
                                           const void* k_codes, const void* v_codes, const void* k_scales,
                                           const void* v_scales, const int64_t* positions, int32_t n_queries,
                                           int32_t n_tokens, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                           int32_t block_tokens, double scale, void* workspace,
                                           int64_t workspace_bytes, int32_t* err, void* stream) {
  using namespace ckv;
  if (head_dim != 64 && head_dim != 128) return CKV_ERR_INVALID_ARGUMENT;
  if (block_tokens != 32 && block_tokens != 64 && block_tokens != 128) return CKV_ERR_INVALID_ARGUMENT;
  if (n_queries < 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || !(scale > 0.0))
    return CKV_ERR_INVALID_ARGUMENT;
  if (n_queries == 0) return CKV_OK;
  if (out == nullptr || q == nullptr || k_codes == nullptr || v_codes == nullptr || k_scales == nullptr ||
      v_scales == nullptr || positions == nullptr)
    return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride % 8 || q_head_stride % 8) return CKV_ERR_INVALID_ARGUMENT;  // 16-byte rows
  if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes) % 16) return CKV_ERR_INVALID_ARGUMENT;
  if (q_token_stride < head_dim) return CKV_ERR_OUT_OF_RANGE;
  if (n_q_heads > 65535) return CKV_ERR_TOO_LARGE;
  const int block_log = block_tokens == 32 ? 5 : block_tokens == 64 ? 6 : 7;
  const int blocks = (int)(((int64_t)n_tokens + block_tokens - 1) >> block_log);
  hipStream_t st = (hipStream_t)stream;
  if (workspace == nullptr || (uintptr_t)workspace % 16) workspace_bytes = 0;

  const int64_t decoded = decoded_bytes(n_tokens, n_kv_heads, head_dim);
  if (workspace_bytes >= decoded && decode_first(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim)) {
    char* kd = (char*)workspace;
    char* vd = kd + decoded / 2;
    const int64_t pieces = (int64_t)n_tokens * (head_dim / 16);
    const dim3 grid((unsigned)((pieces + 255) / 256), (unsigned)n_kv_heads, 2);
    auto decode = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, kd, vd, (const char*)k_codes, (const char*)v_codes,
                         (const uint8_t*)k_scales, (const uint8_t*)v_scales, n_tokens, blocks, block_log);
    };
    if (head_dim == 128) decode(decode_rows_kernel<128>);
    else decode(decode_rows_kernel<64>);
    CKV_RETURN_IF_LAUNCH_FAILED();
    return ckv_attention_active(out, q, q_head_stride, q_token_stride, kd, vd, (int64_t)n_tokens * head_dim, positions,
                                n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, CKV_DTYPE_BF16, scale,
                                vd + decoded / 2, workspace_bytes - decoded, err, stream);
  }

  const float scale_log2 = (float)(scale * 1.4426950408889634);  // exp(x) = exp2(x log2 e)
  const int group = n_q_heads / n_kv_heads;
  const AttnPlan plan = attn_wave_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, workspace_bytes, wave_fill(n_tokens));
  const AttnMap& map = plan.map;
  float* ws = plan.splits > 1 ? (float*)workspace : nullptr;
  const CacheScales scales = {(const uint8_t*)k_scales, (const uint8_t*)v_scales, blocks, block_log - 5};
  static_assert(kWaveChunk == 32, "a chunk has one scale");
  const uint32_t inv_gqa = inverse_of((int64_t)n_queries * group, group);
  auto launch = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(waves * 64), 0, st, map.nqb, map.group, map.xpk_log, map.items,
                       map.inv_group, map.inv_nqb, positions, n_queries, n_tokens, (const char*)k_codes,
                       (const char*)v_codes, (int64_t)n_tokens * head_dim, (const char*)q, q_head_stride * 2,
                       q_token_stride * 2, n_q_heads, group, inv_gqa, scale_log2, plan.split_chunks, (char*)out, ws, err, scales);
  };
#define CKV_WAVE(HD, QG, W, GR) \
  else if (head_dim == HD && plan.qg == QG && plan.waves == W && plan.grouped == GR) \
    launch(attn_wave_kernel<HD, QG, W, GR, true>, W);
  if (false) {
  }
  CKV_WAVE_FORMS(CKV_WAVE)
  else return CKV_ERR_INVALID_ARGUMENT;  // a plan outside the list
#undef CKV_WAVE
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
