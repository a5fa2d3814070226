// A cache cut to its heaviest rows. Per KV head: the first n_sink rows and the last n_recent stay, and of the others
// those of the largest weight (what attention_weights.hip adds up) until n_keep stay, the lower row first among
// equals; a NaN ranks below every number. The kept rows move to the front of new caches, in order.
//
// Design: evict_select_kernel, one workgroup of 1024 threads a head, maps the weights to integers that order as they
// do and finds the smallest one kept by three passes of a radix histogram in LDS (11, 11 and 10 bits), the keys
// held in registers (read again from L2 above 36,864 rows). A wavefront owns a run of consecutive rows, so the ranks
// that place kept rows in order are ballots and one scan over 16 wavefronts. evict_gather_kernel then copies the
// rows, a 16-byte piece a thread.
// Bound: the selection's latency on one CU of a head; the copy is HBM's.
#include <algorithm>

#include "ckv_common.hpp"

namespace ckv {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;
constexpr int kEvictBins = 2048;

// An integer that orders as the weight does; 0 for a NaN, below -infinity's.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);  // -0 and 0 are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Lane-wise sum over a wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
  for (int m = 32; m > 0; m >>= 1) x += (uint32_t)__shfl_xor((int)x, m);
  return x;
}

// PER: 64-row steps of a wavefront's run held in registers; 0: any number, read again for each pass.
template <int PER>
__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(const float* __restrict__ weights,
                                                                     int64_t w_hs, int N, int n_keep, int n_sink,
                                                                     int n_recent, int run_steps,
                                                                     int64_t* __restrict__ rows_out,
                                                                     float* __restrict__ weights_out) {
  __shared__ uint32_t hist[kEvictBins];
  __shared__ uint32_t wave_tot[2][kEvictWaves];
  __shared__ uint32_t found[2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const float* w = weights + (int64_t)blockIdx.x * w_hs;
  const int64_t run = (int64_t)wave * run_steps * kWave;
  auto row_of = [&](int i) { return run + (int64_t)i * kWave + lane; };
  float reg[PER > 0 ? PER : 1];
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t r = row_of(i);
      reg[i] = i < run_steps && r < N ? w[r] : 0.f;
    }
  }
  const int tail = N - n_recent;
  // f(row, weight) for each of this thread's rows, wavefront-uniformly (rows past the cache too)
  auto each = [&](auto f) {
    if constexpr (PER > 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < run_steps) f(row_of(i), reg[i]);
    } else {
      for (int i = 0; i < run_steps; ++i) {
        const int64_t r = row_of(i);
        f(r, r < N ? w[r] : 0.f);
      }
    }
  };
  auto candidate = [&](int64_t r) { return r >= n_sink && r < tail; };

  uint32_t need = (uint32_t)(n_keep - n_sink - n_recent);  // of the candidates; the caller has fixed rows apart
  uint32_t prefix = 0;                                     // the threshold's bits found so far
  int shift = 32;
  if (need > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10, next = shift - bits;
      for (int b = tid; b < kEvictBins; b += kEvictThreads) hist[b] = 0;
      __syncthreads();
      each([&](int64_t r, float x) {
        const uint32_t k = weight_key(x);
        if (candidate(r) && (shift == 32 || k >> shift == prefix)) atomicAdd(&hist[(k >> next) & ((1u << bits) - 1)], 1u);
      });
      __syncthreads();
      // the bin, from the top, in which the need-th candidate lies: two bins a thread
      const int top = (1 << bits) - 1 - 2 * tid;
      const uint32_t a = top >= 0 ? hist[top] : 0u, b = top >= 1 ? hist[top - 1] : 0u;
      const uint32_t incl = wave_incl_scan(a + b);
      if (lane == kWave - 1) wave_tot[0][wave] = incl;
      __syncthreads();
      uint32_t before = incl - (a + b);
      for (int v = 0; v < wave; ++v) before += wave_tot[0][v];
      if (before < need && need <= before + a) {
        found[0] = (uint32_t)top;
        found[1] = need - before;
      } else if (before + a < need && need <= before + a + b) {
        found[0] = (uint32_t)(top - 1);
        found[1] = need - before - a;
      }
      __syncthreads();
      prefix = (prefix << bits) | found[0];
      need = found[1];
      shift = next;
      __syncthreads();
    }
  }
  // Kept: fixed rows, candidates above the threshold, and the first `need` candidates equal to it.
  const bool some = n_keep > n_sink + n_recent;
  uint32_t n_above = 0, n_equal = 0;
  each([&](int64_t r, float x) {
    const uint32_t k = weight_key(x);
    const bool in = r < N, c = candidate(r);
    n_above += in && (!c || (some && k > prefix)) ? 1u : 0u;
    n_equal += in && c && some && k == prefix ? 1u : 0u;
  });
  n_above = wave_sum(n_above);
  n_equal = wave_sum(n_equal);
  if (lane == 0) {
    wave_tot[0][wave] = n_above;
    wave_tot[1][wave] = n_equal;
  }
  __syncthreads();
  uint32_t equal_before = 0, at = 0;
  for (int v = 0; v < wave; ++v) {  // kept rows of the wavefronts before this one
    const uint32_t left = need > equal_before ? need - equal_before : 0u;
    at += wave_tot[0][v] + (wave_tot[1][v] < left ? wave_tot[1][v] : left);
    equal_before += wave_tot[1][v];
  }
  int64_t* rows = rows_out + (int64_t)blockIdx.x * n_keep;
  float* out = weights_out + (int64_t)blockIdx.x * n_keep;
  const uint64_t below = (1ull << lane) - 1;
  each([&](int64_t r, float x) {
    const uint32_t k = weight_key(x);
    const bool in = r < N, c = candidate(r);
    const bool equal = in && c && some && k == prefix;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(equal);
    const bool keep = (in && (!c || (some && k > prefix))) || (equal && equal_before + (uint32_t)__popcll(eq & below) < need);
    const uint64_t kept = __builtin_amdgcn_ballot_w64(keep);
    if (keep) {
      const uint32_t to = at + (uint32_t)__popcll(kept & below);
      rows[to] = r;
      out[to] = x;
    }
    at += (uint32_t)__popcll(kept);
    equal_before += (uint32_t)__popcll(eq);
  });
}

// out[h, i] = in[h, rows[h, i]] of K (z = 0) and V: a 16-byte piece a thread, rows of `pieces` pieces.
__global__ __launch_bounds__(256) void evict_gather_kernel(const int64_t* __restrict__ rows, int n_keep, int pieces,
                                                           int piece_log, const char* __restrict__ k, int64_t k_hs_b,
                                                           const char* __restrict__ v, int64_t v_hs_b,
                                                           char* __restrict__ ko, int64_t ko_hs_b,
                                                           char* __restrict__ vo, int64_t vo_hs_b) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i >> piece_log;
  if (row >= n_keep) return;
  const int h = blockIdx.y;
  const int64_t b = (i & (pieces - 1)) * 16, from = rows[(int64_t)h * n_keep + row];
  const bool is_v = blockIdx.z != 0;
  const char* src = (is_v ? v + (int64_t)h * v_hs_b : k + (int64_t)h * k_hs_b) + from * pieces * 16 + b;
  char* dst = (is_v ? vo + (int64_t)h * vo_hs_b : ko + (int64_t)h * ko_hs_b) + row * pieces * 16 + b;
  st16(dst, ld16_stream(src));
}

}  // namespace ckv

extern "C" int32_t ckv_evict_rows(void* k_out, int64_t ko_head_stride, void* v_out, int64_t vo_head_stride,
                                  int64_t* rows_out, float* weights_out, const void* k_cache, int64_t k_head_stride,
                                  const void* v_cache, int64_t v_head_stride, const float* weights,
                                  int64_t weights_head_stride, int32_t n_tokens, int32_t n_keep, int32_t n_sink,
                                  int32_t n_recent, int32_t n_heads, int32_t head_dim, int32_t dtype, void* stream) {
  using namespace ckv;
  if (n_tokens <= 0 || n_heads <= 0 || n_sink < 0 || n_recent < 0 || n_keep < 0) return CKV_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return CKV_ERR_INVALID_ARGUMENT;
  if (dtype != CKV_DTYPE_F32 && dtype != CKV_DTYPE_BF16) return CKV_ERR_INVALID_ARGUMENT;
  if (n_keep > n_tokens || (int64_t)n_sink + n_recent > n_keep) return CKV_ERR_OUT_OF_RANGE;
  if (n_keep == 0) return CKV_OK;
  if (k_out == nullptr || v_out == nullptr || rows_out == nullptr || weights_out == nullptr || k_cache == nullptr ||
      v_cache == nullptr || weights == nullptr)
    return CKV_ERR_INVALID_ARGUMENT;
  const int eb = dtype == CKV_DTYPE_BF16 ? 2 : 4, vec = 16 / eb;
  if (k_head_stride % vec || v_head_stride % vec || ko_head_stride % vec || vo_head_stride % vec) return CKV_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16) return CKV_ERR_INVALID_ARGUMENT;
  if (k_head_stride < (int64_t)n_tokens * head_dim || v_head_stride < (int64_t)n_tokens * head_dim ||
      weights_head_stride < n_tokens || ko_head_stride < (int64_t)n_keep * head_dim || vo_head_stride < (int64_t)n_keep * head_dim)
    return CKV_ERR_OUT_OF_RANGE;
  if (n_heads > 65535) return CKV_ERR_TOO_LARGE;
  hipStream_t s = (hipStream_t)stream;
  const int steps = (int)(((int64_t)n_tokens + kEvictThreads - 1) / kEvictThreads);
  auto select = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_heads), dim3(kEvictThreads), 0, s, weights, weights_head_stride, n_tokens, n_keep, n_sink,
                       n_recent, steps, rows_out, weights_out);
  };
  if (steps <= 8) select(evict_select_kernel<8>);
  else if (steps <= 16) select(evict_select_kernel<16>);
  else if (steps <= 36) select(evict_select_kernel<36>);
  else select(evict_select_kernel<0>);
  CKV_RETURN_IF_LAUNCH_FAILED();
  const int pieces = head_dim * eb / 16;  // 8 to 64, a power of two
  const int64_t blocks = ((int64_t)n_keep * pieces + 255) / 256;
  hipLaunchKernelGGL(evict_gather_kernel, dim3((unsigned)blocks, (unsigned)n_heads, 2), dim3(256), 0, s, rows_out, n_keep, pieces,
                     __builtin_ctz((unsigned)pieces), (const char*)k_cache, k_head_stride * eb, (const char*)v_cache,
                     v_head_stride * eb, (char*)k_out, ko_head_stride * eb, (char*)v_out, vo_head_stride * eb);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}
