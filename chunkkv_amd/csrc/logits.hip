// Logits adjusted before a token is chosen (no counterpart in the reference, whose decode takes the plain argmax of
// src/chunkkv/engine/torch_engine.py:197): penalties for tokens that are there already, a bias, a grammar's mask.
//   c = how often v was generated, seen = c > 0 or v is in the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * c - presence            (c > 0 only)
//   x = x + bias[v];   x = -inf where v is not allowed
// in fp32, each step rounded once. The token is the first of the largest (a NaN above every number, as torch's argmax).
//
// A workgroup has a slice of a row's vocabulary: it counts the row's tokens that fall into the slice in LDS (integer
// atomics: any order gives the same counts), while its logits are on their way, then reads each logit once. No table of
// counts over the vocabulary exists in memory, so there is no state to keep, and a step reads the logits and the
// tokens. Bound: latency up to a few rows (one row of 152064 behind 8302 + 256 tokens 6.0 us traced and 1.4 for the
// joined slices: 8.4 in a graph), the logits' bytes and the result's beyond (64 rows under a grammar with a bias, 61
// MB, 15.4 us: 4.0 TB/s).
#include "attention_common.hpp"

namespace ckv {

// Sixteen bytes wherever an element may lie. Loads and stores here are of this kind: rows of an odd vocabulary start
// anywhere, and the device takes 16 bytes at any address.
__device__ __forceinline__ vec16 ld16_any(const void* p) {
  vec16 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

struct RowValue {  // of a row: rows[b], or one for all
  const float* rows;
  float all;
  __device__ float at(int b) const { return rows != nullptr ? rows[b] : all; }
};
struct Tokens {
  const int64_t* at;
  int64_t stride;
  int n;
};
struct Adjust {
  Tokens prompt, generated;
  RowValue repetition, frequency, presence;
  const float* bias;
  int64_t bias_stride;
  const uint32_t* allowed;
  int64_t allowed_stride;
};

constexpr int kLogitsThreads = 512, kLogitsEach = 8;  // logits of a thread
constexpr int kLogitsSlice = kLogitsThreads * kLogitsEach;
constexpr uint32_t kInPrompt = 1u << 31;
// Pairs of tokens that a thread, and a workgroup, has in flight.
constexpr int kPairsEach = 4, kPairsStep = kPairsEach * kLogitsThreads;

// Counts the row's tokens that lie in [v0, v0 + kLogitsSlice) into count[]: occurrences in generated, kInPrompt where
// it is in the prompt. Both lists are one of pairs, whose loads go out U at a time for each thread, the last of them
// too (past the end they read the last pair again, which is passed over).
__device__ __forceinline__ void count_tokens(const Tokens& prompt, const Tokens& generated, int row, int64_t v0, uint32_t* count) {
  const int64_t* pt = prompt.at + row * prompt.stride;
  const int64_t* gt = generated.at + row * generated.stride;
  const int pp = prompt.n / 2, pairs = pp + generated.n / 2;
  constexpr int NT = kLogitsThreads, U = kPairsEach;
  auto take = [&](int64_t v, bool in_prompt) {
    const uint64_t o = (uint64_t)v - (uint64_t)v0;  // any token
    if (o >= (uint64_t)kLogitsSlice) return;
    if (in_prompt) atomicOr(&count[o], kInPrompt);
    else atomicAdd(&count[o], 1u);
  };
  for (int i0 = 0; i0 < pairs; i0 += kPairsStep) {
    vec16 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * NT >= pairs) continue;  // uniform
      const int i = min(i0 + u * NT + (int)threadIdx.x, pairs - 1);
      v[u] = ld16_any(i < pp ? pt + 2 * i : gt + 2 * (i - pp));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT + (int)threadIdx.x;
      if (i0 + u * NT >= pairs || i >= pairs) continue;
      take((int64_t)((uint64_t)v[u][1] << 32 | v[u][0]), i < pp);
      take((int64_t)((uint64_t)v[u][3] << 32 | v[u][2]), i < pp);
    }
  }
  if ((prompt.n & 1) != 0 && threadIdx.x == 0) take(pt[prompt.n - 1], true);
  if ((generated.n & 1) != 0 && threadIdx.x == 64) take(gt[generated.n - 1], false);
}

// A logit as a number whose order is argmax's: a NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t logit_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 + 0 is 0
  return x != x ? UINT32_MAX : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
// And with its place: of equal ones the first is the larger.
__device__ __forceinline__ uint64_t logit_key(uint32_t order, int v) { return (uint64_t)order << 32 | (uint32_t)(INT32_MAX - v); }
// The key of the wavefront's largest, for places that ascend with the lanes.
__device__ __forceinline__ uint64_t wave_best(uint32_t order, int v) {
  auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  uint32_t m = row16_reduce(order, up);
  auto pair = [&](auto r) { return up(r[0], r[1]); };
  m = pair(__builtin_amdgcn_permlane16_swap(m, m, false, false));
  m = pair(__builtin_amdgcn_permlane32_swap(m, m, false, false));
  const int first = __builtin_ctzll(__builtin_amdgcn_ballot_w64(order == m));
  return logit_key(m, __builtin_amdgcn_readlane(v, first));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    const uint64_t y = (uint64_t)__shfl_xor((unsigned long long)x, d);
    x = y > x ? y : x;
  }
  return x;
}
__device__ __forceinline__ void store_token(int64_t* to, uint64_t key, int32_t* err) {
  constexpr uint32_t kNegInf = ~0xff800000u;
  *to = INT32_MAX - (uint32_t)key;
  if ((uint32_t)(key >> 32) == kNegInf) flag_error(err, CKV_DEVICE_ERR_NO_TOKEN);
}

// WRITE: the adjusted logits to out; else each slice's best key to keys, or the token where a row is one slice. A
// thread's logits are vectors of W, a workgroup's threads side by side: 16 bytes of what is written, or else of what is
// read.
template <typename E, bool WRITE>
__global__ __launch_bounds__(kLogitsThreads) void adjust_logits_kernel(const char* __restrict__ logits, int64_t row_b, int V, Adjust a,
                                                                       float* __restrict__ out, uint64_t* __restrict__ keys,
                                                                       int64_t* __restrict__ tokens, int32_t* __restrict__ err) {
  constexpr int NT = kLogitsThreads, W = WRITE ? 4 : E::kVec, NV = kLogitsEach / W;
  __shared__ __attribute__((aligned(16))) uint32_t s_count[kLogitsSlice];
  const int row = blockIdx.y, v0 = blockIdx.x * kLogitsSlice, tid = threadIdx.x;
  const char* p = logits + row * row_b;
  const float* bias = a.bias != nullptr ? a.bias + row * a.bias_stride : nullptr;
  const uint32_t* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
  auto first = [&](int k) { return v0 + (k * NT + tid) * W; };
  float x[NV][W], add[NV][W];
  uint32_t bits[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int v = first(k);
    if (v + W <= V) {
      uint32_t w[W * E::kBytes / 4];
      __builtin_memcpy(w, p + (int64_t)v * E::kBytes, sizeof(w));
#pragma unroll
      for (int i = 0; i < W; ++i)
        x[k][i] = E::kBytes == 4 ? __uint_as_float(w[i]) : __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      if (bias != nullptr) __builtin_memcpy(add[k], bias + v, sizeof(add[k]));
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        x[k][i] = add[k][i] = 0.f;
        if (v + i >= V) continue;
        if constexpr (E::kBytes == 2) x[k][i] = bf16_bits_to_f32(((const uint16_t*)p)[v + i]);
        else x[k][i] = ((const float*)p)[v + i];
        if (bias != nullptr) add[k][i] = bias[v + i];
      }
    }
    bits[k] = ~0u;
    if (allowed != nullptr && v < V) bits[k] = allowed[v / 32] >> (v % 32);
  }

  if (a.prompt.n > 0 || a.generated.n > 0) {
#pragma unroll
    for (int i = 0; i < kLogitsEach / 4; ++i) ((vec16*)s_count)[i * NT + tid] = vec16{0, 0, 0, 0};
    __syncthreads();
    count_tokens(a.prompt, a.generated, row, v0, s_count);
    __syncthreads();
    const float r = a.repetition.at(row), f = a.frequency.at(row), pr = a.presence.at(row);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      uint32_t s[W], any = 0;
#pragma unroll
      for (int i = 0; i < W / 4; ++i) *(vec16*)(s + 4 * i) = *(const vec16*)(s_count + (k * NT + tid) * W + 4 * i);
#pragma unroll
      for (int i = 0; i < W; ++i) any |= s[i];
      if (__builtin_amdgcn_ballot_w64(any != 0) == 0) continue;  // uniform: most of a vocabulary
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (__builtin_amdgcn_ballot_w64(s[i] != 0) == 0) continue;
        const float y = x[k][i] > 0.f ? x[k][i] / r : x[k][i] * r;
        const uint32_t c = s[i] & ~kInPrompt;
        x[k][i] = s[i] == 0 ? x[k][i] : c == 0 ? y : y - f * (float)c - pr;
      }
    }
  }
  if (bias != nullptr) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) x[k][i] += add[k][i];
  }
  if (allowed != nullptr) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (!(bits[k] >> i & 1)) x[k][i] = -INFINITY;
  }

  if constexpr (WRITE) {
    // non-temporal: 64 rows of 152064, 61 MB, take 15.4 us in place of 18.2 (without a history 9.8 and 12.2)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = first(k);
      float* to = out + (int64_t)row * V + v;
      if (v + W <= V) {
        typedef float any4 __attribute__((ext_vector_type(4), aligned(4)));
        static_assert(W == 4, "one store");
        __builtin_nontemporal_store(any4{x[k][0], x[k][1], x[k][2], x[k][3]}, (any4*)to);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (v + i < V) to[i] = x[k][i];
      }
    }
  } else {
    uint64_t best = 0;  // below every logit
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      uint32_t top = 0;
      int place = first(k);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint32_t o = first(k) + i < V ? logit_order(x[k][i]) : 0;
        place = o > top ? first(k) + i : place;
        top = o > top ? o : top;
      }
      const uint64_t key = wave_best(top, place);
      best = key > best ? key : best;
    }
    __shared__ uint64_t s_best[NT / kWave];
    if (tid % kWave == 0) s_best[tid / kWave] = best;
    __syncthreads();
    if (tid >= kWave) return;
    best = wave_max(tid < NT / kWave ? s_best[tid] : 0);
    if (tid != 0) return;
    if (gridDim.x == 1) store_token(tokens + row, best, err);
    else keys[(int64_t)row * gridDim.x + blockIdx.x] = best;
  }
}

// A wavefront a row: the largest of its slices' keys.
__global__ __launch_bounds__(kWave) void best_token_kernel(const uint64_t* __restrict__ keys, int slices,
                                                           int64_t* __restrict__ tokens, int32_t* __restrict__ err) {
  const int row = blockIdx.x;
  uint64_t best = 0;
  for (int i = threadIdx.x; i < slices; i += kWave) best = max(best, keys[(int64_t)row * slices + i]);
  best = wave_max(best);
  if (threadIdx.x == 0) store_token(tokens + row, best, err);
}

static inline int64_t logits_slices(int64_t vocab) { return (vocab + kLogitsSlice - 1) / kLogitsSlice; }

static int32_t check_adjust(const void* logits, int64_t row_stride, int32_t n_rows, int32_t vocab, int32_t dtype, const Adjust& a) {
  if (n_rows < 0 || vocab <= 0 || (dtype != CKV_DTYPE_BF16 && dtype != CKV_DTYPE_F32)) return CKV_ERR_INVALID_ARGUMENT;
  if (n_rows == 0) return CKV_OK;
  const int e = dtype == CKV_DTYPE_BF16 ? 2 : 4;
  if (logits == nullptr || (uintptr_t)logits % e) return CKV_ERR_INVALID_ARGUMENT;
  for (const Tokens* t : {&a.prompt, &a.generated}) {
    if (t->n < 0 || (t->n > 0 && (t->at == nullptr || (uintptr_t)t->at % 8))) return CKV_ERR_INVALID_ARGUMENT;
    if (t->n > 0 && n_rows > 1 && t->stride < 0) return CKV_ERR_OUT_OF_RANGE;
  }
  if ((uintptr_t)a.bias % 4 || (uintptr_t)a.allowed % 4) return CKV_ERR_INVALID_ARGUMENT;
  if (n_rows > 1 && (row_stride < vocab || a.bias_stride < 0 || a.allowed_stride < 0)) return CKV_ERR_OUT_OF_RANGE;
  if (n_rows > 65535 || vocab > INT32_MAX - kLogitsSlice) return CKV_ERR_TOO_LARGE;
  if ((int64_t)a.prompt.n / 2 + a.generated.n / 2 > INT32_MAX - kPairsStep) return CKV_ERR_TOO_LARGE;  // count_tokens' numbers
  return CKV_OK;
}

template <bool WRITE>
static int32_t adjust_launch(const void* logits, int64_t row_stride, int32_t n_rows, int32_t vocab, int32_t dtype, const Adjust& a,
                             float* out, uint64_t* keys, int64_t* tokens, int32_t* err, hipStream_t st) {
  const dim3 grid((unsigned)logits_slices(vocab), (unsigned)n_rows);
  const int e = dtype == CKV_DTYPE_BF16 ? 2 : 4;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kLogitsThreads), 0, st, (const char*)logits, row_stride * e, vocab, a, out, keys, tokens, err);
  };
  if (e == 2) launch(adjust_logits_kernel<Elem<CKV_DTYPE_BF16>, WRITE>);
  else launch(adjust_logits_kernel<Elem<CKV_DTYPE_F32>, WRITE>);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}

}  // namespace ckv

#define CKV_ADJUST_ARGS                                                                                              \
  const void *logits, int64_t logits_row_stride, int32_t n_rows, int32_t vocab, int32_t dtype, const int64_t *prompt, \
      int64_t prompt_row_stride, int32_t n_prompt, const int64_t *generated, int64_t generated_row_stride,            \
      int32_t n_generated, const float *repetition_rows, float repetition, const float *frequency_rows,               \
      float frequency, const float *presence_rows, float presence, const float *bias, int64_t bias_row_stride,        \
      const int32_t *allowed, int64_t allowed_row_stride
#define CKV_ADJUST                                                                                                  \
  Adjust {                                                                                                          \
    {prompt, prompt_row_stride, n_prompt}, {generated, generated_row_stride, n_generated}, {repetition_rows, repetition}, \
        {frequency_rows, frequency}, {presence_rows, presence}, bias, bias_row_stride, (const uint32_t*)allowed,    \
        allowed_row_stride                                                                                          \
  }

extern "C" int32_t ckv_adjust_logits(float* out, CKV_ADJUST_ARGS, void* stream) {
  using namespace ckv;
  const Adjust a = CKV_ADJUST;
  const int32_t bad = check_adjust(logits, logits_row_stride, n_rows, vocab, dtype, a);
  if (bad != CKV_OK || n_rows == 0) return bad;
  if (out == nullptr || (uintptr_t)out % 4) return CKV_ERR_INVALID_ARGUMENT;
  return adjust_launch<true>(logits, logits_row_stride, n_rows, vocab, dtype, a, out, nullptr, nullptr, nullptr, (hipStream_t)stream);
}

extern "C" int64_t ckv_next_tokens_workspace_bytes(int32_t n_rows, int32_t vocab) {
  if (n_rows <= 0 || vocab <= 0) return 0;
  const int64_t slices = ckv::logits_slices(vocab);
  return slices > 1 ? n_rows * slices * 8 : 0;
}

extern "C" int32_t ckv_next_tokens(int64_t* tokens, CKV_ADJUST_ARGS, void* workspace, int64_t workspace_bytes, int32_t* err,
                                   void* stream) {
  using namespace ckv;
  const Adjust a = CKV_ADJUST;
  const int32_t bad = check_adjust(logits, logits_row_stride, n_rows, vocab, dtype, a);
  if (bad != CKV_OK || n_rows == 0) return bad;
  if (tokens == nullptr || (uintptr_t)tokens % 8) return CKV_ERR_INVALID_ARGUMENT;
  const int64_t need = ckv_next_tokens_workspace_bytes(n_rows, vocab);
  if (need > 0 && (workspace == nullptr || (uintptr_t)workspace % 8 || workspace_bytes < need)) return CKV_ERR_INVALID_ARGUMENT;
  const int32_t st = adjust_launch<false>(logits, logits_row_stride, n_rows, vocab, dtype, a, nullptr, (uint64_t*)workspace, tokens,
                                          err, (hipStream_t)stream);
  if (st != CKV_OK || need == 0) return st;
  hipLaunchKernelGGL(best_token_kernel, dim3((unsigned)n_rows), dim3(kWave), 0, (hipStream_t)stream, (const uint64_t*)workspace,
                     (int)logits_slices(vocab), tokens, err);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}
