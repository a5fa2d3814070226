// Logits adjusted before a token is chosen (no counterpart in the reference, whose decode takes the plain argmax of
// src/chunkkv/engine/torch_engine.py:197): penalties for tokens that are there already, a bias, a grammar's mask.
//   c = how often v was generated, seen = c > 0 or v is in the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * c - presence            (c > 0 only)
//   x = x + bias[v];   x = -inf where v is not allowed
// in fp32, each step rounded once. The token is the first of the largest (a NaN above every number, as torch's argmax).
//
// A workgroup has a slice of a row's vocabulary: it counts the row's tokens that fall into the slice in LDS (integer
// atomics: any order gives the same counts), while its logits are on their way, then reads each logit once.
// No table of counts over the vocabulary exists in memory, so there is no state to keep, and a step reads the logits and
// the tokens. Bound: latency up to a few rows, the logits' bytes (and the result's) beyond.
#include "ckv_common.hpp"

namespace ckv {

// Loads and stores of 16 bytes wherever an element may lie: rows of an odd vocabulary start anywhere.
__device__ __forceinline__ vec16 ld16_any(const void* p) {
  vec16 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void st16_any(void* p, const vec16& v) { __builtin_memcpy(p, &v, 16); }

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

constexpr int kLogitsEach = 8;  // logits of a thread
constexpr uint32_t kInPrompt = 1u << 31;

// f over the row's tokens that lie in [v0, v0 + count), as offsets. A batch's loads go out together, the last one's too
// (past the row's end they read its last pair again, which is passed over).
template <int NT, typename F>
__device__ __forceinline__ void each_token(const Tokens& t, int row, int64_t v0, int count, F f) {
  const int64_t* p = t.at + row * t.stride;
  constexpr int U = 4;
  auto take = [&](int64_t v) {
    const uint64_t o = (uint64_t)(v - v0);
    if (o < (uint64_t)count) f((int)o);
  };
  const int pairs = t.n / 2;
  for (int i0 = 0; i0 < pairs; i0 += U * NT) {
    vec16 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = ld16_any(p + 2 * min(i0 + u * NT + (int)threadIdx.x, pairs - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * NT + (int)threadIdx.x >= pairs) continue;
      take((int64_t)((uint64_t)v[u][1] << 32 | v[u][0]));
      take((int64_t)((uint64_t)v[u][3] << 32 | v[u][2]));
    }
  }
  if ((t.n & 1) != 0 && threadIdx.x == 0) take(p[t.n - 1]);
}

// A logit as a key whose order is argmax's: larger logits first, a NaN above all, -0 as 0; then the lower index.
__device__ __forceinline__ uint64_t logit_key(float x, int v) {
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t order = x != x ? UINT32_MAX : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)order << 32 | (uint32_t)(INT32_MAX - v);
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

// WRITE: the adjusted logits to out; else each slice's best key to keys, or the token where a row is one slice.
template <typename E, int NT, bool WRITE>
__global__ __launch_bounds__(NT) void adjust_logits_kernel(const char* __restrict__ logits, int64_t row_b, int V, Adjust a,
                                                           float* __restrict__ out, uint64_t* __restrict__ keys,
                                                           int64_t* __restrict__ tokens, int32_t* __restrict__ err) {
  constexpr int N = kLogitsEach, SLICE = NT * N, VN = N / E::kVec;
  __shared__ uint32_t s_count[SLICE];
  const int row = blockIdx.y, v0 = blockIdx.x * SLICE, v = v0 + threadIdx.x * N;
  const int here = min(N, V - v);  // <= 0: past the vocabulary
  const char* p = logits + row * row_b + (int64_t)v * E::kBytes;
  float x[N];
  vec16 raw[VN];
  if (here >= N) {
#pragma unroll
    for (int i = 0; i < VN; ++i) raw[i] = ld16_any(p + 16 * i);
  }
  const float* bias = a.bias != nullptr ? a.bias + row * a.bias_stride + v : nullptr;
  vec16 b[N / 4];
  if (bias != nullptr && here >= N) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) b[i] = ld16_any(bias + 4 * i);
  }
  uint32_t bits = ~0u;
  if (a.allowed != nullptr && here > 0) bits = a.allowed[row * a.allowed_stride + v / 32] >> (v % 32);

  const bool history = a.prompt.n > 0 || a.generated.n > 0;
  if (history) {
#pragma unroll
    for (int i = 0; i < N; ++i) s_count[i * NT + threadIdx.x] = 0;
    __syncthreads();
    // a thread's N logits are N words NT apart, so that its reads below spread over the banks
    auto word = [](int o) { return (o % N) * NT + o / N; };
    if (a.prompt.n > 0) each_token<NT>(a.prompt, row, v0, SLICE, [&](int o) { atomicOr(&s_count[word(o)], kInPrompt); });
    if (a.generated.n > 0) each_token<NT>(a.generated, row, v0, SLICE, [&](int o) { atomicAdd(&s_count[word(o)], 1u); });
    __syncthreads();
  }
  if (here >= N) {
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      float f[E::kVec];
      E::unpack(raw[i], f);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) x[i * E::kVec + j] = f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = 0.f;
      if (i < here) {
        if constexpr (E::kBytes == 2) x[i] = bf16_bits_to_f32(((const uint16_t*)p)[i]);
        else x[i] = ((const float*)p)[i];
      }
    }
  }
  if (history) {
    const float r = a.repetition.at(row), f = a.frequency.at(row), pr = a.presence.at(row);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t s = s_count[i * NT + threadIdx.x];
      if (s == 0) continue;
      x[i] = x[i] > 0.f ? x[i] / r : x[i] * r;
      const uint32_t c = s & ~kInPrompt;
      if (c > 0) x[i] = x[i] - f * (float)c - pr;
    }
  }
  if (bias != nullptr) {
    if (here >= N) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += __uint_as_float(b[i / 4][i % 4]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < here) x[i] += bias[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (!(bits >> i & 1)) x[i] = -INFINITY;

  if constexpr (WRITE) {
    float* to = out + (int64_t)row * V + v;
    if (here >= N) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        st16_any(to + 4 * i, vec16{__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]),
                                   __float_as_uint(x[4 * i + 3])});
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < here) to[i] = x[i];
    }
  } else {
    uint64_t best = 0;  // below every logit's key
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < here) best = max(best, logit_key(x[i], v + i));
    __shared__ uint64_t s_best[NT / kWave];
    best = wave_max(best);
    if (threadIdx.x % kWave == 0) s_best[threadIdx.x / kWave] = best;
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    best = wave_max(threadIdx.x < NT / kWave ? s_best[threadIdx.x] : 0);
    if (threadIdx.x != 0) return;
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

constexpr int kLogitsThreads = 512;
static inline int64_t logits_slices(int64_t vocab) { return (vocab + kLogitsThreads * kLogitsEach - 1) / (kLogitsThreads * kLogitsEach); }

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
  if (n_rows > 65535 || vocab > INT32_MAX - kLogitsThreads * kLogitsEach) return CKV_ERR_TOO_LARGE;
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
  if (e == 2) launch(adjust_logits_kernel<Elem<CKV_DTYPE_BF16>, kLogitsThreads, WRITE>);
  else launch(adjust_logits_kernel<Elem<CKV_DTYPE_F32>, kLogitsThreads, WRITE>);
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
