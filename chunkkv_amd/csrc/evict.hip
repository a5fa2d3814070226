// A cache cut to its heaviest rows. Per KV head: the first n_sink rows and the last n_recent stay, and of the others
// those of the largest weight (what attention_weights.hip adds up) until n_keep stay, the lower row first among
// equals; a NaN ranks below every number. The kept rows move to the front of new caches, in order.
//
// Design: a row becomes an integer that orders as its weight does, above all of them for a row that stays anyway, and
// the n_keep-th largest (with how many of its equals stay) comes out of a radix histogram in LDS of 11, 11 and 10 bits.
// Up to 34,816 rows one launch does everything: the integers of a head's rows stay in LDS (in registers they unroll every pass,
// for the same time), a wavefront has a run of consecutive rows, so that the places of kept rows are ballots and a scan over
// 16 wavefronts. Many workgroups a head
// find the same threshold, each for a slice of the kept rows that it then copies: the selection is the latency of
// one CU whatever is done, and this way no launch waits for it. Longer caches: one workgroup a head reads the weights
// again for each pass, and evict_gather_kernel copies.
// Weights of 0, as rows that no query reached have, are counted by ballots: atomics on one address queue (a fifth of 32832 rows at 0
// 19.1 -> 17.6 us). The first histogram counts a row as it arrives (32832 rows of 4 heads of 128 cut to 4104 20.1 -> 19.1 us), and a bin that stays whole
// needs no further pass (20.9 -> 20.1; 60000 to 4000, where each pass reads the weights again, 52 -> 49).
// Bound: the issue of the CU that selects. Those 17.6 us by phase, about: rows and first pass 5, the other two 3, count 2, list
// and copy 2, the rest start and launch; 1103 fp32 rows of 2 heads of 64 cut to 300 take 5.5 (eager calls 6.4, the host's time), mostly the
// passes' scans and barriers.
// One workgroup a head with a copy launch behind it took 46 and 11.4.
#include <algorithm>

#include "ckv_common.hpp"

namespace ckv {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;
constexpr int kEvictBins = 2048;
constexpr int kEvictCopies = 2;                 // of the first histogram: a lane counts into lane % 2's
constexpr int kEvictPitch = kEvictBins + 16;    // copies of a bin on banks of their own
constexpr int kEvictList = 2048;                // kept rows that a workgroup lists at a time
constexpr int kEvictKeys = 34 * 1024;           // rows whose integers LDS holds, at most
constexpr uint32_t kKeyZero = 0x80000000u;   // of the weight 0
constexpr uint32_t kKeyFixed = 0xffffffffu;     // a row that stays, above every weight's key

// An integer that orders as the weight does: 1 for a NaN, below -infinity's; 0 is no row's.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t b = __float_as_uint(w + 0.f);  // -0 becomes 0
  const uint32_t k = b ^ (uint32_t)((int32_t)b >> 31 | (int32_t)0x80000000);
  return w != w ? 1u : k;
}

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // four floats on any float's address

// How many bits of the mask are below this lane, plus `more`.
__device__ __forceinline__ uint32_t bits_below(uint64_t mask, uint32_t more) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, more));
}

// A workgroup barrier behind which LDS writes are seen; global loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct EvictCopy {
  const char *k, *v;
  char *ko, *vo;
  int64_t k_hs_b, v_hs_b, ko_hs_b, vo_hs_b;
  int piece_log;  // log2 of the 16-byte pieces of a row
};

// PER: 256-row steps of a wavefront's run, at most; 0: any number, the weights read again for each pass, and no copy
// (copy.ko unused). KEYS: rows whose integers LDS holds. A lane has four consecutive rows of a step. blockIdx.x: the slice of `slice` kept rows,
// blockIdx.y: the head.
template <int PER, int KEYS>
__global__ __launch_bounds__(kEvictThreads) void evict_kernel(const float* __restrict__ weights, int64_t w_hs, int N,
                                                              int n_keep, int n_sink, int n_recent, int run_steps,
                                                              int slice, int64_t* __restrict__ rows_out,
                                                              float* __restrict__ weights_out, EvictCopy copy) {
  constexpr int STEP = 4 * kWave;
  __shared__ __attribute__((aligned(16))) uint32_t keys[PER > 0 ? KEYS : 4];
  __shared__ uint32_t hist0[kEvictCopies * kEvictPitch];  // the first pass's copies; a copy each of the later passes
  static_assert(kEvictCopies == 2, "the passes' histograms");
  static_assert(KEYS % STEP == 0 && PER * STEP * kEvictWaves >= KEYS, "whole steps");
  __shared__ uint32_t wave_tot[3][kEvictWaves];
  __shared__ uint32_t wave_gt[kEvictWaves], wave_eq[kEvictWaves];
  __shared__ uint32_t step_count[kEvictWaves][PER > 0 ? PER : 1];
  __shared__ uint32_t found[3][3];  // the bin, the kept keys in it, its keys
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int h = blockIdx.y;
  const float* w = weights + (int64_t)h * w_hs;
  const int64_t run = (int64_t)wave * run_steps * STEP;  // this wavefront's first row
  const int tail = N - n_recent;
  const int steps = (int)max((int64_t)0, min((int64_t)run_steps, (N - run + STEP - 1) / STEP));  // with a row
  auto load4 = [&](int i, float(&x)[4]) {
    const int64_t r = run + (int64_t)i * STEP + 4 * lane;
    if (run + (int64_t)(i + 1) * STEP <= N) {  // uniform: a whole step
      const f32x4_any v = *(const f32x4_any*)(w + r);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = w[min(r + j, (int64_t)N - 1)];
    }
  };
  auto keys4 = [&](int i, const float(&x)[4], uint32_t(&k)[4]) {
    const int64_t s0 = run + (int64_t)i * STEP;
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = weight_key(x[j]);
    if (s0 < n_sink || s0 + STEP > tail) {  // uniform: rows that stay, or past the cache, among them
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t r = s0 + 4 * lane + j;
        if (r < n_sink || r >= tail) k[j] = r < N ? kKeyFixed : 0u;
      }
    }
  };
  uint32_t* mine = hist0 + (lane % kEvictCopies) * kEvictPitch;
  uint32_t zeros = 0;  // of this wavefront
  auto count4 = [&](const uint32_t(&k)[4]) {  // the first pass; key 0 counts below every row's
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool zero = k[j] == kKeyZero;
      zeros += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(zero));
      if (!zero) atomicAdd(&mine[k[j] >> 21], 1u);
    }
  };
  auto clear = [&] {
    for (int b = tid; b < kEvictCopies * kEvictPitch; b += kEvictThreads) hist0[b] = 0;
    lds_barrier();
  };
  if constexpr (PER > 0) {
    float x[PER][4];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < steps) load4(i, x[i]);
    clear();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < steps) {
        uint32_t k[4];
        keys4(i, x[i], k);
        const int at = (wave * run_steps + i) * STEP + 4 * lane;  // only this wavefront reads them
        *(vec16*)(keys + at) = vec16{k[0], k[1], k[2], k[3]};
        count4(k);
      }
  } else {
    clear();
  }
  // f(step, keys) for each of this thread's steps (key 0: no row)
  auto each = [&](auto f) {
    if constexpr (PER > 0) {
      const vec16* at = (const vec16*)(keys + wave * run_steps * STEP) + lane;
      vec16 next = *at;  // a step ahead of its use
#pragma unroll 1
      for (int i = 0; i < steps; ++i) {
        const uint32_t k[4] = {next.x, next.y, next.z, next.w};
        next = at[min(i + 1, steps - 1) * kWave];
        f(i, k);
      }
    } else {
      for (int i = 0; i < steps; ++i) {
        float x[4];
        uint32_t k[4];
        load4(i, x);
        keys4(i, x, k);
        f(i, k);
      }
    }
  };

  uint32_t need = (uint32_t)n_keep, prefix = 0;  // kept among the keys that start with the bits found
  bool whole = false;                             // all of them are: the bits behind need not be known
  auto pass = [&](int p, int bits, uint32_t a, uint32_t b) {
    // the bin, from the top, in which the need-th key lies: two bins (a, then b) a thread
    const int top = (1 << bits) - 1 - 2 * tid;
    const uint32_t incl = wave_incl_scan(a + b);
    if (lane == kWave - 1) wave_tot[p][wave] = incl;
    __syncthreads();
    // of the wavefronts before this one: lane v has wavefront v's total
    const uint32_t tots = wave_incl_scan(lane < kEvictWaves ? wave_tot[p][lane % kEvictWaves] : 0u);
    const uint32_t before = incl - (a + b) + (wave > 0 ? (uint32_t)__builtin_amdgcn_readlane((int)tots, wave - 1) : 0u);
    if (before < need && need <= before + a) {
      found[p][0] = (uint32_t)top;
      found[p][1] = need - before;
      found[p][2] = a;
    } else if (before + a < need && need <= before + a + b) {
      found[p][0] = (uint32_t)(top - 1);
      found[p][1] = need - before - a;
      found[p][2] = b;
    }
    __syncthreads();
    prefix = (prefix << bits) | (uint32_t)__builtin_amdgcn_readfirstlane((int)found[p][0]);
    need = (uint32_t)__builtin_amdgcn_readfirstlane((int)found[p][1]);
    whole = need == (uint32_t)__builtin_amdgcn_readfirstlane((int)found[p][2]) && prefix != 0;  // (0: among keys of no row)
    if (whole && p < 2) {  // then the keys above the bin's last predecessor stay, and none of that
      prefix = (prefix << (p == 0 ? 21 : 10)) - 1u;
      need = 0;
    }
  };
  {
    if constexpr (PER == 0) each([&](int, const uint32_t(&k)[4]) { count4(k); });
    if (lane == 0) atomicAdd(&mine[kKeyZero >> 21], zeros);
    __syncthreads();
    const int top = kEvictBins - 1 - 2 * tid;
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int c = 0; c < kEvictCopies; ++c) {
      a += hist0[c * kEvictPitch + top];
      b += hist0[c * kEvictPitch + top - 1];
      hist0[c * kEvictPitch + top] = hist0[c * kEvictPitch + top - 1] = 0;  // this thread's own, for the next passes
    }
    pass(0, 11, a, b);
  }
#pragma unroll 1
  for (int p = 1; p < 3 && !whole; ++p) {
    const int bits = p == 1 ? 11 : 10, shift = p == 1 ? 21 : 10, next = p == 1 ? 10 : 0;
    const uint32_t low = prefix << shift, span = 1u << shift;
    uint32_t* bins = hist0 + (p - 1) * kEvictPitch;
    each([&](int, const uint32_t(&k)[4]) {
      uint32_t d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = k[j] - low;
      if (min(min(d[0], d[1]), min(d[2], d[3])) < span) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d[j] < span) atomicAdd(&bins[d[j] >> next], 1u);
      }
    });
    __syncthreads();
    const int top = (1 << bits) - 1 - 2 * tid;
    pass(p, bits, top >= 0 ? bins[max(top, 0)] : 0u, top >= 1 ? bins[max(top - 1, 0)] : 0u);
  }
  // Kept: keys above prefix, and of those equal to it the first `need`.
  uint32_t n_gt = 0, n_eq = 0;
  each([&](int i, const uint32_t(&k)[4]) {
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      gt += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(k[j] > prefix));
      eq += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(k[j] == prefix));
    }
    n_gt += gt;
    n_eq += eq;
    if constexpr (PER > 0) {
      if (lane == 0) step_count[wave][i] = gt | eq << 16;
    }
  });
  if (lane == 0) {
    wave_gt[wave] = n_gt;
    wave_eq[wave] = n_eq;
  }
  __syncthreads();
  // equals, and kept rows, of the wavefronts before this one: lane v has wavefront v's
  const uint32_t v_eq = lane < kEvictWaves ? wave_eq[lane % kEvictWaves] : 0u, v_gt = lane < kEvictWaves ? wave_gt[lane % kEvictWaves] : 0u;
  const uint32_t eq_incl = wave_incl_scan(v_eq), eq_excl = eq_incl - v_eq;
  const uint32_t v_kept = v_gt + min(v_eq, need > eq_excl ? need - eq_excl : 0u);
  const uint32_t kept_incl = wave_incl_scan(v_kept);
  const uint32_t eq_before = (uint32_t)__builtin_amdgcn_readlane((int)eq_excl, wave);
  const uint32_t kept_end = (uint32_t)__builtin_amdgcn_readlane((int)kept_incl, wave);
  const uint32_t kept_before = kept_end - (uint32_t)__builtin_amdgcn_readlane((int)v_kept, wave);

  // Where the kept rows of each step start, a step a lane, and the steps that have some in [o0, o1).
  uint32_t step_at = 0, step_eq = 0, step_end = 0;
  if constexpr (PER > 0) {
    const uint32_t c = lane < steps ? step_count[wave][lane % PER] : 0u, eq = c >> 16;
    step_eq = eq_before + wave_incl_scan(eq) - eq;
    const uint32_t kept = (c & 0xffffu) + min(eq, need > step_eq ? need - step_eq : 0u);
    step_end = kept_before + wave_incl_scan(kept);
    step_at = step_end - kept;
  }
  auto step_mask = [&](uint32_t o0, uint32_t o1) { return __builtin_amdgcn_ballot_w64(lane < steps && step_end > o0 && step_at < o1); };

  int* list = (int*)hist0;  // every wavefront is past the histograms' last read
  static_assert(kEvictList <= kEvictCopies * kEvictPitch, "the list");
  // This workgroup's slice, kEvictList rows at a time: listed by the wavefronts that have them, then copied by all.
  const uint32_t slice_end = (uint32_t)min((int64_t)n_keep, ((int64_t)blockIdx.x + 1) * slice);
  for (uint32_t o0 = (uint32_t)((int64_t)blockIdx.x * slice); o0 < slice_end; o0 += kEvictList) {
    const uint32_t o1 = min(o0 + (uint32_t)kEvictList, slice_end);
    if (kept_before < o1 && kept_end > o0) {  // uniform per wavefront
      uint32_t at = kept_before, eq_at = eq_before;
      const uint64_t wanted = step_mask(o0, o1);
      each([&](int i, const uint32_t(&k)[4]) {
        if constexpr (PER > 0) {
          if (!(wanted >> i & 1)) return;  // uniform
          at = (uint32_t)__builtin_amdgcn_readlane((int)step_at, i);
          eq_at = (uint32_t)__builtin_amdgcn_readlane((int)step_eq, i);
        }
        if (at >= o1) return;  // uniform
        uint64_t kept[4], eq[4], any_eq = 0;
        uint32_t count = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kept[j] = __builtin_amdgcn_ballot_w64(k[j] > prefix);
          eq[j] = __builtin_amdgcn_ballot_w64(k[j] == prefix);
          any_eq |= eq[j];
        }
        if (any_eq != 0) {  // uniform: the first `need` equals stay
          uint32_t rank = eq_at;
#pragma unroll
          for (int j = 0; j < 4; ++j) rank = bits_below(eq[j], rank);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            kept[j] |= __builtin_amdgcn_ballot_w64(k[j] == prefix && rank < need);
            rank += k[j] == prefix ? 1u : 0u;
            eq_at += (uint32_t)__popcll(eq[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) count += (uint32_t)__popcll(kept[j]);
        if (at + count > o0) {  // uniform
          uint32_t to = at;
#pragma unroll
          for (int j = 0; j < 4; ++j) to = bits_below(kept[j], to);
          const int row = (int)(run + (int64_t)i * STEP) + 4 * lane;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool mine = kept[j] >> lane & 1;
            if (mine && to >= o0 && to < o1) list[to - o0] = row + j;
            to += mine ? 1u : 0u;
          }
        }
        at += count;
      });
    }
    __syncthreads();
    const int count = (int)(o1 - o0);
    const int64_t out0 = (int64_t)h * n_keep + o0;
    for (int i = tid; i < count; i += kEvictThreads) {
      rows_out[out0 + i] = list[i];
      weights_out[out0 + i] = w[list[i]];
    }
    if constexpr (PER > 0) {
      const int pieces = 1 << copy.piece_log;
      const char* ks = copy.k + (int64_t)h * copy.k_hs_b;
      const char* vs = copy.v + (int64_t)h * copy.v_hs_b;
      char* kd = copy.ko + (int64_t)h * copy.ko_hs_b + (int64_t)o0 * pieces * 16;
      char* vd = copy.vo + (int64_t)h * copy.vo_hs_b + (int64_t)o0 * pieces * 16;
      for (int i = tid; i < count << copy.piece_log; i += kEvictThreads) {
        const int64_t from = ((int64_t)list[i >> copy.piece_log] * pieces + (i & (pieces - 1))) * 16;
        const vec16 a = ld16_stream(ks + from), b = ld16_stream(vs + from);
        st16(kd + (int64_t)i * 16, a);
        st16(vd + (int64_t)i * 16, b);
      }
    }
    __syncthreads();
  }
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
  const int steps = (int)(((int64_t)n_tokens + 4 * kEvictThreads - 1) / (4 * kEvictThreads));  // 256-row steps a wavefront
  const int pieces = head_dim * eb / 16;  // 8 to 64, a power of two
  const EvictCopy copy = {(const char*)k_cache, (const char*)v_cache, (char*)k_out, (char*)v_out, k_head_stride * eb,
                          v_head_stride * eb, ko_head_stride * eb, vo_head_stride * eb, __builtin_ctz((unsigned)pieces)};
  auto select = [&](auto kernel, int slices) {
    const int slice = (int)(((int64_t)n_keep + slices - 1) / slices);
    const unsigned grid = (unsigned)(((int64_t)n_keep + slice - 1) / slice);
    hipLaunchKernelGGL(kernel, dim3(grid, (unsigned)n_heads), dim3(kEvictThreads), 0, s, weights, weights_head_stride, n_tokens, n_keep,
                       n_sink, n_recent, steps, slice, rows_out, weights_out, copy);
  };
  if (n_tokens <= kEvictKeys) {
    const int slices = (int)std::max<int64_t>(1, std::min<int64_t>(256 / n_heads, ((int64_t)n_keep + 31) / 32));
    if (steps <= 1) select(evict_kernel<1, 4096>, slices);
    else if (steps <= 3) select(evict_kernel<3, 12288>, slices);
    else select(evict_kernel<9, kEvictKeys>, slices);
    CKV_RETURN_IF_LAUNCH_FAILED();
    return CKV_OK;
  }
  select(evict_kernel<0, 0>, 1);
  CKV_RETURN_IF_LAUNCH_FAILED();
  const int64_t blocks = ((int64_t)n_keep * pieces + 255) / 256;
  hipLaunchKernelGGL(evict_gather_kernel, dim3((unsigned)blocks, (unsigned)n_heads, 2), dim3(256), 0, s, rows_out, n_keep, pieces,
                     copy.piece_log, copy.k, copy.k_hs_b, copy.v, copy.v_hs_b, copy.ko, copy.ko_hs_b, copy.vo, copy.vo_hs_b);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}
