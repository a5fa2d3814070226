// Rows written into an 8-bit K/V cache, and such a cache read back as bf16.
//
// A cache holds e4m3 codes (one sign, four exponent, three fraction bits, largest value 448) and, for every block of
// `block` tokens of a head, K and V apart, one power of two s = 2^e as its exponent byte e + 127:
//   e = the least integer with max |x| <= 448 * 2^e over the block's rows,   code = e4m3(x / s), to nearest even.
// A power of two because e4m3 is a floating type, which gains nothing from a finer scale, while this one makes
// every step but the rounding exact: x / s, code * s (a bf16 value), and a kept row's new codes when a row that
// is appended to its block raises s (codes move by whole exponents; only those that fall below 2^-6 lose bits).
// So a cache that grew row by row has the scales of one written at once (unless rows were dropped and written again from the
// middle of a block: its stored scale stands, which the dropped ones may have raised).
//
// Design: one workgroup per block, head and tensor holds the block's new rows in registers between the
// maximum and the codes: each element is read once and written once. Bound: HBM for a prefill's rows (32832 bf16 rows of 4
// heads of 128, 101 MB: 19.0 us, 5.3 TB/s; a torch copy reaches 5.1), the launch for one token's (2.4 us in a graph),
// where the workgroup touches the kept rows of its block only if they need a new scale.
#include <algorithm>

#include "ckv_common.hpp"

namespace ckv {

constexpr int kQuantThreads = 256;
constexpr int kPiece = 16;  // elements of a row that make 16 bytes of codes

struct QuantTensor {
  char* codes;
  uint8_t* scales;
  const char* x;
  int64_t x_hs_b, x_ts_b;
};

// The exponent byte of the least power of two that maps amax (bits of a value >= 0) into [0, 448];
// 448 = 1.75 * 2^8. 255 (no number) for an infinity or a NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 1);
}

// Four fp32 values as e4m3 codes.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

template <int DTYPE>
__device__ __forceinline__ void unpack_piece(const vec16* raw, float (&f)[kPiece]) {
  using E = Elem<DTYPE>;
#pragma unroll
  for (int i = 0; i < kPiece / E::kVec; ++i) {
    float v[E::kVec];
    E::unpack(raw[i], v);
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) f[i * E::kVec + e] = v[e];
  }
}

// UNITS: pieces of a whole block per thread, rounded up.
template <int DTYPE, int D, int UNITS>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(QuantTensor k, QuantTensor v, int64_t start,
                                                                      const int64_t* __restrict__ start_dev, int n,
                                                                      int N, int blocks, int block_log,
                                                                      int32_t* __restrict__ err) {
  using E = Elem<DTYPE>;
  constexpr int VP = kPiece / E::kVec;  // 16-byte loads per piece
  constexpr int PR = D / kPiece;        // pieces per row
  __shared__ uint32_t wave_max[kQuantThreads / kWave];
  const QuantTensor& t = blockIdx.z == 0 ? k : v;
  const int h = blockIdx.y, tid = threadIdx.x;
  if (start_dev != nullptr) start = *start_dev;
  if (start < 0 || start > N - n) {  // uniform
    if (tid == 0) flag_error(err, CKV_DEVICE_ERR_RANGE);
    return;
  }
  const int s = (int)start, first = (s >> block_log) + (int)blockIdx.x;
  const int lo = first << block_log, hi = min(lo + (1 << block_log), s + n);  // rows of this block
  if (lo >= s + n) return;  // uniform: fewer blocks than the grid allows for
  const int from = max(lo, s);
  char* codes = t.codes + ((int64_t)h * N + lo) * D;
  const char* x = t.x + (int64_t)h * t.x_hs_b;
  const int64_t at = (int64_t)h * blocks + first;
  const uint32_t old = from > lo ? t.scales[at] : 0u;

  vec16 raw[UNITS][VP];
  uint32_t amax = 0;
  const int units = (hi - from) * PR;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int p = u * kQuantThreads + tid;
    if (p < units) {
      const char* src = x + (int64_t)(from - s + p / PR) * t.x_ts_b + (p % PR) * kPiece * E::kBytes;
#pragma unroll
      for (int i = 0; i < VP; ++i) raw[u][i] = ld16_stream(src + i * 16);
    }
  }
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (u * kQuantThreads + tid < units) {
      float f[kPiece];
      unpack_piece<DTYPE>(raw[u], f);
#pragma unroll
      for (int e = 0; e < kPiece; ++e) amax = max(amax, __float_as_uint(f[e]) & 0x7fffffffu);
    }
  }
  // bits of values >= 0 order as the values do, and those of a NaN above all of them
  for (int m = 32; m > 0; m >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, m));
  if (tid % kWave == 0) wave_max[tid / kWave] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / kWave; ++w) amax = max(amax, wave_max[w]);
  const uint32_t b = max(scale_byte(amax), old);
  const int up = 127 - (int)b;  // x / s = ldexp(x, up)
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int p = u * kQuantThreads + tid;
    if (p < units) {
      float f[kPiece];
      unpack_piece<DTYPE>(raw[u], f);
#pragma unroll
      for (int e = 0; e < kPiece; ++e) f[e] = __builtin_amdgcn_ldexpf(f[e], up);
      vec16 c;
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = codes4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
      if (b == 255u) c = vec16{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
      st16(codes + (int64_t)(from - lo) * D + (int64_t)p * kPiece, c);
    }
  }
  if (from > lo && b != old) {  // uniform: the kept rows under their new scale
    for (int p = tid; p < (from - lo) * PR; p += kQuantThreads) {
      vec16 c = ld16(codes + (int64_t)p * kPiece);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto l = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), g = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
        const int d = (int)old - (int)b;
        c[i] = b == 255u ? 0x7f7f7f7fu
                         : codes4(__builtin_amdgcn_ldexpf(l[0], d), __builtin_amdgcn_ldexpf(l[1], d),
                                  __builtin_amdgcn_ldexpf(g[0], d), __builtin_amdgcn_ldexpf(g[1], d));
      }
      st16(codes + (int64_t)p * kPiece, c);
    }
  }
  if (tid == 0 && (from == lo || b != old)) t.scales[at] = (uint8_t)b;
}

}  // namespace ckv

extern "C" int32_t ckv_quantize_rows(void* k_codes, void* v_codes, void* k_scales, void* v_scales, const void* k,
                                     int64_t k_head_stride, int64_t k_token_stride, const void* v,
                                     int64_t v_head_stride, int64_t v_token_stride, int64_t start,
                                     const int64_t* start_dev, int32_t n_rows, int32_t n_tokens, int32_t n_heads,
                                     int32_t head_dim, int32_t block_tokens, int32_t dtype, int32_t* err,
                                     void* stream) {
  using namespace ckv;
  if (n_rows < 0 || n_tokens <= 0 || n_heads <= 0) return CKV_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return CKV_ERR_INVALID_ARGUMENT;
  if (block_tokens != 32 && block_tokens != 64 && block_tokens != 128) return CKV_ERR_INVALID_ARGUMENT;
  if (dtype != CKV_DTYPE_F32 && dtype != CKV_DTYPE_BF16) return CKV_ERR_INVALID_ARGUMENT;
  if (n_rows > n_tokens || (start_dev == nullptr && (start < 0 || start > n_tokens - n_rows))) return CKV_ERR_OUT_OF_RANGE;
  if (n_rows == 0) return CKV_OK;
  if (k_codes == nullptr || v_codes == nullptr || k_scales == nullptr || v_scales == nullptr || k == nullptr || v == nullptr)
    return CKV_ERR_INVALID_ARGUMENT;
  const int vec = dtype == CKV_DTYPE_BF16 ? 8 : 4;
  if (k_head_stride % vec || k_token_stride % vec || v_head_stride % vec || v_token_stride % vec)
    return CKV_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k | (uintptr_t)v) % 16) return CKV_ERR_INVALID_ARGUMENT;
  if (n_heads > 65535) return CKV_ERR_TOO_LARGE;
  const int log = block_tokens == 32 ? 5 : block_tokens == 64 ? 6 : 7;
  const int blocks = (int)(((int64_t)n_tokens + block_tokens - 1) >> log);
  // blocks that n_rows rows touch: from a known start, or at most
  const int64_t grid = start_dev == nullptr ? ((start + n_rows - 1) >> log) - (start >> log) + 1
                                            : std::min<int64_t>(((int64_t)n_rows + block_tokens - 2) / block_tokens + 1, blocks);
  const int eb = dtype == CKV_DTYPE_BF16 ? 2 : 4;
  const QuantTensor kt = {(char*)k_codes, (uint8_t*)k_scales, (const char*)k, k_head_stride * eb, k_token_stride * eb};
  const QuantTensor vt = {(char*)v_codes, (uint8_t*)v_scales, (const char*)v, v_head_stride * eb, v_token_stride * eb};
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid, (unsigned)n_heads, 2), dim3(kQuantThreads), 0, (hipStream_t)stream, kt,
                       vt, start, start_dev, n_rows, n_tokens, blocks, log, err);
  };
  // pieces of a thread: min(block, n_rows) rows of head_dim / 16
  const int most = std::min(block_tokens, n_rows) * (head_dim / kPiece);
  auto by_units = [&](auto dt, auto hd) {
    constexpr int T = decltype(dt)::value, D = decltype(hd)::value;
    if (most <= kQuantThreads) launch(quantize_rows_kernel<T, D, 1>);
    else if (most <= 2 * kQuantThreads) launch(quantize_rows_kernel<T, D, 2>);
    else if constexpr (D == 128) launch(quantize_rows_kernel<T, D, 4>);
  };
  auto by_dim = [&](auto dt) {
    if (head_dim == 128) by_units(dt, std::integral_constant<int, 128>{});
    else by_units(dt, std::integral_constant<int, 64>{});
  };
  if (dtype == CKV_DTYPE_BF16) by_dim(std::integral_constant<int, CKV_DTYPE_BF16>{});
  else by_dim(std::integral_constant<int, CKV_DTYPE_F32>{});
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}
