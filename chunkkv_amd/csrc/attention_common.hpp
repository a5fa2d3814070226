// Device helpers that the attention kernels share (attention.hip, attention_wave.hpp, attention_weights.hip): matrix
// operand types, reductions over the lanes of a query, LDS layouts of cache rows, work items.
#pragma once

#include "attention_plan.hpp"
#include "ckv_common.hpp"

namespace ckv {

// What an 8-bit cache has beside its codes: for head h and 32-row chunk c the scale byte e + 127 of 2^e
// is at [h * blocks + (c >> chunk_log)], of K and of V.
struct CacheScales {
  const uint8_t* k;
  const uint8_t* v;
  int blocks, chunk_log;
};
// The same for a launch whose query rows are the (token, query head) pairs of a KV head; inv_gqa: for div_by of its heads.
struct GroupedCacheScales : CacheScales {
  uint32_t inv_gqa;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Combine a lane's value with the lanes 16 and 32 away (the four lane groups of one query), with
// gfx950's row-swap permutes (VALU, no LDS round trip): each returns the lane's own value and
// its partner's, in an order that depends on the lane, so only order-free combinations are used.
__device__ __forceinline__ float group_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// f over the 16 lanes of a row, in every lane (row rotations: VALU, no LDS round trip).
template <typename T, typename F>
__device__ __forceinline__ T row16_reduce(T v, F f) {
  static_assert(sizeof(T) == 4, "one VGPR");
  auto from = [](T x, auto ctrl) {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v = f(v, from(v, std::integral_constant<int, 0x128>{}));
  v = f(v, from(v, std::integral_constant<int, 0x124>{}));
  v = f(v, from(v, std::integral_constant<int, 0x122>{}));
  return f(v, from(v, std::integral_constant<int, 0x121>{}));
}

typedef short v4i16 __attribute__((ext_vector_type(4)));

// LDS tiles (K and V, 64 cache rows each) are unpadded rows of D x 2 bytes, CPR 16-byte chunks,
// filled by direct-to-LDS loads. Spreading over the banks comes from swizzles of the chunk index:
// chunk c of slot s holds logical chunk c ^ swz(s).
//  - K: swz_k(s) = s % CPR. The 16 lanes of one lane group read one logical chunk of 16
//    consecutive slots for an S^T operand (16-byte reads): 16 distinct physical chunks.
//  - V: swz_v(s) = 2 (s % 4) + 8 ((s / 8) % 2) (CPR = 16; 2 (s % 4) for CPR = 8). A transposing
//    read of a lane group covers 4 consecutive slots x 2 adjacent chunks x 2 halves; the swizzle
//    puts them, and the next lane group's 4 slots 8 rows on, on distinct 8-byte bank ranges.
//  - K slot s of a 32-row block holds cache row kslot_row(s): slot 16 t + 4 a + b <- row
//    8 a + 4 t + b, so the 16 slots one S^T operand reads give each lane 8 consecutive rows of
//    the output (the rows its P^T operand pairs with V). V slots hold rows in order.
// Without the swizzles the kernel takes 0.405 ms instead of 0.220 ms on the 2976-row case.
template <int CPR>
__device__ __forceinline__ int swz_k(int s) { return s % CPR; }
template <int CPR>
__device__ __forceinline__ int swz_v(int s) { return CPR >= 16 ? 2 * (s % 4) + 8 * ((s / 8) % 2) : 2 * (s % 4); }
__device__ __forceinline__ int kslot_row(int s) {
  const int k = s & 31;
  return (s & ~31) + 8 * ((k >> 2) & 3) + 4 * (k >> 4) + (k & 3);
}

// The A operand of O^T = V^T P^T for columns 16 dt .. + 16 of 32 V rows at vb (swizzled, row-major),
// through transposing 64-bit LDS loads: in each 16-lane group, lane m names row 4 h + m / 4 (of the
// group's 8 keys 8 g ..) at column 4 (m % 4) of the 16-column tile, and lane 4a + b receives column
// 4a + b of rows 4h + 0..3. So lane (g, lm) holds V[8 g + 4 h + e][16 dt + lm], e = 0..3: two loads
// (h = 0, 1) give the eight keys 8 g + e' the B operand (P^T) pairs with that lane. Element
// 16 dt + 4 (lm % 4) is logical chunk 2 dt + (lm % 4) / 2, byte 8 (lm % 2).
template <int CPR>
__device__ __forceinline__ bf16x8 v_operand(const char* vb, int dt, int g, int lm) {
  typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
  auto rd = [&](int h) {
    const int row = 8 * g + 4 * h + lm / 4;
    return row * CPR * 16 + (((2 * dt + (lm % 4) / 2) ^ swz_v<CPR>(row)) * 16) + 8 * (lm % 2);
  };
  const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vb + rd(0)));
  const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vb + rd(1)));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// x / d for d > 0, with inv = inverse_of(.., d).
__device__ __forceinline__ int div_by(int x, int d, uint32_t inv) {
  return inv != 0 ? (int)__umulhi((uint32_t)x, inv) : d == 1 ? x : x / d;
}
__device__ __forceinline__ bool attn_work_item(int nqb, int group, int xpk_log, int items, uint32_t inv_group,
                                               uint32_t inv_nqb, int& qb, int& h, int& z) {
  const int L = (int)blockIdx.x, xcd = L % kXcds;
  const int j = ((L / kXcds) << xpk_log) + (xcd & ((1 << xpk_log) - 1));
  const int rest = div_by(j, group, inv_group);
  h = (xcd >> xpk_log) * group + (j - rest * group);
  z = div_by(rest, nqb, inv_nqb);
  qb = nqb - 1 - (rest - z * nqb);
  return j < items;
}

// Between the stages in which a wavefront's lanes exchange rows through LDS (and before a stage's rows
// are overwritten): LDS runs one wavefront's operations in order, so this is no instruction, only an
// order of stores and loads that the compiler has to keep though no lane reads its own bytes.
__device__ __forceinline__ void wave_lds_stage() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

}  // namespace ckv
