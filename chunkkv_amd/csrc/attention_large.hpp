// The attention of launches that 128-query workgroups fill (attention.hip describes it; attention_quantized.hip runs it over
// 8-bit caches).
#pragma once

#include "attention_common.hpp"

namespace ckv {

// With a CacheScales argument at the end the cache holds e4m3 codes: a thread takes its pieces of the next tile into registers while
// this one is worked on, and makes them bf16 on their way into the other buffer, once for the workgroup's 128 queries. The
// same occupancy (230 and 144 registers at head_dim 128 and 64) and about a tenth more time (us, codes and bf16 rows: 28 / 4 heads
// of 128, 128 queries over 28787 rows 67 and 62, 300 177 and 163; 14 / 2 heads of 64, 500 over 65536 136 and 126).
// SPLIT: split z of the cache's tiles per workgroup, unnormalised rows with their max and sum to ws.
template <int D, bool SPLIT, typename... Scales>
__global__ __launch_bounds__(kAttnWaves * 64) void attn_active_kernel(
    int nqb, int map_group, int xpk_log, int items, uint32_t inv_group, uint32_t inv_nqb,
    const int64_t* __restrict__ pos, int n, int N, const char* __restrict__ kc, const char* __restrict__ vc,
    int64_t kv_hs_b, const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b, int Hq, int group, float scale_log2,
    char* __restrict__ out, int32_t* __restrict__ err, float* __restrict__ ws, int split_tiles, Scales... scales) {
  constexpr bool CODES = sizeof...(Scales) == 1, GROUPED = (std::is_same_v<Scales, GroupedCacheScales> || ...);
  constexpr int DS = D / 32;          // k-steps of S^T = K Q^T
  constexpr int DT = D / 16;          // 16-row tiles of O^T
  constexpr int CPR = D / 8;          // 16-byte chunks per cache row
  constexpr int ROWB = D * 2;        // bytes per cache row (and LDS slot)
  constexpr int NT = kAttnWaves * 64;
  static_assert(D % 32 == 0, "head_dim must be a multiple of 32");
  static_assert((kAttnBN * CPR) % NT == 0, "tile loads must tile the workgroup");
  static_assert((CPR & (CPR - 1)) == 0 && CPR >= 8, "swizzles need a power-of-two chunk count");

  // Two buffers per tensor: tile t + 1 loads into one while tile t is read from the other.
  __shared__ __attribute__((aligned(1024))) char k_lds0[kAttnBN * ROWB];
  __shared__ __attribute__((aligned(1024))) char k_lds1[kAttnBN * ROWB];
  __shared__ __attribute__((aligned(1024))) char v_lds0[kAttnBN * ROWB];
  __shared__ __attribute__((aligned(1024))) char v_lds1[kAttnBN * ROWB];
  __shared__ int blk_max_s[kAttnWaves];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  int qb, hq, z;
  if (!attn_work_item(nqb, map_group, xpk_log, items, inv_group, inv_nqb, qb, hq, z)) return;
  const int hk = GROUPED ? hq : hq / group;
  const int rows = GROUPED ? n * group : n;
  auto token_of = [&](int m) {  // of row m
    if constexpr (GROUPED) return div_by(m, group, (scales.inv_gqa, ...));
    else return m;
  };
  auto head_of = [&](int m, int t) { return GROUPED ? hk * group + m - t * group : hq; };
  const int q0 = qb * kAttnBM + wave * kAttnQG * 16;
  // Positions of this lane's queries (-1 = no query); out-of-range positions are flagged and
  // clamped so that every read stays inside the cache.
  int my_pos[kAttnQG];
  int wmax = -1, wmin = N;
#pragma unroll
  for (int qg = 0; qg < kAttnQG; ++qg) {
    const int m = q0 + qg * 16 + lm;
    int p = -1;
    if (m < rows) {
      const int64_t p64 = pos[token_of(m)];
      if (p64 < 0 || p64 >= N) {
        flag_error(err, CKV_DEVICE_ERR_RANGE);
        p = p64 < 0 ? 0 : N - 1;
      } else {
        p = (int)p64;
      }
      wmin = min(wmin, p);
    }
    my_pos[qg] = p;
    wmax = max(wmax, p);
  }
  wmax = __builtin_amdgcn_readfirstlane(row16_reduce(wmax, [](int a, int b) { return max(a, b); }));
  wmin = __builtin_amdgcn_readfirstlane(row16_reduce(wmin, [](int a, int b) { return min(a, b); }));
  if (lane == 0) blk_max_s[wave] = wmax;
  __syncthreads();
  int bmax = blk_max_s[0];
#pragma unroll
  for (int w = 1; w < kAttnWaves; ++w) bmax = max(bmax, blk_max_s[w]);
  bmax = __builtin_amdgcn_readfirstlane(bmax);
  int n_tiles = bmax < 0 ? 0 : bmax / kAttnBN + 1;
  const int tile_begin = SPLIT ? z * split_tiles : 0;
  if (SPLIT) n_tiles = min(n_tiles, tile_begin + split_tiles);

  // Q fragments (B operand of S^T): query q0 + 16 qg + lm, head-dim 32 s + 8 g .. + 8.
  bf16x8 qf[kAttnQG][DS];
#pragma unroll
  for (int qg = 0; qg < kAttnQG; ++qg) {
    const int m = q0 + qg * 16 + lm;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      vec16 v = {0, 0, 0, 0};
      if (m < rows) {
        const int t = token_of(m);
        v = ld16(q + (int64_t)head_of(m, t) * q_hs_b + (int64_t)t * q_ts_b + (32 * s + 8 * g) * 2);
      }
      qf[qg][s] = __builtin_bit_cast(bf16x8, v);
    }
  }

  f32x4 o[kAttnQG][DT];
  float m_run[kAttnQG], m_sub[kAttnQG];
  // The row sums come from one more MFMA per key block with an all-ones A operand: every row of its output is sum_k P^T[k][query], the sum of the bf16 weights that
  // multiply V (lane (g, lm) gets query lm's sum in each of its four values).
  f32x4 l_acc[kAttnQG];
  const bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f,
                       (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int qg = 0; qg < kAttnQG; ++qg) {
    m_run[qg] = -INFINITY;
    m_sub[qg] = 0.f;
    l_acc[qg] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[qg][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const char* kh = kc + (int64_t)hk * kv_hs_b;
  const char* vh = vc + (int64_t)hk * kv_hs_b;

  // Tile loads go straight from global memory to LDS (global_load_lds_dwordx4): load
  // instruction i of wavefront w fills the 1 KB block w * KI + i of a tile buffer, lane l its 16
  // bytes at l * 16, i.e. position P = (w KI + i) 64 + l = slot P / CPR, chunk P % CPR. No
  // registers stage the tile and no LDS store instructions run; rows past every query's position
  // load the last one's row instead: they are masked, but their zero weights meet the values, and a
  // cache row not written yet may hold a NaN (nor is there a row past the cache to read).
  constexpr int KI = (kAttnBN * CPR) / NT;  // load instructions per wavefront, tile and tensor
  static_assert(KI >= 1 && (kAttnBN * CPR) % NT == 0, "a tile must fill whole load instructions");
  // A lane's offsets in a tile are kept (K slots hold rows in kslot_row's order) and added to the
  // tile's uniform address: two 64-bit addresses built per load were a quarter of a tile's vector
  // instructions. Only a workgroup's last tile clamps its rows.
  int off_k[KI], off_v[KI];
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int P = (wave * KI + i) * 64 + lane;
    const int slot = P / CPR, pc = P % CPR;
    off_k[i] = kslot_row(slot) * ROWB + (pc ^ swz_k<CPR>(slot)) * 16;
    off_v[i] = slot * ROWB + (pc ^ swz_v<CPR>(slot)) * 16;
  }
  typedef __attribute__((address_space(1))) void gvoid;
  typedef __attribute__((address_space(3))) void lvoid;
  auto issue = [&](int n0, char* kb, char* vb) {
    const char* kt = kh + (int64_t)n0 * ROWB;
    const char* vt = vh + (int64_t)n0 * ROWB;
    const int last = bmax - n0;  // >= 0: only tiles that some query sees are issued
    auto load = [&](const char* t, int off, char* to) {
      __builtin_amdgcn_global_load_lds((gvoid*)(t + (uint32_t)off), (lvoid*)to, 16, 0, 0);
    };
    if (last >= kAttnBN - 1) {  // uniform: a whole tile
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        load(kt, off_k[i], kb + (wave * KI + i) * 1024);
        load(vt, off_v[i], vb + (wave * KI + i) * 1024);
      }
    } else {
      auto clamp = [&](int off) { return min(off / ROWB, last) * ROWB + off % ROWB; };
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        load(kt, clamp(off_k[i]), kb + (wave * KI + i) * 1024);
        load(vt, clamp(off_v[i]), vb + (wave * KI + i) * 1024);
      }
    }
  };
  // Codes: a thread's 16-byte pieces of a tile, 256 apart, and the scale byte of each piece's row.
  constexpr int GP = D / 16, KC = kAttnBN * GP / NT;
  [[maybe_unused]] vec16 kcode[KC], vcode[KC];
  [[maybe_unused]] uint8_t kbyte[KC], vbyte[KC];
  [[maybe_unused]] auto load_codes = [&](int n0, const CacheScales& sc) {
    const char* kt = kh + (int64_t)n0 * D;
    const char* vt = vh + (int64_t)n0 * D;
    const int last = bmax - n0;  // as for bf16 rows
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int P = i * NT + (int)threadIdx.x;
      const uint32_t off = min(P / GP, last) * D + P % GP * 16;
      kcode[i] = ld16(kt + off);
      vcode[i] = ld16(vt + off);
      // 32 rows are whole wavefronts' pieces: one scale for each
      const int chunk = min((n0 + __builtin_amdgcn_readfirstlane(P / GP)) >> 5, bmax >> 5);
      const int64_t b = (int64_t)hk * sc.blocks + (chunk >> sc.chunk_log);
      kbyte[i] = sc.k[b];
      vbyte[i] = sc.v[b];
    }
  };
  [[maybe_unused]] auto store_codes = [&](char* kb, char* vb) {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int P = i * NT + (int)threadIdx.x, row = P / GP, p = P % GP;
      const int slot = (row & ~31) + 16 * ((row >> 2) & 1) + 4 * ((row >> 3) & 3) + (row & 3);  // kslot_row's inverse
      vec16 lo, hi;
      decode16(kcode[i], __uint_as_float((uint32_t)kbyte[i] << 23), lo, hi);
      *(vec16*)(kb + slot * ROWB + ((2 * p) ^ swz_k<CPR>(slot)) * 16) = lo;
      *(vec16*)(kb + slot * ROWB + ((2 * p + 1) ^ swz_k<CPR>(slot)) * 16) = hi;
      decode16(vcode[i], __uint_as_float((uint32_t)vbyte[i] << 23), lo, hi);
      *(vec16*)(vb + row * ROWB + ((2 * p) ^ swz_v<CPR>(row)) * 16) = lo;
      *(vec16*)(vb + row * ROWB + ((2 * p + 1) ^ swz_v<CPR>(row)) * 16) = hi;
    }
  };
  // S^T operand of (kb, t, ds) for lane (g, lm): slot 32 kb + 16 t + lm, logical chunk 4 ds + g.
  int k_rd[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) k_rd[ds] = lm * ROWB + (((4 * ds + g) ^ swz_k<CPR>(lm)) * 16);
  if constexpr (CODES) {
    if (tile_begin < n_tiles) {
      (load_codes(tile_begin * kAttnBN, scales), ...);
      store_codes(k_lds0, v_lds0);
    }
  } else {
    if (tile_begin < n_tiles) issue(tile_begin * kAttnBN, k_lds0, v_lds0);
  }

  // One tile; the loop below alternates the buffers (each call names its buffers directly, so
  // the compiler sees that the loads in flight never alias the buffer being read).
  auto body = [&](int tile, const char* k_lds, const char* v_lds, char* k_nxt, char* v_nxt) {
    const int n0 = tile * kAttnBN;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's loads of the tile landed
    __syncthreads();  // every wavefront's loads landed and every wavefront is done with the other buffer
    if constexpr (CODES) {
      if (tile + 1 < n_tiles) (load_codes(n0 + kAttnBN, scales), ...);
    } else {
      if (tile + 1 < n_tiles) issue(n0 + kAttnBN, k_nxt, v_nxt);  // lands during the MFMAs below
    }

    if (n0 > wmax) return;  // uniform per wavefront: no query of this wavefront reaches the tile
    const bool need_mask = n0 + kAttnBN - 1 > wmin;

    // S^T for the tile: lane (g, lm) gets query lm, rows n0 + 32 kb + 8 g + 4 t + e.
    constexpr int KB = kAttnBN / 32;
    f32x4 s[kAttnQG][KB][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {  // the halves inside: dependent products four apart
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bf16x8 a = *(const bf16x8*)(k_lds + (kb * 32 + 16 * t) * ROWB + k_rd[ds]);
#pragma unroll
          for (int qg = 0; qg < kAttnQG; ++qg)
            s[qg][kb][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[qg][ds], ds == 0 ? f32x4{0.f, 0.f, 0.f, 0.f}
                                                                                       : s[qg][kb][t], 0, 0, 0);
        }
      }

    // Online softmax over the tile. The running max is only raised when a query's tile max
    // exceeds it by more than 2^8 (log2 domain): weights stay <= 256, the output rescale is
    // skipped for the whole wavefront otherwise, and the result is unchanged (the final division
    // uses the same max).
    bf16x8 pb[kAttnQG][KB];
#pragma unroll
    for (int qg = 0; qg < kAttnQG; ++qg) {
      // Raw scores of this lane (query lm, rows n0 + 32 kb + 8 g + 4 t + e); rows past the query's
      // position become -inf, on the tiles that reach past the lowest position only (uniform).
      float x[KB][8];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[kb][4 * t + e] = s[qg][kb][t][e];
      if (need_mask) {
        const int lim = my_pos[qg] - n0 - 8 * g;  // row offset 32 kb + 4 t + e must stay <= lim
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (32 * kb + j > lim) x[kb][j] = -INFINITY;
      }
      float bm = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 8; ++j) bm = fmaxf(bm, x[kb][j]);
      // A lane asks for its own scores; the four lanes of a query agree on its max inside the branch.
      if (__builtin_amdgcn_ballot_w64(bm * scale_log2 > m_run[qg] + 8.f)) {  // uniform branch
        bm = group_max(bm) * scale_log2;           // the scale is > 0: max commutes
        const bool raise = bm > m_run[qg] + 8.f;  // also true on the first visible tile (m_run = -inf)
        const float m_new = raise ? bm : m_run[qg];
        const float alpha = m_run[qg] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[qg] - m_new);
        l_acc[qg] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[qg][dt] *= alpha;
        m_run[qg] = m_new;
        // with no visible row yet (absent queries) every score is -inf and subtracting 0 keeps p = 0
        m_sub[qg] = m_new == -INFINITY ? 0.f : m_new;
      }
      // p = 2^(score * scale - max) in one fma
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pb[qg][kb][e] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[kb][e], scale_log2, -m_sub[qg]));
        }
    }

    // O^T += V^T P^T: A = V^T rows dt*16 + lm, columns 32 kb + 8 g .. + 8.
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 a = v_operand<CPR>(v_lds + kb * 32 * ROWB, dt, g, lm);
#pragma unroll
        for (int qg = 0; qg < kAttnQG; ++qg)
          o[qg][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[qg][kb], o[qg][dt], 0, 0, 0);
        if (dt == DT - 1) {
#pragma unroll
          for (int qg = 0; qg < kAttnQG; ++qg)
            l_acc[qg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[qg][kb], l_acc[qg], 0, 0, 0);
        }
      }
  };
  for (int tile = tile_begin; tile < n_tiles; tile += 2) {
    body(tile, k_lds0, v_lds0, k_lds1, v_lds1);
    if constexpr (CODES) {
      if (tile + 1 < n_tiles) store_codes(k_lds1, v_lds1);
    }
    if (tile + 1 < n_tiles) body(tile + 1, k_lds1, v_lds1, k_lds0, v_lds0);
    if constexpr (CODES) {
      if (tile + 2 < n_tiles) store_codes(k_lds0, v_lds0);
    }
  }

  // Normalise and write: lane (g, lm) holds O[query][dt*16 + 4g + e], 4 bf16 = 8 bytes per tile.
#pragma unroll
  for (int qg = 0; qg < kAttnQG; ++qg) {
    const float l = l_acc[qg][0];
    const int m = q0 + qg * 16 + lm;
    if (m >= rows) continue;
    const int t = token_of(m), h = head_of(m, t);
    if constexpr (GROUPED && SPLIT) {
      if (my_pos[qg] < tile_begin * kAttnBN) continue;  // nothing of this split: its row is not read
    }
    if (SPLIT) {
      float* prow = ws + (((int64_t)z * Hq + h) * n + t) * (D + 4);  // 16-byte aligned rows
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *(f32x4*)(prow + dt * 16 + 4 * g) = o[qg][dt];
      if (g == 0) {
        prow[D] = m_run[qg];
        prow[D + 1] = l;
      }
      continue;
    }
    const float inv = 1.f / l;
    char* orow = out + ((int64_t)t * Hq + h) * (D * 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      unsigned w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) w[h] = f32x2_to_bf16x2_bits(o[qg][dt][2 * h] * inv, o[qg][dt][2 * h + 1] * inv);
      *(uint2*)(orow + (dt * 16 + 4 * g) * 2) = uint2{w[0], w[1]};
    }
  }
}

}  // namespace ckv
