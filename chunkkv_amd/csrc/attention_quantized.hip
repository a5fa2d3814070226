// Attention of the active rows over an 8-bit cache (quantize.hip): the function of attention.hip on the rows
// that codes and scales stand for. A code times its power of two is a bf16 value, so both forms here compute
// with exactly the rows a bf16 cache would hold, and scores, softmax and output are attention.hip's.
//
//  - One token's rows: attn_codes_kernel below.
//  - Few query rows (some tokens, short prompts): attention_wave.hpp's kernel reads the codes and makes them bf16
//    on their way into LDS, a wavefront its own 32 rows.
//  - More, as attention_plan.hpp decides for bf16 rows: attention_large.hpp's workgroups of 128 queries, which convert a tile on
//    its way into LDS. Over a long cache (attn_grouped_plan) a workgroup has 128 of the (token, query head) rows of a KV head instead.
//  - Every workgroup that reads a row converts it again, about a tenth of the kernel's time, so launches of many rows first write
//    the cache as bf16 into the workspace, one pass, and attention.hip runs on that (kDecodeRows has both sides).
#include "attention_large.hpp"
#include "attention_quantized_plan.hpp"
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

// ---- one token's rows ------------------------------------------------------------------------------------------
// Up to 16 (token, query head) rows of a KV head: one matrix tile that streams the cache. attention_wave.hpp's split of
// the work (a wavefront its own 32-row chunks and softmax, partial rows of the cache's splits joined by a second
// launch), but the codes go from global memory straight into LDS and become bf16 behind it, as each operand is read: half
// the LDS traffic, and loads that no register waits for. Four stages a wavefront, three chunks in flight, no barrier in
// the loop. Bound: from about 30 MB of codes their bytes, below the two launches. Measured (us, 28 / 4 heads of 128, one row,
// with attention_wave.hpp's kernel on codes before): over 131072 rows 41.3 -> 29.8 (134 MB; reading as much and nothing else
// takes 25), 65536 20.6 -> 17.0, 32832 15.2 -> 12.4, 8302 9.4 and 9.5; 8 heads of 64 over 65536 21.7 -> 15.7.
// LDS rows of D code bytes, PP = D / 16 pieces of 16: piece p of row r is at p ^ swz_code(r). The 16 rows that one S^T
// operand reads, 8 a + 4 t + b (a, b < 4), and the 16 that two lane groups of a transposing read name, r and r + 1 .. + 15,
// fall on distinct 16-byte places of 256 bytes.
template <int D>
__device__ __forceinline__ int swz_code(int r) {
  return D == 128 ? ((r >> 1) ^ (((r >> 4) & 1) << 1)) & 7 : ((r >> 2) ^ ((r >> 4) & 1)) & 3;
}

// A chunk's operands out of LDS, and the wait for them: NK 16-byte pieces of K, and NV transposing 64-bit loads of V, lane
// (g, lm) of which receives column lm of the eight code rows that its lane group names. Written out because the compiler
// takes such reads for ones that may meet the loads into other stages, and waits for all of those first.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int NK, int NV>
__device__ __forceinline__ void read_chunk(const uint32_t (&k_at)[NK], const uint32_t (&v_at)[NV], vec16 (&k)[NK], u32x2 (&v)[NV]) {
  static_assert((NK == 4 && NV == 8) || (NK == 2 && NV == 4), "a row of 128 or 64 codes");
  if constexpr (NK == 4)
    asm volatile(
        "ds_read_b128 %0, %12\n\t" "ds_read_b128 %1, %13\n\t"
        "ds_read_b128 %2, %14\n\t" "ds_read_b128 %3, %15\n\t"
        "ds_read_b64_tr_b8 %4, %16\n\t" "ds_read_b64_tr_b8 %5, %17\n\t"
        "ds_read_b64_tr_b8 %6, %18\n\t" "ds_read_b64_tr_b8 %7, %19\n\t"
        "ds_read_b64_tr_b8 %8, %20\n\t" "ds_read_b64_tr_b8 %9, %21\n\t"
        "ds_read_b64_tr_b8 %10, %22\n\t" "ds_read_b64_tr_b8 %11, %23\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
        : "v"(k_at[0]), "v"(k_at[1]), "v"(k_at[2]), "v"(k_at[3]), "v"(v_at[0]), "v"(v_at[1]), "v"(v_at[2]), "v"(v_at[3]), "v"(v_at[4]), "v"(v_at[5]), "v"(v_at[6]), "v"(v_at[7])
        : "memory");
  else
    asm volatile(
        "ds_read_b128 %0, %6\n\t" "ds_read_b128 %1, %7\n\t"
        "ds_read_b64_tr_b8 %2, %8\n\t" "ds_read_b64_tr_b8 %3, %9\n\t"
        "ds_read_b64_tr_b8 %4, %10\n\t" "ds_read_b64_tr_b8 %5, %11\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0]), "=&v"(k[1]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
        : "v"(k_at[0]), "v"(k_at[1]), "v"(v_at[0]), "v"(v_at[1]), "v"(v_at[2]), "v"(v_at[3])
        : "memory");
}

template <int D>
__global__ __launch_bounds__(kCodeWaves * 64) void attn_codes_kernel(
    const int64_t* __restrict__ pos, int n, int N, const char* __restrict__ kc, const char* __restrict__ vc,
    const char* __restrict__ q, int64_t q_hs_b, int64_t q_ts_b, int Hq, int group, float scale_log2, int split_chunks,
    char* __restrict__ out, float* __restrict__ ws, int32_t* __restrict__ err, CacheScales scales) {
  constexpr int W = kCodeWaves, CH = kWaveChunk, PP = D / 16, DJ = D / 64, DT = D / 16;
  constexpr int LI = CH * PP / 64;  // 1 KB loads of K, and of V, a chunk
  __shared__ __attribute__((aligned(1024))) char lds0[W * 2 * CH * D];  // per wavefront K rows, then V rows
  __shared__ __attribute__((aligned(1024))) char lds1[W * 2 * CH * D];
  __shared__ __attribute__((aligned(1024))) char lds2[W * 2 * CH * D];
  __shared__ __attribute__((aligned(1024))) char lds3[W * 2 * CH * D];
  __shared__ float s_m[W][kCodeRows], s_l[W][kCodeRows];
  static_assert(W * 2 * CH * D == W * kCodeRows * D * 4, "partial rows take a stage's place");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int g = lane / 16, lm = lane % 16;
  const int z = blockIdx.x, hk = blockIdx.y, rows = n * group;
  const char* kh = kc + (int64_t)hk * N * D;
  const char* vh = vc + (int64_t)hk * N * D;
  const uint8_t* ksb = scales.k + (int64_t)hk * scales.blocks;
  const uint8_t* vsb = scales.v + (int64_t)hk * scales.blocks;
  typedef __attribute__((address_space(1))) void gvoid;
  typedef __attribute__((address_space(3))) void lvoid;
  int off_row[LI], off_col[LI];
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int P = i * 64 + lane;
    off_row[i] = P / PP;
    off_col[i] = ((P % PP) ^ swz_code<D>(P / PP)) * 16;
  }
  auto issue = [&](int c, char* to) {
    c = min(c, (N - 1) / CH);
    const int64_t base = (int64_t)c * (CH * D);
    const int last = N - 1 - c * CH;  // rows past the cache load its last one
    char* wl = to + wave * 2 * CH * D;
#pragma unroll
    for (int i = 0; i < LI; ++i) {
      const uint32_t o = (uint32_t)(min(off_row[i], last) * D + off_col[i]);
      __builtin_amdgcn_global_load_lds((gvoid*)(kh + base + o), (lvoid*)(wl + i * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gvoid*)(vh + base + o), (lvoid*)(wl + CH * D + i * 1024), 16, 0, 0);
    }
  };
  const int begin = ws != nullptr ? z * split_chunks : 0;
  int c = begin + wave;
  issue(c, lds0);  // known before the positions are
  // Scale bytes of a wavefront's next 64 chunks, a chunk a lane.
  uint32_t k_bytes, v_bytes;
  auto load_scales = [&](int c) {
    const int at = min(c + lane * W, (N - 1) / CH) >> scales.chunk_log;
    k_bytes = ksb[at];
    v_bytes = vsb[at];
    asm volatile("" : "+v"(k_bytes), "+v"(v_bytes));  // waited for here, not at every use
  };

  const int r = min(lm, rows - 1), t_of = r / group;
  const char* qr = q + (int64_t)(hk * group + r - t_of * group) * q_hs_b + (int64_t)t_of * q_ts_b;
  bf16x8 qf[DJ][2];  // step (j, u): the dims 16 (4 j + g) + 8 u .. + 8, as a 16-code piece has them
#pragma unroll
  for (int j = 0; j < DJ; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u) qf[j][u] = __builtin_bit_cast(bf16x8, ld16(qr + (16 * (4 * j + g) + 8 * u) * 2));
  const int64_t p64 = pos[t_of];
  const int my_pos = p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64;
  if (my_pos != p64 && lm < rows) flag_error(err, CKV_DEVICE_ERR_RANGE);
  const int wmax = __builtin_amdgcn_readfirstlane(row16_reduce(my_pos, [](int a, int b) { return max(a, b); }));
  const int wmin = __builtin_amdgcn_readfirstlane(row16_reduce(my_pos, [](int a, int b) { return min(a, b); }));
  int c_end = wmax / CH + 1;
  if (ws != nullptr) c_end = min(c_end, begin + split_chunks);

  f32x4 o[DT], l_acc = {0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY;
  const bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f,
                       (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  load_scales(c);
  constexpr int AHEAD = 3;  // chunks in flight behind the one that is worked on
  if (c + W < c_end) issue(c + W, lds1);
  if (c + 2 * W < c_end) issue(c + 2 * W, lds2);
  int step = 0;
  // A lane's reads in a stage: row slot lm of S^T tile t is row 8 (lm / 4) + 4 t + lm % 4, so that the tiles' outputs are
  // a lane's rows 8 g .. + 7, which its V operands hold too.
  uint32_t k_off[2 * DJ], v_off[DT];
#pragma unroll
  for (int i = 0; i < 2 * DJ; ++i) {
    const int row = 8 * (lm >> 2) + 4 * (i % 2) + (lm & 3);
    k_off[i] = (uint32_t)(row * D + (((4 * (i / 2) + g) ^ swz_code<D>(row)) * 16));
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int row = 8 * g + lm / 2;
    v_off[dt] = (uint32_t)(CH * D + row * D + 8 * (lm % 2) + ((dt ^ swz_code<D>(row)) * 16));
  }
  auto body = [&](const char* cur, char* far) {
    const char* wl = cur + wave * 2 * CH * D;
    if (c + AHEAD * W < c_end) {  // into the stage whose reads the last step waited for
      issue(c + AHEAD * W, far);
      // all but the loads of the AHEAD later chunks have landed (2 LI each, in order)
      if constexpr (LI == 4) asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
      static_assert((LI == 4 || LI == 2) && AHEAD == 3, "the counts above");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const int n0 = c * CH;
    const float ks = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)k_bytes, step) << 23);
    const float vs = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)v_bytes, step) << 23);
    uint32_t k_at[2 * DJ], v_at[DT];
    vec16 kc16[2 * DJ];
    u32x2 v[DT];
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)wl;
#pragma unroll
    for (int i = 0; i < 2 * DJ; ++i) k_at[i] = at + k_off[i];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) v_at[dt] = at + v_off[dt];
    read_chunk<2 * DJ, DT>(k_at, v_at, kc16, v);
    f32x4 s[2];
#pragma unroll
    for (int j = 0; j < DJ; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        vec16 lo, hi;
        decode16(kc16[2 * j + t], ks, lo, hi);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lo), qf[j][0],
                                                       j == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, hi), qf[j][1], s[t], 0, 0, 0);
      }
    float x[8];  // cache rows n0 + 8 g + j of row lm
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = s[j / 4][j % 4];
    if (n0 + CH - 1 > wmin) {
      const int lim = my_pos - n0 - 8 * g;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j > lim) x[j] = -INFINITY;
    }
    float bm = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) bm = fmaxf(bm, x[j]);
    bm *= scale_log2;  // > 0: max commutes
    if (__builtin_amdgcn_ballot_w64(bm > m_run + 8.f)) {  // weights up to 2^8 need no new maximum
      bm = group_max(bm);
      const bool raise = bm > m_run + 8.f;
      const float m_new = raise ? bm : m_run;
      const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_acc *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      m_run = m_new;
    }
    const float sub = m_run == -INFINITY ? 0.f : m_run;
    bf16x8 pb;
#pragma unroll
    for (int j = 0; j < 8; ++j) pb[j] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[j], scale_log2, -sub));
    // codes of rows past every position become 0: their weights are, and a row not written yet may hold a NaN
    uint32_t keep_lo = 0xffffffffu, keep_hi = 0xffffffffu;
    if (n0 + CH - 1 > wmax) {
      const int lim = wmax - n0 - 8 * g;  // rows 0 .. lim of this lane's eight
      const uint64_t keep = lim < 0 ? 0ull : lim >= 7 ? ~0ull : (1ull << (8 * (lim + 1))) - 1;
      keep_lo = (uint32_t)keep;
      keep_hi = (uint32_t)(keep >> 32);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      vec16 w, none;
      decode16(vec16{v[dt][0] & keep_lo, v[dt][1] & keep_hi, 0, 0}, vs, w, none);
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), pb, o[dt], 0, 0, 0);
    }
    l_acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb, l_acc, 0, 0, 0);
    c += W;
    if (++step == 64) {
      step = 0;
      load_scales(c);
    }
  };
  while (c < c_end) {
    body(lds0, lds3);
    if (c < c_end) body(lds1, lds0);
    if (c < c_end) body(lds2, lds1);
    if (c < c_end) body(lds3, lds2);
  }

  // Join the wavefronts: each scales its rows to the common maximum and leaves them in the first stage's place (all
  // loads into it have landed and been read), column group j of row r at j ^ r % 8 of its 16-byte places' eighths.
  if (g == 0) s_m[wave][lm] = m_run;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // a wavefront without chunks has its first loads in flight
  __syncthreads();
  float* so = reinterpret_cast<float*>(lds0);
  auto place = [](int w, int row, int col) { return (w * kCodeRows + row) * D + (col ^ ((row % 8) * (D / 8))); };
  {
    float mx = s_m[0][lm];
#pragma unroll
    for (int w = 1; w < W; ++w) mx = fmaxf(mx, s_m[w][lm]);
    const float sc = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - mx);
    if (g == 0) s_l[wave][lm] = l_acc[0] * sc;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *(f32x4*)(so + place(wave, lm, dt * 16 + 4 * g)) = o[dt] * sc;
  }
  __syncthreads();
  for (int it = threadIdx.x; it < rows * (D / 8); it += W * 64) {
    const int row = it / (D / 8), col = (it % (D / 8)) * 8;
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    float l = 0.f, mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a += *(const f32x4*)(so + place(w, row, col));
      b += *(const f32x4*)(so + place(w, row, col + 4));
      l += s_l[w][row];
      mx = fmaxf(mx, s_m[w][row]);
    }
    const int m = row / group, h = hk * group + row - m * group;
    if (ws != nullptr) {
      float* prow = ws + (((int64_t)z * Hq + h) * n + m) * (D + 4);  // 16-byte aligned rows
      *(f32x4*)(prow + col) = a;
      *(f32x4*)(prow + col + 4) = b;
      if (col == 0) {
        prow[D] = mx;
        prow[D + 1] = l;
      }
    } else {
      const float inv = 1.f / l;
      a *= inv;
      b *= inv;
      *(vec16*)(out + ((int64_t)m * Hq + h) * (D * 2) + col * 2) =
          vec16{f32x2_to_bf16x2_bits(a[0], a[1]), f32x2_to_bf16x2_bits(a[2], a[3]), f32x2_to_bf16x2_bits(b[0], b[1]),
                f32x2_to_bf16x2_bits(b[2], b[3])};
    }
  }
}

// ---- the splits of (token, query head) rows joined ---------------------------------------------------------------
// attn_combine_kernel's merge for launches of many rows: a row a wavefront, D / 4 lanes a partial row (16-byte loads) and 64 / (D / 4)
// partials side by side, four of each in flight. Only the splits that begin at or before the row's position are written and
// read: half of them where positions are spread over the cache.
template <int D>
__global__ __launch_bounds__(256) void join_rows_kernel(char* __restrict__ out, const float* __restrict__ ws,
                                                        const int64_t* __restrict__ pos, int n, int N, int Hq, int splits,
                                                        int split_rows) {
  constexpr int LR = D / 4, P = 64 / LR, U = 4;
  const int lane = threadIdx.x % 64, sub = lane / LR, col = lane % LR * 4;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (row >= (int64_t)n * Hq) return;  // uniform
  const int h = (int)(row / n), m = (int)(row - (int64_t)h * n);
  const int64_t p64 = pos[m], stride = (int64_t)Hq * n * (D + 4);
  const int p = p64 < 0 ? 0 : p64 >= N ? N - 1 : (int)p64;
  const int live = __builtin_amdgcn_readfirstlane(min(splits, p / split_rows + 1));
  const float* base = ws + row * (D + 4);
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int z0 = 0; z0 < live; z0 += P * U) {
    f32x4 o[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      ml[u] = make_float2(-INFINITY, 0.f);
      if (z0 + u * P >= live) continue;  // uniform
      const float* pz = base + (int64_t)min(z0 + u * P + sub, live - 1) * stride;
      o[u] = *(const f32x4*)(pz + col);
      ml[u] = *(const float2*)(pz + D);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool mine = z0 + u * P + sub < live;
      const float mz = mine ? ml[u].x : -INFINITY, mn = fmaxf(M, mz), ref = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(M - ref), b = __builtin_amdgcn_exp2f(mz - ref);  // 0 of -inf
      L = L * a + (mine ? ml[u].y : 0.f) * b;
      acc = acc * a + o[u] * b;
      M = mn;
    }
  }
  float mx = M;
#pragma unroll
  for (int d = LR; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
  const float s = __builtin_amdgcn_exp2f(M - mx);  // the first split has a visible row
  L *= s;
  acc *= s;
#pragma unroll
  for (int d = LR; d < 64; d *= 2) {
    L += __shfl_xor(L, d);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], d);
  }
  const float inv = 1.f / L;
  if (sub == 0)
    *(uint2*)(out + ((int64_t)m * Hq + h) * (D * 2) + col * 2) =
        uint2{f32x2_to_bf16x2_bits(acc[0] * inv, acc[1] * inv), f32x2_to_bf16x2_bits(acc[2] * inv, acc[3] * inv)};
}

}  // namespace ckv

extern "C" int64_t ckv_attention_quantized_workspace_bytes(int32_t n_queries, int32_t n_tokens, int32_t n_q_heads,
                                                           int32_t n_kv_heads, int32_t head_dim) {
  using namespace ckv;
  if (n_queries <= 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_q_heads % n_kv_heads) return 0;
  if (few_rows(n_queries, n_q_heads, n_kv_heads)) {
    const int splits = codes_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, INT64_MAX).splits;
    return splits > 1 ? (int64_t)splits * n_q_heads * n_queries * (head_dim + 4) * 4 : 0;
  }
  if (const GroupedPlan p = attn_grouped_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, INT64_MAX); p.splits > 0)
    return (int64_t)p.splits * n_q_heads * n_queries * (head_dim + 4) * 4;
  return attn_workspace_bytes(n_queries, n_tokens, n_q_heads, head_dim) +
         (decode_first(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim) ? decoded_bytes(n_tokens, n_kv_heads, head_dim) : 0);
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
  if (n_queries < 0 || n_tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || log2_scale(scale) == 0.f)
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

  const float scale_log2 = log2_scale(scale);
  const int group = n_q_heads / n_kv_heads;
  const CacheScales scales = {(const uint8_t*)k_scales, (const uint8_t*)v_scales, blocks, block_log - 5};
  static_assert(kWaveChunk == 32, "a chunk has one scale");
  auto join = [&](float* ws, int splits) {
    const dim3 grid((unsigned)n_queries, (unsigned)n_q_heads);
    const dim3 block(64 * (unsigned)std::min((splits + kCombineParts - 1) / kCombineParts, kCombineMaxWaves));
    auto merge = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, (char*)out, ws, n_queries, n_q_heads, splits); };
    if (head_dim == 128) merge(attn_combine_kernel<128>);
    else merge(attn_combine_kernel<64>);
  };
  if (few_rows(n_queries, n_q_heads, n_kv_heads)) {
    const CodesPlan p = codes_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, workspace_bytes);
    float* ws = p.splits > 1 ? (float*)workspace : nullptr;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)p.splits, (unsigned)n_kv_heads), dim3(kCodeWaves * 64), 0, st, positions, n_queries,
                         n_tokens, (const char*)k_codes, (const char*)v_codes, (const char*)q, q_head_stride * 2, q_token_stride * 2,
                         n_q_heads, group, scale_log2, p.split_chunks, (char*)out, ws, err, scales);
    };
    if (head_dim == 128) launch(attn_codes_kernel<128>);
    else launch(attn_codes_kernel<64>);
    CKV_RETURN_IF_LAUNCH_FAILED();
    if (ws != nullptr) {
      join(ws, p.splits);
      CKV_RETURN_IF_LAUNCH_FAILED();
    }
    return CKV_OK;
  }
  if (const GroupedPlan p = attn_grouped_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, workspace_bytes); p.splits > 0) {
    float* ws = (float*)workspace;
    const GroupedCacheScales gs = {scales, inverse_of((int64_t)n_queries * group, group)};
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(p.map.blocks), dim3(kAttnWaves * 64), 0, st, p.map.nqb, p.map.group, p.map.xpk_log,
                         p.map.items, p.map.inv_group, p.map.inv_nqb, positions, n_queries, n_tokens, (const char*)k_codes,
                         (const char*)v_codes, (int64_t)n_tokens * head_dim, (const char*)q, q_head_stride * 2,
                         q_token_stride * 2, n_q_heads, group, scale_log2, (char*)out, err, ws, p.split_tiles, gs);
    };
    if (head_dim == 128) launch(attn_active_kernel<128, true, GroupedCacheScales>);
    else launch(attn_active_kernel<64, true, GroupedCacheScales>);
    CKV_RETURN_IF_LAUNCH_FAILED();
    const dim3 grid((unsigned)(((int64_t)n_queries * n_q_heads + 3) / 4));
    auto merge = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, (char*)out, (const float*)ws, positions, n_queries, n_tokens, n_q_heads, p.splits,
                         p.split_tiles * kAttnBN);
    };
    if (head_dim == 128) merge(join_rows_kernel<128>);
    else merge(join_rows_kernel<64>);
    CKV_RETURN_IF_LAUNCH_FAILED();
    return CKV_OK;
  }
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

  const AttnPlan plan = attn_plan(n_queries, n_tokens, n_q_heads, n_kv_heads, head_dim, workspace_bytes);
  const AttnMap& map = plan.map;
  float* ws = plan.splits > 1 ? (float*)workspace : nullptr;
  if (plan.wave) {
    const uint32_t inv_gqa = inverse_of((int64_t)n_queries * group, group);
    auto launch = [&](auto kernel, int waves) {
      hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(waves * 64), 0, st, map.nqb, map.group, map.xpk_log, map.items,
                         map.inv_group, map.inv_nqb, positions, n_queries, n_tokens, (const char*)k_codes,
                         (const char*)v_codes, (int64_t)n_tokens * head_dim, (const char*)q, q_head_stride * 2,
                         q_token_stride * 2, n_q_heads, group, inv_gqa, scale_log2, plan.split_chunks, (char*)out, ws, err, scales);
    };
#define CKV_WAVE(HD, QG, W, GR) \
  else if (head_dim == HD && plan.qg == QG && plan.waves == W && plan.grouped == GR) \
    launch(attn_wave_kernel<HD, QG, W, GR, CacheScales>, W);
    if (false) {
    }
    CKV_WAVE_FORMS(CKV_WAVE)
    else return CKV_ERR_INVALID_ARGUMENT;  // a plan outside the list
#undef CKV_WAVE
  } else {
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(map.blocks), dim3(kAttnWaves * 64), 0, st, map.nqb, map.group, map.xpk_log, map.items,
                         map.inv_group, map.inv_nqb, positions, n_queries, n_tokens, (const char*)k_codes,
                         (const char*)v_codes, (int64_t)n_tokens * head_dim, (const char*)q, q_head_stride * 2,
                         q_token_stride * 2, n_q_heads, group, scale_log2, (char*)out, err, ws,
                         plan.split_chunks / (kAttnBN / kWaveChunk), scales);
    };
    if (head_dim == 128) ws != nullptr ? launch(attn_active_kernel<128, true, CacheScales>) : launch(attn_active_kernel<128, false, CacheScales>);
    else ws != nullptr ? launch(attn_active_kernel<64, true, CacheScales>) : launch(attn_active_kernel<64, false, CacheScales>);
  }
  CKV_RETURN_IF_LAUNCH_FAILED();
  if (ws != nullptr) {
    join(ws, plan.splits);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  return CKV_OK;
}
