// The pages of a cache that several sequences share (no counterpart in the reference): sequences grow, continue one
// another, end, and the pages that stay move together, all on the device, so that a captured decode step takes its
// pages itself and nothing is read back.
//
// A pool is an ordinary cache (layers, heads, pages * page_tokens, head_dim): page p is the rows [p * page_tokens, (p +
// 1) * page_tokens) of every layer and head, so the kernels that write rows of a cache write into pages as they are.
// The book beside it: table[s][j], the page of sequence s's rows j * page_tokens ..; lengths[s], its rows; refs[p], how
// often the table names page p (free: 0). Pages are taken lowest first, so a book's next state follows from its last.
//
// Bookkeeping runs in one workgroup: which page is the r-th free one is a prefix sum over all of them, a few
// microseconds for tens of thousands of pages, and a second launch would cost as much. Bound: latency, of dependent
// loads and barriers. Traced: a decode step of 32 sequences over 1704 pages 3.6-3.7 us, 63255 tokens of 16 prompts that
// take about 2000 pages 6.7-7.0 (and 4.8 for the launch that writes their rows), 16 forks among 197 pages 6.3, 634
// pages moved together 4.6. Copies of pages run in a launch of their own over (layer, head, K or V) x page; bound:
// their bytes (1.17 GB read and written in 235 us, 5.0 TB/s, what a large torch copy reaches; the 117 MB of 16 forks
// 17.5).
#include <algorithm>

#include "ckv_common.hpp"

namespace ckv {

constexpr int kBookThreads = 1024, kBookWaves = kBookThreads / kWave;
constexpr int kMostSequences = 4096;  // of a book: a workgroup holds two words for each in LDS

struct Book {
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int S, M, P, T_log;
};

// Inclusive prefix sums of K values over the workgroup's threads, in x, and the totals.
template <int K>
struct ScanRoom {
  uint64_t of_wave[kBookWaves][K];
};
template <int K>
__device__ __forceinline__ void book_scan(uint64_t (&x)[K], uint64_t (&total)[K], ScanRoom<K>& s) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    x[k] = wave_incl_scan(x[k]);
    if (lane == kWave - 1) s.of_wave[wave][k] = x[k];
  }
  __syncthreads();
  auto at = [](uint64_t v, int l) {
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), l), lo = __builtin_amdgcn_readlane((uint32_t)v, l);
    return (uint64_t)hi << 32 | lo;
  };
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint64_t w = wave_incl_scan(lane < kBookWaves ? s.of_wave[lane][k] : (uint64_t)0);
    total[k] = at(w, kBookWaves - 1);
    if (wave > 0) x[k] += at(w, wave - 1);
  }
  __syncthreads();
}

// The i with pre[i] <= x < pre[i + 1], for ascending pre[0 .. n] and pre[0] <= x < pre[n].
__device__ __forceinline__ int interval_of(const uint32_t* pre, int n, uint32_t x) {
  int lo = 0, hi = n;  // pre[lo] <= x < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    (pre[mid] <= x ? lo : hi) = mid;
  }
  return lo;
}

// The pages that thread t of a workgroup looks at: [t * n, (t + 1) * n) for n = span_of(P), four at a time.
__device__ __forceinline__ int span_of(int P) { return (((P + kBookThreads - 1) / kBookThreads) + 3) & ~3; }
// f(page, refs) for the pages of this thread, ascending.
template <typename F>
__device__ __forceinline__ void each_page(const Book& b, F f) {
  const int n = span_of(b.P);
  const int64_t first = (int64_t)threadIdx.x * n;
  const int end = (int)min((int64_t)n, b.P - first);  // <= 0: none
  int i = 0;
  for (; i + 4 <= end; i += 4) {
    int r[4];  // 16 bytes at any word
    __builtin_memcpy(r, b.refs + first + i, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) f((int)first + i + j, r[j]);
  }
  for (; i < end; ++i) f((int)first + i, b.refs[first + i]);
}

__device__ __forceinline__ int rows_of(const Book& b, int s) { return min(max(b.lengths[s], 0), b.M << b.T_log); }

// The pool's row of row `pos` of sequence s; -1, flagged, where the table names no page of the pool.
__device__ __forceinline__ int64_t pool_row(const Book& b, int s, int64_t pos, int32_t* err) {
  const int p = b.table[(int64_t)s * b.M + (pos >> b.T_log)];
  if ((uint32_t)p < (uint32_t)b.P) return ((int64_t)p << b.T_log) + (pos & ((1 << b.T_log) - 1));
  flag_error(err, CKV_DEVICE_ERR_RANGE);
  return -1;
}

// Sequence s grows by counts[s] rows, or not at all (flagged): where the count is negative or past its table, the
// tokens past n, or its pages past the free ones.
__global__ __launch_bounds__(kBookThreads) void extend_pages_kernel(int64_t* __restrict__ positions, int64_t* __restrict__ rows,
                                                                    int32_t* __restrict__ starts, int n,
                                                                    const int32_t* __restrict__ counts, Book b,
                                                                    int32_t* __restrict__ err) {
  __shared__ uint32_t s_need[kMostSequences + 1], s_start[kMostSequences + 1];  // pages and tokens of the sequences before
  __shared__ ScanRoom<2> s_scan2;
  __shared__ ScanRoom<1> s_scan1;
  const int T = 1 << b.T_log, tid = threadIdx.x;
  auto pages_of = [&](int64_t r) { return (int)((r + T - 1) >> b.T_log); };
  auto count_of = [&](int s, int len) {
    const int c = counts[s];
    if (c >= 0 && c <= (b.M << b.T_log) - len) return c;
    flag_error(err, CKV_DEVICE_ERR_RANGE);
    return 0;
  };
  uint64_t needed = 0, tokens = 0;
  for (int s0 = 0; s0 < b.S; s0 += kBookThreads) {
    const int s = s0 + tid;
    uint64_t x[2] = {0, 0}, total[2];
    if (s < b.S) {
      const int len = rows_of(b, s), c = count_of(s, len);
      x[0] = pages_of(len + c) - pages_of(len);
      x[1] = c;
    }
    book_scan(x, total, s_scan2);
    if (s < b.S) {
      s_need[s + 1] = (uint32_t)min(needed + x[0], (uint64_t)UINT32_MAX);
      s_start[s + 1] = (uint32_t)min(tokens + x[1], (uint64_t)UINT32_MAX);
    }
    needed += total[0];
    tokens += total[1];
  }
  uint64_t free_pages = 0, free_before = 0;  // before this thread's own
  if (needed > 0) {  // uniform; a decode step often needs none
    uint64_t x[1] = {0}, total[1];
    each_page(b, [&](int, int r) { x[0] += r <= 0; });
    const uint64_t mine = x[0];
    book_scan(x, total, s_scan1);
    free_pages = total[0];
    free_before = x[0] - mine;
  }
  if (tid == 0) s_need[0] = s_start[0] = 0;
  __syncthreads();
  if (needed > free_pages || tokens > (uint64_t)n) {  // uniform: not all of them fit
    tokens = 0;
    for (int s0 = 0; s0 < b.S; s0 += kBookThreads) {
      const int s = s0 + tid;
      uint64_t x[1] = {0}, total[1];
      if (s < b.S) {
        const int len = rows_of(b, s), c = count_of(s, len);
        x[0] = c;
        if (pages_of(len + c) > pages_of(len) && s_need[s + 1] > free_pages) {  // its own need, not s_need's step: that saturates
          x[0] = 0;
          flag_error(err, CKV_DEVICE_ERR_PAGES);
        }
      }
      const bool any = x[0] > 0;
      book_scan(x, total, s_scan1);
      if (s < b.S) {
        if (any && tokens + x[0] > (uint64_t)n) flag_error(err, CKV_DEVICE_ERR_RANGE);
        s_start[s + 1] = (uint32_t)min(tokens + x[0], (uint64_t)n + 1);
      }
      tokens += total[0];
    }
    __syncthreads();
    // Ends past n are n + 1, so of the sequences that reach there the first still has tokens before them: none of it
    // stays.
    if (tokens > (uint64_t)n) {
      const int fit = interval_of(s_start, b.S, (uint32_t)n);  // uniform; s_start[fit] <= n < s_start[fit + 1]
      const uint32_t end = s_start[fit];
      __syncthreads();
      for (int s = fit + 1 + tid; s <= b.S; s += kBookThreads) s_start[s] = end;
      __syncthreads();
    }
  }
  const int total = (int)s_start[b.S];

  if (needed > 0) {
    uint64_t r = free_before;
    each_page(b, [&](int p, int refs) {
      if (refs > 0) return;
      const uint64_t rank = r++;
      if (rank >= needed) return;
      const int s = interval_of(s_need, b.S, (uint32_t)rank);
      if (s_start[s + 1] == s_start[s]) return;  // did not grow
      const int j = pages_of(rows_of(b, s)) + (int)((uint32_t)rank - s_need[s]);
      b.table[(int64_t)s * b.M + j] = p;
      b.refs[p] = 1;
    });
    __syncthreads();
  }
  for (int i = tid; positions != nullptr && i < n; i += kBookThreads) {
    int64_t pos = 0, row = -1;
    if (i < total) {
      const int s = interval_of(s_start, b.S, (uint32_t)i);
      pos = rows_of(b, s) + i - (int)s_start[s];
      row = pool_row(b, s, pos, err);
    }
    positions[i] = pos;
    rows[i] = row;
  }
  __syncthreads();
  for (int s = tid; s <= b.S; s += kBookThreads) {
    starts[s] = (int32_t)s_start[s];
    if (s < b.S) b.lengths[s] = rows_of(b, s) + (int)(s_start[s + 1] - s_start[s]);
  }
}

// The positions and rows of many tokens, after extend_pages_kernel without them (kRowsAlone).
constexpr int kRowsThreads = 256, kRowsEach = 4;
__global__ __launch_bounds__(kRowsThreads) void token_rows_kernel(int64_t* __restrict__ positions, int64_t* __restrict__ rows,
                                                                  const int32_t* __restrict__ starts, int n, Book b,
                                                                  int32_t* __restrict__ err) {
  __shared__ uint32_t s_start[kMostSequences + 1];
  for (int s = threadIdx.x; s <= b.S; s += kRowsThreads) s_start[s] = (uint32_t)starts[s];
  __syncthreads();
  const int total = (int)s_start[b.S];
#pragma unroll
  for (int e = 0; e < kRowsEach; ++e) {
    const int64_t i = ((int64_t)blockIdx.x * kRowsEach + e) * kRowsThreads + threadIdx.x;
    if (i >= n) return;
    int64_t pos = 0, row = -1;
    if (i < total) {
      const int s = interval_of(s_start, b.S, (uint32_t)i);
      pos = b.lengths[s] - (int64_t)s_start[s + 1] + i;
      row = pool_row(b, s, pos, err);
    }
    positions[i] = pos;
    rows[i] = row;
  }
}

// ---- copies of pages -------------------------------------------------------------------------------------------

struct Pool {
  char* k;
  char* v;
  int64_t layer_b, head_b;  // strides, bytes
  int layers, heads, page_b;  // page_b: of a layer, head and K or V; a multiple of 4096
};
constexpr int kCopyThreads = 256;

// Part `part` of 2 * layers * heads (K's, then V's) of page src to page dst. ONCE: no other block reads it
// (non-temporal loads: 1.2 GB of pages moved in 235 us, with ordinary ones 242); a page that 16 sequences get a copy of
// comes out of the L2 (118 MB 27 us, 34 without).
template <bool ONCE>
__device__ __forceinline__ void copy_page(const Pool& pool, int part, int src, int dst) {
  const int lh = pool.layers * pool.heads, at = part % lh;
  char* base = (part < lh ? pool.k : pool.v) + (int64_t)(at / pool.heads) * pool.layer_b + (int64_t)(at % pool.heads) * pool.head_b;
  const char* from = base + (int64_t)src * pool.page_b + threadIdx.x * 16;
  char* to = base + (int64_t)dst * pool.page_b + threadIdx.x * 16;
  constexpr int STEP = kCopyThreads * 16, U = 4;
  auto load = [](const char* p) { return ONCE ? ld16_stream(p) : ld16(p); };
  int off = 0;
  for (; off + U * STEP <= pool.page_b; off += U * STEP) {
    vec16 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load(from + off + u * STEP);
#pragma unroll
    for (int u = 0; u < U; ++u) st16_stream(to + off + u * STEP, v[u]);
  }
  for (; off < pool.page_b; off += STEP) st16_stream(to + off, load(from + off));
}

// ---- continuing sequences --------------------------------------------------------------------------------------

struct Fork {
  int32_t source, target, rows, whole;  // source -1: none; whole pages are shared, ..
  int32_t last, copy;                   // .. page `last` (-1: none) is copied into `copy`
};

// Which pairs are taken, and the free page of each one's partial last page.
__global__ __launch_bounds__(kBookThreads) void fork_book_kernel(Fork* __restrict__ forks, const int32_t* __restrict__ sources,
                                                                 const int32_t* __restrict__ targets, int n, Book b,
                                                                 int32_t* __restrict__ err) {
  __shared__ int s_first[kMostSequences];        // the first pair that names this target
  __shared__ uint32_t s_need[kMostSequences + 1];  // partial pages of the pairs before
  __shared__ ScanRoom<2> s_scan;
  const int T = 1 << b.T_log, tid = threadIdx.x;
  for (int s = tid; s < b.S; s += kBookThreads) s_first[s] = n;
  __syncthreads();
  for (int i = tid; i < n; i += kBookThreads)
    if ((uint32_t)targets[i] < (uint32_t)b.S) atomicMin(&s_first[targets[i]], i);
  if (tid == 0) s_need[0] = 0;
  __syncthreads();
  auto taken = [&](int i) {  // pair i names two sequences, its target is empty and named by no pair before
    const uint32_t s = (uint32_t)sources[i], t = (uint32_t)targets[i];
    return s < (uint32_t)b.S && t < (uint32_t)b.S && s != t && s_first[t] == i && b.lengths[t] == 0;
  };
  uint64_t mine = 0;
  each_page(b, [&](int, int r) { mine += r <= 0; });
  uint64_t needed = 0, free_pages = 0, free_before = 0;  // before this thread's own
  for (int i0 = 0; i0 < n; i0 += kBookThreads) {
    const int i = i0 + tid;
    uint64_t x[2] = {0, i0 == 0 ? mine : 0}, total[2];
    if (i < n) {
      if (taken(i)) x[0] = rows_of(b, sources[i]) % T > 0;
      else flag_error(err, CKV_DEVICE_ERR_RANGE);
    }
    book_scan(x, total, s_scan);
    if (i < n) s_need[i + 1] = (uint32_t)(needed + x[0]);
    if (i0 == 0) {
      free_pages = total[1];
      free_before = x[1] - mine;
    }
    needed += total[0];
  }
  __syncthreads();
  for (int i = tid; i < n; i += kBookThreads) {
    Fork f = {-1, -1, 0, 0, -1, -1};
    if (taken(i)) {
      const int len = rows_of(b, sources[i]);
      if (len % T == 0 || s_need[i + 1] <= free_pages) {
        f = {sources[i], targets[i], len, len >> b.T_log, -1, -1};
        if (len % T > 0) {
          f.last = b.table[(int64_t)f.source * b.M + f.whole];
          if ((uint32_t)f.last >= (uint32_t)b.P) {  // a broken book: nothing outside the pool is read
            f.last = 0;
            flag_error(err, CKV_DEVICE_ERR_RANGE);
          }
        }
      } else {
        flag_error(err, CKV_DEVICE_ERR_PAGES);
      }
    }
    forks[i] = f;
  }
  __syncthreads();
  if (needed > 0) {
    uint64_t r = free_before;
    each_page(b, [&](int p, int refs) {
      if (refs > 0) return;
      const uint64_t rank = r++;
      if (rank >= needed) return;
      const int i = interval_of(s_need, n, (uint32_t)rank);
      if (forks[i].source < 0) return;
      forks[i].copy = p;
      b.refs[p] = 1;
    });
  }
  __syncthreads();
  for (int i = tid; i < n; i += kBookThreads)
    if (forks[i].source >= 0) b.lengths[forks[i].target] = forks[i].rows;
}

// Block (x, i): part x of pair i's partial page; the last x its table row and the shared pages' counts.
__global__ __launch_bounds__(kCopyThreads) void fork_copy_kernel(const Fork* __restrict__ forks, Pool pool, Book b,
                                                                 int32_t* __restrict__ err) {
  const Fork f = forks[blockIdx.y];
  if (f.source < 0) return;
  if ((int)blockIdx.x < 2 * pool.layers * pool.heads) {
    if (f.last >= 0) copy_page<false>(pool, blockIdx.x, f.last, f.copy);
    return;
  }
  const int32_t* from = b.table + (int64_t)f.source * b.M;
  int32_t* to = b.table + (int64_t)f.target * b.M;
  for (int j = threadIdx.x; j < f.whole; j += kCopyThreads) {
    const int p = from[j];
    to[j] = p;
    if ((uint32_t)p < (uint32_t)b.P) atomicAdd(&b.refs[p], 1);
    else flag_error(err, CKV_DEVICE_ERR_RANGE);
  }
  if (threadIdx.x == 0 && f.copy >= 0) to[f.whole] = f.copy;
}

// ---- ending sequences ------------------------------------------------------------------------------------------

// The rows that sequence sequences[i] keeps, into rows[i]: at most keep[i], -1 (all of them, flagged by the next launch,
// which knows whether the sequence was named before) where keep[i] is negative or its last row would be one of several
// in a page that others share, which the next rows would then be written into.
__global__ __launch_bounds__(kCopyThreads) void keep_rows_kernel(int32_t* __restrict__ rows, const int32_t* __restrict__ sequences,
                                                                 const int32_t* __restrict__ keep, int n, Book b) {
  const int i = blockIdx.x * kCopyThreads + threadIdx.x;
  if (i >= n) return;
  const int s = sequences[i];
  if ((uint32_t)s >= (uint32_t)b.S) return;  // flagged there too
  const int len = rows_of(b, s);
  int left = min(keep[i], len);
  if (left < len && (left & ((1 << b.T_log) - 1)) != 0) {
    const int p = left < 0 ? -1 : b.table[(int64_t)s * b.M + (left >> b.T_log)];
    if ((uint32_t)p >= (uint32_t)b.P || b.refs[p] > 1) left = -1;
  }
  rows[i] = max(left, -1);
}

// A block a sequence; of two that are the same the first one's. rows NULL: no row is kept.
__global__ __launch_bounds__(kCopyThreads) void free_pages_kernel(const int32_t* __restrict__ sequences, const int32_t* __restrict__ rows,
                                                                  Book b, int32_t* __restrict__ err) {
  const int s = sequences[blockIdx.x];
  if ((uint32_t)s >= (uint32_t)b.S) {
    if (threadIdx.x == 0) flag_error(err, CKV_DEVICE_ERR_RANGE);
    return;
  }
  int before = 0;
  for (int i = threadIdx.x; i < (int)blockIdx.x; i += kCopyThreads) before |= sequences[i] == s;
  if (__syncthreads_or(before)) return;
  auto pages_of = [&](int r) { return (int)(((uint32_t)r + (1u << b.T_log) - 1) >> b.T_log); };
  const int len = rows_of(b, s), pages = pages_of(len);
  int left = rows != nullptr ? rows[blockIdx.x] : 0;
  if (left < 0) {
    if (threadIdx.x == 0) flag_error(err, CKV_DEVICE_ERR_RANGE);
    left = len;
  }
  int32_t* row = b.table + (int64_t)s * b.M;
  for (int j = pages_of(left) + threadIdx.x; j < pages; j += kCopyThreads) {
    const int p = row[j];
    if ((uint32_t)p < (uint32_t)b.P) atomicSub(&b.refs[p], 1);
    else flag_error(err, CKV_DEVICE_ERR_RANGE);
    row[j] = -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) b.lengths[s] = left;
}

// ---- moving pages together -------------------------------------------------------------------------------------

// Workspace words: [0] moves, then per move its source and target, then the new name of each page.
__host__ __device__ inline int64_t compact_words(int64_t P) { return 1 + (P / 2) * 2 + P; }
struct Moves {
  int32_t* words;
  int P;
  __device__ int32_t& count() const { return words[0]; }
  __device__ int32_t& source(int i) const { return words[1 + i]; }
  __device__ int32_t& target(int i) const { return words[1 + P / 2 + i]; }
  __device__ int32_t& name(int p) const { return words[1 + P / 2 * 2 + p]; }
};

// Of U used pages the i-th at U or above moves to the i-th free one below U: targets and sources are apart, so the
// copies need no order.
__global__ __launch_bounds__(kBookThreads) void compact_book_kernel(Moves m, int32_t* __restrict__ used_out, Book b) {
  __shared__ ScanRoom<1> s_scan;
  __shared__ int s_below;  // used pages below U
  int mine = 0;
  each_page(b, [&](int, int r) { mine += r > 0; });
  uint64_t x[1] = {(uint64_t)mine}, total[1];
  book_scan(x, total, s_scan);
  const int first = (int)x[0] - mine, U = (int)total[0];
  if (threadIdx.x == 0) s_below = U;  // where all of them are, U = P among it
  __syncthreads();
  int used = first;
  each_page(b, [&](int p, int r) {
    if (p == U) s_below = used;
    used += r > 0;
  });
  __syncthreads();
  const int below = s_below;
  used = first;
  each_page(b, [&](int p, int r) {
    if (p < U && r <= 0) m.target(p - used) = p;
    if (p >= U && r > 0) m.source(used - below) = p;
    used += r > 0;
  });
  __syncthreads();
  const int count = U - below;
  used = first;
  each_page(b, [&](int p, int r) {
    m.name(p) = p >= U && r > 0 ? m.target(used - below) : p;
    used += r > 0;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBookThreads) {
    b.refs[m.target(i)] = b.refs[m.source(i)];
    b.refs[m.source(i)] = 0;
  }
  if (threadIdx.x == 0) {
    m.count() = count;
    *used_out = U;
  }
}

// Block (x, y): part x of the moves y, y + gridDim.y, ..; the last x the table rows y, y + gridDim.y, ..
__global__ __launch_bounds__(kCopyThreads) void compact_copy_kernel(Moves m, Pool pool, Book b, int32_t* __restrict__ err) {
  if ((int)blockIdx.x < 2 * pool.layers * pool.heads) {
    const int count = m.count();
    for (int i = blockIdx.y; i < count; i += gridDim.y) copy_page<true>(pool, blockIdx.x, m.source(i), m.target(i));
    return;
  }
  for (int s = blockIdx.y; s < b.S; s += gridDim.y) {
    const int pages = (rows_of(b, s) + (1 << b.T_log) - 1) >> b.T_log;
    int32_t* row = b.table + (int64_t)s * b.M;
    for (int j = threadIdx.x; j < pages; j += kCopyThreads) {
      const int p = row[j];
      if ((uint32_t)p < (uint32_t)b.P) row[j] = m.name(p);
      else flag_error(err, CKV_DEVICE_ERR_RANGE);
    }
  }
}

// New tokens from which their rows get a launch of their own: one workgroup writes 1024 in 0.7 us, a launch costs about
// three.
constexpr int kRowsAlone = 4096;

// ---- arguments -------------------------------------------------------------------------------------------------

static int32_t make_book(Book& b, int32_t* table, int32_t* lengths, int32_t* refs, int32_t S, int32_t M, int32_t P, int32_t T) {
  if (table == nullptr || lengths == nullptr || refs == nullptr) return CKV_ERR_INVALID_ARGUMENT;
  if (S <= 0 || M <= 0 || P <= 0 || (T != 32 && T != 64 && T != 128)) return CKV_ERR_INVALID_ARGUMENT;
  if (S > kMostSequences || (int64_t)M * T > INT32_MAX || (int64_t)P * T > INT32_MAX) return CKV_ERR_TOO_LARGE;
  b = {table, lengths, refs, S, M, P, T == 32 ? 5 : T == 64 ? 6 : 7};
  return CKV_OK;
}
static int32_t make_pool(Pool& pool, void* k, void* v, int64_t layer_stride, int64_t head_stride, int32_t layers, int32_t heads,
                         int32_t head_dim, int32_t dtype, const Book& b) {
  if (k == nullptr || v == nullptr || ((uintptr_t)k | (uintptr_t)v) % 16) return CKV_ERR_INVALID_ARGUMENT;
  if (dtype != CKV_DTYPE_BF16 && dtype != CKV_DTYPE_F32) return CKV_ERR_INVALID_ARGUMENT;
  if (layers <= 0 || heads <= 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return CKV_ERR_INVALID_ARGUMENT;
  const int e = dtype == CKV_DTYPE_BF16 ? 2 : 4;
  if (layer_stride * e % 16 || head_stride * e % 16) return CKV_ERR_INVALID_ARGUMENT;
  const int64_t rows = ((int64_t)b.P << b.T_log) * head_dim;
  if ((heads > 1 && head_stride < rows) || (layers > 1 && layer_stride < (heads - 1) * head_stride + rows)) return CKV_ERR_OUT_OF_RANGE;
  if ((int64_t)layers * heads > INT32_MAX / 2 - 1) return CKV_ERR_TOO_LARGE;
  pool = {(char*)k, (char*)v, layer_stride * e, head_stride * e, layers, heads, (int)((head_dim * e) << b.T_log)};
  return CKV_OK;
}

}  // namespace ckv

#define CKV_RETURN_IF_BAD(call)              \
  do {                                       \
    const int32_t st_ = (call);              \
    if (st_ != CKV_OK) return st_;           \
  } while (0)

extern "C" int32_t ckv_extend_pages(int64_t* positions, int64_t* rows, int32_t* starts, int32_t n_new, const int32_t* counts,
                                    int32_t* table, int32_t* lengths, int32_t* refs, int32_t n_sequences, int32_t n_entries,
                                    int32_t n_pages, int32_t page_tokens, int32_t* err, void* stream) {
  using namespace ckv;
  Book b;
  CKV_RETURN_IF_BAD(make_book(b, table, lengths, refs, n_sequences, n_entries, n_pages, page_tokens));
  if (n_new < 0 || counts == nullptr || starts == nullptr || (n_new > 0 && (positions == nullptr || rows == nullptr)))
    return CKV_ERR_INVALID_ARGUMENT;
  const bool alone = n_new > kRowsAlone;
  hipLaunchKernelGGL(extend_pages_kernel, dim3(1), dim3(kBookThreads), 0, (hipStream_t)stream, alone ? nullptr : positions, rows,
                     starts, n_new, counts, b, err);
  CKV_RETURN_IF_LAUNCH_FAILED();
  if (alone) {
    constexpr int each = kRowsThreads * kRowsEach;
    hipLaunchKernelGGL(token_rows_kernel, dim3((unsigned)(((int64_t)n_new + each - 1) / each)), dim3(kRowsThreads), 0,
                       (hipStream_t)stream, positions, rows, starts, n_new, b, err);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  return CKV_OK;
}

extern "C" int64_t ckv_fork_pages_workspace_bytes(int32_t n_pairs) {
  return n_pairs > 0 ? (int64_t)n_pairs * (int64_t)sizeof(ckv::Fork) : 0;
}

extern "C" int32_t ckv_fork_pages(void* k_pool, void* v_pool, int64_t layer_stride, int64_t head_stride, int32_t n_layers,
                                  int32_t n_heads, int32_t head_dim, int32_t dtype, const int32_t* sources,
                                  const int32_t* targets, int32_t n_pairs, int32_t* table, int32_t* lengths, int32_t* refs,
                                  int32_t n_sequences, int32_t n_entries, int32_t n_pages, int32_t page_tokens,
                                  void* workspace, int64_t workspace_bytes, int32_t* err, void* stream) {
  using namespace ckv;
  Book b;
  Pool pool;
  CKV_RETURN_IF_BAD(make_book(b, table, lengths, refs, n_sequences, n_entries, n_pages, page_tokens));
  CKV_RETURN_IF_BAD(make_pool(pool, k_pool, v_pool, layer_stride, head_stride, n_layers, n_heads, head_dim, dtype, b));
  if (n_pairs < 0) return CKV_ERR_INVALID_ARGUMENT;
  if (n_pairs == 0) return CKV_OK;
  if (sources == nullptr || targets == nullptr) return CKV_ERR_INVALID_ARGUMENT;
  if (n_pairs > kMostSequences) return CKV_ERR_TOO_LARGE;
  if (workspace == nullptr || (uintptr_t)workspace % 4 || workspace_bytes < ckv_fork_pages_workspace_bytes(n_pairs))
    return CKV_ERR_INVALID_ARGUMENT;
  Fork* forks = (Fork*)workspace;
  hipLaunchKernelGGL(fork_book_kernel, dim3(1), dim3(kBookThreads), 0, (hipStream_t)stream, forks, sources, targets, n_pairs, b, err);
  CKV_RETURN_IF_LAUNCH_FAILED();
  hipLaunchKernelGGL(fork_copy_kernel, dim3(2u * n_layers * n_heads + 1, (unsigned)n_pairs), dim3(kCopyThreads), 0,
                     (hipStream_t)stream, forks, pool, b, err);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}

extern "C" int32_t ckv_free_pages(const int32_t* sequences, const int32_t* keep, int32_t n, int32_t* table, int32_t* lengths,
                                  int32_t* refs, int32_t n_sequences, int32_t n_entries, int32_t n_pages, int32_t page_tokens,
                                  void* workspace, int64_t workspace_bytes, int32_t* err, void* stream) {
  using namespace ckv;
  Book b;
  CKV_RETURN_IF_BAD(make_book(b, table, lengths, refs, n_sequences, n_entries, n_pages, page_tokens));
  if (n < 0) return CKV_ERR_INVALID_ARGUMENT;
  if (n == 0) return CKV_OK;
  if (sequences == nullptr) return CKV_ERR_INVALID_ARGUMENT;
  if (n > kMostSequences) return CKV_ERR_TOO_LARGE;
  int32_t* rows = nullptr;
  if (keep != nullptr) {
    if (workspace == nullptr || (uintptr_t)workspace % 4 || workspace_bytes < (int64_t)n * 4) return CKV_ERR_INVALID_ARGUMENT;
    rows = (int32_t*)workspace;
    hipLaunchKernelGGL(keep_rows_kernel, dim3((unsigned)((n + kCopyThreads - 1) / kCopyThreads)), dim3(kCopyThreads), 0,
                       (hipStream_t)stream, rows, sequences, keep, n, b);
    CKV_RETURN_IF_LAUNCH_FAILED();
  }
  hipLaunchKernelGGL(free_pages_kernel, dim3((unsigned)n), dim3(kCopyThreads), 0, (hipStream_t)stream, sequences, rows, b, err);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}

extern "C" int64_t ckv_compact_pages_workspace_bytes(int32_t n_pages) {
  return n_pages > 0 ? ckv::compact_words(n_pages) * 4 : 0;
}

extern "C" int32_t ckv_compact_pages(void* k_pool, void* v_pool, int64_t layer_stride, int64_t head_stride, int32_t n_layers,
                                     int32_t n_heads, int32_t head_dim, int32_t dtype, int32_t* used, int32_t* table,
                                     int32_t* lengths, int32_t* refs, int32_t n_sequences, int32_t n_entries, int32_t n_pages,
                                     int32_t page_tokens, void* workspace, int64_t workspace_bytes, int32_t* err, void* stream) {
  using namespace ckv;
  Book b;
  Pool pool;
  CKV_RETURN_IF_BAD(make_book(b, table, lengths, refs, n_sequences, n_entries, n_pages, page_tokens));
  CKV_RETURN_IF_BAD(make_pool(pool, k_pool, v_pool, layer_stride, head_stride, n_layers, n_heads, head_dim, dtype, b));
  if (used == nullptr || workspace == nullptr || (uintptr_t)workspace % 4 || workspace_bytes < ckv_compact_pages_workspace_bytes(n_pages))
    return CKV_ERR_INVALID_ARGUMENT;
  const Moves m = {(int32_t*)workspace, n_pages};
  hipLaunchKernelGGL(compact_book_kernel, dim3(1), dim3(kBookThreads), 0, (hipStream_t)stream, m, used, b);
  CKV_RETURN_IF_LAUNCH_FAILED();
  const unsigned parts = 2u * n_layers * n_heads;
  const unsigned per_part = std::max(1u, std::min((unsigned)(n_pages / 2 + 1), 32768 / parts + 1));
  hipLaunchKernelGGL(compact_copy_kernel, dim3(parts + 1, per_part), dim3(kCopyThreads), 0, (hipStream_t)stream, m, pool, b, err);
  CKV_RETURN_IF_LAUNCH_FAILED();
  return CKV_OK;
}
