// Walks the launch plans of attention over a paged cache (attention_paged_plan.hpp) and shares out the work of random batches as the
// kernels do: the items fit the launch, and a sequence's splits cover its rows.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "attention_paged_plan.hpp"

using namespace ckv;

int main() {
  std::mt19937_64 rng(5);
  auto log_int = [&](double lo, double hi) {
    return (int64_t)std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi + 1))(rng));
  };
  const int heads[][3] = {{28, 4, 128}, {14, 2, 64}, {8, 8, 64}, {32, 1, 64}, {3, 1, 128}, {64, 8, 128}, {24, 24, 64}, {128, 2, 128}};
  long checked = 0, split = 0, bad = 0;
  for (const auto& h : heads) {
    for (int k = 0; k < 4000; ++k) {
      const int64_t S = log_int(1, 4096), M = log_int(1, 4000), T = 32 << (rng() % 3);
      std::vector<int64_t> count(S), rows(S);
      int64_t n = 0, most = 0;
      const int64_t top = rng() % 2 ? 1 : log_int(1, 3000);
      for (int64_t s = 0; s < S; ++s) {
        count[s] = rng() % 8 == 0 ? 0 : top == 1 ? 1 : log_int(1, top);
        rows[s] = rng() % 8 == 0 ? 0 : log_int(1, M * T);
        n += count[s];
        most = std::max(most, count[s]);
      }
      if (n == 0) continue;
      for (int64_t hint : {most, n, (int64_t)1}) {  // a hint below the truth too
        const int64_t longest = rng() % 2 ? M * T : log_int(1, M * T);  // and of the rows
        const int64_t total = rng() % 2 ? 0 : log_int(1, S * M * T);
        const PagedPlan p = paged_plan(n, S, hint, longest, total, M * T, h[0], h[1], h[2], INT64_MAX);
        const bool large = p.rows == kAttnBM;
        ++checked;
        split += p.target > 0;
        bool ok = (p.rows == 16 || p.rows == 32 || large) && p.map.blocks > 0 && (p.target == 0) == (p.ws_bytes == 0);
        ok = ok && p.ws_bytes == (p.target > 0 ? (large ? p.items : 2 * p.items) * h[1] * p.rows * (h[2] + 4) * 4 : 0);
        const int64_t group = h[0] / h[1], unit = large ? kAttnBN : kPagedUnit;
        float work = 0.f;
        int64_t all_tiles = 0, all_units = 0;
        std::vector<int64_t> tiles(S), units(S);
        for (int64_t s = 0; s < S; ++s) {
          tiles[s] = (count[s] * group + p.rows - 1) / p.rows;
          units[s] = std::max<int64_t>(1, (rows[s] + unit - 1) / unit);
          work += (float)tiles[s] * (float)units[s];
          all_tiles += tiles[s];
          all_units += tiles[s] * units[s];
        }
        int64_t items = 0;
        if (large) {
          const int su = p.target > 0 ? paged_split_units(work, 1.f / (float)p.target, p.min_units) : 1 << 30;
          const float inv = 1.f / (float)su;
          for (int64_t s = 0; s < S; ++s) {
            const int z = paged_splits((int)units[s], su, inv);
            ok = ok && z >= 1 && (tiles[s] == 0 || ((int64_t)z * su >= units[s] && (p.target > 0 || z == 1)));
            items += tiles[s] * z;
          }
          ok = ok && items <= p.items;
        } else if (p.target > 0) {  // equal shares: they are all of the units, which are counted in 32 bits
          const int64_t share = paged_split_units((float)(uint32_t)all_units, 1.f / (float)p.target, p.min_units);
          ok = ok && p.items == p.target && share * p.items >= all_units && all_units <= INT32_MAX / 2 && share * (p.items + 1) < (1ll << 32);
          items = (all_units + share - 1) / share;
        } else {
          items = all_tiles;
          ok = ok && items <= p.items;
        }
        // less workspace than asked for: a form that needs none or less
        const PagedPlan q = paged_plan(n, S, hint, longest, total, M * T, h[0], h[1], h[2], p.ws_bytes - 1);
        ok = ok && (p.target == 0 || q.ws_bytes < p.ws_bytes) && (q.target == 0) == (q.ws_bytes == 0);
        if (!ok) {
          ++bad;
          if (bad < 10) std::printf("S %ld n %ld most %ld rows %ld heads %d/%d: items %ld of %ld\n", (long)S, (long)n, (long)hint, (long)(M * T), h[0], h[1], (long)items, (long)p.items);
        }
      }
    }
  }
  std::printf("%ld %ld %ld\n", checked, split, bad);
  return 0;
}
