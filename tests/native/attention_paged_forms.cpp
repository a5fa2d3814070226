// The kernel form of each launch named on standard input, one a line: tokens, sequences, most tokens of one, rows that the table has room for, rows of all (0: not told),
// query heads, KV heads, head size, and whether there is a workspace. Prints the head size, the tile's rows, and whether tiles are split, their
// joins spread and the sequences more than 64.
#include <cstdio>

#include "attention_paged_plan.hpp"

int main() {
  long n, S, most, rows, total;
  int Hq, Hkv, D, split;
  while (std::scanf("%ld %ld %ld %ld %ld %d %d %d %d", &n, &S, &most, &rows, &total, &Hq, &Hkv, &D, &split) == 9) {
    const ckv::PagedPlan p = ckv::paged_plan(n, S, most, rows, total, rows, Hq, Hkv, D, split ? INT64_MAX : 0);
    std::printf("%d %d %d %d %d\n", D, p.rows, p.target > 0, p.target > 0 && p.spread_join, p.rows < ckv::kAttnBM && S > 64);
  }
  return 0;
}
