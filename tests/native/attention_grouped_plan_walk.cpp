// Walks attn_grouped_plan, the plan of the 128-query kernel over an 8-bit cache with a KV head's (token, query head) pairs as rows: its
// blocks hold every row, its splits cover the cache, none empty, and fit the workspace, its work items cover every (block, head,
// split) once. Prints the plans checked, those that take the form, and the bad ones.
#include "attention_plan.hpp"

#include <cstdio>
#include <vector>

using namespace ckv;

static int divided(int x, int d, uint32_t inv) {
  return inv != 0 ? (int)(((uint64_t)(uint32_t)x * inv) >> 32) : d == 1 ? x : x / d;
}

int main() {
  long checked = 0, taken_form = 0, bad = 0;
  for (int D : {64, 128})
    for (int hkv : {1, 2, 3, 4, 5, 8, 16, 64, 600})
      for (int group : {1, 2, 3, 7, 8, 16, 64})
        for (int n : {1, 3, 17, 25, 33, 64, 84, 128, 129, 251, 300, 500, 915, 1100, 2000, 2976, 8256})
          for (int N : {1, 33, 1103, 3999, 4000, 6999, 7000, 8256, 8302, 28787, 65536, 131072, 1000000, 2147483647})
            for (int share : {0, 1, 2, 3}) {
              const int Hq = hkv * group;
              const int64_t row_b = (int64_t)Hq * n * (D + 4) * 4, ws = share == 3 ? INT64_MAX : row_b * share * 2;
              const GroupedPlan p = attn_grouped_plan(n, N, Hq, hkv, D, ws);
              ++checked;
              if (p.splits == 0) continue;
              ++taken_form;
              const int64_t tiles = ((int64_t)N + kAttnBN - 1) / kAttnBN, rows = (int64_t)n * group;
              const AttnMap& m = p.map;
              bool ok = p.splits >= 2 && (int64_t)m.nqb * kAttnBM >= rows && (int64_t)p.splits * p.split_tiles >= tiles &&
                        (int64_t)(p.splits - 1) * p.split_tiles < tiles && p.splits * row_b <= ws;
              std::vector<char> taken((size_t)hkv * m.nqb * p.splits, 0);
              size_t count = 0;
              for (uint32_t L = 0; ok && L < m.blocks; ++L) {
                const int xcd = L % kXcds, j = (int)((L / kXcds) << m.xpk_log) + (xcd & ((1 << m.xpk_log) - 1));
                if (j >= m.items) continue;
                const int rest = divided(j, m.group, m.inv_group), h = (xcd >> m.xpk_log) * m.group + (j - rest * m.group);
                const int z = divided(rest, m.nqb, m.inv_nqb), qb = m.nqb - 1 - (rest - z * m.nqb);
                ok = h >= 0 && h < hkv && z >= 0 && z < p.splits && qb >= 0 && qb < m.nqb;
                if (!ok) break;
                char& t = taken[((size_t)z * m.nqb + qb) * hkv + h];
                ok = !t;
                t = 1, ++count;
              }
              ok = ok && count == taken.size();
              if (!ok && ++bad <= 10)
                std::printf("D %d hkv %d group %d n %d N %d ws %lld: splits %d x %d, %d blocks\n", D, hkv, group, n, N, (long long)ws, p.splits,
                            p.split_tiles, m.nqb);
            }
  std::printf("%ld %ld %ld\n", checked, taken_form, bad);
}
