// Walks attn_wave_plan, attn_wave_kernel's plan, over launches of any size (attn_plan asks it for small ones): its form exists, its splits cover the cache, none empty, and fit the workspace, its work items
// cover every (query block, head, split) once. Prints the plans checked and the bad ones.
#include "attention_plan.hpp"

#include <cstdio>
#include <vector>

using namespace ckv;

static int divided(int x, int d, uint32_t inv) {
  return inv != 0 ? (int)(((uint64_t)(uint32_t)x * inv) >> 32) : d == 1 ? x : x / d;
}
static bool form_exists(const AttnPlan& p, int D) {
#define CKV_IS(HD, QG, W, GR) if (D == HD && p.qg == QG && p.waves == W && p.grouped == GR) return true;
  CKV_WAVE_FORMS(CKV_IS)
#undef CKV_IS
  return false;
}

int main() {
  long checked = 0, bad = 0;
  for (int D : {64, 128})
    for (int hkv : {1, 2, 3, 4, 5, 8, 16, 64})
      for (int group : {1, 2, 7, 8, 16, 64})
        for (int n : {1, 2, 3, 5, 16, 17, 33, 64, 127, 128, 129, 300, 1000, 2976, 8256})
          for (int N : {1, 31, 32, 33, 500, 1103, 2048, 8256, 32832, 131072, 1000000})
            for (int share : {0, 1, 2}) {
              const int Hq = hkv * group;
              const int64_t ws = attn_workspace_bytes(n, N, Hq, D) * share / 2;
              const AttnPlan p = attn_wave_plan(n, N, Hq, hkv, D, ws);
              ++checked;
              const int chunks = (N + kWaveChunk - 1) / kWaveChunk, rows = p.grouped ? n * group : n, heads = p.grouped ? hkv : Hq;
              bool ok = form_exists(p, D) && p.wave && (int64_t)p.map.nqb * 16 * p.qg >= rows;
              ok = ok && p.splits >= 1 && (p.splits == 1 || ((int64_t)p.splits * p.split_chunks >= chunks &&
                                                             (int64_t)(p.splits - 1) * p.split_chunks < chunks &&
                                                             (int64_t)p.splits * Hq * n * (D + 4) * 4 <= ws));
              const AttnMap& m = p.map;
              if (ok && (int64_t)heads * m.nqb * p.splits < 200000) {
                std::vector<char> taken((size_t)heads * m.nqb * p.splits, 0);
                size_t count = 0;
                for (uint32_t L = 0; ok && L < m.blocks; ++L) {
                  const int xcd = L % kXcds, j = (int)((L / kXcds) << m.xpk_log) + (xcd & ((1 << m.xpk_log) - 1));
                  if (j >= m.items) continue;
                  const int rest = divided(j, m.group, m.inv_group), h = (xcd >> m.xpk_log) * m.group + (j - rest * m.group);
                  const int z = divided(rest, m.nqb, m.inv_nqb), qb = m.nqb - 1 - (rest - z * m.nqb);
                  ok = h >= 0 && h < heads && z >= 0 && z < p.splits && qb >= 0 && qb < m.nqb;
                  if (!ok) break;
                  char& t = taken[((size_t)z * m.nqb + qb) * heads + h];
                  ok = !t;
                  t = 1, ++count;
                }
                ok = ok && count == taken.size();
              }
              if (!ok && ++bad <= 10)
                std::printf("D %d hkv %d group %d n %d N %d ws %lld: qg %d waves %d grouped %d splits %d x %d\n", D, hkv, group, n, N,
                            (long long)ws, p.qg, p.waves, (int)p.grouped, p.splits, p.split_chunks);
            }
  std::printf("%ld %ld\n", checked, bad);
}
