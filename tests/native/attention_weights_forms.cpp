// The kernels that an attention_weights launch takes, by attention_weights_plan.hpp. Shapes on the input, one a line as
// "Hq Hkv D N n": the forms of each, one a line. Without input: every form that any shape of a wide walk takes, and checks of each plan:
// splits and parts cover the cache and the query rows, none empty, joined rows fit what a workgroup holds, workspace regions hold what
// the kernels write; the last line is the shapes walked and the bad ones.
#include "attention_weights_plan.hpp"

#include <cstdio>
#include <set>
#include <string>
#include <vector>

using namespace ckv;

static std::string text(const char* f, int a, int b, int c, int d) {
  char s[64];
  std::snprintf(s, sizeof s, f, a, b, c, d);
  return s;
}

static std::vector<std::string> forms(int Hq, int Hkv, int D, int N, int n, bool& ok) {
  const int rows = n * (Hq / Hkv);
  if (rows <= kWtFewRows && N <= kWtWholeRows) return {text("scores D%d whole", D, 0, 0, 0)};
  if (rows <= kWtFewRows) {
    const FewPlan p = few_plan(rows, N, Hkv);
    ok = p.splits >= 1 && p.splits <= kWtMostParts && (int64_t)p.splits * p.split_chunks >= p.chunks &&
         (int64_t)(p.splits - 1) * p.split_chunks < p.chunks && p.score_stride >= N &&
         p.bytes >= (int64_t)Hkv * rows * (p.score_stride * 4 + p.splits * 8);
    return {text("scores D%d split", D, 0, 0, 0)};
  }
  if (short_cache(rows, N)) return {text("short D%d T%d", D, N <= 64 ? 4 : 16, 0, 0)};
  const WeightsPlan p = weights_plan(n, N, Hq, Hkv, D);
  const int tiles = (N + kWtTile - 1) / kWtTile, row_tiles = p.stat_rows / kWtTile;
  const int64_t total = (int64_t)Hkv * p.stat_rows;
  ok = p.stat_rows >= rows && p.stat_rows % kWtTile == 0 && p.stat_rows - rows < kWtTile && p.row_blocks * 64 * p.qg >= p.stat_rows &&
       p.splits >= 1 && p.splits <= 64 && (p.splits == 1 || ((int64_t)p.splits * p.split_tiles >= tiles && (int64_t)(p.splits - 1) * p.split_tiles < tiles)) &&
       (int64_t)p.key_blocks * 64 * p.kg >= N && p.parts >= 1 && (int64_t)p.parts * p.part_tiles >= row_tiles &&
       (int64_t)(p.parts - 1) * p.part_tiles < row_tiles && p.stat_bytes >= total * (int64_t)sizeof(RowStat) && p.stat_bytes % 16 == 0 &&
       (p.splits == 1 || (p.part_bytes >= total * 8 * p.splits && p.part_bytes % 16 == 0)) &&
       (p.parts == 1 || p.sum_bytes >= (int64_t)Hkv * N * 4 * p.parts) &&
       (!p.join || (p.splits > 1 && p.splits <= kWtJoinSplits && p.part_tiles * kWtTile <= kWtJoinRows));
  std::vector<std::string> f = {text("lse D%d QG%d split%d", D, p.qg, p.splits > 1, 0), text("sum D%d KG%d parts%d join%d", D, p.kg, p.parts > 1, p.join)};
  if (p.splits > 1 && !p.join) f.push_back("join kernel");
  if (p.parts > 1) f.push_back("reduce kernel");
  return f;
}

int main() {
  int hq, hkv, d, N, n;
  bool any = false;
  while (std::scanf("%d %d %d %d %d", &hq, &hkv, &d, &N, &n) == 5) {
    any = true;
    bool ok = true;
    std::string line;
    for (const std::string& f : forms(hq, hkv, d, N, n, ok)) line += (line.empty() ? "" : "; ") + f;
    std::printf("%s\n", line.c_str());
  }
  if (any) return 0;
  std::set<std::string> all;
  long walked = 0, bad = 0;
  for (int D : {64, 128})
    for (int kv : {1, 2, 3, 4, 5, 8, 16, 32, 64, 300})
      for (int group : {1, 2, 3, 4, 7, 8, 14, 16, 17, 64})
        for (int q : {1, 2, 3, 5, 9, 13, 17, 25, 33, 64, 65, 91, 128, 129, 200, 251, 300, 450, 512, 700, 1000, 1500, 2976, 5000, 8256, 20000, 65536, 131072})
          for (int rows_n : {1, 33, 64, 65, 128, 200, 256, 257, 400, 513, 700, 1024, 1025, 1103, 2048, 2050, 4100, 5120, 5121, 8256, 8302, 11999, 12000, 16400,
                             32832, 40960, 41000, 65536, 81920, 131072, 1000000, 2147483000}) {
            bool ok = true;
            for (const std::string& f : forms(kv * group, kv, D, rows_n, q, ok)) all.insert(f);
            ++walked;
            if (!ok && ++bad <= 10) std::printf("bad: %d / %d heads of %d, %d rows, %d queries\n", kv * group, kv, D, rows_n, q);
          }
  for (const std::string& f : all) std::printf("%s\n", f.c_str());
  std::printf("%ld %ld\n", walked, bad);
}
