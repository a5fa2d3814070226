// The kernels that a launch of attention over an 8-bit cache takes, by attention_quantized_plan.hpp and attention_plan.hpp. Shapes on the
// input, one a line as "Hq Hkv D N n workspace" (workspace 1: all that the launch asks for, 0: none): the forms of each, one a line. Without
// input: every form that any shape of a wide walk takes, and whether workspaces hold what the kernels write; the last line is the
// shapes walked and the bad ones.
#include "attention_quantized_plan.hpp"

#include <cstdio>
#include <set>
#include <string>
#include <vector>

using namespace ckv;

static std::string text(const char* f, int a, int b, int c, int d, int e) {
  char s[64];
  std::snprintf(s, sizeof s, f, a, b, c, d, e);
  return s;
}

// As ckv_attention_quantized and its workspace size decide, in their order.
static std::vector<std::string> forms(int Hq, int Hkv, int D, int N, int n, bool workspace, bool& ok) {
  const int64_t row_b = (int64_t)Hq * n * (D + 4) * 4;
  if (few_rows(n, Hq, Hkv)) {
    const int asked = codes_plan(n, N, Hq, Hkv, D, INT64_MAX).splits;
    const int64_t ws = workspace && asked > 1 ? asked * row_b : 0;
    const CodesPlan p = codes_plan(n, N, Hq, Hkv, D, ws);
    const int chunks = (int)(((int64_t)N + kWaveChunk - 1) / kWaveChunk);
    ok = p.splits >= 1 && (p.splits == 1 || p.splits * row_b <= ws) && (int64_t)p.splits * p.split_chunks >= chunks &&
         (int64_t)(p.splits - 1) * p.split_chunks < chunks;
    return {text("codes D%d split%d", D, p.splits > 1, 0, 0, 0)};
  }
  const int asked = attn_grouped_plan(n, N, Hq, Hkv, D, INT64_MAX).splits;
  const int64_t ws = !workspace   ? 0
                     : asked > 0 ? asked * row_b
                                 : attn_workspace_bytes(n, N, Hq, D) + (decode_first(n, N, Hq, Hkv, D) ? decoded_bytes(N, Hkv, D) : 0);
  if (const GroupedPlan p = attn_grouped_plan(n, N, Hq, Hkv, D, ws); p.splits > 0) {
    ok = p.splits * row_b <= ws;
    return {text("grouped D%d", D, 0, 0, 0, 0)};
  }
  const int64_t decoded = decoded_bytes(N, Hkv, D);
  if (ws >= decoded && decode_first(n, N, Hq, Hkv, D)) {
    const AttnPlan p = attn_plan(n, N, Hq, Hkv, D, ws - decoded);
    ok = !p.wave && (p.splits <= 1 || decoded + p.splits * row_b <= ws);
    return {text("bf16 copy D%d split%d", D, p.splits > 1, 0, 0, 0)};
  }
  const AttnPlan p = attn_plan(n, N, Hq, Hkv, D, ws);
  ok = p.splits <= 1 || p.splits * row_b <= ws;
  if (p.wave) return {text("wave D%d QG%d W%d grouped%d split%d", D, p.qg, p.waves, p.grouped, p.splits > 1)};
  return {text("large D%d split%d", D, p.splits > 1, 0, 0, 0)};
}

int main() {
  int hq, hkv, d, N, n, w;
  bool any = false;
  while (std::scanf("%d %d %d %d %d %d", &hq, &hkv, &d, &N, &n, &w) == 6) {
    any = true;
    bool ok = true;
    std::printf("%s\n", forms(hq, hkv, d, N, n, w != 0, ok)[0].c_str());
  }
  if (any) return 0;
  std::set<std::string> all;
  long walked = 0, bad = 0;
  for (int D : {64, 128})
    for (int kv : {1, 2, 3, 4, 5, 8, 16, 32, 64})
      for (int group : {1, 2, 3, 4, 7, 8, 14, 16, 17, 64})
        for (int q : {1, 2, 3, 4, 5, 9, 13, 17, 18, 25, 33, 40, 64, 65, 84, 91, 128, 129, 160, 200, 251, 300, 450, 512, 700, 1000, 1500, 2100, 2976, 4128,
                      5000, 8256, 20000})
          for (int rows : {1, 33, 64, 300, 513, 545, 700, 768, 800, 1024, 1025, 1103, 1500, 1537, 1600, 2050, 3000, 3999, 4000, 4100, 5120, 5121, 6999, 7000,
                           8256, 8302, 16400, 28787, 32832, 65536, 131072, 1000000})
            for (bool ws : {false, true}) {
              bool ok = true;
              for (const std::string& f : forms(kv * group, kv, D, rows, q, ws, ok)) all.insert(f);
              ++walked;
              if (!ok && ++bad <= 10) std::printf("bad: %d / %d heads of %d, %d rows, %d queries, workspace %d\n", kv * group, kv, D, rows, q, ws);
            }
  for (const std::string& f : all) std::printf("%s\n", f.c_str());
  std::printf("%ld %ld\n", walked, bad);
}
