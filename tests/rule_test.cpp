// csrc/mx_rule.h as a filter: a line of sizes in, the form that the library takes out.
#include "mx_rule.h"

#include <cstdio>

using namespace tinyoai_rule;

int main() {
  char kind;
  while (std::scanf(" %c", &kind) == 1) {
    if (kind == 'r') {  // tokens, experts, choices
      long n, experts, k;
      if (std::scanf("%ld %ld %ld", &n, &experts, &k) != 3) return 1;
      static const char *names[] = {"one_block", "by_expert", "by_tokens"};
      std::printf("%s %d\n", names[(int)sort_path(n, k)], lane_experts((int)experts));
      continue;
    }
    int bf16, planes, gate, grouped;
    long experts, n, rows, cols;
    if (std::scanf("%d %d %d %d %ld %ld %ld %ld", &bf16, &planes, &gate, &grouped, &experts, &n, &rows, &cols) != 8) return 1;
    const Sizes s{bf16 != 0, planes, gate != 0, grouped != 0, experts, n, rows, cols};
    if (few_rows(s)) {
      const Few f = few_form(s);
      std::printf("few %d %d %d\n", f.waves, f.column_tiles, f.wave_chunks);
    } else {
      const int ks = parts(s, 256);
      const Tile t = tile(s, ks, 256);
      if (ks > 1 && t.bm != 32) return 2;  // only the smallest tiles come in parts
      std::printf("tile %d %d %d\n", t.bm, t.bn, (int)t.runs);
    }
  }
}
