// Prints which tiles the launches of dense products have (csrc/mmoe_dense_rules.h), for the tests.  Host code only.
// stdin: a launch a line, "<pairs> <products> " and of each product "<type> <kind> <m> <n> <k> <A transposed> <B transposed>".
// stdout: of each product "<columns> <tiles> ", then the launch's stages.
#include <stdio.h>

#include "../vllm_plugin_b200/csrc/mmoe_dense_rules.h"

using namespace mmoe;

int main() {
  int pairs, parts;
  while (scanf("%d %d", &pairs, &parts) == 2 && parts <= kMaxParts) {
    DenseProduct p[kMaxParts] = {};
    for (int i = 0; i < parts; ++i) {
      int a, b;
      if (scanf("%d %d %d %d %d %d %d", &p[i].type, &p[i].kind, &p[i].m, &p[i].n, &p[i].k, &a, &b) != 7) return 1;
      p[i].a.k_rows = a != 0, p[i].b.k_rows = b != 0;
    }
    int cols[kMaxParts] = {}, bytes = 0;
    choose_cols(p, parts, pairs, cols);
    for (int i = 0; i < parts; ++i) {
      printf("%d %lld ", cols[i], (long long)tile_cost(p[i], cols[i]).tiles);
      bytes = std::max(bytes, kStageA + stage_b_bytes(p[i], cols[i]));
    }
    printf("%d\n", std::min(kPairStageRoom / bytes, kMaxStages));
  }
  return 0;
}
