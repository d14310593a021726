// Prints which kernel takes a product of the experts, for the tests: compiled with the source that decides it.  Nothing is launched.
// stdin: "<multiprocessors> <type> <kind> <rows> <experts> <n> <k>" a line.  stdout: 1 for few rows, 0 for pairs.
#include <stdio.h>

#include "../vllm_plugin_b200/csrc/mmoe_grouped_few.cu"

namespace mmoe {
bool chained() { return false; }
EncodeFn dense_encoder() { return nullptr; }
}  // namespace mmoe

int main() {
  mmoe::GroupedProduct p = {};
  int sms;
  while (scanf("%d %d %d %d %d %d %d", &sms, &p.type, &p.kind, &p.rows, &p.experts, &p.n, &p.k) == 7) printf("%d\n", mmoe::grouped_few_rows(p, sms) ? 1 : 0);
  return 0;
}
