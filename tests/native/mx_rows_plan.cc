// Prints the plan of every problem on stdin: "weight_only M N K cus" -> "groups chunk waves lds".
#include <cstdio>

#include "mx_rows_plan.h"

int main() {
  int weight_only, M, N, K, cus;
  while (std::scanf("%d %d %d %d %d", &weight_only, &M, &N, &K, &cus) == 5) {
    const cdit::MxRowsPlan p = cdit::mx_rows_plan(weight_only != 0, M, N, K, cus);
    std::printf("%d %d %d %d\n", p.groups, p.chunk, p.waves, p.lds);
  }
}
