// Every plan of an 8-bit product has a kernel, and plans without one are told apart.
#include <cstdio>

#include "re_int8_plan.h"

int main() {
  using namespace re;
  long plans = 0, kinds[5][5] = {}, cut = 0, bad = 0;
  for (int64_t tokens = 1; tokens < 70000; tokens += 1 + tokens / 9)
    for (int64_t inner = 16; inner < 1 << 17; inner += 16 * (1 + inner / 200))
      for (int64_t outer = 1; outer < 300000; outer += 1 + outer / 5) {
        const LinearPlan p = linear_plan(tokens, inner, outer);
        ++plans;
        const int64_t steps = ceil_div(inner, kInt8StepBytes);
        if (!has_kernel(p) || p.ranges > steps || (p.few_rows != 0) != (tokens <= kFewTokens)) {
          if (++bad <= 20) std::printf("%ld x %ld -> %ld: %d x %d, %d ranges, %d\n", long(tokens), long(inner), long(outer), p.mj, p.gn, p.ranges, p.few_rows);
        } else if (p.few_rows == 0) {
          ++kinds[p.mj][p.gn / 64];
          cut += p.ranges > 1;
        }
      }
  // No tile without a call that reaches it.
  long unused = 0;
  for (int mj = 1; mj <= 4; ++mj)
    for (int wide = 1; wide <= 4; ++wide) unused += has_kernel({mj, 64 * wide, 1, 0}) && kinds[mj][wide] == 0;
  // What a broken plan could ask for.
  const LinearPlan none[] = {{0, 0, 3, 97}, {0, 0, 27, 102}, {0, 0, 1, -1}, {0, 0, 0, 16}, {0, 0, 1, 0}, {5, 256, 1, 0}, {4, 192, 1, 0},
                             {3, 128, 1, 0}, {3, 64, 1, 0}, {0, 64, 1, 0}, {2, 320, 1, 0}, {2, 128, 2, 0}, {1, 256, 0, 0}};
  long taken = 0;
  for (const LinearPlan& p : none) taken += has_kernel(p);
  std::printf("%ld plans, %ld cut, %ld without a kernel, %ld tiles unused, %ld broken plans taken\n", plans, cut, bad, unused, taken);
  return bad == 0 && unused == 0 && taken == 0 && cut > 0 ? 0 : 1;
}
