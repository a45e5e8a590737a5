// The plans of the 8-bit products of up to 64 tokens, on the host: a workgroup has as
// many channels as its kernel has room for, whatever the sizes.
#include <cstdio>

#include "re_int8_plan.h"

int main() {
  using namespace re;
  long plans = 0, cut = 0, bad = 0;
  const auto check = [&](int64_t tokens, int64_t inner, int64_t outer) {
    const LinearPlan p = few_plan(tokens, inner, outer);
    ++plans;
    cut += p.ranges > 1;
    const int64_t steps = ceil_div(inner, kInt8StepBytes);
    const bool fits = p.few_rows >= 1 && p.few_rows <= kFewRows && p.few_rows <= outer && p.ranges >= 1 && p.ranges <= steps;
    if (!fits && ++bad <= 20)
      std::printf("%ld x %ld -> %ld: %d channels a workgroup, %d ranges\n", long(tokens), long(inner), long(outer), p.few_rows, p.ranges);
  };
  // The plan goes by whole tiles of 16 tokens.  Above 16,384 channels no K is cut.
  for (int64_t tokens = 16; tokens <= kFewTokens; tokens += 16)
    for (int64_t inner = 16; inner < 1 << 17; inner += 16)
      for (int64_t outer = 1; outer <= 16640; outer += outer < 4200 || outer > 8100 ? 1 : 3) check(tokens, inner, outer);
  for (int64_t tokens = 1; tokens <= kFewTokens; ++tokens)
    for (int64_t inner = 16; inner < 1 << 17; inner += 16 * 511)
      for (int64_t outer = 1; outer < int64_t{1} << 29; outer += 1 + outer / 97) check(tokens, inner, outer);
  std::printf("%ld plans, %ld with ranges, %ld of them without a kernel\n", plans, cut, bad);
  return bad == 0 && cut > 0 ? 0 : 1;
}
