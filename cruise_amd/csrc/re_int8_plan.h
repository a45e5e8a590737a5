// How a product of re_int8.hip is cut: the kernel, its tiles and its ranges of K.
// Plain functions of the sizes, so that the host runs them alone too.
#pragma once

#include <algorithm>
#include <cstdint>

#include "re_sizes.h"

namespace re {

constexpr int kFewTokens = 64;       // k_int8_few takes up to so many
constexpr int kFewRows = 96;         // and up to so many channels a workgroup, 6 tiles of 16
constexpr int kInt8StepBytes = 128;  // of K
constexpr int kInt8Waves = 8;

struct LinearPlan {
  int mj, gn, ranges;  // tiles of 64 mj tokens by gn channels
  int few_rows;        // not 0: k_int8_few with so many channels a workgroup
};

// The plans that there are kernels for: any other is an error and not a launch.
constexpr bool has_kernel(const LinearPlan& p) {
  if (p.ranges < 1) return false;
  if (p.few_rows != 0) return p.few_rows > 0 && p.few_rows <= kFewRows;
  const bool tile = p.gn == 256 ? p.mj >= 1 && p.mj <= 4 : p.gn == 192 ? p.mj >= 1 && p.mj <= 3 : (p.gn == 64 || p.gn == 128) && (p.mj == 1 || p.mj == 2);
  return tile && (p.ranges == 1 || p.gn == 256);
}

// Few tokens: as many channels a workgroup as give every CU one workgroup, or equal
// rounds of them.  K is cut where the tokens' bytes, which every workgroup reads, are
// several hundred KB and more than the weights': 64 tokens of 18,944 by 3,584 channels
// take 29, 25 and 24 us in one, two and four ranges, of 3,584 by 3,584 8.5 and 11.6
// in one and two.  A round has a whole number of workgroups for each range, so channels
// that fit the rounds by their number alone can take one round more (64 tokens of 14,336 in
// three ranges: 8,160 channels 34.5 us, 8,192 in two rounds 40.7).
inline LinearPlan few_plan(int64_t tokens, int64_t inner, int64_t outer) {
  constexpr int64_t kCus = 256;
  const int64_t steps = ceil_div(inner, kInt8StepBytes);
  const int64_t bytes = round_up(tokens, 16) * inner, weights = ceil_div(outer, kCus) * inner;
  const int64_t ranges = std::clamp<int64_t>(std::min(bytes / 300000, 2 * bytes / weights), 1, std::max<int64_t>(1, steps / kInt8Waves));
  for (int64_t rounds = ceil_div(outer * ranges, kCus * kFewRows);; ++rounds) {
    const int64_t rows = ceil_div(outer, std::clamp<int64_t>(kCus * rounds / ranges, 1, outer));
    if (rows <= kFewRows) return LinearPlan{0, 0, static_cast<int>(ranges), static_cast<int>(rows)};
  }
}

// The tile and the K ranges of a product: those of least estimated time, rounds of one
// workgroup a CU x (steps of a range x time per step + start and end) plus the partial
// sums' launch, write and read; K is cut with 256-channel tiles only.  The times are fits to
// one MI355X at 65 to 4,096 tokens of the 7B projections, in us a step of 128 bytes; what
// the plan chooses is mostly within 5 % of the best of all there.  Smaller tiles against
// 256 channels alone: 333 x 1,104 x 1,001 7.7 us (64 x 64) and 11.4, 1,000 x 3,584 x 4,608
// 26 (128 x 192) and 31, 256 x 3,584 x 3,584 14 (64 x 64) and 21.
inline LinearPlan linear_plan(int64_t tokens, int64_t inner, int64_t outer) {
  if (tokens <= kFewTokens) return few_plan(tokens, inner, outer);
  constexpr int64_t kCus = 256;
  constexpr double kStep[4][4] = {{0.38, 0.48, 0.6, 0.68}, {0.5, 0.64, 0.84, 0.92}, {0, 0, 1.02, 1.27}, {0, 0, 0, 1.55}};  // 0: no such tile
  constexpr double kFixed = 4.0, kSum = 4.0, kPartBytesPerUs = 2.2e6;
  const int64_t steps = ceil_div(inner, kInt8StepBytes);
  LinearPlan best{4, 256, 1, 0};
  double best_us = 0;
  for (int mj = 4; mj >= 1; --mj)
    for (int wide = 4; wide >= 1; --wide) {
      const double step = kStep[mj - 1][wide - 1];
      if (step == 0) continue;
      const int64_t tiles = ceil_div(tokens, 64 * mj) * ceil_div(outer, 64 * wide);
      for (int s = 1; s <= steps; ++s) {
        if (s > 1 && (wide != 4 || tiles * s > kCus)) break;
        const double bytes = s > 1 ? 4.0 * s * tokens * outer : 0;
        const double us = static_cast<double>(ceil_div(tiles * s, kCus)) * (ceil_div(steps, s) * step + kFixed) + (s > 1 ? kSum + bytes / kPartBytesPerUs : 0);
        if (best_us == 0 || us < best_us) {
          best = LinearPlan{mj, 64 * wide, s, 0};
          best_us = us;
        }
      }
    }
  return best;
}

}  // namespace re
