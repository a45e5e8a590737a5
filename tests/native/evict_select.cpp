// kv_evict's selection on the host, with the kernel's own arithmetic
// (re_evict_select.h) and its passes, against a sort.  A lane without a slot takes
// part with the key that the kernel gives it.  Prints the first case that differs
// and returns 1.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <limits>
#include <random>
#include <vector>

#include "re_evict_select.h"

namespace {

using re::kProtected;

struct Selected {
  uint32_t last;
  int ties;
};

// What k_kv_evict does between its keys and its ranks; `lanes` slots at a time.
Selected select(const std::vector<uint32_t>& keys, int budget, int lanes) {
  const int n = static_cast<int>(keys.size());
  uint32_t least = kProtected, most = 0;
  int shield = 0;
  for (uint32_t k : keys) {
    shield += k == kProtected;
    least = std::min(least, k);
    most = std::max(most, k + 1);
  }
  if (shield >= budget) return {kProtected, budget};
  Selected got{kProtected, budget};
  int need = budget - shield;
  re::KeyRange range{least, most - 1 - least};
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = range.shift();
    std::vector<int> bins(1 << re::kBinBits, 0);
    for (int j = 0; j < (n + lanes - 1) / lanes * lanes; ++j) {
      const uint32_t key = j < n ? keys[j] : kProtected;
      if (!range.holds(key)) continue;
      const uint32_t bin = range.bin(key, shift);
      if (bin >= bins.size()) return {0, -1};  // past the bins
      ++bins[bin];
    }
    int b = static_cast<int>(bins.size()) - 1, before = 0;
    while (b >= 0 && before + bins[b] < need) before += bins[b--];
    if (b < 0) return {0, -2};  // fewer keys than needed
    need -= before;
    range = range.part(static_cast<uint32_t>(b), shift);
    if (bins[b] == need) return {range.low - 1, 0};
    got = {range.low, need};
    if (shift == 0) break;
  }
  return got;
}

// Empty: the same slots as a sort's, in lists that cover one another.
const char* check(const std::vector<uint32_t>& keys, int budget, int bound) {
  const int n = static_cast<int>(keys.size()), moves_most = std::max(0, std::min(budget, bound - budget));
  const Selected s = select(keys, budget, 1024);
  if (s.ties == -1) return "a key lies past the bins";
  if (s.ties == -2) return "fewer keys than places";
  std::vector<int> order(n);
  for (int j = 0; j < n; ++j) order[j] = j;
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return keys[x] > keys[y]; });
  std::vector<bool> stays(n, false);
  for (int i = 0; i < budget; ++i) stays[order[i]] = true;
  std::vector<int> list(2 * moves_most, -1), holes, sources;
  int rank = 0, equal = 0, below = 0;
  for (int j = 0; j < n; ++j) {
    const bool kept = keys[j] > s.last || (s.ties > 0 && keys[j] == s.last && equal < s.ties);
    if (kept != stays[j]) return "another slot stays";
    if (j == budget) below = rank;
    if (kept != (j < budget)) {
      const uint32_t at = re::list_entry(j, rank, budget, moves_most);
      if (at >= list.size()) return "an entry lies past the lists";
      list[at] = j;
      (j < budget ? holes : sources).push_back(j);
    }
    equal += keys[j] == s.last;
    rank += kept;
  }
  const int moves = re::moves_of(rank, below, budget, moves_most);
  if (moves != static_cast<int>(holes.size()) || holes.size() != sources.size()) return "moves miscounted";
  for (int i = 0; i < moves; ++i)
    if (list[i] != holes[i] || list[moves_most + moves - 1 - i] != sources[i]) return "lists miss a slot";
  return nullptr;
}

// Whatever a selection said (any slots may stay, as many as it likes): entries lie
// within the lists, and what the moves read was written.
const char* check_bounds(std::mt19937& rng) {
  for (int i = 0; i < 20000; ++i) {
    const int n = 2 + static_cast<int>(rng() % 60), budget = 1 + static_cast<int>(rng() % (n - 1)), bound = n + static_cast<int>(rng() % 5);
    const int moves_most = std::min(budget, bound - budget), often = static_cast<int>(rng() % 11);
    std::vector<int> list(2 * moves_most, -1);
    int rank = 0, below = 0;
    for (int j = 0; j < n; ++j) {
      const bool kept = static_cast<int>(rng() % 10) < often;
      if (j == budget) below = rank;
      const uint32_t at = re::list_entry(j, rank, budget, moves_most);
      if (kept != (j < budget) && at < 2 * static_cast<uint32_t>(moves_most)) list.at(at) = j;
      rank += kept;
    }
    const int moves = re::moves_of(rank, below, budget, moves_most);
    if (moves < 0 || moves > moves_most) return "more moves than the lists hold";
    for (int m = 0; m < moves; ++m)
      if (list[m] < 0 || list[moves_most + moves - 1 - m] < 0) return "a move reads what nobody wrote";
  }
  return nullptr;
}

}  // namespace

int main() {
  std::mt19937 rng(5);
  if (const char* why = check_bounds(rng)) return std::printf("bounds: %s\n", why), 1;
  const float nan = std::numeric_limits<float>::quiet_NaN(), inf = std::numeric_limits<float>::infinity();
  const float least_of[] = {-inf, -1.f, -1e-45f, 0.f, 1e-45f, 1e-3f, 0.5f, 0.7f, 1.f, 3e38f, inf};
  long cases = 0;
  for (int n : {2, 65, 300, 600, 1024, 1025, 1152, 4097})
    for (int budget : {1, n / 3 + 1, n - n / 9 - 1, n - 1}) {
      if (budget >= n) continue;
      for (int shield : {0, 1, budget / 4, budget - 1, budget}) {
        const int places = budget - std::min(budget, shield);
        for (int nans : {0, 1, places - 1, places, places + 1, (places + n) / 2, n - shield - 1, n - shield})
          for (float least : least_of) {
            if (nans < 0 || shield + nans > n) continue;
            std::vector<uint32_t> keys(n);
            for (int j = 0; j < n; ++j) {
              const float above = static_cast<float>(rng() % 1000) / 500.f;
              const float weight = j < shield + nans ? (rng() % 2 ? nan : -nan) : rng() % 3 == 0 ? least : least + above;
              keys[j] = j < shield ? kProtected : re::weight_key(weight);
            }
            std::shuffle(keys.begin(), keys.end(), rng);
            ++cases;
            if (const char* why = check(keys, budget, n + static_cast<int>(rng() % 50)))
              return std::printf("n %d budget %d protected %d NaN %d least %g: %s\n", n, budget, shield, nans, least, why), 1;
          }
      }
    }
  // Keys of any bits.
  for (int i = 0; i < 2000; ++i) {
    const int n = 2 + static_cast<int>(rng() % 3000), budget = 1 + static_cast<int>(rng() % (n - 1));
    std::vector<uint32_t> keys(n);
    const uint32_t mask = rng() % 2 ? 0xffffffffu : 0xffu << rng() % 25;
    for (uint32_t& k : keys) {
      const uint32_t bits = rng() & mask;
      float weight;
      std::memcpy(&weight, &bits, 4);
      k = rng() % 20 == 0 ? kProtected : re::weight_key(weight);
    }
    ++cases;
    if (const char* why = check(keys, budget, n)) return std::printf("random case %d, n %d budget %d: %s\n", i, n, budget, why), 1;
  }
  std::printf("%ld selections\n", cases);
  return 0;
}
