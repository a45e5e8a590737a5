// The arithmetic by which kv_evict finds which slots stay (re_kv_evict.hip).
// Plain functions of integers, so that the host runs them too.
#pragma once

#include <cstdint>

namespace re {

// The order in which slots are kept, as a number: protected slots above all, then
// NaN, then the weights by value (-0 as 0).  No number gets 0.
constexpr uint32_t kProtected = 0xffffffffu, kNanKey = 0xfffffffeu;
constexpr uint32_t weight_key(float weight) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, weight + 0.f);
  const uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
  return weight != weight ? kNanKey : key;
}

// The unprotected keys among which the last one to be kept is looked for, low ..
// low + span, in bins of equal width.  Ranges go by their span: the end of the bin
// that holds a NaN's key would not fit 32 bits, and a range that wraps there would
// take in the protected keys.
constexpr int kBinBits = 11;
struct KeyRange {
  uint32_t low, span;

  constexpr int shift() const {
    const int width = span == 0 ? 0 : 32 - __builtin_clz(span);
    return width > kBinBits ? width - kBinBits : 0;
  }
  constexpr bool holds(uint32_t key) const { return key - low <= span; }
  constexpr uint32_t bin(uint32_t key, int shift) const { return (key - low) >> shift; }
  // The keys of one bin.
  constexpr KeyRange part(uint32_t bin, int shift) const {
    const uint32_t from = bin << shift, width = (1u << shift) - 1;
    return {low + from, span - from < width ? span - from : width};
  }
};

// Where a slot is listed: the i-th slot to fill at i, the slots to take from behind
// the `moves` entries of that list, the last one first.  `rank`: kept slots before
// slot j.  An entry that is not below 2 * moves is none.
constexpr uint32_t list_entry(int j, int rank, int budget, int moves) {
  return static_cast<uint32_t>((j < budget ? j : moves + budget - 1) - rank);
}

// Moves of a row with `kept` slots that stay, `below` of them below the budget.  Of
// fewer than `budget` the lists would lack entries, and none is read.
constexpr int moves_of(int kept, int below, int budget, int moves) {
  const int holes = budget - below;
  return kept < budget || holes < 0 ? 0 : holes < moves ? holes : moves;
}

}  // namespace re
