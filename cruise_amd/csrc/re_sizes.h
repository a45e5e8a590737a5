// Quotients and multiples of sizes, on the host.
#pragma once

#include <cstdint>

namespace re {

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

}  // namespace re
