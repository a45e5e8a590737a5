// Shared parts of the serving operators over a caller's paged cache
// (re_kv_write.hip, re_kv_attention.hip, re_kv_evict.hip, re_logits.hip): the
// host's argument checks, launches on the caller's device and stream, and the
// device's addressing of pages.
#pragma once

#include <algorithm>
#include <numeric>

#include "re_device.h"
#include "resident_epoch.h"

namespace re {

// ---- host ----

// The caller's device current while a call queues its work.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (device < 0) return;
    int now = 0;
    error_ = hipGetDevice(&now);
    if (error_ != hipSuccess || now == device) return;
    error_ = hipSetDevice(device);
    if (error_ == hipSuccess) before_ = now;
  }
  ~DeviceScope() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  bool ok() const { return error_ == hipSuccess; }

 private:
  int before_ = -1;
  hipError_t error_ = hipSuccess;
};

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Strides that keep every row of elements at a multiple of 16 bytes.  The stride
// of a dimension of extent 1 is never used, so it may be anything.
template <int N>
inline bool row_strides_ok(const int64_t (&s)[N], const int32_t (&extents)[N], int dtype_bytes) {
  for (int i = 0; i < N; ++i)
    if (extents[i] > 1 && (s[i] < 0 || s[i] * dtype_bytes % 16 != 0)) return false;
  return true;
}
template <int N>
inline bool strides_ok(const int64_t (&s)[N]) {
  for (int i = 0; i < N; ++i)
    if (s[i] < 0) return false;
  return true;
}

inline bool cache_ok(const ResidentKvCache& c) {
  if (c.keys == nullptr || c.values == nullptr) return false;
  if (c.dtype_bytes != 2 && c.dtype_bytes != 4) return false;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return false;
  if (c.pages <= 0 || c.block_size <= 0 || c.kv_heads <= 0) return false;
  if (static_cast<int64_t>(c.pages) * c.block_size > INT32_MAX) return false;
  return aligned(c.keys, 16) && aligned(c.values, 16) && aligned(c.weights, 4) && aligned(c.positions, 4) &&
         row_strides_ok(c.key_strides, {c.pages, c.block_size, c.kv_heads}, c.dtype_bytes) &&
         row_strides_ok(c.value_strides, {c.pages, c.block_size, c.kv_heads}, c.dtype_bytes) &&
         strides_ok(c.weight_strides) && strides_ok(c.position_strides);
}

// The heads of some tokens or rows, `bytes` each, in memory.
struct HeadRows {
  const void* base;
  int64_t stride[2], extent[2], bytes;  // token, head; the stride of a single one is 0

  HeadRows(const void* p, const int64_t (&s)[2], int64_t rows, int64_t heads, int head_dim, int dtype_bytes)
      : base(p),
        stride{rows > 1 ? s[0] * dtype_bytes : 0, heads > 1 ? s[1] * dtype_bytes : 0},
        extent{rows, heads},
        bytes(static_cast<int64_t>(head_dim) * dtype_bytes) {}
  int outer() const { return stride[0] >= stride[1] ? 0 : 1; }
  // From the start of the first to the end of the last along the inner dimension, and along both.
  __int128 run() const { return static_cast<__int128>(extent[1 - outer()] - 1) * stride[1 - outer()] + bytes; }
  __int128 span() const { return static_cast<__int128>(extent[outer()] - 1) * stride[outer()] + run(); }
  // No two of them overlap.
  bool distinct() const {
    const int o = outer();
    return (extent[1 - o] == 1 || stride[1 - o] >= bytes) && (extent[o] == 1 || stride[o] >= run());
  }
  bool same(const HeadRows& b) const { return base == b.base && stride[0] == b.stride[0] && stride[1] == b.stride[1]; }
};

// None of a's heads overlaps one of b's: one lies behind the other, or both repeat
// in a period in which they have places of their own (parts of one projection, or
// heads side by side).
inline bool apart(const HeadRows& a, const HeadRows& b) {
  const __int128 from = reinterpret_cast<uintptr_t>(a.base), to = reinterpret_cast<uintptr_t>(b.base);
  if (from + a.span() <= to || to + b.span() <= from) return true;
  const auto places = [&](int64_t period, __int128 width_a, __int128 width_b) {
    if (period == 0) return false;
    const __int128 at = ((to - from) % period + period) % period;
    return at >= width_a && at + width_b <= period;
  };
  const int64_t rows = std::gcd(a.stride[a.outer()], b.stride[b.outer()]);
  return places(rows, a.run(), b.run()) || places(std::gcd(rows, std::gcd(a.stride[1 - a.outer()], b.stride[1 - b.outer()])), a.bytes, b.bytes);
}

// An output may take the place of what it is made of, head by head.
inline bool output_ok(const HeadRows& out, const HeadRows& in) { return out.distinct() && (out.same(in) || apart(out, in)); }

// The most slots that a row of a call can have.  Up to 2^30 of them are taken, so
// that the kernels step past the last one in 32 bits.
inline int64_t row_bound(int32_t max_length, int32_t table_width, int32_t block_size) {
  return std::min<int64_t>(max_length, static_cast<int64_t>(table_width) * block_size);
}
constexpr int64_t kMostSlots = 1 << 30;

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// A launch that reports its own error and no earlier one's.
template <typename Args>
inline hipError_t launch(void (*kernel)(Args), int64_t blocks, int threads, size_t lds, hipStream_t stream, const Args& args) {
  void* params[] = {const_cast<Args*>(&args)};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(static_cast<unsigned>(blocks)), dim3(threads), params, lds,
                         stream);
}

// ---- device ----

// The row's slots: its length cut to the call's bound.
__device__ __forceinline__ int cut_length(const int32_t* lengths, int row, int bound) {
  return max(0, min(lengths[row], bound));
}

}  // namespace re
