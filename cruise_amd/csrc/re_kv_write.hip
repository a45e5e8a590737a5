// New tokens into a paged cache: the norm of each query and key head, the
// rotation by the token's position, and the write of keys and values.
#include "re_ops.h"

namespace re {
namespace {

constexpr int kWriteThreads = 256;
constexpr int64_t kWriteMaxBlocks = 1 << 16;  // the kernel strides over the rest

// One wave per (token, head): lane i holds the pairs (i, i + d/2), i + 64, ...
template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) k_kv_write(ResidentKvWrite a) {
  constexpr int kPairs = (D / 2 + 63) / 64;
  const ResidentKvCache& c = a.cache;
  const int lane = threadIdx.x & 63, per_token = a.heads + 2 * c.kv_heads;
  const int64_t units = static_cast<int64_t>(a.tokens) * per_token;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kWriteThreads / 64) + wave_index(threadIdx.x); u < units;
       u += static_cast<int64_t>(gridDim.x) * (kWriteThreads / 64)) {
    const int64_t t = u / per_token;
    const int part = static_cast<int>(u - t * per_token);
    const bool is_q = part < a.heads, is_v = part >= a.heads + c.kv_heads;
    const int h = is_q ? part : (part - a.heads) % c.kv_heads;
    const T* src = is_q   ? static_cast<const T*>(a.q) + t * a.q_strides[0] + h * a.q_strides[1]
                   : is_v ? static_cast<const T*>(a.v) + t * a.v_strides[0] + h * a.v_strides[1]
                          : static_cast<const T*>(a.k) + t * a.k_strides[0] + h * a.k_strides[1];
    T* dst = nullptr;
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + t * a.q_out_strides[0] + h * a.q_out_strides[1];
    } else {
      const int slot = a.slots[t];
      if (slot < 0 || slot >= c.pages * c.block_size) continue;
      const int page = slot / c.block_size, at = slot - page * c.block_size;
      dst = is_v ? static_cast<T*>(c.values) + page * c.value_strides[0] + at * c.value_strides[1] + h * c.value_strides[2]
                 : static_cast<T*>(c.keys) + page * c.key_strides[0] + at * c.key_strides[1] + h * c.key_strides[2];
      if (!is_v && lane == 0) {
        if (c.weights != nullptr) c.weights[page * c.weight_strides[0] + h * c.weight_strides[1] + at] = 0.f;
        if (c.positions != nullptr)
          c.positions[page * c.position_strides[0] + h * c.position_strides[1] + at] = static_cast<int32_t>(a.positions[t]);
      }
    }
    float x[kPairs], y[kPairs], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int e = lane + 64 * i;
      x[i] = e < D / 2 ? Elt<T>::f(src[e]) : 0.f;
      y[i] = e < D / 2 ? Elt<T>::f(src[e + D / 2]) : 0.f;
      sum += x[i] * x[i] + y[i] * y[i];
    }
    if (!is_v) {
      const T* norm = static_cast<const T*>(is_q ? a.q_norm : a.k_norm);
      const float r = norm != nullptr ? 1.f / sqrtf(wave_sum(sum) / D + a.eps) : 1.f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int e = lane + 64 * i;
        if (e >= D / 2) continue;
        if (norm != nullptr) {
          x[i] *= r * Elt<T>::f(norm[e]);
          y[i] *= r * Elt<T>::f(norm[e + D / 2]);
        }
        const double turns = static_cast<double>(a.positions[t]) * a.inv_freq[e] * 0.15915494309189533577;  // / 2 pi
        float s, co;
        sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &co);
        const float n = x[i];
        x[i] = n * co - y[i] * s;
        y[i] = y[i] * co + n * s;
      }
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int e = lane + 64 * i;
      if (e >= D / 2) continue;
      dst[e] = Elt<T>::t(x[i]);
      dst[e + D / 2] = Elt<T>::t(y[i]);
    }
  }
}

template <typename T>
hipError_t launch_write(const ResidentKvWrite& a, hipStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.tokens) * (a.heads + 2 * a.cache.kv_heads);
  const int64_t blocks = std::min(ceil_div(units, kWriteThreads / 64), kWriteMaxBlocks);
  const auto kernel = a.cache.head_dim == 64 ? k_kv_write<T, 64> : a.cache.head_dim == 128 ? k_kv_write<T, 128> : k_kv_write<T, 256>;
  return launch(kernel, blocks, kWriteThreads, 0, stream, a);
}

bool write_ok(const ResidentKvWrite& a) {
  if (!cache_ok(a.cache) || a.tokens < 0 || a.heads <= 0 || a.heads > (1 << 20) || a.cache.kv_heads > (1 << 20) || a.reserved != 0)
    return false;
  if (!(a.eps >= 0.f) || a.inv_freq == nullptr) return false;
  if (a.tokens == 0) return true;
  const int T = a.cache.dtype_bytes;
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.q_out == nullptr || a.positions == nullptr || a.slots == nullptr)
    return false;
  return aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.q_out, 16) && aligned(a.q_norm, 16) &&
         aligned(a.k_norm, 16) && aligned(a.inv_freq, 4) && aligned(a.positions, 8) && aligned(a.slots, 4) &&
         row_strides_ok(a.q_strides, {a.tokens, a.heads}, T) && row_strides_ok(a.q_out_strides, {a.tokens, a.heads}, T) &&
         row_strides_ok(a.k_strides, {a.tokens, a.cache.kv_heads}, T) &&
         row_strides_ok(a.v_strides, {a.tokens, a.cache.kv_heads}, T);
}

}  // namespace
}  // namespace re

extern "C" int32_t resident_kv_write(const ResidentKvWrite* args, void* stream) {
  using namespace re;
  if (args == nullptr || !write_ok(*args)) return -1;
  if (args->tokens == 0) return 0;
  const DeviceScope device(args->cache.device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_write<bf16_t>(*args, s) : launch_write<float>(*args, s);
  return e == hipSuccess ? 0 : -2;
}
