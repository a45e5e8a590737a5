// One new token of every row over the row's slots of a paged cache.
#include "re_ops.h"

namespace re {
namespace {

constexpr int kAttendThreads = 256;
constexpr int kAttendWaves = kAttendThreads / 64;

struct AttendArgs {
  ResidentKvAttention a;
  int bound;  // slots that a row can have
};

// One workgroup per (row, KV head), its query heads one after the other, each
// wave the slots j = wave, wave + 4, ...: a running maximum and sum with the
// output so far, joined over the waves at the end.  The weights take a second
// pass over the keys, once the head's maximum and sum are known.
template <typename T, int D>
__global__ void __launch_bounds__(kAttendThreads) k_kv_attention(AttendArgs args) {
  constexpr int E = D / 64;
  const ResidentKvAttention& a = args.a;
  const ResidentKvCache& c = a.cache;
  __shared__ float wave_max_s[kAttendWaves], wave_sum_s[kAttendWaves], out_s[kAttendWaves][D];
  __shared__ int any_s[kAttendWaves];
  extern __shared__ float head_max_s[];  // each query head's maximum, then its sum
  const int lane = threadIdx.x & 63, w = wave_index(threadIdx.x);
  const int row = blockIdx.x / c.kv_heads, g = blockIdx.x % c.kv_heads, group = a.heads / c.kv_heads;
  const int n = cut_length(a.lengths, row, args.bound);
  const int32_t* table = a.block_table + row * a.table_stride;
  for (int i = 0; i < group; ++i) {
    const int h = g * group + i;
    const T* q = static_cast<const T*>(a.q) + row * a.q_strides[0] + h * a.q_strides[1];
    float qf[E], acc[E] = {}, m = -INFINITY, sum = 0.f;
    int any = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) qf[e] = Elt<T>::f(q[lane + 64 * e]) * a.scale;
    for (int j = w; j < n; j += kAttendWaves) {
      const int page = table[j / c.block_size], at = j % c.block_size;
      if (page < 0 || page >= c.pages) continue;
      const T* k = static_cast<const T*>(c.keys) + page * c.key_strides[0] + at * c.key_strides[1] + g * c.key_strides[2];
      const T* v = static_cast<const T*>(c.values) + page * c.value_strides[0] + at * c.value_strides[1] + g * c.value_strides[2];
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += qf[e] * Elt<T>::f(k[lane + 64 * e]);
      s = wave_sum(s);
      any = 1;
      const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
      const float keep = expf(m - base), p = expf(s - base);
      m = top;
      sum = sum * keep + p;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + p * Elt<T>::f(v[lane + 64 * e]);
    }
    if (lane == 0) {
      wave_max_s[w] = m;
      wave_sum_s[w] = sum;
      any_s[w] = any;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out_s[w][lane + 64 * e] = acc[e];
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    any = 0;
    for (int x = 0; x < kAttendWaves; ++x) top = fmaxf(top, wave_max_s[x]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int x = 0; x < kAttendWaves; ++x) {
      total += wave_sum_s[x] * expf(wave_max_s[x] - base);
      any |= any_s[x];
    }
    T* out = static_cast<T*>(a.out) + row * a.out_strides[0] + h * a.out_strides[1];
    __syncthreads();  // out may be q
    for (int e = threadIdx.x; e < D; e += kAttendThreads) {
      float o = 0.f;
      for (int x = 0; x < kAttendWaves; ++x) o += out_s[x][e] * expf(wave_max_s[x] - base);
      out[e] = Elt<T>::t(any ? o / total : 0.f);
    }
    if (threadIdx.x == 0) {
      head_max_s[i] = base;
      head_max_s[group + i] = total;
    }
    __syncthreads();
  }
  if (c.weights == nullptr) return;
  for (int j = w; j < n; j += kAttendWaves) {
    const int page = table[j / c.block_size], at = j % c.block_size;
    if (page < 0 || page >= c.pages) continue;
    const T* k = static_cast<const T*>(c.keys) + page * c.key_strides[0] + at * c.key_strides[1] + g * c.key_strides[2];
    float p = 0.f;
    for (int i = 0; i < group; ++i) {
      const T* q = static_cast<const T*>(a.q) + row * a.q_strides[0] + (g * group + i) * a.q_strides[1];
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += Elt<T>::f(q[lane + 64 * e]) * a.scale * Elt<T>::f(k[lane + 64 * e]);
      p += expf(wave_sum(s) - head_max_s[i]) / head_max_s[group + i];
    }
    if (lane == 0) c.weights[page * c.weight_strides[0] + g * c.weight_strides[1] + at] += p;
  }
}

template <typename T>
hipError_t launch_attention(const AttendArgs& a, hipStream_t stream) {
  const ResidentKvCache& c = a.a.cache;
  const auto kernel = c.head_dim == 64 ? k_kv_attention<T, 64> : c.head_dim == 128 ? k_kv_attention<T, 128> : k_kv_attention<T, 256>;
  return launch(kernel, static_cast<int64_t>(a.a.rows) * c.kv_heads, kAttendThreads,
                static_cast<size_t>(a.a.heads / c.kv_heads) * 8, stream, a);
}

bool attention_ok(const ResidentKvAttention& a) {
  const ResidentKvCache& c = a.cache;
  if (!cache_ok(c) || a.rows < 0 || a.heads <= 0 || a.heads % c.kv_heads != 0 || a.table_width < 0 || a.max_length < 0 ||
      a.table_stride < 0 || a.workspace_bytes < 0 || a.reserved != 0)
    return false;
  if (a.heads / c.kv_heads > 1024) return false;
  if (static_cast<int64_t>(a.rows) * a.heads > (1 << 22)) return false;  // launches stay below 2^32 threads
  if (a.rows == 0) return true;
  if (a.q == nullptr || a.out == nullptr || a.lengths == nullptr || (a.block_table == nullptr && a.table_width > 0)) return false;
  return aligned(a.q, 16) && aligned(a.out, 16) && aligned(a.block_table, 4) && aligned(a.lengths, 4) && aligned(a.workspace, 16) &&
         row_strides_ok(a.q_strides, {a.rows, a.heads}, c.dtype_bytes) && row_strides_ok(a.out_strides, {a.rows, a.heads}, c.dtype_bytes);
}

int attention_bound(const ResidentKvAttention& a) {
  return static_cast<int>(std::min<int64_t>(a.max_length, static_cast<int64_t>(a.table_width) * a.cache.block_size));
}

}  // namespace
}  // namespace re

extern "C" int64_t resident_kv_attention_workspace(const ResidentKvAttention* args) {
  return args != nullptr && re::attention_ok(*args) ? 0 : -1;
}

extern "C" int32_t resident_kv_attention(const ResidentKvAttention* args, void* stream) {
  using namespace re;
  if (args == nullptr || !attention_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  const DeviceScope device(args->cache.device);
  if (!device.ok()) return -2;
  const AttendArgs a{*args, attention_bound(*args)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_attention<bf16_t>(a, s) : launch_attention<float>(a, s);
  return e == hipSuccess ? 0 : -2;
}
