// One new token of every row over the row's slots of a paged cache: the launches
// and the entry point of what re_kv_attend.h describes.
#include "re_kv_attend.h"

namespace re {
namespace {

template <typename T, int D, bool EVEN>
__global__ void __launch_bounds__(kAttendThreads) k_kv_attention(AttendArgs args) {
  extern __shared__ __align__(16) unsigned char smem[];
  attend_chunk<T, D, EVEN>(args, blockIdx.x, smem);
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) k_kv_attention_join(AttendArgs args) {
  extern __shared__ __align__(16) unsigned char smem[];
  attend_join<T, D>(args, blockIdx.x, 0, smem);
}

template <typename T, int D>
hipError_t launch_attention(const AttendArgs& p, hipStream_t stream) {
  const ResidentKvCache& c = p.a.cache;
  const bool even = even_pages(c);
  const size_t lds = shared_lds(c, p.chunk) + (p.local_scores != 0 ? score_lds(p.a, p.bound) : 0);
  const int64_t blocks = static_cast<int64_t>(p.a.rows) * c.kv_heads * p.head_tiles * p.chunks;
  hipError_t e = launch(even ? k_kv_attention<T, D, true> : k_kv_attention<T, D, false>, blocks, kAttendThreads, lds, stream, p);
  if (e == hipSuccess && p.joined) {
    const int64_t adds = c.weights != nullptr ? p.a.rows * c.kv_heads * ceil_div(p.bound, 4 * kJoinThreads) : 0;
    e = launch(k_kv_attention_join<T, D>, adds + static_cast<int64_t>(p.a.rows) * p.a.heads, kJoinThreads,
               std::max<size_t>(kJoinThreads * 16, static_cast<size_t>(p.a.heads / c.kv_heads) * 8), stream, p);
  }
  return e;
}

template <typename T>
hipError_t launch_attention(const AttendArgs& p, hipStream_t stream) {
  const int d = p.a.cache.head_dim;
  return d == 64 ? launch_attention<T, 64>(p, stream) : d == 128 ? launch_attention<T, 128>(p, stream) : launch_attention<T, 256>(p, stream);
}

}  // namespace
}  // namespace re

extern "C" int64_t resident_kv_attention_workspace(const ResidentKvAttention* args) {
  using namespace re;
  if (args == nullptr || !attention_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  const AttendBytes b = attention_bytes(attention_plan(*args));
  return b.parts + b.stats + b.scores;
}

extern "C" int32_t resident_kv_attention(const ResidentKvAttention* args, void* stream) {
  using namespace re;
  if (args == nullptr || !attention_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  AttendArgs p = attention_plan(*args);
  const AttendBytes b = attention_bytes(p);
  const int64_t need = b.parts + b.stats + b.scores;
  if (need > 0 && (args->workspace == nullptr || args->workspace_bytes < need)) return -1;
  char* base = static_cast<char*>(args->workspace);
  p.parts = reinterpret_cast<float*>(base);
  p.stats = reinterpret_cast<float*>(base + b.parts);
  p.scores = reinterpret_cast<float*>(base + b.parts + b.stats);
  const DeviceScope device(args->cache.device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_attention<bf16_t>(p, s) : launch_attention<float>(p, s);
  return e == hipSuccess ? 0 : -2;
}
