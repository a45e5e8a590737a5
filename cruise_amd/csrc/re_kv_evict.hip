// Eviction from a paged cache by the attention weight that its slots gathered.
#include "re_ops.h"

namespace re {
namespace {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;

struct EvictArgs {
  ResidentKvEvict a;
  int bound;      // slots that a row can have
  int32_t* lists; // [rows][kv_heads][2][budget]: evicted slots below the budget, kept slots by rank
};

// Where slot j of a row lies, for one KV head.
struct SlotAddress {
  int page, at;
};
__device__ __forceinline__ SlotAddress slot_address(const int32_t* table, int block_size, int j) {
  const int p = j / block_size;
  return {table[p], j - p * block_size};
}

// The order in which slots are kept, as a number: protected slots above all,
// then NaN, then the weights by value (-0 as 0).
__device__ __forceinline__ uint32_t keep_key(float weight, int position, int64_t recent_from, int sinks) {
  if (position >= 0 && (position < sinks || position >= recent_from)) return 0xffffffffu;
  if (weight != weight) return 0xfffffffeu;
  const uint32_t bits = __float_as_uint(weight == 0.f ? 0.f : weight);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ int block_sum(int v, int* red, int tid) {
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = v;
  __syncthreads();
  int sum = 0;
  for (int w = 0; w < kEvictWaves; ++w) sum += red[w];
  return sum;
}

// One workgroup per (row, KV head).  The key of the last slot kept is found bit
// by bit (the greatest one that `budget` slots reach), ties in slot order; then
// the evicted slots below the budget and the kept ones behind it are listed in
// order and paired.
template <typename T, int D>
__global__ void __launch_bounds__(kEvictThreads) k_kv_evict(EvictArgs args) {
  const ResidentKvEvict& a = args.a;
  const ResidentKvCache& c = a.cache;
  __shared__ int red[kEvictWaves], gt_s[kEvictWaves], tie_s[kEvictWaves], below_s;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_index(tid);
  const int row = blockIdx.x / c.kv_heads, g = blockIdx.x % c.kv_heads, budget = a.budget;
  const int n = cut_length(a.lengths, row, args.bound);
  const int32_t* table = a.block_table + row * a.table_stride;
  int bad = 0;
  for (int p = tid; p < (n + c.block_size - 1) / c.block_size; p += kEvictThreads) bad |= table[p] < 0 || table[p] >= c.pages;
  bad = block_sum(bad, red, tid);
  if (g == 0 && tid == 0) a.out_lengths[row] = bad ? n : min(n, budget);
  if (bad != 0 || n <= budget) return;

  const int64_t recent_from = a.next_positions[row] - a.recent;
  auto key_of = [&](int j) {
    const SlotAddress s = slot_address(table, c.block_size, j);
    return keep_key(c.weights[s.page * c.weight_strides[0] + g * c.weight_strides[1] + s.at],
                    c.positions[s.page * c.position_strides[0] + g * c.position_strides[1] + s.at], recent_from, a.sinks);
  };
  uint32_t last = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t probe = last | (1u << b);
    int count = 0;
    for (int j = tid; j < n; j += kEvictThreads) count += key_of(j) >= probe;
    if (block_sum(count, red, tid) >= budget) last = probe;
  }
  int above = 0;
  for (int j = tid; j < n; j += kEvictThreads) above += key_of(j) > last;
  const int ties = budget - block_sum(above, red, tid);  // of the slots with the last key, the lowest so many stay

  int32_t* holes = args.lists + static_cast<int64_t>(blockIdx.x) * 2 * budget;
  int32_t* kept_slots = holes + budget;
  int gt_before = 0, tie_before = 0;
  for (int j0 = 0; j0 < n; j0 += kEvictThreads) {
    const int j = j0 + tid;
    const uint32_t key = j < n ? key_of(j) : 0;
    const bool gt = j < n && key > last, tie = j < n && key == last;
    const uint64_t gts = __ballot(gt), tys = __ballot(tie), lower = (1ull << lane) - 1;
    __syncthreads();
    if (lane == 0) {
      gt_s[w] = __popcll(gts);
      tie_s[w] = __popcll(tys);
    }
    __syncthreads();
    int gt_at = gt_before + __popcll(gts & lower), tie_at = tie_before + __popcll(tys & lower);
    for (int x = 0; x < kEvictWaves; ++x) {
      if (x < w) {
        gt_at += gt_s[x];
        tie_at += tie_s[x];
      }
      gt_before += gt_s[x];
      tie_before += tie_s[x];
    }
    const bool kept = gt || (tie && tie_at < ties);
    const int rank = gt_at + min(tie_at, ties);  // kept slots before j
    if (j < budget && !kept) holes[j - rank] = j;
    if (j >= budget && kept) kept_slots[rank] = j;
    if (j == budget) below_s = rank;
  }
  __syncthreads();
  const int below = below_s, moves = budget - below;

  constexpr int kLanes = D * sizeof(T) / 16;
  for (int i = tid / kLanes; i < moves; i += kEvictThreads / kLanes) {
    const SlotAddress to = slot_address(table, c.block_size, holes[i]), from = slot_address(table, c.block_size, kept_slots[below + i]);
    const int e = tid % kLanes * (16 / sizeof(T));
    const T* k = static_cast<const T*>(c.keys) + g * c.key_strides[2] + e;
    const T* v = static_cast<const T*>(c.values) + g * c.value_strides[2] + e;
    const re_u32x4 kx = *reinterpret_cast<const re_u32x4*>(k + from.page * c.key_strides[0] + from.at * c.key_strides[1]);
    const re_u32x4 vx = *reinterpret_cast<const re_u32x4*>(v + from.page * c.value_strides[0] + from.at * c.value_strides[1]);
    *reinterpret_cast<re_u32x4*>(const_cast<T*>(k) + to.page * c.key_strides[0] + to.at * c.key_strides[1]) = kx;
    *reinterpret_cast<re_u32x4*>(const_cast<T*>(v) + to.page * c.value_strides[0] + to.at * c.value_strides[1]) = vx;
  }
  float* weights = c.weights + g * c.weight_strides[1];
  int32_t* positions = c.positions + g * c.position_strides[1];
  for (int i = tid; i < moves; i += kEvictThreads) {
    const SlotAddress to = slot_address(table, c.block_size, holes[i]), from = slot_address(table, c.block_size, kept_slots[below + i]);
    weights[to.page * c.weight_strides[0] + to.at] = weights[from.page * c.weight_strides[0] + from.at];
    positions[to.page * c.position_strides[0] + to.at] = positions[from.page * c.position_strides[0] + from.at];
  }
  __syncthreads();
  for (int j = budget + tid; j < n; j += kEvictThreads) {
    const SlotAddress s = slot_address(table, c.block_size, j);
    weights[s.page * c.weight_strides[0] + s.at] = 0.f;
    positions[s.page * c.position_strides[0] + s.at] = -1;
  }
}

template <typename T>
hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  const ResidentKvCache& c = a.a.cache;
  const auto kernel = c.head_dim == 64 ? k_kv_evict<T, 64> : c.head_dim == 128 ? k_kv_evict<T, 128> : k_kv_evict<T, 256>;
  return launch(kernel, static_cast<int64_t>(a.a.rows) * c.kv_heads, kEvictThreads, 0, stream, a);
}

bool evict_ok(const ResidentKvEvict& a) {
  const ResidentKvCache& c = a.cache;
  if (!cache_ok(c) || c.weights == nullptr || c.positions == nullptr || a.rows < 0 || a.table_width < 0 || a.max_length < 0 ||
      a.table_stride < 0 || a.workspace_bytes < 0 || a.budget <= 0 || a.recent < 0 || a.sinks < 0)
    return false;
  if (static_cast<int64_t>(a.recent) + a.sinks > a.budget) return false;
  if (static_cast<int64_t>(a.rows) * c.kv_heads > (1 << 21)) return false;  // launches stay below 2^32 threads
  if (a.rows == 0) return true;
  if (a.lengths == nullptr || a.next_positions == nullptr || a.out_lengths == nullptr || (a.block_table == nullptr && a.table_width > 0))
    return false;
  const uintptr_t in = reinterpret_cast<uintptr_t>(a.lengths), out = reinterpret_cast<uintptr_t>(a.out_lengths);
  const uintptr_t bytes = static_cast<uintptr_t>(a.rows) * 4;
  if (in < out + bytes && out < in + bytes) return false;
  return aligned(a.block_table, 4) && aligned(a.lengths, 4) && aligned(a.next_positions, 8) && aligned(a.out_lengths, 4) &&
         aligned(a.workspace, 16);
}

int evict_bound(const ResidentKvEvict& a) {
  return static_cast<int>(std::min<int64_t>(a.max_length, static_cast<int64_t>(a.table_width) * a.cache.block_size));
}

int64_t evict_bytes(const ResidentKvEvict& a) {
  return evict_bound(a) <= a.budget ? 0 : static_cast<int64_t>(a.rows) * a.cache.kv_heads * 2 * a.budget * 4;
}

}  // namespace
}  // namespace re

extern "C" int64_t resident_kv_evict_workspace(const ResidentKvEvict* args) {
  return args != nullptr && re::evict_ok(*args) ? re::evict_bytes(*args) : -1;
}

extern "C" int32_t resident_kv_evict(const ResidentKvEvict* args, void* stream) {
  using namespace re;
  if (args == nullptr || !evict_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  const int64_t need = evict_bytes(*args);
  if (need > 0 && (args->workspace == nullptr || args->workspace_bytes < need)) return -1;
  const DeviceScope device(args->cache.device);
  if (!device.ok()) return -2;
  const EvictArgs a{*args, evict_bound(*args), static_cast<int32_t*>(args->workspace)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_evict<bf16_t>(a, s) : launch_evict<float>(a, s);
  return e == hipSuccess ? 0 : -2;
}
