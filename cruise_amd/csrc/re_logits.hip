// Penalties, biases and a grammar mask on a step's logits, and the greedy token.
#include "re_ops.h"

// Every step of the formula is rounded by itself, so a product and a sum are
// never made one.
#pragma clang fp contract(off)

namespace re {
namespace {

// What LDS holds of an id: whether it was seen, whether it has a bias, and how
// often it was generated.
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u;
constexpr int kMostEntries = (1 << 30) - 1;  // of a row's history, and of its biases
// How the biases of a row are found again when an id passes: a few are listed
// and the ids that have one are marked; for more, every id has room for a number.
// (64 rows of 152,064 ids, 16 biases: 21.9 us listed, 25.0 numbered, which
// doubles the LDS.)
enum Biases { kNoBias, kListedBias, kNumberedBias };
constexpr int kListed = 64;
constexpr int kIdsOfThread = 16;  // vocabulary ids of a thread, in groups of four
constexpr int kChooseThreads = 256;

struct LogitsArgs {
  ResidentLogits a;
  int parts;       // workgroups of a row
  uint64_t* best;  // [rows][parts], if there are several
};

// Four neighbouring elements of a row that may begin at any element.
template <typename T>
struct Four;
template <>
struct Four<float> {
  typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
  __device__ __forceinline__ static re_f32x4 load(const float* p) { return *reinterpret_cast<const Vec*>(p); }
  __device__ __forceinline__ static void store(float* p, re_f32x4 v) { __builtin_nontemporal_store(static_cast<Vec>(v), reinterpret_cast<Vec*>(p)); }
};
template <>
struct Four<bf16_t> {
  typedef uint16_t Vec __attribute__((ext_vector_type(4), aligned(2)));
  __device__ __forceinline__ static re_f32x4 load(const bf16_t* p) {
    const Vec v = *reinterpret_cast<const Vec*>(p);
    return re_f32x4{bf16_to_f(v[0]), bf16_to_f(v[1]), bf16_to_f(v[2]), bf16_to_f(v[3])};
  }
};

// A logit's place in the order of choices: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t choice_order(float x) {
  const uint32_t bits = __float_as_uint(x == 0.f ? 0.f : x);
  return x != x ? 0xffffffffu : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
constexpr uint32_t kOrderNegInf = 0x007fffffu, kOrderPosInf = 0xff800000u;
// With the id, as one number whose maximum is the greatest logit's lowest id.
__device__ __forceinline__ uint64_t choice_key(uint32_t order, int id) {
  return static_cast<uint64_t>(order) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ int64_t choice_of(uint64_t key) {
  const uint32_t order = static_cast<uint32_t>(key >> 32);
  return order > kOrderNegInf && order < kOrderPosInf ? static_cast<int64_t>(~static_cast<uint32_t>(key)) : -1;
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(v >> 32), m, 64)) << 32 |
                       static_cast<uint32_t>(__shfl_xor(static_cast<uint32_t>(v), m, 64));
    v = o > v ? o : v;
  }
  return v;
}

// The logits pass once, and HBM bounds that (64 rows of 152,064 in fp32 with a
// mask and no history to speak of, 79 MB in and out: 19.4 us, 4.1 TB/s); what the
// history and the biases say of an id has to be known when its logit passes.  So
// a workgroup owns THREADS * 16 ids of a row, requests their logits and mask bits
// first, and gathers what its ids need in LDS while those are on the way.  Every workgroup of a row reads
// the whole history (from L2, but for the first).
template <typename T, int THREADS, Biases BIAS>
__global__ void __launch_bounds__(THREADS) k_logits(LogitsArgs args) {
  constexpr int kIds = THREADS * kIdsOfThread, kGroups = kIdsOfThread / 4;
  const ResidentLogits& a = args.a;
  __shared__ __align__(16) uint32_t count[kIds], bias[BIAS == kNumberedBias ? kIds : 4];
  __shared__ int listed_id[kListed];
  __shared__ float listed_value[kListed];
  __shared__ uint64_t best_s[THREADS / 64];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / args.parts, part = blockIdx.x % args.parts;
  const int first = part * kIds, ids = min(kIds, a.vocab - first);
  const T* logits = static_cast<const T*>(a.logits) + row * a.logits_stride + first;

  re_f32x4 x[kGroups];
  uint32_t allowed[kGroups];
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    const int i = (q * THREADS + tid) * 4;
    allowed[q] = 0xffffffffu;
    x[q] = re_f32x4{};
    if (i + 4 <= ids) {
      x[q] = Four<T>::load(logits + i);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (i + e < ids) x[q][e] = Elt<T>::f(logits[i + e]);
    }
    if (a.allowed != nullptr && i < ids) allowed[q] = a.allowed[row * a.allowed_stride + ((first + i) >> 5)] >> ((first + i) & 31);
  }
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    *reinterpret_cast<re_u32x4*>(&count[(q * THREADS + tid) * 4]) = re_u32x4{};
    if constexpr (BIAS == kNumberedBias) *reinterpret_cast<re_u32x4*>(&bias[(q * THREADS + tid) * 4]) = re_u32x4{};
  }
  lds_barrier();
  if (a.history != nullptr) {
    const int n = max(0, min(a.history_lengths[row], a.history_width));
    const int prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
    const int64_t* history = a.history + row * a.history_stride;
    constexpr int kAhead = 4;
    for (int i0 = tid; i0 < n; i0 += kAhead * THREADS) {
      int64_t id[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) id[u] = history[min(i0 + u * THREADS, n - 1)] - first;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * THREADS;
        if (i >= n || id[u] < 0 || id[u] >= ids) continue;
        if (i < prompt) atomicOr(&count[id[u]], kSeen);
        else atomicAdd(&count[id[u]], 1u);
      }
    }
  }
  if constexpr (BIAS != kNoBias) {
    for (int i = tid; i < a.biases; i += THREADS) {
      const int64_t id = a.bias_ids[row * a.bias_id_stride + i] - first;
      const bool mine = id >= 0 && id < ids;
      if constexpr (BIAS == kListedBias) {
        listed_id[i] = mine ? static_cast<int>(id) : -1;
        listed_value[i] = a.bias_values[row * a.bias_value_stride + i];
        if (mine) atomicOr(&count[id], kBiased);
      } else {
        if (mine) atomicMax(&bias[id], static_cast<uint32_t>(i) + 1);
      }
    }
  }
  lds_barrier();
  const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
  const float presence = a.presence != nullptr ? a.presence[row] : 0.f;
  const float frequency = a.frequency != nullptr ? a.frequency[row] : 0.f;
  uint32_t best = 0;
  int best_id = 0;
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    const int i = (q * THREADS + tid) * 4;
    const re_u32x4 seen = *reinterpret_cast<const re_u32x4*>(&count[i]);
    re_u32x4 biased = {};
    if constexpr (BIAS == kNumberedBias) biased = *reinterpret_cast<const re_u32x4*>(&bias[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = x[q][e];
      const uint32_t c = seen[e], made = c & ~(kSeen | kBiased);
      if ((c & ~kBiased) != 0) {
        v = v > 0.f ? v / rep : v * rep;
        if (made != 0) v = v - frequency * static_cast<float>(made) - presence;
      }
      if constexpr (BIAS == kListedBias) {
        if ((c & kBiased) != 0) {
          int number = a.biases - 1;  // the last one counts, and there is one
          while (number > 0 && listed_id[number] != i + e) --number;
          v = v + listed_value[number];
        }
      }
      if constexpr (BIAS == kNumberedBias) {
        const uint32_t number = biased[e];
        if (number != 0) v = v + a.bias_values[row * a.bias_value_stride + number - 1];
      }
      if ((allowed[q] >> e & 1) == 0) v = -INFINITY;
      x[q][e] = v;
      const uint32_t order = choice_order(v);
      if (order > best && i + e < ids) {  // ids rise along the loops, so equals keep the lower one
        best = order;
        best_id = first + i + e;
      }
    }
    if (a.out == nullptr) continue;
    float* out = a.out + row * a.out_stride + first + i;
    if (i + 4 <= ids) {
      Four<float>::store(out, x[q]);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (i + e < ids) out[e] = x[q][e];
    }
  }
  if (a.tokens == nullptr) return;
  uint64_t key = wave_max_u64(choice_key(best, best_id));
  if ((tid & 63) == 0) best_s[tid >> 6] = key;
  lds_barrier();
  if (tid != 0) return;
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) key = best_s[w] > key ? best_s[w] : key;
  if (args.parts > 1) args.best[blockIdx.x] = key;
  else a.tokens[row] = choice_of(key);
}

// The row's choice among its workgroups': one wave per row.
__global__ void __launch_bounds__(kChooseThreads) k_logits_choose(LogitsArgs args) {
  const int row = blockIdx.x * (kChooseThreads / 64) + wave_index(threadIdx.x), lane = threadIdx.x & 63;
  if (row >= args.a.rows) return;
  uint64_t best = 0;
  for (int i = lane; i < args.parts; i += 64) {
    const uint64_t v = args.best[static_cast<int64_t>(row) * args.parts + i];
    best = v > best ? v : best;
  }
  best = wave_max_u64(best);
  if (lane == 0) args.a.tokens[row] = choice_of(best);
}

// Threads of a workgroup, sixteen ids each.  Long histories want few workgroups
// of a row, since each reads all of it, short ones many (152,064 ids, 256 and 512
// threads: 64 rows with histories of 8,192 30.4 and 26.7 us, 4 rows 11.3 and 10.1;
// 16 rows with 1,024 11.9 and 12.4, 4 rows with 256 8.2 and 8.5).
int logits_threads(const ResidentLogits& a) { return a.history != nullptr && a.history_width >= 2048 ? 512 : 256; }
int logits_parts(const ResidentLogits& a) { return static_cast<int>(ceil_div(a.vocab, logits_threads(a) * kIdsOfThread)); }
int64_t logits_bytes(const ResidentLogits& a) {
  const int parts = logits_parts(a);
  return a.tokens == nullptr || parts == 1 ? 0 : static_cast<int64_t>(a.rows) * parts * 8;
}

template <typename T>
hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
  const int threads = logits_threads(a.a);
  const int biases = a.a.bias_ids != nullptr ? a.a.biases : 0;
  const auto kernel = threads == 256
                          ? (biases == 0 ? k_logits<T, 256, kNoBias> : biases <= kListed ? k_logits<T, 256, kListedBias>
                                                                                        : k_logits<T, 256, kNumberedBias>)
                          : (biases == 0 ? k_logits<T, 512, kNoBias> : biases <= kListed ? k_logits<T, 512, kListedBias>
                                                                                        : k_logits<T, 512, kNumberedBias>);
  hipError_t e = launch(kernel, static_cast<int64_t>(a.a.rows) * a.parts, threads, 0, stream, a);
  if (e == hipSuccess && a.a.tokens != nullptr && a.parts > 1)
    e = launch(k_logits_choose, ceil_div(a.a.rows, kChooseThreads / 64), kChooseThreads, 0, stream, a);
  return e;
}

bool logits_ok(const ResidentLogits& a) {
  if (a.rows < 0 || a.vocab <= 0 || a.history_width < 0 || a.history_width > kMostEntries || a.biases < 0 || a.biases > kMostEntries || (a.dtype_bytes != 2 && a.dtype_bytes != 4) ||
      a.workspace_bytes < 0)
    return false;
  if (a.logits_stride < 0 || a.out_stride < 0 || a.history_stride < 0 || a.bias_id_stride < 0 || a.bias_value_stride < 0 ||
      a.allowed_stride < 0)
    return false;
  if (static_cast<int64_t>(a.rows) * logits_parts(a) > (1 << 21)) return false;  // launches stay below 2^32 threads
  if (a.rows == 0) return true;
  if (a.logits == nullptr || (a.out == nullptr && a.tokens == nullptr) || (a.history != nullptr && a.history_lengths == nullptr) ||
      (a.bias_ids != nullptr && a.bias_values == nullptr))
    return false;
  // The output is the logits themselves or apart from them.
  if (a.out != nullptr) {
    const uintptr_t in = reinterpret_cast<uintptr_t>(a.logits), out = reinterpret_cast<uintptr_t>(a.out);
    const uintptr_t in_bytes = (static_cast<uintptr_t>(a.rows - 1) * a.logits_stride + a.vocab) * a.dtype_bytes;
    const uintptr_t out_bytes = (static_cast<uintptr_t>(a.rows - 1) * a.out_stride + a.vocab) * 4;
    const bool same = in == out && a.dtype_bytes == 4 && (a.logits_stride == a.out_stride || a.rows == 1);
    if (!same && in < out + out_bytes && out < in + in_bytes) return false;
    if (a.rows > 1 && a.out_stride < a.vocab) return false;
  }
  return aligned(a.logits, a.dtype_bytes) && aligned(a.out, 4) && aligned(a.tokens, 8) && aligned(a.history, 8) &&
         aligned(a.history_lengths, 4) && aligned(a.prompt_lengths, 4) && aligned(a.repetition, 4) && aligned(a.presence, 4) &&
         aligned(a.frequency, 4) && aligned(a.bias_ids, 8) && aligned(a.bias_values, 4) && aligned(a.allowed, 4) && aligned(a.workspace, 16);
}

}  // namespace
}  // namespace re

extern "C" int64_t resident_logits_process_workspace(const ResidentLogits* args) {
  return args != nullptr && re::logits_ok(*args) ? re::logits_bytes(*args) : -1;
}

extern "C" int32_t resident_logits_process(const ResidentLogits* args, void* stream) {
  using namespace re;
  if (args == nullptr || !logits_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  const int64_t need = logits_bytes(*args);
  if (need > 0 && (args->workspace == nullptr || args->workspace_bytes < need)) return -1;
  const DeviceScope device(args->device);
  if (!device.ok()) return -2;
  const LogitsArgs a{*args, logits_parts(*args), static_cast<uint64_t*>(args->workspace)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->dtype_bytes == 2 ? launch_logits<bf16_t>(a, s) : launch_logits<float>(a, s);
  return e == hipSuccess ? 0 : -2;
}
