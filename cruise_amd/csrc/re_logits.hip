// Penalties, biases and a grammar mask on a step's logits, and the greedy token.
#include "re_ops.h"

// Every step of the formula is rounded by itself, so a product and a sum are
// never made one.
#pragma clang fp contract(off)

namespace re {
namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsIds = 4096;  // vocabulary ids of one workgroup
constexpr uint32_t kSeen = 0x80000000u;

struct LogitsArgs {
  ResidentLogits a;
  int parts;       // workgroups of a row
  uint64_t* best;  // [rows][parts]
};

// A logit and its id as one number whose maximum is the greatest logit's lowest
// id; NaN above all.
__device__ __forceinline__ uint64_t choice_key(float x, int id) {
  const uint32_t bits = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t order = x != x ? 0xffffffffu : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return static_cast<uint64_t>(order) << 32 | static_cast<uint32_t>(~id);
}
constexpr uint32_t kOrderNegInf = 0x007fffffu, kOrderPosInf = 0xff800000u;

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(v >> 32), m, 64)) << 32 |
                       static_cast<uint32_t>(__shfl_xor(static_cast<uint32_t>(v), m, 64));
    v = o > v ? o : v;
  }
  return v;
}

// One workgroup per (row, 4,096 ids): what the history and the biases say of
// those ids is gathered in LDS (a count with a bit for "seen", the last bias's
// number), then the logits pass once.
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) k_logits(LogitsArgs args) {
  const ResidentLogits& a = args.a;
  __shared__ uint32_t count[kLogitsIds], bias[kLogitsIds];
  __shared__ uint64_t best_s[kLogitsThreads / 64];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / args.parts, part = blockIdx.x % args.parts;
  const int first = part * kLogitsIds, ids = min(kLogitsIds, a.vocab - first);
  for (int i = tid; i < kLogitsIds; i += kLogitsThreads) count[i] = bias[i] = 0;
  __syncthreads();
  if (a.history != nullptr) {
    const int n = max(0, min(a.history_lengths[row], a.history_width));
    const int prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
    for (int i = tid; i < n; i += kLogitsThreads) {
      const int64_t id = a.history[row * a.history_stride + i] - first;
      if (id < 0 || id >= ids) continue;
      atomicOr(&count[id], kSeen);
      if (i >= prompt) atomicAdd(&count[id], 1u);
    }
  }
  if (a.bias_ids != nullptr) {
    for (int i = tid; i < a.biases; i += kLogitsThreads) {
      const int64_t id = a.bias_ids[row * a.bias_id_stride + i] - first;
      if (id >= 0 && id < ids) atomicMax(&bias[id], static_cast<uint32_t>(i) + 1);
    }
  }
  __syncthreads();
  const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
  const float presence = a.presence != nullptr ? a.presence[row] : 0.f;
  const float frequency = a.frequency != nullptr ? a.frequency[row] : 0.f;
  uint64_t best = 0;
  for (int i = tid; i < ids; i += kLogitsThreads) {
    const int id = first + i;
    float x = Elt<T>::f(static_cast<const T*>(a.logits)[row * a.logits_stride + id]);
    const uint32_t seen = count[i];
    if (seen != 0) {
      x = x > 0.f ? x / rep : x * rep;
      if ((seen & ~kSeen) != 0) x = x - frequency * static_cast<float>(seen & ~kSeen) - presence;
    }
    if (bias[i] != 0) x += a.bias_values[row * a.bias_value_stride + bias[i] - 1];
    if (a.allowed != nullptr && (a.allowed[row * a.allowed_stride + (id >> 5)] >> (id & 31) & 1) == 0) x = -INFINITY;
    if (a.out != nullptr) a.out[row * a.out_stride + id] = x;
    const uint64_t key = choice_key(x, id);
    best = key > best ? key : best;
  }
  if (a.tokens == nullptr) return;
  best = wave_max_u64(best);
  if ((tid & 63) == 0) best_s[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLogitsThreads / 64; ++w) best = best_s[w] > best ? best_s[w] : best;
    args.best[blockIdx.x] = best;
  }
}

// The row's choice among its workgroups': one wave per row.
__global__ void __launch_bounds__(64) k_logits_choose(LogitsArgs args) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < args.parts; i += 64) {
    const uint64_t v = args.best[static_cast<int64_t>(blockIdx.x) * args.parts + i];
    best = v > best ? v : best;
  }
  best = wave_max_u64(best);
  const uint32_t order = static_cast<uint32_t>(best >> 32);
  if (threadIdx.x == 0)
    args.a.tokens[blockIdx.x] = order > kOrderNegInf && order < kOrderPosInf ? static_cast<int64_t>(~static_cast<uint32_t>(best)) : -1;
}

int logits_parts(const ResidentLogits& a) { return static_cast<int>(ceil_div(a.vocab, kLogitsIds)); }
int64_t logits_bytes(const ResidentLogits& a) {
  return a.tokens == nullptr ? 0 : static_cast<int64_t>(a.rows) * logits_parts(a) * 8;
}

bool logits_ok(const ResidentLogits& a) {
  if (a.rows < 0 || a.vocab <= 0 || a.history_width < 0 || a.biases < 0 || (a.dtype_bytes != 2 && a.dtype_bytes != 4) ||
      a.workspace_bytes < 0)
    return false;
  if (a.logits_stride < 0 || a.out_stride < 0 || a.history_stride < 0 || a.bias_id_stride < 0 || a.bias_value_stride < 0 ||
      a.allowed_stride < 0)
    return false;
  if (static_cast<int64_t>(a.rows) * logits_parts(a) > (1 << 23)) return false;  // launches stay below 2^32 threads
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
  hipError_t e = launch(args->dtype_bytes == 2 ? k_logits<bf16_t> : k_logits<float>, static_cast<int64_t>(a.a.rows) * a.parts,
                        kLogitsThreads, 0, s, a);
  if (e == hipSuccess && args->tokens != nullptr) e = launch(k_logits_choose, args->rows, 64, 0, s, a);
  return e == hipSuccess ? 0 : -2;
}
