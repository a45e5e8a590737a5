// Eviction from a paged cache by the attention weight that its slots gathered.
//
// Weights and positions are read once (8 bytes a slot), and of keys and values
// only those slots move that are kept but lie behind the budget: attention over
// rotated keys does not depend on the slots' order, so every slot that stays
// below the budget keeps its place.  Sources lie behind the budget and
// destinations below it, so the moves are independent of one another.
//   select  one workgroup per (row, KV head): every slot's key (its order as a
//           number) goes to LDS, the budget-th greatest one is found by
//           histograms of 2,048 bins between the least and the greatest key
//           left, and the slots to fill and to take from are listed in order;
//           a few moves (a page or two over the budget) are made right here,
//   move    a second launch over all of the chip for more of them.
#include <type_traits>

#include "re_ops.h"

namespace re {
namespace {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kBins = 2 * kEvictThreads;
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;  // rows of one lane group in flight
// Moves that the selecting workgroup makes itself: up to here they take it less
// time than a second launch.
constexpr int kOwnMoves = 256;

struct EvictArgs {
  ResidentKvEvict a;
  int bound;       // slots that a row can have
  int moves;       // that a (row, KV head) can have
  int pieces;      // workgroups of a (row, KV head) in the second launch; 0: none
  int32_t* lists;  // [rows][kv_heads][1 + 2 moves], for a second launch: how many (-1: the row stays as it is), slots
                   // to fill, slots to take from, last one first
};

struct SlotAddress {
  int page, at;
};
// A slot from a list.  Rows of a call that another call changes at the same time
// (or that share pages) may list anything, but reach no address outside the row.
__device__ __forceinline__ int listed_slot(int32_t j, int n) { return static_cast<int>(min(static_cast<unsigned>(j), static_cast<unsigned>(n - 1))); }

__device__ __forceinline__ SlotAddress slot_address(const int32_t* table, int block_size, int j) {
  const int p = static_cast<int>(static_cast<unsigned>(j) / static_cast<unsigned>(block_size));
  return {table[p], j - p * block_size};
}

// The order in which slots are kept, as a number: protected slots above all,
// then NaN, then the weights by value (-0 as 0).  No number gets 0.  Protected
// are the positions in [0, sinks) and in [recent_from, 2^31).
constexpr uint32_t kProtected = 0xffffffffu;
__device__ __forceinline__ uint32_t keep_key(float weight, int position, uint32_t recent_from, int sinks) {
  const uint32_t p = static_cast<uint32_t>(position), bits = __float_as_uint(weight + 0.f);
  uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
  key = weight != weight ? 0xfffffffeu : key;
  return p < static_cast<uint32_t>(sinks) || p - recent_from < 0x80000000u - recent_from ? kProtected : key;
}

// One value over the wave, by an operation on pairs: lane exchanges inside rows
// of 16, then across them.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_move_bits(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
template <typename Op>
__device__ __forceinline__ uint32_t wave_join(uint32_t v, Op op) {
  v = op(v, dpp_move_bits<kDppQuadXor1>(v));
  v = op(v, dpp_move_bits<kDppQuadXor2>(v));
  v = op(v, dpp_move_bits<kDppRowHalfMirror>(v));
  v = op(v, dpp_move_bits<kDppRowMirror>(v));
  const auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = op(x[0], x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return op(y[0], y[1]);
}
// Set bits of a wave's mask below this lane.
__device__ __forceinline__ int bits_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}
// The waves' values before wave w, added up.
__device__ __forceinline__ int sum_before(const int* values, int w) {
  int sum = 0;
#pragma unroll
  for (int x = 0; x < kEvictWaves; ++x) sum += x < w ? values[x] : 0;
  return sum;
}

template <typename T, int D>
struct Rows {
  static constexpr int kLanes = D * sizeof(T) / 16;  // 16 bytes each
  const ResidentKvCache& c;
  const int32_t* table;
  int g, e;  // KV head, first byte's element of this lane

  __device__ __forceinline__ Rows(const ResidentKvCache& cache, const int32_t* t, int head, int tid)
      : c(cache), table(t), g(head), e(tid % kLanes * (16 / static_cast<int>(sizeof(T)))) {}
  __device__ __forceinline__ void load(int j, re_u32x4& k, re_u32x4& v) const {
    const SlotAddress s = slot_address(table, c.block_size, j);
    k = *reinterpret_cast<const re_u32x4*>(static_cast<const T*>(c.keys) + s.page * c.key_strides[0] + s.at * c.key_strides[1] +
                                           g * c.key_strides[2] + e);
    v = *reinterpret_cast<const re_u32x4*>(static_cast<const T*>(c.values) + s.page * c.value_strides[0] + s.at * c.value_strides[1] +
                                           g * c.value_strides[2] + e);
  }
  __device__ __forceinline__ void store(int j, re_u32x4 k, re_u32x4 v) const {
    const SlotAddress s = slot_address(table, c.block_size, j);
    *reinterpret_cast<re_u32x4*>(static_cast<T*>(c.keys) + s.page * c.key_strides[0] + s.at * c.key_strides[1] + g * c.key_strides[2] + e) = k;
    *reinterpret_cast<re_u32x4*>(static_cast<T*>(c.values) + s.page * c.value_strides[0] + s.at * c.value_strides[1] +
                                 g * c.value_strides[2] + e) = v;
  }
};

// Moves i0, i0 + step, ... below `moves` of the lists, UNROLL of them in flight
// (the slots to take from are listed last one first).
template <int UNROLL, typename R>
__device__ __forceinline__ void move_rows(const R& rows, const int32_t* fill, const int32_t* take, int moves, int n, int i0, int step) {
  for (int i = i0; i < moves; i += UNROLL * step) {
    re_u32x4 k[UNROLL], v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * step < moves) rows.load(listed_slot(take[moves - 1 - i - u * step], n), k[u], v[u]);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * step < moves) rows.store(listed_slot(fill[i + u * step], n), k[u], v[u]);
  }
}

// Slots j, j + step, ... below n hold nothing any more.
__device__ __forceinline__ void clear_slots(const ResidentKvCache& c, const int32_t* table, int g, int j, int n, int step) {
  for (; j < n; j += step) {
    const SlotAddress s = slot_address(table, c.block_size, j);
    c.weights[s.page * c.weight_strides[0] + g * c.weight_strides[1] + s.at] = 0.f;
    c.positions[s.page * c.position_strides[0] + g * c.position_strides[1] + s.at] = -1;
  }
}

// KEYS: slots whose keys LDS holds; LONGER: rows may have more, whose keys are
// made again from memory in every pass.
template <typename T, int D, int KEYS, bool LONGER>
__global__ void __launch_bounds__(kEvictThreads) k_kv_evict(EvictArgs args) {
  const ResidentKvEvict& a = args.a;
  const ResidentKvCache& c = a.cache;
  __shared__ uint32_t keys_s[KEYS], bins[kBins];
  __shared__ uint32_t least_s[kEvictWaves], most_s[kEvictWaves];
  __shared__ int count_s[kEvictWaves], other_s[kEvictWaves], found_s[3], moves_s;
  __shared__ int32_t fill_s[kOwnMoves], take_s[kOwnMoves];
  const int tid = threadIdx.x, lane = tid & 63, w = wave_index(tid);
  const int row = blockIdx.x / c.kv_heads, g = blockIdx.x % c.kv_heads, budget = a.budget;
  const int n = cut_length(a.lengths, row, args.bound);
  const int32_t* table = a.block_table + row * a.table_stride;
  int32_t* list = args.lists + static_cast<int64_t>(blockIdx.x) * (1 + 2 * static_cast<int64_t>(args.moves));
  if (n <= budget) {
    if (tid == 0) {
      if (g == 0) a.out_lengths[row] = n;
      if (args.pieces > 0) list[0] = -1;
    }
    return;
  }
  float* weights = c.weights + g * c.weight_strides[1];
  int32_t* positions = c.positions + g * c.position_strides[1];
  const uint32_t recent_from =
      static_cast<uint32_t>(max(INT64_C(0), min(a.next_positions[row] - a.recent, INT64_C(0x80000000))));
  auto key_of = [&](int j) {
    if (!LONGER || j < KEYS) return keys_s[j];
    const SlotAddress s = slot_address(table, c.block_size, j);
    return keep_key(weights[s.page * c.weight_strides[0] + s.at], positions[s.page * c.position_strides[0] + s.at], recent_from, a.sinks);
  };

  // Keys, how many slots are protected, and the range of the others' keys.
  int shield = 0, bad = 0;
  uint32_t least = kProtected, most = 0;  // most: one above the greatest
  // The thread's slots tid, tid + 1024, ..., kAhead of them requested together
  // (pages, then weights and positions).  ALIGNED: the 64 slots of a wave lie on
  // one page, so their address is the wave's; else every slot has its own.
  // Stepping the page and the offset along spares a division per slot.
  constexpr int kAhead = KEYS > 4096 ? 16 : 2;
  auto read_keys = [&](auto aligned) {
    constexpr bool ALIGNED = decltype(aligned)::value;
    const int first = ALIGNED ? w * 64 : tid, pages_on = kEvictThreads / c.block_size, slots_on = kEvictThreads % c.block_size;
    int p = first / c.block_size, at = first % c.block_size;
    const int last_page = (n - 1) / c.block_size;
    for (int j0 = 0; j0 < n; j0 += kAhead * kEvictThreads) {
      int page[kAhead], offset[kAhead];
      float weight[kAhead];
      int position[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        // behind the row: its last page, whose slots are all there to read
        page[u] = table[min(p, last_page)];
        offset[u] = at;
        p += pages_on;
        at += slots_on;
        if (at >= c.block_size) {
          at -= c.block_size;
          ++p;
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if constexpr (ALIGNED) page[u] = __builtin_amdgcn_readfirstlane(page[u]);
        const bool there = page[u] >= 0 && page[u] < c.pages;
        bad |= !there;
        page[u] = there ? page[u] : 0;
        const int more = ALIGNED ? lane : 0;
        weight[u] = (weights + page[u] * c.weight_strides[0] + offset[u])[more];
        position[u] = (positions + page[u] * c.position_strides[0] + offset[u])[more];
      }
      auto take_keys = [&](auto whole) {  // whole: all of the batch lies in the row
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int j = j0 + u * kEvictThreads + tid;
          const uint32_t key = keep_key(weight[u], position[u], recent_from, a.sinks);
          if (!decltype(whole)::value && j >= n) continue;
          if (!LONGER || j < KEYS) keys_s[j] = key;
          shield += key == kProtected;
          least = min(least, key);
          most = max(most, key + 1);  // of the unprotected ones: the greatest key wraps to 0
        }
      };
      if (j0 + kAhead * kEvictThreads <= n) take_keys(std::true_type{});
      else take_keys(std::false_type{});
    }
  };
  if (c.block_size % 64 == 0) read_keys(std::true_type{});
  else read_keys(std::false_type{});
  least = wave_join(least, [](uint32_t x, uint32_t y) { return min(x, y); });
  most = wave_join(most, [](uint32_t x, uint32_t y) { return max(x, y); });
  shield = wave_join(shield, [](uint32_t x, uint32_t y) { return x + y; });
  bad = __any(bad);
  if (lane == 0) {
    least_s[w] = least;
    most_s[w] = most;
    count_s[w] = shield;
    other_s[w] = bad;
  }
  __syncthreads();
  shield = bad = 0;
#pragma unroll
  for (int x = 0; x < kEvictWaves; ++x) {
    least = min(least, least_s[x]);
    most = max(most, most_s[x]);
    shield += count_s[x];
    bad |= other_s[x];
  }
  if (tid == 0) {
    if (g == 0) a.out_lengths[row] = bad ? n : budget;
    if (args.pieces > 0 && bad) list[0] = -1;
  }
  if (bad) return;

  constexpr int kTogether = 4;  // keys that a thread reads before it works on them

  // Kept: keys above `last`, and the `ties` lowest slots of those equal to it.
  uint32_t last = kProtected;
  int ties = budget;
  if (shield < budget) {
    int need = budget - shield;
    uint32_t low = least, high = most - 1;
    for (int pass = 0; pass < 3; ++pass) {  // 11 bits each
      const int width = 32 - __clz(high - low), shift = max(0, width - 11);  // 2,048 bins
      __syncthreads();
      bins[tid] = bins[tid + kEvictThreads] = 0;
      __syncthreads();
      for (int j0 = tid; j0 < n; j0 += kTogether * kEvictThreads) {
        uint32_t at[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) at[u] = (j0 + u * kEvictThreads < n ? key_of(j0 + u * kEvictThreads) : kProtected) - low;
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
          if (at[u] <= high - low) atomicAdd(&bins[at[u] >> shift], 1u);  // no protected key lies in the range
      }
      __syncthreads();
      // The bin, from the greatest down, in which the need is met.
      const int b = kBins - 1 - 2 * tid;
      const int upper = bins[b], lower = bins[b - 1];
      int sum = upper + lower;
      for (int m = 1; m < 64; m <<= 1) {
        const int v = __shfl_up(sum, m, 64);
        if (lane >= m) sum += v;
      }
      if (lane == 63) count_s[w] = sum;
      __syncthreads();
      sum += sum_before(count_s, w);
      const int before = sum - upper - lower;
      if (before < need && need <= sum) {
        const bool first = need <= before + upper;
        found_s[0] = first ? b : b - 1;
        found_s[1] = first ? before : before + upper;
        found_s[2] = first ? upper : lower;
      }
      __syncthreads();
      need -= found_s[1];
      low += static_cast<uint32_t>(found_s[0]) << shift;
      if (found_s[2] == need) {  // all of this bin
        last = low - 1;
        ties = 0;
        break;
      }
      last = low;
      ties = need;
      if (shift == 0) break;
      high = min(high, low + ((1u << shift) - 1));
    }
  }

  // Wave w goes over a run of slots: what it holds first, then every slot's rank.
  const int run = ((n + 63) / 64 + kEvictWaves - 1) / kEvictWaves * 64;
  const int from = min(n, w * run), to = min(n, from + run);
  int above = 0, equal = 0;
  for (int j0 = from + lane; j0 - lane < to; j0 += 64 * kTogether) {
    uint32_t key[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) key[u] = j0 + 64 * u < to ? key_of(j0 + 64 * u) : 0;  // no slot's key
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      above += __popcll(__ballot(key[u] > last));
      equal += __popcll(__ballot(key[u] == last));
    }
  }
  __syncthreads();
  if (lane == 0) {
    count_s[w] = above;
    other_s[w] = equal;
  }
  __syncthreads();
  above = sum_before(count_s, w);
  equal = sum_before(other_s, w);
  // The i-th slot to fill and the i-th last one to take from: in LDS where this
  // workgroup makes the moves itself (at most kOwnMoves).
  const bool own = args.pieces == 0;
  for (int j0 = from + lane; j0 - lane < to; j0 += 64 * kTogether) {
    uint32_t key[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) key[u] = j0 + 64 * u < to ? key_of(j0 + 64 * u) : 0;
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int j = j0 + 64 * u;
      const uint64_t gts = __ballot(key[u] > last), eqs = ties > 0 ? __ballot(key[u] == last) : 0;
      bool kept = key[u] > last;
      int rank = above + bits_below(gts);  // kept slots before j
      if (ties > 0) {
        const int equal_at = equal + bits_below(eqs);
        kept = kept || (key[u] == last && equal_at < ties);
        rank += min(equal_at, ties);
      }
      if (j < to && j == budget) moves_s = max(0, min(budget - rank, args.moves));
      above += __popcll(gts);
      equal += __popcll(eqs);
      if (j < to && kept != (j < budget)) {
        const int i = j < budget ? j - rank : budget - 1 - rank;
        if (i < 0 || i >= args.moves) continue;  // another call changes the weights meanwhile
        if (own) (j < budget ? fill_s : take_s)[i] = j;
        else list[(j < budget ? 1 : 1 + args.moves) + i] = j;
      }
    }
  }
  __syncthreads();
  const int moves = moves_s;
  const int32_t* fill = own ? fill_s : list + 1;
  const int32_t* take = own ? take_s : list + 1 + args.moves;
  if (own) {
    const Rows<T, D> rows(c, table, g, tid);
    move_rows<2>(rows, fill_s, take_s, moves, n, tid / rows.kLanes, kEvictThreads / rows.kLanes);
  } else if (tid == 0) {
    list[0] = moves;
  }
  for (int i0 = tid; i0 < moves; i0 += kMoveUnroll * kEvictThreads) {
    float weight[kMoveUnroll];
    int position[kMoveUnroll];
    SlotAddress dest[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = min(i0 + u * kEvictThreads, moves - 1);
      const SlotAddress source = slot_address(table, c.block_size, listed_slot(take[moves - 1 - i], n));
      dest[u] = slot_address(table, c.block_size, listed_slot(fill[i], n));
      weight[u] = weights[source.page * c.weight_strides[0] + source.at];
      position[u] = positions[source.page * c.position_strides[0] + source.at];
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      if (i0 + u * kEvictThreads >= moves) break;
      weights[dest[u].page * c.weight_strides[0] + dest[u].at] = weight[u];
      positions[dest[u].page * c.position_strides[0] + dest[u].at] = position[u];
    }
  }
  if (args.pieces > 0) return;
  __syncthreads();  // the sources are read before they are cleared
  clear_slots(c, table, g, budget + tid, n, kEvictThreads);
}

// The moves of the keys and values, and the slots behind the budget.  Whether a
// row moves anything or not, it has slots to clear exactly if it was selected
// from: its list says so.
template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) k_kv_evict_move(EvictArgs args) {
  const ResidentKvEvict& a = args.a;
  const ResidentKvCache& c = a.cache;
  const int pair = blockIdx.x / args.pieces, piece = blockIdx.x % args.pieces, row = pair / c.kv_heads, g = pair % c.kv_heads;
  const int32_t* list = args.lists + static_cast<int64_t>(pair) * (1 + 2 * static_cast<int64_t>(args.moves));
  const int moves = list[0];
  if (moves < 0) return;
  const int32_t* table = a.block_table + row * a.table_stride;
  const Rows<T, D> rows(c, table, g, threadIdx.x);
  constexpr int kGroups = kMoveThreads / Rows<T, D>::kLanes;
  const int n = cut_length(a.lengths, row, args.bound);
  move_rows<kMoveUnroll>(rows, list + 1, list + 1 + args.moves, moves, n, piece * kGroups + threadIdx.x / rows.kLanes,
                         args.pieces * kGroups);
  clear_slots(c, table, g, a.budget + piece * kMoveThreads + threadIdx.x, n, args.pieces * kMoveThreads);
}

int evict_bound(const ResidentKvEvict& a) {
  return static_cast<int>(std::min<int64_t>(a.max_length, static_cast<int64_t>(a.table_width) * a.cache.block_size));
}

template <typename T, int D>
hipError_t launch_evict(EvictArgs a, hipStream_t stream) {
  const ResidentKvCache& c = a.a.cache;
  const int64_t pairs = static_cast<int64_t>(a.a.rows) * c.kv_heads;
  constexpr int kPieceRows = kMoveUnroll * kMoveThreads / Rows<T, D>::kLanes;
  a.pieces = a.moves <= kOwnMoves ? 0 : static_cast<int>(std::clamp<int64_t>((1 << 22) / pairs, 1, ceil_div(a.moves, kPieceRows)));
  hipError_t e = launch(a.bound <= 4096    ? k_kv_evict<T, D, 4096, false>
                        : a.bound <= 32768 ? k_kv_evict<T, D, 32768, false>
                                           : k_kv_evict<T, D, 32768, true>,
                        pairs, kEvictThreads, 0, stream, a);
  if (e == hipSuccess && a.pieces > 0) e = launch(k_kv_evict_move<T, D>, pairs * a.pieces, kMoveThreads, 0, stream, a);
  return e;
}

template <typename T>
hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  const int d = a.a.cache.head_dim;
  return d == 64 ? launch_evict<T, 64>(a, stream) : d == 128 ? launch_evict<T, 128>(a, stream) : launch_evict<T, 256>(a, stream);
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

// What a (row, KV head) can move: the kept slots behind the budget.
int evict_moves(const ResidentKvEvict& a) { return std::max(0, std::min(a.budget, evict_bound(a) - a.budget)); }

int64_t evict_bytes(const ResidentKvEvict& a) {
  const int64_t moves = evict_moves(a);
  return moves <= kOwnMoves ? 0 : static_cast<int64_t>(a.rows) * a.cache.kv_heads * (1 + 2 * moves) * 4;
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
  const EvictArgs a{*args, evict_bound(*args), evict_moves(*args), 0, static_cast<int32_t*>(args->workspace)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_evict<bf16_t>(a, s) : launch_evict<float>(a, s);
  return e == hipSuccess ? 0 : -2;
}
