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
//   move    a launch over all of the chip for more of them,
//   keys    one before the selection for rows of more slots than LDS holds.
// The selection is a chain of passes with barriers between them, and its latency
// is what a small call costs: 11 us for 64 workgroups of 1,152 slots, of which
// reading takes 1.5, the histograms 2 to 3, ranks and lists 2, the moves 2.  8 rows
// of up to 32,768 slots cut to 4,096 take 30 us to select (the instructions of one
// CU for each row and KV head) and 24 to move (119 MB, 5 TB/s).
#include <type_traits>

#include "re_evict_select.h"
#include "re_ops.h"

namespace re {
namespace {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kBins = 2 * kEvictThreads;
static_assert(kBins == 1 << kBinBits, "two bins a thread");
constexpr int kMoveThreads = 256;
// Moves that the selecting workgroup makes itself: up to here they take it less
// time than a second launch (16 rows of 4 KV heads, 128 moves: 14.4 and 15.9 us,
// 512 moves: 19.9 and 20.9; 64 rows, 256 moves: 23.0 and 27.0).
constexpr int kOwnMoves = 512;

constexpr int kKeyThreads = 256, kKeySlots = 4096;
// Keys that the selecting workgroup holds in LDS: 16 KB, so that two share a CU
// and a short row asks for no more than it has, or 128 (16 rows of 1,152 slots:
// 14.4 and 15.7 us, 128 rows 28.0 and 30.4).
constexpr int kShortKeys = 4096, kLongKeys = 32768;

struct KeyStats {
  uint32_t least, most;  // of unprotected keys, the greatest plus one
  int shield, bad;       // protected slots; whether a page is not there
};

struct EvictArgs {
  ResidentKvEvict a;
  int bound;       // slots that a row can have
  int moves;       // that a (row, KV head) can have
  int pieces;      // workgroups of a (row, KV head) in the second launch; 0: none
  int key_pieces;  // workgroups of a (row, KV head) that make keys ahead; 0: the selecting one does
  uint32_t* keys;  // [rows][kv_heads][key_pieces * kKeySlots]
  KeyStats* key_stats;  // [rows][kv_heads][key_pieces]
  int32_t* lists;  // [rows][kv_heads][1 + 2 moves], for a second launch: how many (-1: the row stays as it is), slots
                   // to fill, slots to take from, last one first
};

struct SlotAddress {
  int page, at;
};
__device__ __forceinline__ SlotAddress slot_address(const int32_t* table, int block_size, int j) {
  const int p = static_cast<int>(static_cast<unsigned>(j) / static_cast<unsigned>(block_size));
  return {table[p], j - p * block_size};
}

// A slot's place in the order (re_evict_select.h).  Protected are the positions in
// [0, sinks) and in [recent_from, 2^31).
__device__ __forceinline__ uint32_t keep_key(float weight, int position, uint32_t recent_from, int sinks) {
  const uint32_t p = static_cast<uint32_t>(position);
  return p < static_cast<uint32_t>(sinks) || p - recent_from < 0x80000000u - recent_from ? kProtected : weight_key(weight);
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
    T* key = static_cast<T*>(c.keys) + s.page * c.key_strides[0] + s.at * c.key_strides[1] + g * c.key_strides[2] + e;
    T* value = static_cast<T*>(c.values) + s.page * c.value_strides[0] + s.at * c.value_strides[1] + g * c.value_strides[2] + e;
    __builtin_nontemporal_store(k, reinterpret_cast<re_u32x4*>(key));
    __builtin_nontemporal_store(v, reinterpret_cast<re_u32x4*>(value));
  }
};

// Moves i, i + step, ... below `moves` of the lists (the slots to take from are
// listed last one first).  One row at a time: two or four of a lane group in
// flight take longer (8 rows of 32,768 cut to 4,096: 74, 76 and 80 us).  The rows
// are not read again soon, and stores past the caches leave those to the others
// (71 us instead of 74).
template <typename R>
__device__ __forceinline__ void move_rows(const R& rows, const int32_t* fill, const int32_t* take, int moves, int i, int step) {
  for (; i < moves; i += step) {
    re_u32x4 k, v;
    rows.load(take[moves - 1 - i], k, v);
    rows.store(fill[i], k, v);
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

// W neighbouring values at any address.
template <typename V, int W>
struct Values {
  typedef V Vec __attribute__((ext_vector_type(W), aligned(4)));
  V v[W];
  __device__ __forceinline__ static Values load(const V* p) {
    Values r;
    if constexpr (W == 1) {
      r.v[0] = *p;
    } else {
      const Vec x = *reinterpret_cast<const Vec*>(p);
#pragma unroll
      for (int i = 0; i < W; ++i) r.v[i] = x[i];
    }
    return r;
  }
};

// The keys of a row's slots [begin, end) for one KV head: store(j, keys) takes W
// neighbours (the last ones may lie behind the end), the result is what this
// thread saw of the others.  Groups of W slots, which lie on one page, AHEAD of
// them requested together (pages, then weights and positions); stepping page and
// offset along spares a division per group, and a group of four, where pages hold
// whole ones, most of the address (8 rows of 32,768: 64 us, 73 slot by slot).
template <int THREADS, int AHEAD, int W, typename Store>
__device__ __forceinline__ KeyStats read_keys(const ResidentKvEvict& a, int row, int g, int n, int begin, int end, Store store) {
  const ResidentKvCache& c = a.cache;
  const int tid = threadIdx.x;
  const int32_t* table = a.block_table + row * a.table_stride;
  const float* weights = c.weights + g * c.weight_strides[1];
  const int32_t* positions = c.positions + g * c.position_strides[1];
  const uint32_t recent_from =
      static_cast<uint32_t>(max(INT64_C(0), min(max(INT64_C(0), a.next_positions[row]) - a.recent, INT64_C(0x80000000))));
  constexpr int kStep = THREADS * W;
  const int pages_on = kStep / c.block_size, slots_on = kStep % c.block_size;
  int p = (begin + tid * W) / c.block_size, at = (begin + tid * W) % c.block_size;
  const int last_page = (n - 1) / c.block_size;
  KeyStats seen{kProtected, 0, 0, 0};
  for (int j0 = begin; j0 < end; j0 += AHEAD * kStep) {
    int page[AHEAD], offset[AHEAD];
    Values<float, W> weight[AHEAD];
    Values<int32_t, W> position[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
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
    for (int u = 0; u < AHEAD; ++u) {
      const bool there = page[u] >= 0 && page[u] < c.pages;
      seen.bad |= !there;
      page[u] = there ? page[u] : 0;
      weight[u] = Values<float, W>::load(weights + page[u] * c.weight_strides[0] + offset[u]);
      position[u] = Values<int32_t, W>::load(positions + page[u] * c.position_strides[0] + offset[u]);
    }
    auto take = [&](auto whole) {  // whole: all of the batch lies in the range
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int j = j0 + u * kStep + tid * W;
        if (!decltype(whole)::value && j >= end) continue;
        uint32_t keys[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
          keys[i] = keep_key(weight[u].v[i], position[u].v[i], recent_from, a.sinks);
          if (!decltype(whole)::value && j + i >= end) continue;
          seen.shield += keys[i] == kProtected;
          seen.least = min(seen.least, keys[i]);
          seen.most = max(seen.most, keys[i] + 1);  // a protected key wraps to 0
        }
        store(j, keys);
      }
    };
    if (j0 + AHEAD * kStep <= end) take(std::true_type{});
    else take(std::false_type{});
  }
  return seen;
}

// W neighbouring keys to where they are kept, a multiple of W from its start.
template <int W>
__device__ __forceinline__ void store_keys(uint32_t* to, const uint32_t (&keys)[W]) {
  if constexpr (W == 1) *to = keys[0];
  else *reinterpret_cast<re_u32x4*>(to) = re_u32x4{keys[0], keys[1], keys[2], keys[3]};
}

// What the workgroup's threads saw, together.  Every thread gets it.
template <int WAVES>
__device__ __forceinline__ KeyStats join_stats(KeyStats s, KeyStats* waves, int lane, int w) {
  s.least = wave_join(s.least, [](uint32_t x, uint32_t y) { return min(x, y); });
  s.most = wave_join(s.most, [](uint32_t x, uint32_t y) { return max(x, y); });
  s.shield = wave_join(s.shield, [](uint32_t x, uint32_t y) { return x + y; });
  s.bad = __any(s.bad);
  if (lane == 0) waves[w] = s;
  __syncthreads();
  s = waves[0];
#pragma unroll
  for (int x = 1; x < WAVES; ++x) {
    s.least = min(s.least, waves[x].least);
    s.most = max(s.most, waves[x].most);
    s.shield += waves[x].shield;
    s.bad |= waves[x].bad;
  }
  return s;
}

// Keys ahead of the selection: one workgroup per (row, KV head, 4,096 slots).
template <int W>
__global__ void __launch_bounds__(kKeyThreads) k_kv_evict_keys(EvictArgs args) {
  const ResidentKvEvict& a = args.a;
  __shared__ KeyStats waves[kKeyThreads / 64];
  const int pair = blockIdx.x / args.key_pieces, piece = blockIdx.x % args.key_pieces, row = pair / a.cache.kv_heads;
  const int n = cut_length(a.lengths, row, args.bound), begin = piece * kKeySlots;
  if (n <= a.budget || begin >= n) return;
  uint32_t* keys = args.keys + static_cast<int64_t>(pair) * args.key_pieces * kKeySlots;
  const KeyStats seen =
      read_keys<kKeyThreads, kKeySlots / kKeyThreads / W, W>(a, row, pair % a.cache.kv_heads, n, begin, min(n, begin + kKeySlots),
                                                             [&](int j, const uint32_t (&k)[W]) { store_keys<W>(keys + j, k); });
  const KeyStats all = join_stats<kKeyThreads / 64>(seen, waves, threadIdx.x & 63, wave_index(threadIdx.x));
  if (threadIdx.x == 0) args.key_stats[blockIdx.x] = all;
}

// KEYS: slots whose keys LDS holds; AHEAD_OF: the keys were made by a launch
// before this one, and rows may have more of them than LDS holds.
template <typename T, int D, int KEYS, bool AHEAD_OF>
__global__ void __launch_bounds__(kEvictThreads) k_kv_evict(EvictArgs args) {
  const ResidentKvEvict& a = args.a;
  const ResidentKvCache& c = a.cache;
  __shared__ __align__(16) uint32_t keys_s[KEYS];
  __shared__ uint32_t bins[kBins];
  __shared__ KeyStats waves[kEvictWaves];
  __shared__ int count_s[kEvictWaves], other_s[kEvictWaves], found_s[3], moves_s;
  __shared__ int32_t lists_s[2 * kOwnMoves];
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
  const uint32_t* keys = AHEAD_OF ? args.keys + static_cast<int64_t>(blockIdx.x) * args.key_pieces * kKeySlots : nullptr;
  auto key_of = [&](int j) { return !AHEAD_OF || j < KEYS ? keys_s[j] : keys[j]; };

  // Keys, how many slots are protected, and the range of the others' keys.
  KeyStats seen{kProtected, 0, 0, 0};
  if constexpr (AHEAD_OF) {
    constexpr int kAhead = 8;
    for (int j0 = 4 * tid; j0 < min(n, KEYS); j0 += 4 * kAhead * kEvictThreads) {
      re_u32x4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = j0 + 4 * u * kEvictThreads;
        v[u] = *reinterpret_cast<const re_u32x4*>(keys + (j < n ? j : j0));  // pieces are whole: their ends may be read
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = j0 + 4 * u * kEvictThreads;
        if (j < min(n, KEYS)) *reinterpret_cast<re_u32x4*>(keys_s + j) = v[u];
      }
    }
    for (int i = tid; i < (n + kKeySlots - 1) / kKeySlots; i += kEvictThreads) {
      const KeyStats s = args.key_stats[static_cast<int64_t>(blockIdx.x) * args.key_pieces + i];
      seen = KeyStats{min(seen.least, s.least), max(seen.most, s.most), seen.shield + s.shield, seen.bad | s.bad};
    }
  } else {
    constexpr int kAhead = KEYS > kShortKeys ? 16 : 2, kFours = KEYS > kShortKeys ? 4 : 1;
    if (c.block_size % 4 == 0)
      seen = read_keys<kEvictThreads, kFours, 4>(a, row, g, n, 0, n, [&](int j, const uint32_t (&k)[4]) { store_keys<4>(keys_s + j, k); });
    else
      seen = read_keys<kEvictThreads, kAhead, 1>(a, row, g, n, 0, n, [&](int j, const uint32_t (&k)[1]) { store_keys<1>(keys_s + j, k); });
  }
  seen = join_stats<kEvictWaves>(seen, waves, lane, w);
  if (tid == 0) {
    if (g == 0) a.out_lengths[row] = seen.bad ? n : budget;
    if (args.pieces > 0 && seen.bad) list[0] = -1;
  }
  if (seen.bad) return;

  // Keys that a thread reads before it works on them: from LDS few, from memory
  // more.
  constexpr int kTogether = AHEAD_OF ? 16 : KEYS > kShortKeys ? 4 : 2;

  // Kept: keys above `last`, and the `ties` lowest slots of those equal to it.
  uint32_t last = kProtected;
  int ties = budget;
  if (seen.shield < budget) {
    int need = budget - seen.shield;
    KeyRange range{seen.least, seen.most - 1 - seen.least};
    for (int pass = 0; pass < 3; ++pass) {  // 11 bits each
      const int shift = range.shift();
      __syncthreads();
      bins[tid] = bins[tid + kEvictThreads] = 0;
      __syncthreads();
      for (int j0 = tid; j0 < n; j0 += kTogether * kEvictThreads) {
        uint32_t key[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) key[u] = j0 + u * kEvictThreads < n ? key_of(j0 + u * kEvictThreads) : kProtected;
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
          if (range.holds(key[u])) atomicAdd(&bins[range.bin(key[u], shift)], 1u);  // no protected key lies in the range
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
      range = range.part(static_cast<uint32_t>(found_s[0]), shift);
      if (found_s[2] == need) {  // all of this bin
        last = range.low - 1;
        ties = 0;
        break;
      }
      last = range.low;
      ties = need;
      if (shift == 0) break;
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
  const int kept_all = sum_before(count_s, kEvictWaves) + min(sum_before(other_s, kEvictWaves), ties);
  // The i-th slot to fill and the i-th last one to take from: in LDS where this
  // workgroup makes the moves itself (at most kOwnMoves).  Every entry that a move
  // reads was written, and none lies past the lists, whatever was selected.
  const bool own = args.pieces == 0;
  int32_t* lists_out = list + 1;
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
      if (j < to && j == budget) moves_s = moves_of(kept_all, rank, budget, args.moves);
      above += __popcll(gts);
      equal += __popcll(eqs);
      const uint32_t i = list_entry(j, rank, budget, args.moves);
      if (j < to && kept != (j < budget) && i < 2 * static_cast<uint32_t>(args.moves)) {
        if (own) lists_s[i] = j;
        else lists_out[i] = j;
      }
    }
  }
  __syncthreads();
  const int moves = moves_s;
  const int32_t* fill = own ? lists_s : lists_out;
  const int32_t* take = fill + args.moves;
  if (own) {
    const Rows<T, D> rows(c, table, g, tid);
    move_rows(rows, lists_s, lists_s + args.moves, moves, tid / rows.kLanes, kEvictThreads / rows.kLanes);
  } else if (tid == 0) {
    list[0] = moves;
  }
  for (int i = tid; i < moves; i += kEvictThreads) {
    const SlotAddress source = slot_address(table, c.block_size, take[moves - 1 - i]), dest = slot_address(table, c.block_size, fill[i]);
    weights[dest.page * c.weight_strides[0] + dest.at] = weights[source.page * c.weight_strides[0] + source.at];
    positions[dest.page * c.position_strides[0] + dest.at] = positions[source.page * c.position_strides[0] + source.at];
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
  move_rows(rows, list + 1, list + 1 + args.moves, moves, piece * kGroups + threadIdx.x / rows.kLanes, args.pieces * kGroups);
  clear_slots(c, table, g, a.budget + piece * kMoveThreads + threadIdx.x, n, args.pieces * kMoveThreads);
}

int evict_bound(const ResidentKvEvict& a) {
  return static_cast<int>(row_bound(a.max_length, a.table_width, a.cache.block_size));
}

template <typename T, int D>
hipError_t launch_evict(EvictArgs a, hipStream_t stream) {
  const ResidentKvCache& c = a.a.cache;
  const int64_t pairs = static_cast<int64_t>(a.a.rows) * c.kv_heads;
  constexpr int kPieceRows = kMoveThreads / Rows<T, D>::kLanes;
  a.pieces = a.moves <= kOwnMoves ? 0 : static_cast<int>(std::clamp<int64_t>((1 << 22) / pairs, 1, ceil_div(a.moves, kPieceRows)));
  hipError_t e = hipSuccess;
  if (a.key_pieces > 0)
    e = launch(c.block_size % 4 == 0 ? k_kv_evict_keys<4> : k_kv_evict_keys<1>, pairs * a.key_pieces, kKeyThreads, 0, stream, a);
  if (e == hipSuccess)
    e = launch(a.key_pieces > 0        ? k_kv_evict<T, D, kLongKeys, true>
               : a.bound <= kShortKeys ? k_kv_evict<T, D, kShortKeys, false>
                                       : k_kv_evict<T, D, kLongKeys, false>,
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
      a.table_stride < 0 || a.workspace_bytes < 0 || a.budget <= 0 || a.recent < 0 || a.sinks < 0 ||
      row_bound(a.max_length, a.table_width, c.block_size) > kMostSlots)
    return false;
  if (static_cast<int64_t>(a.recent) + a.sinks > a.budget) return false;
  const int64_t pairs = static_cast<int64_t>(a.rows) * c.kv_heads;  // launches stay below 2^32 threads
  if (pairs > (1 << 21) || pairs * ceil_div(evict_bound(a), kKeySlots) > (1 << 23))
    return false;
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

// Workgroups that make a (row, KV head)'s keys ahead, where rows may have more
// slots than the selecting workgroup's LDS has room for: every pass over the rest
// then reads 4 bytes a slot and no pages (one row of 65,536 cut to 8,192: 70 us,
// 162 with those keys made again in every pass).  Below that the launch costs more
// than it saves (8 rows of 32,768: 64 us without, 72 with).
int evict_key_pieces(const ResidentKvEvict& a) {
  const int bound = evict_bound(a);
  return bound > kLongKeys ? static_cast<int>(ceil_div(bound, kKeySlots)) : 0;
}

struct EvictBytes {
  int64_t keys, stats, lists;
  int64_t sum() const { return keys + stats + lists; }
};
EvictBytes evict_bytes(const ResidentKvEvict& a) {
  const int64_t pairs = static_cast<int64_t>(a.rows) * a.cache.kv_heads, pieces = pairs * evict_key_pieces(a), moves = evict_moves(a);
  if (moves == 0) return {0, 0, 0};
  return {pieces * kKeySlots * 4, pieces * static_cast<int64_t>(sizeof(KeyStats)), moves <= kOwnMoves ? 0 : pairs * (1 + 2 * moves) * 4};
}

}  // namespace
}  // namespace re

extern "C" int64_t resident_kv_evict_workspace(const ResidentKvEvict* args) {
  return args != nullptr && re::evict_ok(*args) ? re::evict_bytes(*args).sum() : -1;
}

extern "C" int32_t resident_kv_evict(const ResidentKvEvict* args, void* stream) {
  using namespace re;
  if (args == nullptr || !evict_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  const EvictBytes b = evict_bytes(*args);
  if (b.sum() > 0 && (args->workspace == nullptr || args->workspace_bytes < b.sum())) return -1;
  EvictArgs a{};
  a.a = *args;
  a.bound = evict_bound(*args);
  a.moves = evict_moves(*args);
  a.key_pieces = b.keys > 0 ? evict_key_pieces(*args) : 0;
  char* base = static_cast<char*>(args->workspace);
  a.keys = reinterpret_cast<uint32_t*>(base);
  a.key_stats = reinterpret_cast<KeyStats*>(base + b.keys);
  a.lists = reinterpret_cast<int32_t*>(base + b.keys + b.stats);
  const DeviceScope device(args->cache.device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_evict<bf16_t>(a, s) : launch_evict<float>(a, s);
  return e == hipSuccess ? 0 : -2;
}
