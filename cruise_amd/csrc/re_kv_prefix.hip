// One new token of every row over a prefix that all rows share and over the row's
// own slots.
//
// The prefix's slots are the same for every row, so its KV heads see the queries of
// all rows at once: rows * group of them, cut into tiles of 16 QT whatever row
// they are of.  A workgroup takes one tile and one chunk of the prefix, its waves
// every fourth step of it, with the products of re_kv_attend.h; what it leaves is a
// part of each of its queries, as a chunk of a row's own slots does, and one launch
// joins them all.
#include "re_kv_attend.h"

namespace re {
namespace {

struct PrefixArgs {
  AttendArgs own;
  const int32_t* table;
  const int32_t* length;
  int bound;          // slots that the prefix can have
  int chunk, chunks;  // slots of one workgroup at most, workgroups of a tile
  int tiles;
  int blocks;         // of the prefix; the own slots' come behind them
};

// The prefix's slots, and those of each of its chunks: an even share of what is there.
__device__ __forceinline__ int prefix_slots(const PrefixArgs& args) { return max(0, min(args.length[0], args.bound)); }
__device__ __forceinline__ int prefix_chunk(const PrefixArgs& args, int n) {
  const int share = (n + args.chunks - 1) / args.chunks;
  return max(kLeastChunk, (share + kLeastChunk - 1) / kLeastChunk * kLeastChunk);
}

template <typename T, int D, bool EVEN, int QT>
__device__ __forceinline__ void prefix_part(const PrefixArgs& args, int block, unsigned char* smem) {
  using S = Step<T, D>;
  constexpr int kPiece = EVEN ? 16 : 1, kRows = 4 * S::kHalves;
  const ResidentKvAttention& a = args.own.a;
  const ResidentKvCache& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_index(tid), x = lane & 15, y = lane >> 4;
  // A chunk's tiles follow each other on one XCD, whose L2 then has its slots.
  const int local = block >> 3, unit = (local / args.tiles << 3) + (block & 7), tile = local % args.tiles;
  const int g = unit % c.kv_heads, chunk = unit / c.kv_heads, group = a.heads / c.kv_heads, queries = a.rows * group;
  const int n = prefix_slots(args), size = prefix_chunk(args, n), first = chunk * size, count = min(size, n - first);
  if (chunk >= args.chunks || count <= 0) return;

  int2* place = reinterpret_cast<int2*>(smem);
  for (int e = tid; e * kPiece < count; e += kAttendThreads) {
    const int j = first + e * kPiece, p = j / c.block_size;
    int page = args.table[p];
    if (page < 0 || page >= c.pages) page = -1;
    place[e] = make_int2(page, j - p * c.block_size);
  }
  S step[QT];  // the queries of each; the slots are step[0]'s
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int m = (tile * QT + t) * kHeadTile + x, row = m / group;
    step[t].load_q(static_cast<const T*>(a.q) + row * a.q_strides[0] + (g * group + m - row * group) * a.q_strides[1], y, m < queries);
  }
  __syncthreads();

  const T* keys = static_cast<const T*>(c.keys) + g * c.key_strides[2];
  const T* values = static_cast<const T*>(c.values) + g * c.value_strides[2];
  const float scale = a.scale * kLog2e;
  float top[QT], sum[QT];
  bool seen = false;
  re_f32x4 out[QT][S::kCols] = {};
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = -INFINITY;
    sum[t] = 0.f;
  }
  auto place_of = [&](int j) {
    int2 p = place[min(j, count - 1) / kPiece];
    if constexpr (EVEN) {
      p.x = __builtin_amdgcn_readfirstlane(p.x);
      p.y = __builtin_amdgcn_readfirstlane(p.y);
    }
    return p;
  };
  auto load_keys = [&](int j0) {
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half) {
      const int2 p = place_of(EVEN ? j0 + 16 * half : j0 + 16 * half + x);
      const T* at = keys + max(p.x, 0) * c.key_strides[0] + p.y * c.key_strides[1];
      step[0].load_k(half, EVEN ? at + x * c.key_strides[1] : at, y);
    }
  };
  const int stride = kAttendWaves * S::kSlots;
  if (w * S::kSlots < count) load_keys(w * S::kSlots);
  for (int j0 = w * S::kSlots; j0 < count; j0 += stride) {
    uint32_t valid = 0;  // of the lane's slots, 4 y + i of every half
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + 16 * half + 4 * y + i;
        const int2 p = place_of(EVEN ? j0 + 16 * half : j);
        step[0].load_v(4 * half + i, values + max(p.x, 0) * c.value_strides[0] + (p.y + (EVEN ? 4 * y + i : 0)) * c.value_strides[1], x);
        if (p.x >= 0 && j < count) valid |= 1u << (4 * half + i);
      }
    re_f32x4 s[QT][S::kHalves];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int half = 0; half < S::kHalves; ++half) s[t][half] = step[0].scores(half, step[t].q);
    if (j0 + stride < count) load_keys(j0 + stride);
    if (!__all(valid == (1u << kRows) - 1)) {  // a probability of 0 does not silence a NaN
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (!(valid >> i & 1)) step[0].clear_v(i);
    }
    seen = seen || __any(valid != 0);
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float peak = -INFINITY;
#pragma unroll
      for (int half = 0; half < S::kHalves; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[t][half][i] = valid >> (4 * half + i) & 1 ? s[t][half][i] * scale : -INFINITY;
          peak = fmaxf(peak, s[t][half][i]);
        }
      peak = xor_max<32>(xor_max<16>(peak, lane), lane);
      if (__any(peak > top[t])) {
        const float next = fmaxf(top[t], peak), keep = exp2_of(top[t] - base_of(next));
        top[t] = next;
        sum[t] *= keep;
#pragma unroll
        for (int i = 0; i < S::kCols; ++i) out[t][i] *= keep;
      }
      const float base = base_of(top[t]);
#pragma unroll
      for (int half = 0; half < S::kHalves; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[t][half][i] = exp2_of(s[t][half][i] - base);
          sum[t] += s[t][half][i];
        }
      step[0].output(s[t], out[t]);
    }
  }

  // Join the waves, 16 queries and 8 columns of every 16th part of the head at a time.
  constexpr int kCols = S::kCols < 8 ? S::kCols : 8, kWidth = 16 * kCols;
  float* stat = reinterpret_cast<float*>(smem);       // [waves][16][2]
  float* part = stat + kAttendWaves * kHeadTile * 2;  // [waves][16][kWidth]
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int m0 = (tile * QT + t) * kHeadTile, heads = min(kHeadTile, queries - m0);
    if (heads <= 0) break;
    const float whole = xor_add<32>(xor_add<16>(sum[t], lane), lane);
#pragma unroll
    for (int c0 = 0; c0 < S::kCols; c0 += kCols) {
      __syncthreads();  // the places, or the columns before, are no longer read
      if (c0 == 0 && y == 0) {
        stat[(w * kHeadTile + x) * 2] = top[t];
        stat[(w * kHeadTile + x) * 2 + 1] = seen ? whole : -1.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < kCols; q += 4)
          *reinterpret_cast<re_f32x4*>(part + (w * kHeadTile + x) * kWidth + kCols * (4 * y + i) + q) =
              re_f32x4{out[t][c0 + q][i], out[t][c0 + q + 1][i], out[t][c0 + q + 2][i], out[t][c0 + q + 3][i]};
      __syncthreads();
      for (int u = tid; u < heads * (kWidth / 4); u += kAttendThreads) {
        const int h = u / (kWidth / 4), at_part = u % (kWidth / 4) * 4;
        const int e = at_part / kCols * S::kCols + c0 + at_part % kCols;  // of the head
        float top_of = -INFINITY, total = 0.f;
        bool any = false;
#pragma unroll
        for (int i = 0; i < kAttendWaves; ++i) top_of = fmaxf(top_of, stat[(i * kHeadTile + h) * 2]);
        const float base = base_of(top_of);
        re_f32x4 o = {};
#pragma unroll
        for (int i = 0; i < kAttendWaves; ++i) {
          const float l = stat[(i * kHeadTile + h) * 2 + 1];
          if (l < 0.f) continue;  // a wave without a slot (a NaN is a slot's)
          const float r = exp2_of(stat[(i * kHeadTile + h) * 2] - base);
          any = true;
          total += l * r;
          o += *reinterpret_cast<const re_f32x4*>(part + (i * kHeadTile + h) * kWidth + at_part) * r;
        }
        const int m = m0 + h, row = m / group;
        const int64_t at = (static_cast<int64_t>(row) * a.heads + g * group + m - row * group) * args.own.list + chunk;
        if (e == 0) {
          args.own.stats[at * 2] = top_of;
          args.own.stats[at * 2 + 1] = any ? total : -1.f;
        }
        *reinterpret_cast<re_f32x4*>(args.own.parts + at * D + e) = o;
      }
    }
  }
}

template <typename T, int D, bool EVEN, int QT>
__global__ void __launch_bounds__(kAttendThreads) k_kv_prefix(PrefixArgs args) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (static_cast<int>(blockIdx.x) < args.blocks) {
    prefix_part<T, D, EVEN, QT>(args, blockIdx.x, smem);
  } else {
    attend_chunk<T, D, EVEN>(args.own, blockIdx.x - args.blocks, smem);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) k_kv_prefix_join(PrefixArgs args) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int n = prefix_slots(args), size = prefix_chunk(args, n);
  attend_join<T, D>(args.own, blockIdx.x, (n + size - 1) / size, smem);
}

// Query tiles of 16 of a workgroup.
int query_tiles(const ResidentKvAttention& a) {
  const int64_t queries = static_cast<int64_t>(a.rows) * (a.heads / a.cache.kv_heads);
  const int most = a.cache.dtype_bytes == 2 && a.cache.head_dim <= 128 ? 4 : 2;
  return queries <= 16 ? 1 : queries <= 32 ? 2 : most;
}

PrefixArgs prefix_plan(const ResidentKvPrefixAttention& a) {
  const ResidentKvCache& c = a.own.cache;
  PrefixArgs p{};
  p.own = attention_plan(a.own);
  p.table = a.prefix_table;
  p.length = a.prefix_length;
  p.bound = static_cast<int>(row_bound(a.max_prefix, a.prefix_width, c.block_size));
  const int64_t queries = static_cast<int64_t>(a.own.rows) * (a.own.heads / c.kv_heads);
  p.tiles = static_cast<int>(ceil_div(queries, static_cast<int64_t>(kHeadTile) * query_tiles(a.own)));
  const int64_t units = static_cast<int64_t>(c.kv_heads) * p.tiles, most = even_pages(c) ? 8 * kMostChunk : kMostChunk;
  p.chunk = static_cast<int>(std::clamp<int64_t>(round_up(ceil_div(p.bound * units, 256), kLeastChunk), kLeastChunk, most));
  p.chunks = std::max(1, static_cast<int>(ceil_div(p.bound, p.chunk)));
  p.blocks = static_cast<int>(round_up(static_cast<int64_t>(c.kv_heads) * p.chunks, 8) * p.tiles);
  p.own.joined = 1;
  p.own.local_scores = 0;
  p.own.score_stride = round_up(p.own.bound, 32);
  p.own.shared = p.chunks;
  p.own.list = p.chunks + p.own.chunks;
  return p;
}

template <typename T, int D, bool EVEN, int QT>
hipError_t launch_prefix(const PrefixArgs& p, hipStream_t stream) {
  const ResidentKvAttention& a = p.own.a;
  const size_t lds = std::max(shared_lds(a.cache, p.own.chunk), shared_lds(a.cache, p.chunk));
  const int64_t own = static_cast<int64_t>(a.rows) * a.cache.kv_heads * p.own.head_tiles * p.own.chunks;
  hipError_t e = launch(k_kv_prefix<T, D, EVEN, QT>, p.blocks + own, kAttendThreads, lds, stream, p);
  if (e == hipSuccess) {
    const int64_t adds = a.cache.weights != nullptr ? a.rows * a.cache.kv_heads * ceil_div(p.own.bound, 4 * kJoinThreads) : 0;
    e = launch(k_kv_prefix_join<T, D>, adds + static_cast<int64_t>(a.rows) * a.heads, kJoinThreads,
               std::max<size_t>(kJoinThreads * 16, static_cast<size_t>(a.heads / a.cache.kv_heads) * 8), stream, p);
  }
  return e;
}

template <typename T, int D, bool EVEN>
hipError_t launch_prefix(const PrefixArgs& p, hipStream_t stream) {
  const int tiles = query_tiles(p.own.a);
  if constexpr (sizeof(T) == 2 && D <= 128)
    if (tiles == 4) return launch_prefix<T, D, EVEN, 4>(p, stream);
  return tiles == 1 ? launch_prefix<T, D, EVEN, 1>(p, stream) : launch_prefix<T, D, EVEN, 2>(p, stream);
}

template <typename T>
hipError_t launch_prefix(const PrefixArgs& p, hipStream_t stream) {
  const int d = p.own.a.cache.head_dim;
  if (even_pages(p.own.a.cache))
    return d == 64 ? launch_prefix<T, 64, true>(p, stream) : d == 128 ? launch_prefix<T, 128, true>(p, stream) : launch_prefix<T, 256, true>(p, stream);
  return d == 64 ? launch_prefix<T, 64, false>(p, stream) : d == 128 ? launch_prefix<T, 128, false>(p, stream) : launch_prefix<T, 256, false>(p, stream);
}

bool prefix_ok(const ResidentKvPrefixAttention& a) {
  if (!attention_ok(a.own) || a.prefix_width < 0 || a.max_prefix < 0 ||
      row_bound(a.max_prefix, a.prefix_width, a.own.cache.block_size) > kMostSlots)
    return false;
  if (a.own.rows == 0) return true;
  const PrefixArgs p = prefix_plan(a);  // launches stay below 2^32 threads
  if (p.blocks + static_cast<int64_t>(a.own.rows) * a.own.cache.kv_heads * p.own.head_tiles * p.own.chunks >= 1 << 24) return false;
  return a.prefix_length != nullptr && (a.prefix_table != nullptr || a.prefix_width == 0) && aligned(a.prefix_length, 4) &&
         aligned(a.prefix_table, 4);
}

}  // namespace
}  // namespace re

extern "C" int64_t resident_kv_prefix_attention_workspace(const ResidentKvPrefixAttention* args) {
  using namespace re;
  if (args == nullptr || !prefix_ok(*args)) return -1;
  if (args->own.rows == 0) return 0;
  const AttendBytes b = attention_bytes(prefix_plan(*args).own);
  return b.parts + b.stats + b.scores;
}

extern "C" int32_t resident_kv_prefix_attention(const ResidentKvPrefixAttention* args, void* stream) {
  using namespace re;
  if (args == nullptr || !prefix_ok(*args)) return -1;
  const ResidentKvAttention& own = args->own;
  if (own.rows == 0) return 0;
  PrefixArgs p = prefix_plan(*args);
  const AttendBytes b = attention_bytes(p.own);
  if (own.workspace == nullptr || own.workspace_bytes < b.parts + b.stats + b.scores) return -1;
  char* base = static_cast<char*>(own.workspace);
  p.own.parts = reinterpret_cast<float*>(base);
  p.own.stats = reinterpret_cast<float*>(base + b.parts);
  p.own.scores = reinterpret_cast<float*>(base + b.parts + b.stats);
  const DeviceScope device(own.cache.device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = own.cache.dtype_bytes == 2 ? launch_prefix<bf16_t>(p, s) : launch_prefix<float>(p, s);
  return e == hipSuccess ? 0 : -2;
}
