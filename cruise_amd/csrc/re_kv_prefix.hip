// One new token of every row over a prefix that all rows share and over the row's
// own slots.
//
// The prefix's slots are the same for every row, so its KV heads see the queries of
// all rows at once: rows * group of them, cut into tiles of 16 whatever row they are of.
// A workgroup takes some tiles and one chunk of the prefix; what it leaves is a part of
// each of its queries (output and softmax statistics), as a chunk of a row's own slots
// does in the same launch, and a second launch joins them all.  Two kernels:
//   * up to 16 queries a KV head, and fp32: k_kv_prefix, the products of re_kv_attend.h
//     with one tile a wave (fp32 two), every slot straight from memory to the registers
//     of one wave.  HBM bounds it: 2 rows of 28 over 4 heads of 128 behind 131,071 slots 50 us,
//     5.4 TB/s, 43 in the first launch.
//   * more: k_kv_prefix_wide, four waves that share the slots through LDS (below).  64 rows
//     behind 32,768 slots 69 us, the first launch 62: 16 us before and after its loop
//     (the places, the first tile; the parts' 29 MB), 46 in it.  16 rows behind 131,071 slots
//     77-80 us.  By counters of the whole launch the matrix cores work 22 us in either and
//     vector instructions issue about as long; little of both falls together, although two
//     waves share a SIMD.  From the registers of single waves the same take 176 (with
//     1,000 own slots, 87-89 now) and 114.
//     fp32 with many queries is bound by its products: 64 rows of 28 over 4 heads of 128 behind
//     32,768 slots 560 us (54 TFLOP/s; every two tiles of 16 queries read the prefix again, from
//     the caches), 16 rows 111, one row 32 (4.3 TB/s).
// The own slots' workgroups come first, so that their reads run beside the products of
// the prefix.
#include "re_gemm_tiles.h"
#include "re_kv_attend.h"

namespace re {
namespace {

struct PrefixArgs {
  AttendArgs own;
  const int32_t* table;
  const int32_t* length;
  int bound;          // slots that the prefix can have
  int chunk, chunks;  // slots of one workgroup at most, workgroups of a tile
  int tiles;          // of queries
  int own_blocks;     // the prefix's come behind them
  int wide;           // query tiles of 16 of a workgroup of k_kv_prefix_wide; 0: k_kv_prefix
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
  if (static_cast<int>(blockIdx.x) < args.own_blocks) attend_chunk<T, D, EVEN>(args.own, blockIdx.x, smem);
  else prefix_part<T, D, EVEN, QT>(args, blockIdx.x - args.own_blocks, smem);
}

// ---- many queries ----

// A workgroup of 4 waves takes 16 QT WQ queries, every wave 16 QT of them, and the
// waves share the prefix's slots through LDS: tiles of `kSlots` of them, keys and
// values as they are, by direct loads into two stages.  16-byte piece c of a slot's
// row lies at c ^ swizzle(row), so that both the key fragments (16 rows, one piece) and
// the transposing reads of the values (16 rows, two pieces) touch every bank equally
// often.  128 queries a workgroup (WQ 4) where there are more than 64, else 64 (WQ 2),
// of which two waves each split a tile's slots and are joined in LDS at the end (8
// rows behind 32,768 slots 25 us, as a part of each wave 28; 64 rows 72 us with WQ 4, 74
// with WQ 2).
//   scores  S^T = K Q^T (32 slots: two 16-row products), output O^T = V^T P^T as in
//   re_kv_attend.h, V^T by ds_read_b64_tr_b16: in a group of 16 lanes (y) lane q + 4 r
//   names elements 4 q .. 4 q + 3 of slot 4 y + r, and lane i receives element i of the
//   four slots, which is the order in which the scores leave the probabilities.
// Of the softmax only what every score needs is in the loop: a lane's scores are
// compared with the running base, and the base follows (and what was summed is
// scaled) only when one is more than 2^8 above it; sums stay far from overflow, and any
// base gives the same quotient.  Keys of a tile are requested together, the first values
// ahead of the softmax.  A wave issues its products with a higher priority, so that the
// other wave of its SIMD works on its softmax meanwhile (72 us without, 69 with; the next
// step's softmax laid between the products by hand changes nothing).
// (bf16 probabilities in one part instead of two would save 10 of 72 us, and put 1.4 times
// the stored type's rounding on the output; see re_kv_attend.h.)
template <int D>
struct Wide {
  static constexpr int kQt = D == 256 ? 1 : 2, kSlots = D == 256 ? 32 : 64;
  static constexpr int kRow = 2 * D, kTile = kSlots * kRow;  // bytes
  static constexpr int kLanes = kRow / 16, kRows = 64 / kLanes, kInsts = kTile / 1024 / kAttendWaves;
  static constexpr int kPlaces = 4 * kTile;  // where they lie in LDS
  __device__ __forceinline__ static int swizzle(int row) { return (D == 64 ? row >> 1 & 3 : row & 7) << 1 | (row >> 3 & 1); }
};
constexpr int kWidePlaces = 2040;  // 16 KB of LDS with the flag
__device__ const uint4 kNoSlot = {0, 0, 0, 0};

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16* v4i16_lds;

// A transposing read.  (`__restrict__` says that nothing that is under way writes what
// it reads: without it the compiler waits for every load to LDS in flight, the next
// tile's among them.)
__device__ __forceinline__ v4i16 read_turned(v4i16_lds __restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

template <int D, bool EVEN, int WQ>
__device__ __forceinline__ void prefix_wide(const PrefixArgs& args, int block, unsigned char* smem) {
  using W = Wide<D>;
  constexpr int QT = W::kQt, WS = kAttendWaves / WQ, NS = W::kSlots / 32 / WS, kLoads = D / 32, kCols = D / 16;
  constexpr int kPiece = EVEN ? 16 : 1;
  const ResidentKvAttention& a = args.own.a;
  const ResidentKvCache& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_index(tid), x = lane & 15, y = lane >> 4, wq = w % WQ, ws = w / WQ;
  const int local = block >> 3, unit = (local / args.tiles << 3) + (block & 7), tile = local % args.tiles;
  const int g = unit % c.kv_heads, chunk = unit / c.kv_heads, group = a.heads / c.kv_heads, queries = a.rows * group;
  const int n = prefix_slots(args), size = prefix_chunk(args, n), first = chunk * size, count = min(size, n - first);
  if (chunk >= args.chunks || count <= 0) return;

  int2* place = reinterpret_cast<int2*>(smem + W::kPlaces);
  int* absent = reinterpret_cast<int*>(place + kWidePlaces);
  if (tid == 0) *absent = 0;
  __syncthreads();
  for (int e = tid; e * kPiece < count; e += kAttendThreads) {
    const int j = first + e * kPiece, p = j / c.block_size;
    int page = args.table[p];
    if (page < 0 || page >= c.pages) {
      page = -1;
      *absent = 1;
    }
    place[e] = make_int2(page, j - p * c.block_size);
  }
  // The wave's queries; a negative scale turns them, so that greater scores are greater products,
  // and a scale of 0 makes them 0.
  re_u32x4 q[QT][kLoads];
  const int m0 = (tile * WQ + wq) * 16 * QT;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int m = m0 + 16 * t + x, row = m / group;
    const bf16_t* from = static_cast<const bf16_t*>(a.q) + row * a.q_strides[0] + (g * group + m - row * group) * a.q_strides[1];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      q[t][i] = m < queries && a.scale != 0.f ? *reinterpret_cast<const re_u32x4*>(from + 32 * i + 8 * y) : re_u32x4{};
      if (a.scale < 0.f) q[t][i] ^= re_u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
    }
  }
  __syncthreads();

  const bool holes = *absent != 0;
  const int tiles = (count + W::kSlots - 1) / W::kSlots;
  const char* keys = reinterpret_cast<const char*>(static_cast<const bf16_t*>(c.keys) + g * c.key_strides[2]);
  const char* values = reinterpret_cast<const char*>(static_cast<const bf16_t*>(c.values) + g * c.value_strides[2]);
  // Load i of the wave: rows r .. r + kRows - 1 of a tile, a lane the piece that belongs in its place.
  uint32_t at_key[W::kInsts], at_value[W::kInsts];
#pragma unroll
  for (int i = 0; i < W::kInsts; ++i) {
    const int r = (w * W::kInsts + i) * W::kRows + lane / W::kLanes, piece = lane % W::kLanes ^ W::swizzle(r);
    at_key[i] = (EVEN ? r % 16 * static_cast<uint32_t>(c.key_strides[1]) * 2 : 0) + 16 * piece;
    at_value[i] = (EVEN ? r % 16 * static_cast<uint32_t>(c.value_strides[1]) * 2 : 0) + 16 * piece;
  }
  // (The places are read as 64-bit words: with the type's alias information the compiler
  // knows that a load in flight to LDS does not write them, and does not wait for it.)
  const uint64_t* place_word = reinterpret_cast<const uint64_t*>(place);
  auto place_at = [&](int e) {
    const uint64_t word = place_word[e];
    return make_int2(static_cast<int>(word), static_cast<int>(word >> 32));
  };
  auto issue = [&](int t, int stage) {
    const bool whole = !holes && (t + 1) * W::kSlots <= count;
    const int r0 = w * W::kInsts * W::kRows;  // the wave's rows are of one piece of 16
    unsigned char* to = smem + stage * 2 * W::kTile + w * W::kInsts * 1024;
    const char *k[W::kInsts], *v[W::kInsts];
    if constexpr (EVEN) {
      int2 p = place_at(min(t * W::kSlots + r0, count - 1) / 16);
      p.x = __builtin_amdgcn_readfirstlane(p.x);
      p.y = __builtin_amdgcn_readfirstlane(p.y);
      const char* key = keys + (p.x * c.key_strides[0] + p.y * c.key_strides[1]) * 2;
      const char* value = values + (p.x * c.value_strides[0] + p.y * c.value_strides[1]) * 2;
#pragma unroll
      for (int i = 0; i < W::kInsts; ++i) {
        k[i] = key + at_key[i];
        v[i] = value + at_value[i];
        if (!whole && (p.x < 0 || t * W::kSlots + r0 + i * W::kRows + lane / W::kLanes >= count)) k[i] = v[i] = reinterpret_cast<const char*>(&kNoSlot);
      }
    } else {
      int2 p[W::kInsts];
#pragma unroll
      for (int i = 0; i < W::kInsts; ++i) p[i] = place_at(min(t * W::kSlots + r0 + i * W::kRows + lane / W::kLanes, count - 1));
#pragma unroll
      for (int i = 0; i < W::kInsts; ++i) {
        k[i] = keys + (p[i].x * c.key_strides[0] + p[i].y * c.key_strides[1]) * 2 + at_key[i];
        v[i] = values + (p[i].x * c.value_strides[0] + p[i].y * c.value_strides[1]) * 2 + at_value[i];
        if (!whole && (p[i].x < 0 || t * W::kSlots + r0 + i * W::kRows + lane / W::kLanes >= count)) k[i] = v[i] = reinterpret_cast<const char*>(&kNoSlot);
      }
    }
#pragma unroll
    for (int i = 0; i < W::kInsts; ++i) {
      __builtin_amdgcn_global_load_lds((gemm_gptr)k[i], (gemm_lptr)(to + i * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gemm_gptr)v[i], (gemm_lptr)(to + W::kTile + i * 1024), 16, 0, 0);
    }
  };
  // Where the lane's fragments lie in a step of 32 slots: its key's pieces, its values'.
  int at_k[kLoads], at_v[kCols];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) at_k[i] = x * W::kRow + ((4 * i + y) ^ W::swizzle(x)) * 16;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    const int row = 4 * y + (x >> 2);
    at_v[i] = W::kTile + row * W::kRow + ((2 * i + (x >> 1 & 1)) ^ W::swizzle(row)) * 16 + (x & 1) * 8;
  }

  // (Not 0: masked scores stay -infinity.)
  const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  float base[QT], less[QT], sum[QT];  // less: what is taken off, the base but for none yet
  bool seen = false;
  re_f32x4 out[QT][kCols] = {};
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    base[t] = -INFINITY;
    less[t] = sum[t] = 0.f;
  }
  issue(0, 0);
  for (int t = 0; t < tiles; ++t) {
    gemm_stage_barrier();  // this tile is there, the one before is read
    if (t + 1 < tiles) issue(t + 1, t + 1 & 1);
    const unsigned char* stage = smem + (t & 1) * 2 * W::kTile + ws * NS * 32 * W::kRow;
    // All of the tile's key fragments are requested at once, so that the products
    // wait for the first of them alone.
    re_u32x4 k[NS][2][kLoads];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) k[u][half][i] = *reinterpret_cast<const re_u32x4*>(stage + (32 * u + 16 * half) * W::kRow + at_k[i]);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    re_f32x4 s[NS][QT][2] = {};
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int h = 0; h < QT; ++h)
            s[u][h][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[u][half][i]),
                                                                    __builtin_bit_cast(bf16x8, q[h][i]), s[u][h][half], 0, 0, 0);
    __builtin_amdgcn_s_setprio(0);
    // The first step's values, ahead of the softmax.
    bf16x8 v[kCols];
    auto read_values = [&](int u) {
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const v4i16 v0 = read_turned((v4i16_lds)(stage + 32 * u * W::kRow + at_v[i]));
        const v4i16 v1 = read_turned((v4i16_lds)(stage + (32 * u + 16) * W::kRow + at_v[i]));
        v[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    read_values(0);
    __builtin_amdgcn_sched_barrier(0);
    if (holes || (t + 1) * W::kSlots > count) {
      bool some = false;
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = t * W::kSlots + (ws * NS + u) * 32 + 16 * half + 4 * y + i;
            if (j < count && place_at(j / kPiece).x >= 0) {
              some = true;
              continue;
            }
#pragma unroll
            for (int h = 0; h < QT; ++h) s[u][h][half][i] = -INFINITY;
          }
      seen = seen || __any(some);
    } else {
      seen = true;
    }
#pragma unroll
    for (int h = 0; h < QT; ++h) {
      float peak = s[0][h][0][0];
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 4; ++i) peak = fmaxf(peak, s[u][h][half][i]);
      peak *= scale;
      if (__any(peak > base[h] + 8.f)) {
        peak = xor_max<32>(xor_max<16>(peak, lane), lane);
        const float next = fmaxf(base[h], peak), keep = exp2_of(base[h] - base_of(next));
        base[h] = next;
        less[h] = base_of(next);
        sum[h] *= keep;
#pragma unroll
        for (int i = 0; i < kCols; ++i) out[h][i] *= keep;
      }
    }
    re_u32x4 high[NS][QT], low[NS][QT];
    // Two scores of step u: part i of the 4 QT.
    auto weigh = [&](int u, int part) {
      const int h = part / 4, i = part % 4;
      const float p0 = exp2_of(fmaf(s[u][h][i / 2][2 * (i % 2)], scale, -less[h]));
      const float p1 = exp2_of(fmaf(s[u][h][i / 2][2 * (i % 2) + 1], scale, -less[h]));
      sum[h] += p0 + p1;
      // Two bf16 parts of each, as in re_kv_attend.h; the second is never 0 beside a first that is not.
      high[u][h][i] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
      low[u][h][i] = f2_to_bf16x2_raw(fmaf(p0, 1.f + 0x1p-22f, -__uint_as_float(__float_as_uint(p0) & 0xffff0000u)),
                                      fmaf(p1, 1.f + 0x1p-22f, -__uint_as_float(__float_as_uint(p1) & 0xffff0000u)));
    };
#pragma unroll
    for (int part = 0; part < 4 * QT; ++part)
#pragma unroll
      for (int u = 0; u < NS; ++u) weigh(u, part);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      if (u > 0) read_values(u);
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
#pragma unroll
        for (int h = 0; h < QT; ++h) {
          out[h][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[i], __builtin_bit_cast(bf16x8, low[u][h]), out[h][i], 0, 0, 0);
          out[h][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[i], __builtin_bit_cast(bf16x8, high[u][h]), out[h][i], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
#pragma unroll
  for (int h = 0; h < QT; ++h) sum[h] = xor_add<32>(xor_add<16>(sum[h], lane), lane);
  if constexpr (WS == 2) {
    // The second wave of a query tile hands its slots' share over in LDS.
    re_f32x4* others = reinterpret_cast<re_f32x4*>(smem) + wq * QT * kCols * 64;                     // [QT][kCols][64]
    float2* stats = reinterpret_cast<float2*>(smem + WQ * QT * kCols * 1024) + wq * QT * 64;         // [QT][64]
    __syncthreads();  // the tiles are no longer read
    if (ws == 1) {
#pragma unroll
      for (int h = 0; h < QT; ++h) {
        stats[h * 64 + lane] = make_float2(base[h], seen ? sum[h] : -1.f);
#pragma unroll
        for (int i = 0; i < kCols; ++i) others[(h * kCols + i) * 64 + lane] = out[h][i];
      }
    }
    __syncthreads();
    if (ws == 1) return;
#pragma unroll
    for (int h = 0; h < QT; ++h) {
      const float2 s = stats[h * 64 + lane];
      if (s.y < 0.f) continue;  // it saw no slot (a NaN is a slot's)
      const float next = fmaxf(base[h], s.x), keep = seen ? exp2_of(base[h] - base_of(next)) : 0.f, add = exp2_of(s.x - base_of(next));
      base[h] = next;
      sum[h] = (seen ? sum[h] * keep : 0.f) + s.y * add;
#pragma unroll
      for (int i = 0; i < kCols; ++i) out[h][i] = (seen ? out[h][i] * keep : re_f32x4{}) + others[(h * kCols + i) * 64 + lane] * add;
    }
    seen = seen || !(stats[lane].y < 0.f);
  }
#pragma unroll
  for (int h = 0; h < QT; ++h) {
    const int m = m0 + 16 * h + x, row = m / group;
    if (m >= queries) continue;
    const int64_t at = (static_cast<int64_t>(row) * a.heads + g * group + m - row * group) * args.own.list + chunk;
    if (y == 0) {
      args.own.stats[at * 2] = base[h];
      args.own.stats[at * 2 + 1] = seen ? sum[h] : -1.f;
    }
#pragma unroll
    for (int i = 0; i < kCols; ++i) *reinterpret_cast<re_f32x4*>(args.own.parts + at * D + 16 * i + 4 * y) = out[h][i];
  }
}

template <int D, bool EVEN, int WQ>
__global__ void __launch_bounds__(kAttendThreads, D == 256 ? 1 : 2) k_kv_prefix_wide(PrefixArgs args) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (static_cast<int>(blockIdx.x) < args.own_blocks) attend_chunk<bf16_t, D, EVEN>(args.own, blockIdx.x, smem);
  else prefix_wide<D, EVEN, WQ>(args, blockIdx.x - args.own_blocks, smem);
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) k_kv_prefix_join(PrefixArgs args) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int n = prefix_slots(args), size = prefix_chunk(args, n);
  attend_join<T, D>(args.own, blockIdx.x, (n + size - 1) / size, smem);
}

// Pages of whole 16-slot pieces whose slots a wide load reaches by 32-bit offsets.
bool wide_even(const ResidentKvCache& c) {
  return even_pages(c) && c.key_strides[1] < 1 << 26 && c.value_strides[1] < 1 << 26;
}

PrefixArgs prefix_plan(const ResidentKvPrefixAttention& a) {
  const ResidentKvCache& c = a.own.cache;
  PrefixArgs p{};
  p.own = attention_plan(a.own);
  p.table = a.prefix_table;
  p.length = a.prefix_length;
  p.bound = static_cast<int>(row_bound(a.max_prefix, a.prefix_width, c.block_size));
  const int64_t queries = static_cast<int64_t>(a.own.rows) * (a.own.heads / c.kv_heads);
  // 4 rows of 28 over 4 heads, 28 queries: 15.8 us against 20.2 from single waves behind
  // 8,192 slots, 34 and 37 behind 65,536, 57 and 56 behind 131,072.  2 rows, 14 queries:
  // 14.5 and 13.4, 34 and 31, 56 and 52.
  p.wide = c.dtype_bytes != 2 || queries <= kHeadTile ? 0 : queries <= 64 || c.head_dim == 256 ? 4 : 8;
  const int per = p.wide != 0 ? p.wide : queries <= kHeadTile ? 1 : 2;
  p.tiles = static_cast<int>(ceil_div(queries, static_cast<int64_t>(kHeadTile) * per));
  const int64_t units = static_cast<int64_t>(c.kv_heads) * p.tiles;
  const int64_t most = p.wide != 0 ? (wide_even(c) ? kWidePlaces * 16 : kWidePlaces) / kLeastChunk * kLeastChunk
                                   : even_pages(c) ? 8 * kMostChunk : kMostChunk;
  // One workgroup a CU; two of k_kv_prefix_wide, whose waves then cover each other's
  // waits, where that leaves each about 1,000 slots or more: every part is written and read
  // again (64 rows of 28 over 4 heads, 32,768 slots: 80 us for one, 71 for two;
  // 4,096 slots 28 and 31; 8 rows, 32,768 slots 25 and 30).
  const int64_t workgroups = p.wide != 0 && p.bound * units >= 512 * 1000 ? 512 : 256;
  p.chunk = static_cast<int>(std::clamp<int64_t>(round_up(ceil_div(p.bound * units, workgroups), kLeastChunk), kLeastChunk, most));
  p.chunks = std::max(1, static_cast<int>(ceil_div(p.bound, p.chunk)));
  p.own_blocks = a.own.rows * c.kv_heads * p.own.head_tiles * p.own.chunks;
  p.own.joined = 1;
  p.own.local_scores = 0;
  p.own.score_stride = round_up(p.own.bound, 32);
  p.own.shared = p.chunks;
  p.own.list = p.own.shared + p.own.chunks;
  return p;
}
int64_t prefix_blocks(const PrefixArgs& p) { return round_up(static_cast<int64_t>(p.own.a.cache.kv_heads) * p.chunks, 8) * p.tiles; }

template <typename T, int D>
hipError_t launch_join(const PrefixArgs& p, hipStream_t stream) {
  const ResidentKvAttention& a = p.own.a;
  const int64_t adds = a.cache.weights != nullptr ? a.rows * a.cache.kv_heads * ceil_div(p.own.bound, 4 * kJoinThreads) : 0;
  return launch(k_kv_prefix_join<T, D>, adds + static_cast<int64_t>(a.rows) * a.heads, kJoinThreads,
                std::max<size_t>(kJoinThreads * 16, static_cast<size_t>(a.heads / a.cache.kv_heads) * 8), stream, p);
}

template <typename T, int D, bool EVEN, int QT>
hipError_t launch_prefix(const PrefixArgs& p, hipStream_t stream) {
  const size_t lds = std::max(shared_lds(p.own.a.cache, p.own.chunk), shared_lds(p.own.a.cache, p.chunk));
  const hipError_t e = launch(k_kv_prefix<T, D, EVEN, QT>, p.own_blocks + prefix_blocks(p), kAttendThreads, lds, stream, p);
  return e == hipSuccess ? launch_join<T, D>(p, stream) : e;
}

template <int D, bool EVEN, int WQ>
hipError_t launch_wide(const PrefixArgs& p, hipStream_t stream) {
  constexpr int kLds = Wide<D>::kPlaces + (kWidePlaces + 1) * static_cast<int>(sizeof(int2));
  void (*const kernel)(PrefixArgs) = k_kv_prefix_wide<D, EVEN, WQ>;
  const size_t lds = std::max<size_t>(kLds, shared_lds(p.own.a.cache, p.own.chunk));
  static std::atomic<uint64_t> allowed{0};
  const hipError_t attr = allow_lds(kernel, kLds, allowed);
  if (attr != hipSuccess) return attr;
  const hipError_t e = launch(kernel, p.own_blocks + prefix_blocks(p), kAttendThreads, lds, stream, p);
  return e == hipSuccess ? launch_join<bf16_t, D>(p, stream) : e;
}

template <typename T, int D, bool EVEN>
hipError_t launch_prefix(const PrefixArgs& p, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.wide == 4) return launch_wide<D, EVEN, D == 256 ? 4 : 2>(p, stream);
    if constexpr (D != 256)
      if (p.wide == 8) return launch_wide<D, EVEN, 4>(p, stream);
  } else {
    const int64_t queries = static_cast<int64_t>(p.own.a.rows) * (p.own.a.heads / p.own.a.cache.kv_heads);
    if (queries > kHeadTile) return launch_prefix<T, D, EVEN, 2>(p, stream);
  }
  return launch_prefix<T, D, EVEN, 1>(p, stream);
}

template <typename T>
hipError_t launch_prefix(const PrefixArgs& p, hipStream_t stream) {
  const ResidentKvCache& c = p.own.a.cache;
  const int d = c.head_dim;
  if (p.wide != 0 ? wide_even(c) : even_pages(c))
    return d == 64 ? launch_prefix<T, 64, true>(p, stream) : d == 128 ? launch_prefix<T, 128, true>(p, stream) : launch_prefix<T, 256, true>(p, stream);
  return d == 64 ? launch_prefix<T, 64, false>(p, stream) : d == 128 ? launch_prefix<T, 128, false>(p, stream) : launch_prefix<T, 256, false>(p, stream);
}

bool prefix_ok(const ResidentKvPrefixAttention& a) {
  if (!attention_ok(a.own) || a.prefix_width < 0 || a.max_prefix < 0 ||
      row_bound(a.max_prefix, a.prefix_width, a.own.cache.block_size) > kMostSlots)
    return false;
  if (a.own.rows == 0) return true;
  const PrefixArgs p = prefix_plan(a);  // launches stay below 2^32 threads
  if (p.own_blocks + prefix_blocks(p) >= 1 << 24) return false;
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
