// Attention of one token over paged slots: what re_kv_attention.hip and
// re_kv_prefix.hip share.
//
// The cache is read once and everything else is small: at 7 query heads per KV
// head a slot of 2 x 128 bf16 (512 bytes) takes 3,584 multiply-adds, 14 flops a
// byte, so the bound is HBM, and the work is cut so that every CU streams:
//   * a row's slots in chunks, one workgroup per (row, KV head, chunk), its
//     query heads together, so a KV head's slots are read once for up to 16 of
//     them (more take further workgroups, and read again what L2 does not hold: 16,
//     17, 32 and 64 query heads over one KV head of 128, two rows of 131,071 slots:
//     37, 50, 51 and 86 us);
//   * a chunk's partial outputs and their softmax statistics are joined by a
//     second launch; a call whose rows fit one chunk needs none;
//   * weights need the softmax's sum first, so the scores (4 bytes of each query
//     head beside the slot's 512) are kept until it is known, in LDS or in memory.
// Both products run on the matrix cores with the slots in the order in which
// the loads deliver them, so nothing passes through LDS on the way:
//   scores  S^T = K Q^T   lane (x = lane % 16, y = lane / 16) loads 16 bytes of
//           slot x's key; the result holds query head x, slots 4 y .. 4 y + 3
//   output  O^T = V^T P^T   the same lane's probabilities are the second operand
//           as they are, and the first is column DV x + m of the values of the
//           lane's own slots (DV = head_dim / 16 columns, loaded as one run), so
//           16 lanes read a value row as one contiguous piece.
#pragma once

#include "re_ops.h"

namespace re {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kAttendThreads = 256;
constexpr int kAttendWaves = kAttendThreads / 64;
constexpr int kJoinThreads = 256;
constexpr int kHeadTile = 16;      // query heads of one workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMostChunk = 4096;   // slots of one workgroup at most
constexpr int kWholeRow = 512;     // rows of up to so many slots are not cut

struct AttendArgs {
  ResidentKvAttention a;
  int bound;          // slots that a row can have
  int chunk, chunks;  // slots of one workgroup at most, workgroups of a row
  int head_tiles;
  int joined;         // 1: a second launch joins the chunks and adds the weights
  int local_scores;   // where in LDS a whole row's scores lie, in bytes; 0: in memory
  int64_t score_stride;
  int shared, list;  // parts of a head that lie before its chunks (a shared prefix's), all of its parts
  float* parts;   // [rows][heads][list][head_dim]: outputs relative to the part's maximum
  float* stats;   // [rows][heads][list][2]: maximum (in powers of two), sum; sum -1: no slot
  float* scores;  // [rows][heads][score_stride]: in powers of two
};

// The two products of a step of kSlots slots, and the loads that feed them.
template <typename T, int D>
struct Step;

template <int D>
struct Step<bf16_t, D> {
  static constexpr int kSlots = 32, kHalves = 2, kLoads = D / 32, kCols = D / 16;
  re_u32x4 q[kLoads];
  re_u32x4 k[kHalves][kLoads];
  uint32_t v[8][kCols / 2];

  __device__ __forceinline__ void load_q(const bf16_t* p, int y, bool used) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) q[i] = used ? *reinterpret_cast<const re_u32x4*>(p + 32 * i + 8 * y) : re_u32x4{};
  }
  __device__ __forceinline__ void load_k(int half, const bf16_t* p, int y) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) k[half][i] = *reinterpret_cast<const re_u32x4*>(p + 32 * i + 8 * y);
  }
  // Row i of the lane's eight slots.
  __device__ __forceinline__ void load_v(int i, const bf16_t* p, int x) {
    if constexpr (kCols == 4) {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 r = *reinterpret_cast<const u32x2*>(p + kCols * x);
      v[i][0] = r[0];
      v[i][1] = r[1];
    } else {
#pragma unroll
      for (int c = 0; c < kCols / 8; ++c) {
        const re_u32x4 r = *reinterpret_cast<const re_u32x4*>(p + kCols * x + 8 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][4 * c + e] = r[e];
      }
    }
  }
  __device__ __forceinline__ void clear_v(int i) {
#pragma unroll
    for (int c = 0; c < kCols / 2; ++c) v[i][c] = 0;
  }
  __device__ __forceinline__ re_f32x4 scores(int half) const { return scores(half, q); }
  __device__ __forceinline__ re_f32x4 scores(int half, const re_u32x4 (&of)[kLoads]) const {
    re_f32x4 s = {};
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[half][i]), __builtin_bit_cast(bf16x8, of[i]), s, 0, 0, 0);
    return s;
  }
  // A probability enters this product as two bf16 numbers, its upper half and the
  // rest of it, so that it is off by 2^-15 of itself at most (bf16 alone: 2^-8)
  // and the stored type rounds the output only: the second product takes 128 of
  // the 6,000 cycles that a step's bytes do (64 rows of up to 1,000 slots take 0.6 of
  // 24 us longer than with one part, one row of 131,071 0.1 of 55).  The rest is never 0 beside an upper
  // half that is not (2^-22 of it is added): 0 times an infinite value would be NaN.
  __device__ __forceinline__ static float upper(float p) { return __uint_as_float(__float_as_uint(p) & 0xffff0000u); }
  __device__ __forceinline__ static float rest(float p) { return fmaf(p, 0x1p-22f, p - upper(p)); }
  __device__ __forceinline__ void output(const re_f32x4 (&p)[kHalves], re_f32x4 (&o)[kCols]) const {
    re_u32x4 high, low;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = p[i / 2][2 * (i % 2)], p1 = p[i / 2][2 * (i % 2) + 1];
      high[i] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
      low[i] = f2_to_bf16x2_raw(rest(p0), rest(p1));
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      // column c of the eight rows: low or high halves of two rows' words
      const uint32_t pick = c & 1 ? 0x07060302u : 0x05040100u;
      re_u32x4 col;
#pragma unroll
      for (int e = 0; e < 4; ++e) col[e] = __builtin_amdgcn_perm(v[2 * e + 1][c / 2], v[2 * e][c / 2], pick);
      o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, col), __builtin_bit_cast(bf16x8, low), o[c], 0, 0, 0);
      o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, col), __builtin_bit_cast(bf16x8, high), o[c], 0, 0, 0);
    }
  }
};

template <int D>
struct Step<float, D> {
  static constexpr int kSlots = 16, kHalves = 1, kLoads = D / 16, kCols = D / 16;
  re_f32x4 q[kLoads];
  re_f32x4 k[kHalves][kLoads];
  re_f32x4 v[4][kCols / 4];

  __device__ __forceinline__ void load_q(const float* p, int y, bool used) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) q[i] = used ? *reinterpret_cast<const re_f32x4*>(p + 16 * i + 4 * y) : re_f32x4{};
  }
  __device__ __forceinline__ void load_k(int half, const float* p, int y) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) k[half][i] = *reinterpret_cast<const re_f32x4*>(p + 16 * i + 4 * y);
  }
  __device__ __forceinline__ void load_v(int i, const float* p, int x) {
#pragma unroll
    for (int c = 0; c < kCols / 4; ++c) v[i][c] = *reinterpret_cast<const re_f32x4*>(p + kCols * x + 4 * c);
  }
  __device__ __forceinline__ void clear_v(int i) {
#pragma unroll
    for (int c = 0; c < kCols / 4; ++c) v[i][c] = re_f32x4{};
  }
  __device__ __forceinline__ re_f32x4 scores(int half) const { return scores(half, q); }
  __device__ __forceinline__ re_f32x4 scores(int half, const re_f32x4 (&of)[kLoads]) const {
    // Several sums side by side: one chain of D / 4 roundings puts twice the error of
    // the parts' on the output (heads of 256: 1.4e-6 of it and 5e-7) and is no faster.
    constexpr int kSums = D > 64 ? 4 : 2;
    re_f32x4 s[kSums] = {};
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e % kSums] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[half][i][e], of[i][e], s[e % kSums], 0, 0, 0);
    if constexpr (kSums == 2) return s[0] + s[1];
    else return (s[0] + s[1]) + (s[2] + s[3]);
  }
  __device__ __forceinline__ void output(const re_f32x4 (&p)[kHalves], re_f32x4 (&o)[kCols]) const {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][c / 4][c % 4], p[0][i], o[c], 0, 0, 0);
  }
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// What a maximum is subtracted as: scores of -infinity alone leave no
// difference of infinities behind.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.f : top; }

// The slots of each of a row's workgroups: where there are several, an even
// share of what the row has, so that a call sized for longer rows than it finds
// (a captured one, or a batch of few long ones) still spreads them: one row of
// 2,000 slots in a call for 131,072 takes 9.3 us, as in one for 2,000; with
// chunks of the call's size 25.
constexpr int kLeastChunk = 128;
__device__ __forceinline__ int row_chunk(const AttendArgs& args, int n) {
  if (args.chunks == 1) return args.chunk;
  const int share = (n + args.chunks - 1) / args.chunks;
  return max(kLeastChunk, (share + kLeastChunk - 1) / kLeastChunk * kLeastChunk);
}

// Weights of the row's slots j .. j + 3, j + 4 step .. (j a multiple of four)
// below n, from the scores (scores(h, j): four of query head h) and, in LDS, each
// query head's maximum and 1 / sum.
template <typename Scores>
__device__ __forceinline__ void add_weights(const AttendArgs& args, int row, int g, int group, const float* heads, int j, int n, int step,
                                            Scores scores) {
  const ResidentKvCache& c = args.a.cache;
  const int32_t* table = args.a.block_table + row * args.a.table_stride;
  for (; j < n; j += 4 * step) {
    float* at[4];
    float weight[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = min(j + i, n - 1), p = slot / c.block_size, page = table[p];
      const bool there = j + i < n && page >= 0 && page < c.pages;
      at[i] = there ? c.weights + page * c.weight_strides[0] + g * c.weight_strides[1] + (slot - p * c.block_size) : nullptr;
      weight[i] = there ? *at[i] : 0.f;
    }
    re_f32x4 sum = {};
    constexpr int kAhead = 8;
    for (int h0 = 0; h0 < group; h0 += kAhead) {
      re_f32x4 s[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) s[u] = scores(min(h0 + u, group - 1), j);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (h0 + u >= group) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += exp2_of(s[u][i] - heads[2 * (h0 + u)]) * heads[2 * (h0 + u) + 1];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at[i] != nullptr) *at[i] = weight[i] + sum[i];
  }
}

// Wave w of the workgroup takes the steps w, w + 4, ... of the chunk.  EVEN:
// pages of whole 16-slot pieces, so that a piece has one address; else every
// slot has its own (16 rows of 8,192 slots: 55 us even, 58 not).
template <typename T, int D, bool EVEN>
__device__ __forceinline__ void attend_chunk(const AttendArgs& args, int block, unsigned char* smem) {
  using S = Step<T, D>;
  constexpr int kPiece = EVEN ? 16 : 1, kRows = 4 * S::kHalves;
  const ResidentKvAttention& a = args.a;
  const ResidentKvCache& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_index(tid), x = lane & 15, y = lane >> 4;
  const int units = a.rows * c.kv_heads;
  const int unit = block % units, tile = block / units % args.head_tiles, chunk = block / units / args.head_tiles;
  const int row = unit / c.kv_heads, g = unit % c.kv_heads, group = a.heads / c.kv_heads;
  const int n = cut_length(a.lengths, row, args.bound), size = row_chunk(args, n), first = chunk * size;
  const int count = min(size, n - first);
  if (count <= 0 && chunk > 0) return;
  const int heads = min(kHeadTile, group - tile * kHeadTile), head = g * group + tile * kHeadTile + x;

  // Where the chunk's pieces lie; page -1: absent.
  int2* place = reinterpret_cast<int2*>(smem);
  // (A row that is not cut requests all the pages that it can have, together with
  // its length.)
  const int staged = args.chunks == 1 ? args.bound : count;
  for (int e = tid; e * kPiece < staged; e += kAttendThreads) {
    const int j = first + e * kPiece, p = j / c.block_size;
    int page = a.block_table[row * a.table_stride + p];
    if (page < 0 || page >= c.pages) page = -1;
    place[e] = make_int2(page, j - p * c.block_size);
  }
  S step;
  step.load_q(static_cast<const T*>(a.q) + row * a.q_strides[0] + head * a.q_strides[1], y, x < heads);
  __syncthreads();

  const T* keys = static_cast<const T*>(c.keys) + g * c.key_strides[2];
  const T* values = static_cast<const T*>(c.values) + g * c.value_strides[2];
  const float scale = a.scale * kLog2e;
  float top = -INFINITY, sum = 0.f;
  bool seen = false;
  re_f32x4 out[S::kCols] = {};
  // The chunk's slot at offset j: slots behind the count and on absent pages
  // read a slot that is there, and are masked.
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
      step.load_k(half, EVEN ? at + x * c.key_strides[1] : at, y);
    }
  };
  const int stride = kAttendWaves * S::kSlots;
  if (w * S::kSlots < count) load_keys(w * S::kSlots);
  for (int j0 = w * S::kSlots; j0 < count; j0 += stride) {
    uint32_t valid = 0;  // of the lane's slots, 4 y + i of every half
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half) {
      if constexpr (EVEN) {
        const int2 p = place_of(j0 + 16 * half);
        const T* at = values + max(p.x, 0) * c.value_strides[0] + p.y * c.value_strides[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          step.load_v(4 * half + i, at + (4 * y + i) * c.value_strides[1], x);
          if (p.x >= 0 && j0 + 16 * half + 4 * y + i < count) valid |= 1u << (4 * half + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + 16 * half + 4 * y + i;
          const int2 p = place_of(j);
          step.load_v(4 * half + i, values + max(p.x, 0) * c.value_strides[0] + p.y * c.value_strides[1], x);
          if (p.x >= 0 && j < count) valid |= 1u << (4 * half + i);
        }
      }
    }
    re_f32x4 s[S::kHalves];
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half) s[half] = step.scores(half);
    if (j0 + stride < count) load_keys(j0 + stride);

    float peak = -INFINITY;
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[half][i] = valid >> (4 * half + i) & 1 ? s[half][i] * scale : -INFINITY;
        peak = fmaxf(peak, s[half][i]);
      }
    if (c.weights != nullptr && args.local_scores != 0 && x < heads) {
      float* to = reinterpret_cast<float*>(smem + args.local_scores) + x * static_cast<int>(args.score_stride) + j0 + 4 * y;
#pragma unroll
      for (int half = 0; half < S::kHalves; ++half) *reinterpret_cast<re_f32x4*>(to + 16 * half) = s[half];
    } else if (c.weights != nullptr && x < heads) {
      float* to = args.scores + (static_cast<int64_t>(row) * a.heads + head) * args.score_stride + first + j0 + 4 * y;
#pragma unroll
      for (int half = 0; half < S::kHalves; ++half) *reinterpret_cast<re_f32x4*>(to + 16 * half) = s[half];
    }
    peak = xor_max<32>(xor_max<16>(peak, lane), lane);
    if (__any(peak > top)) {
      const float next = fmaxf(top, peak), keep = exp2_of(top - base_of(next));
      top = next;
      sum *= keep;
#pragma unroll
      for (int i = 0; i < S::kCols; ++i) out[i] *= keep;
    }
    const float base = base_of(top);
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[half][i] = exp2_of(s[half][i] - base);
        sum += s[half][i];
      }
    if (!__all(valid == (1u << kRows) - 1)) {  // a probability of 0 does not silence a NaN
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (!(valid >> i & 1)) step.clear_v(i);
    }
    seen = seen || __any(valid != 0);
    step.output(s, out);
  }

  // Join the waves: statistics and outputs through LDS, the outputs 8 columns
  // of every 16th part of the head at a time.
  sum = xor_add<32>(xor_add<16>(sum, lane), lane);
  constexpr int kCols = S::kCols < 8 ? S::kCols : 8, kWidth = 16 * kCols;
  float* stat = reinterpret_cast<float*>(smem);       // [waves][16][2]
  float* part = stat + kAttendWaves * kHeadTile * 2;  // [waves][16][kWidth]
#pragma unroll
  for (int c0 = 0; c0 < S::kCols; c0 += kCols) {
    __syncthreads();  // the places, or the columns before, are no longer read
    if (c0 == 0 && y == 0) {
      stat[(w * kHeadTile + x) * 2] = top;
      stat[(w * kHeadTile + x) * 2 + 1] = seen ? sum : -1.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < kCols; q += 4)
        *reinterpret_cast<re_f32x4*>(part + (w * kHeadTile + x) * kWidth + kCols * (4 * y + i) + q) =
            re_f32x4{out[c0 + q][i], out[c0 + q + 1][i], out[c0 + q + 2][i], out[c0 + q + 3][i]};
    __syncthreads();
    for (int u = tid; u < heads * (kWidth / 4); u += kAttendThreads) {
      const int h = u / (kWidth / 4), at_part = u % (kWidth / 4) * 4;
      const int e = at_part / kCols * S::kCols + c0 + at_part % kCols;  // of the head
      float m = -INFINITY, total = 0.f;
      bool any = false;
#pragma unroll
      for (int i = 0; i < kAttendWaves; ++i) m = fmaxf(m, stat[(i * kHeadTile + h) * 2]);
      const float base = base_of(m);
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
      const int qh = g * group + tile * kHeadTile + h;
      const int64_t at = (static_cast<int64_t>(row) * a.heads + qh) * args.list + args.shared + chunk;
      if (args.joined) {
        if (e == 0) {
          args.stats[at * 2] = m;
          args.stats[at * 2 + 1] = any ? total : -1.f;
        }
        *reinterpret_cast<re_f32x4*>(args.parts + at * D + e) = o;
      } else {
        T* to = static_cast<T*>(a.out) + row * a.out_strides[0] + qh * a.out_strides[1] + e;
        const float r = 1.f / total;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = Elt<T>::t(any ? o[i] * r : 0.f);
      }
    }
  }
  if (args.joined || c.weights == nullptr) return;

  // The whole row was here: add its weights from the scores that the
  // workgroup's own waves left in LDS or wrote.
  __syncthreads();  // the last columns are read
  if (tid < heads) {
    float m = -INFINITY, total = 0.f;
#pragma unroll
    for (int i = 0; i < kAttendWaves; ++i) m = fmaxf(m, stat[(i * kHeadTile + tid) * 2]);
    const float base = base_of(m);
#pragma unroll
    for (int i = 0; i < kAttendWaves; ++i) {
      const float l = stat[(i * kHeadTile + tid) * 2 + 1];
      total += l < 0.f ? 0.f : l * exp2_of(stat[(i * kHeadTile + tid) * 2] - base);
    }
    part[2 * tid] = base;
    part[2 * tid + 1] = 1.f / total;
  }
  __syncthreads();
  if (args.local_scores != 0) {
    const float* scores = reinterpret_cast<const float*>(smem + args.local_scores);
    add_weights(args, row, g, group, part, 4 * tid, count, kAttendThreads,
                [&](int h, int j) { return *reinterpret_cast<const re_f32x4*>(scores + h * static_cast<int>(args.score_stride) + j); });
  } else {
    const float* scores = args.scores + (static_cast<int64_t>(row) * a.heads + g * group) * args.score_stride;
    add_weights(args, row, g, group, part, 4 * tid, count, kAttendThreads,
                [&](int h, int j) { return *reinterpret_cast<const re_f32x4*>(scores + h * args.score_stride + j); });
  }
}

// Where part i of a head lies, of whose `shared` first places `used` are written.
__device__ __forceinline__ int part_of(int i, int used, int shared) { return i < used ? i : i - used + shared; }

// A head's maximum and sum over its parts, by LANES neighbouring lanes, of
// which this is number `i`; sum -1: no slot.
template <int LANES>
__device__ __forceinline__ float2 join_stats(const float* stats, int parts, int used, int shared, int i, int lane) {
  float top = -INFINITY, sum = 0.f;
  bool any = false;
  // one pass: what was summed so far follows the maximum
  for (int j = i; j < parts; j += LANES) {
    const float2 s = *reinterpret_cast<const float2*>(stats + 2 * part_of(j, used, shared));
    if (s.y < 0.f) continue;
    any = true;
    const float next = fmaxf(top, s.x), base = base_of(next);
    sum = sum * exp2_of(top - base) + s.y * exp2_of(s.x - base);
    top = next;
  }
  float whole = top;
  whole = xor_max<8>(xor_max<4>(xor_max<2>(xor_max<1>(whole, lane), lane), lane), lane);
  if constexpr (LANES == 64) whole = xor_max<32>(xor_max<16>(whole, lane), lane);
  const float base = base_of(whole);
  sum *= exp2_of(top - base);
  float some = any ? 1.f : 0.f;
  sum = xor_add<8>(xor_add<4>(xor_add<2>(xor_add<1>(sum, lane), lane), lane), lane);
  some = xor_add<8>(xor_add<4>(xor_add<2>(xor_add<1>(some, lane), lane), lane), lane);
  if constexpr (LANES == 64) {
    sum = xor_add<32>(xor_add<16>(sum, lane), lane);
    some = xor_add<32>(xor_add<16>(some, lane), lane);
  }
  return make_float2(base, some > 0.f ? sum : -1.f);
}

// The second launch, of calls whose rows take several chunks or more than 16
// query heads per KV head: first the workgroups that add weights, one per (row,
// KV head, 1,024 slots), then one per (row, query head) that joins the chunks'
// outputs.  `used`: how many parts of a shared prefix each head has.
template <typename T, int D>
__device__ __forceinline__ void attend_join(const AttendArgs& args, int block, int used, unsigned char* smem) {
  const ResidentKvAttention& a = args.a;
  const ResidentKvCache& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 63;
  const int pieces = (args.bound + 4 * kJoinThreads - 1) / (4 * kJoinThreads), adds = c.weights != nullptr ? a.rows * c.kv_heads * pieces : 0;
  if (block < adds) {
    const int unit = block / pieces, first = block % pieces * 4 * kJoinThreads;
    const int row = unit / c.kv_heads, g = unit % c.kv_heads, group = a.heads / c.kv_heads;
    const int n = cut_length(a.lengths, row, args.bound), size = row_chunk(args, n), chunks = (n + size - 1) / size;
    if (first >= n) return;
    float* whole = reinterpret_cast<float*>(smem);  // [group]: maximum, 1 / sum
    const int64_t head = static_cast<int64_t>(row) * a.heads + g * group;
    for (int i0 = 0; i0 < group; i0 += kJoinThreads / 16) {  // 16 lanes a head, all of them through the exchanges
      const int i = i0 + tid / 16;
      const float2 s = join_stats<16>(args.stats + (head + min(i, group - 1)) * args.list * 2, used + chunks, used, args.shared, tid % 16, lane);
      if (i < group && tid % 16 == 0) {
        whole[2 * i] = s.x;
        whole[2 * i + 1] = 1.f / s.y;
      }
    }
    __syncthreads();
    const float* scores = args.scores + head * args.score_stride;
    add_weights(args, row, g, group, whole, first + 4 * tid, min(first + 4 * kJoinThreads, n), kJoinThreads,
                [&](int h, int j) { return *reinterpret_cast<const re_f32x4*>(scores + h * args.score_stride + j); });
    return;
  }
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes, kAhead = 4;
  const int b = block - adds, row = b / a.heads, h = b % a.heads;
  const int n = cut_length(a.lengths, row, args.bound), size = row_chunk(args, n), parts = used + (n + size - 1) / size;
  const int64_t at = static_cast<int64_t>(b) * args.list;
  const float* stats = args.stats + at * 2;
  const int e = tid % kLanes * 4;
  re_f32x4 o = {}, v[kAhead];
  float2 s[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = part_of(max(min(i0 + u * kGroups, parts - 1), 0), used, args.shared);
      v[u] = *reinterpret_cast<const re_f32x4*>(args.parts + (at + i) * D + e);
      s[u] = *reinterpret_cast<const float2*>(stats + 2 * i);
    }
  };
  load(tid / kLanes);  // on their way while the statistics are joined
  const float2 whole = join_stats<64>(stats, parts, used, args.shared, lane, lane);
  for (int i0 = tid / kLanes; i0 < parts; i0 += kAhead * kGroups) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u * kGroups < parts && !(s[u].y < 0.f)) o += v[u] * exp2_of(s[u].x - whole.x);
    if (i0 + kAhead * kGroups < parts) load(i0 + kAhead * kGroups);
  }
  re_f32x4* part = reinterpret_cast<re_f32x4*>(smem);  // [groups][D / 4]
  part[tid] = o;
  __syncthreads();
  if (tid >= kLanes) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) o += part[i * kLanes + tid];
  T* to = static_cast<T*>(a.out) + row * a.out_strides[0] + h * a.out_strides[1] + e;
  const float r = 1.f / whole.y;
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i] = Elt<T>::t(whole.y < 0.f ? 0.f : o[i] * r);
}
inline int attention_bound(const ResidentKvAttention& a) {
  return static_cast<int>(row_bound(a.max_length, a.table_width, a.cache.block_size));
}

// Pages of whole 16-slot pieces.
inline bool even_pages(const ResidentKvCache& c) { return c.block_size % 16 == 0; }

// LDS for where a workgroup's slots lie, and later for its waves' statistics and
// outputs.
inline int64_t shared_lds(const ResidentKvCache& c, int chunk) {
  const int64_t places = (chunk / (even_pages(c) ? 16 : 1) + 1) * static_cast<int64_t>(sizeof(int2));
  return round_up(std::max(places, static_cast<int64_t>(kAttendWaves * kHeadTile) * (std::min(c.head_dim, 128) + 2) * 4), 16);
}
// And for the scores of a whole row (four words more a head put the heads on
// different banks).
inline int64_t score_lds(const ResidentKvAttention& a, int bound) {
  return std::min(kHeadTile, a.heads / a.cache.kv_heads) * (round_up(bound, 32) + 4) * 4;
}

// The cut of a call.  A launch streams at the rate of HBM once every CU has one
// workgroup, and the fewer there are, the less is left to join: one row of
// 131,071 slots takes 54 us cut for 256 workgroups, 58 for 512 and 65 for 384,
// which leave some CUs one and some two.  Rows of a batch differ in length,
// which several workgroups to a CU even out (12 rows, a third of them empty: 16
// us for 512, 18 for 256; 3 rows of 65,536 to 131,071: 137 and 153).  Other batches
// of two to four pay for it (2 and 4 equal rows of 131,071: 103.5 and 194 us, 100 and
// 194 for 256; of 16,000: 20.4 and 29.1, 18.4 and 27.7).
// A batch that has one workgroup per CU uncut is not cut: a second launch costs
// more (64 rows of up to 1,000 with weights: 25 us uncut, 32 cut in two).  Short
// rows stay whole for the same reason (4 rows of 4 KV heads, 256 slots: 7.0 us
// whole, 9.2 in two; 512 slots: 9.2 whole, 9.1 in four), longer ones go down to one
// step a wave (1,024 slots in pieces of 128, 256 and 512: 9.5, 10.8 and 12.9 us).
inline AttendArgs attention_plan(const ResidentKvAttention& a) {
  AttendArgs p{};
  p.a = a;
  p.bound = attention_bound(a);
  p.head_tiles = static_cast<int>(ceil_div(a.heads / a.cache.kv_heads, kHeadTile));
  const int64_t units = static_cast<int64_t>(a.rows) * a.cache.kv_heads * p.head_tiles;
  const int64_t workgroups = a.rows == 1 || units >= 256 ? 256 : 512;
  p.chunk = p.bound <= kWholeRow ? kWholeRow
                                 : static_cast<int>(std::clamp<int64_t>(round_up(ceil_div(p.bound * units, workgroups), kLeastChunk), kLeastChunk, kMostChunk));
  p.chunks = std::max(1, static_cast<int>(ceil_div(p.bound, p.chunk)));
  // One chunk cannot hand its weights over to other head tiles: the second
  // launch adds them, and joins outputs of one chunk each.
  p.joined = p.chunks > 1 || (a.cache.weights != nullptr && p.head_tiles > 1);
  // Rows of a launch without a join keep their scores in LDS where 64 KB have
  // room (64 rows of 1,000 slots, 7 query heads: 25.3 us, 27.6 through memory).
  const int64_t base = shared_lds(a.cache, p.chunk);
  p.local_scores = a.cache.weights != nullptr && !p.joined && base + score_lds(a, p.bound) <= 65536 ? static_cast<int>(base) : 0;
  p.score_stride = round_up(p.bound, 32) + (p.local_scores != 0 ? 4 : 0);
  p.list = p.chunks;
  return p;
}

struct AttendBytes {
  int64_t parts, stats, scores;
};
inline AttendBytes attention_bytes(const AttendArgs& p) {
  const int64_t heads = static_cast<int64_t>(p.a.rows) * p.a.heads;
  return {p.joined ? heads * p.list * p.a.cache.head_dim * 4 : 0, p.joined ? round_up(heads * p.list * 8, 16) : 0,
          p.a.cache.weights != nullptr && p.local_scores == 0 ? heads * p.score_stride * 4 : 0};
}

inline bool attention_ok(const ResidentKvAttention& a) {
  const ResidentKvCache& c = a.cache;
  if (!cache_ok(c) || a.rows < 0 || a.heads <= 0 || a.heads % c.kv_heads != 0 || a.table_width < 0 || a.max_length < 0 ||
      a.table_stride < 0 || a.workspace_bytes < 0 || a.reserved != 0 ||
      row_bound(a.max_length, a.table_width, c.block_size) > kMostSlots)
    return false;
  if (a.heads / c.kv_heads > 1024) return false;
  if (static_cast<int64_t>(a.rows) * a.heads > (1 << 22)) return false;
  if (a.rows == 0) return true;
  const AttendArgs p = attention_plan(a);  // launches stay below 2^32 threads
  if (static_cast<int64_t>(a.rows) * c.kv_heads * p.head_tiles * p.chunks >= 1 << 23 ||
      static_cast<int64_t>(a.rows) * (a.heads + c.kv_heads * ceil_div(p.bound, 4 * kJoinThreads)) >= 1 << 24)
    return false;
  if (a.q == nullptr || a.out == nullptr || a.lengths == nullptr || (a.block_table == nullptr && a.table_width > 0)) return false;
  return aligned(a.q, 16) && aligned(a.out, 16) && aligned(a.block_table, 4) && aligned(a.lengths, 4) && aligned(a.workspace, 16) &&
         row_strides_ok(a.q_strides, {a.rows, a.heads}, c.dtype_bytes) && row_strides_ok(a.out_strides, {a.rows, a.heads}, c.dtype_bytes) &&
         output_ok(HeadRows(a.out, a.out_strides, a.rows, a.heads, c.head_dim, c.dtype_bytes),
                   HeadRows(a.q, a.q_strides, a.rows, a.heads, c.head_dim, c.dtype_bytes));
}

}  // namespace
}  // namespace re
