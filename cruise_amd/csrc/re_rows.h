// Whole rows in registers: what re_block_norms.hip and re_int8.hip share.
//
// A row of n elements lies over WAVES waves, P pieces of 16 bytes to a lane.  VEC:
// rows start at multiples of 16 bytes and hold whole pieces.  Otherwise bf16 takes the
// same loads and stores from whatever byte the row starts at (the hardware takes any)
// and the piece that a row ends in by its halves, and a lane's fp32 elements are a row's
// lanes apart, so that a load takes neighbours wherever the row starts (4,097 rows of
// 1,001: 13 us, in loose pieces 16).
//
// Norms of 20,000 bf16 rows: 4,096 elements, aligned, 112 us; 4,095, loose, 199; 4,097 275
// (element by element 1,697).  They move the same bytes to and from memory.  The loose
// pieces' registers (221 and 239, aligned 164) leave two waves a SIMD in place of three, and
// a row of 513 pieces takes four waves of four pieces a lane, half of them empty.
#pragma once

#include "re_ops.h"

namespace re {
namespace {

// Threads of a workgroup: four waves with a row each, or the waves of one row.
constexpr int row_threads(int waves) { return waves == 1 ? 256 : waves * 64; }

// Words at any byte.
typedef uint32_t loose_u32x4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t loose_u32x2 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t loose_u32 __attribute__((aligned(1)));
typedef uint16_t loose_u16 __attribute__((aligned(1)));

template <typename T, int WAVES, int P, bool VEC>
struct RowTile {
  static constexpr int E = Piece<T>::kElems, kLanes = WAVES * 64, kElems = P * E;
  static constexpr int kThreads = row_threads(WAVES);
  static constexpr int kRows = kThreads / kLanes;  // of a workgroup
  int lane;  // of the row

  __device__ __forceinline__ explicit RowTile(int tid) : lane(tid % kLanes) {}
  // The first element of piece p, in the row.
  __device__ __forceinline__ int at(int p) const { return (p * kLanes + lane) * E; }
  static constexpr bool kApart = !VEC && sizeof(T) == 4;
  __device__ __forceinline__ int at(int p, int e) const { return kApart ? (p * E + e) * kLanes + lane : at(p) + e; }
  // Whether a row of n has all of the lane's piece p, and whether it ends in one of the pieces p.
  __device__ __forceinline__ bool full(int p, int n) const { return VEC ? at(p) < n : at(p) + E <= n; }
  __device__ __forceinline__ static bool ends(int p, int n) { return !VEC && n % E != 0 && n / E / kLanes == p; }
  // The lane's elements of a row of n at `row`, 0 behind it.
  __device__ __forceinline__ void load(const T* row, int n, re_u32x4 (&v)[P]) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if constexpr (VEC) {
        v[p] = at(p) < n ? *reinterpret_cast<const re_u32x4*>(row + at(p)) : re_u32x4{};
      } else if constexpr (kApart) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = at(p, e) < n ? __float_as_uint(row[at(p, e)]) : 0;
        v[p] = re_u32x4{w[0], w[1], w[2], w[3]};
      } else {
        v[p] = full(p, n) ? static_cast<re_u32x4>(*reinterpret_cast<const loose_u32x4*>(row + at(p))) : re_u32x4{};
        if (ends(p, n) && at(p) < n && !full(p, n)) v[p] = load_rest(reinterpret_cast<const char*>(row + at(p)), n % E * sizeof(T));
      }
    }
  }
  // The 2 to 14 bytes that a row ends in, by the bits of their number.
  __device__ __forceinline__ static re_u32x4 load_rest(const char* from, int bytes) {
    uint32_t a = 0, b = 0, c = 0, d = 0;
    if (bytes & 8) {
      a = reinterpret_cast<const loose_u32*>(from)[0];
      b = reinterpret_cast<const loose_u32*>(from)[1];
    }
    if (bytes & 4) c = *reinterpret_cast<const loose_u32*>(from + (bytes & 8));
    if (bytes & 2) d = *reinterpret_cast<const loose_u16*>(from + (bytes & 12));
    // The words in their order: those of the bits that are set.
    const bool two = bytes & 8, one = bytes & 4;
    return re_u32x4{two ? a : one ? c : d, two ? b : one ? d : 0, two ? (one ? c : d) : 0, two && one ? d : 0};
  }
  __device__ __forceinline__ static void store_rest(char* to, int bytes, re_u32x4 v) {
    if (bytes & 8) {
      reinterpret_cast<loose_u32*>(to)[0] = v[0];
      reinterpret_cast<loose_u32*>(to)[1] = v[1];
    }
    if (bytes & 4) *reinterpret_cast<loose_u32*>(to + (bytes & 8)) = bytes & 8 ? v[2] : v[0];
    if (bytes & 2) {
      const int i = bytes / 4;
      *reinterpret_cast<loose_u16*>(to + (bytes & 12)) = static_cast<uint16_t>(i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3]);
    }
  }
  __device__ __forceinline__ void store(T* row, int n, const float (&f)[P][E]) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if constexpr (VEC) {
        if (at(p) < n) __builtin_nontemporal_store(Piece<T>::pack(f[p]), reinterpret_cast<re_u32x4*>(row + at(p)));
      } else if constexpr (kApart) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at(p, e) < n) row[at(p, e)] = f[p][e];
      } else {
        if (full(p, n)) *reinterpret_cast<loose_u32x4*>(row + at(p)) = Piece<T>::pack(f[p]);
        else if (ends(p, n) && at(p) < n) store_rest(reinterpret_cast<char*>(row + at(p)), n % E * sizeof(T), Piece<T>::pack(f[p]));
      }
    }
  }
  // Values / step, rounded to nearest even, as bytes; a step of 0 or NaN leaves zeros.
  // The quotient's own rounding to fp32 is part of the format.  From the correctly
  // rounded reciprocal r, t = x r is at most one step off and x - t step is exact, so
  // t + (x - t step) r is the correctly rounded quotient (P. Markstein's theorem): three
  // operations where a division takes about twelve, which bound 64 rows of 18,944 (7.1 us,
  // 4,096 of them 103).  Adding 1.5 * 2^23 leaves the nearest integer in the low byte.
  // Steps so small that the remainder could lose bits are divided by.
  __device__ __forceinline__ void store_bytes(int8_t* row, int n, const float (&f)[P][E], float step) const {
    const bool some = step > 0.f, plain = step < 0x1p-80f;
    const float r = some && !plain ? 1.f / step : 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint32_t q[E];
      if (plain || !some) {
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = some ? static_cast<int>(fminf(fmaxf(rintf(f[p][e] / step), -127.f), 127.f)) : 0;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float t = f[p][e] * r;
          q[e] = __float_as_uint(fmaf(fmaf(-t, step, f[p][e]), r, t) + 12582912.f);
        }
      }
      if constexpr (kApart) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at(p, e) < n) row[at(p, e)] = static_cast<int8_t>(q[e]);
      } else if (full(p, n)) {
        uint32_t w[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          const uint32_t lo = __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0c0c0400u);
          w[i] = lo | hi << 16;
        }
        if constexpr (E == 8 && VEC) *reinterpret_cast<uint2*>(row + at(p)) = make_uint2(w[0], w[1]);
        else if constexpr (E == 8) *reinterpret_cast<loose_u32x2*>(row + at(p)) = loose_u32x2{w[0], w[1]};
        else *reinterpret_cast<uint32_t*>(row + at(p)) = w[0];
      } else if (ends(p, n)) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at(p) + e < n) row[at(p) + e] = static_cast<int8_t>(q[e]);
      }
    }
  }
  // Sums and maxima over the row; `shared` has WAVES words that nothing else uses
  // until every wave has passed the next barrier.
  __device__ __forceinline__ float sum(float v, float* shared) const {
    v = wave_sum_dpp(v);
    if constexpr (WAVES > 1) {
      if (lane % 64 == 0) shared[lane / 64] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) v += shared[i];
    }
    return v;
  }
  // Of magnitudes' bit patterns, in which infinity and then NaN are the greatest.
  __device__ __forceinline__ uint32_t max(uint32_t v, uint32_t* shared) const {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = ::max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m, 64)));
    if constexpr (WAVES > 1) {
      if (lane % 64 == 0) shared[lane / 64] = v;
      __syncthreads();
      v = 0;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) v = ::max(v, shared[i]);
    }
    return v;
  }
};

// The step of a row whose greatest magnitude has these bits: NaN for a row that
// holds an infinity or a NaN, so that nothing of it passes for a number.
__device__ __forceinline__ float step_of(uint32_t top) {
  return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(top) / 127.f;
}

constexpr int kRowElems = 32768;           // of a row in registers
constexpr int64_t kRowMaxBlocks = 1 << 20;  // the kernels stride over the rest

// Waves of a row of `pieces` pieces of `elems` elements, of `rows` rows: as few as
// leave a lane up to four pieces where the rows fill the chip by themselves (with
// eight, two waves a SIMD are left: norms of 64,000 x 3,584 514 us on one wave, 395 on
// two, 415 on four, 416 on eight), one piece a lane where they do not; beyond 8 waves of
// four pieces those of bf16 take up to eight, since 16 waves leave 128 registers.
inline int row_waves(int64_t pieces, int64_t rows, int elems) {
  for (int waves : {1, 2, 4, 8})
    if (pieces <= waves * 256 && (rows * waves >= 1024 || pieces <= waves * 64)) return waves;
  return elems == 8 && rows >= 128 ? 8 : 16;
}

// The kernel of `each` pieces a lane, rounded up to one of Ps.
template <template <typename, int, int, bool> class F, typename T, bool VEC, int WAVES, int... Ps, typename Args>
hipError_t launch_pieces(int64_t each, int64_t rows, const Args& args, hipStream_t stream) {
  hipError_t e = hipErrorInvalidValue;
  (void)((each <= Ps && ((e = F<T, WAVES, Ps, VEC>::go(rows, args, stream)), true)) || ...);
  return e;
}

template <template <typename, int, int, bool> class F, typename T, bool VEC, typename Args>
hipError_t launch_rows(int64_t pieces, int64_t rows, const Args& args, hipStream_t stream) {
  const int waves = row_waves(pieces, rows, Piece<T>::kElems);
  const int64_t each = ceil_div(pieces, waves * 64);
  switch (waves) {
    case 1: return launch_pieces<F, T, VEC, 1, 1, 2, 4>(each, rows, args, stream);
    case 2: return launch_pieces<F, T, VEC, 2, 1, 2, 4>(each, rows, args, stream);
    case 4: return launch_pieces<F, T, VEC, 4, 1, 2, 4>(each, rows, args, stream);
    case 8:
      if constexpr (sizeof(T) == 2) return launch_pieces<F, T, VEC, 8, 1, 2, 3, 4, 5, 6, 8>(each, rows, args, stream);
      else return launch_pieces<F, T, VEC, 8, 1, 2, 4>(each, rows, args, stream);
    default:
      if constexpr (sizeof(T) == 2) return launch_pieces<F, T, VEC, 16, 1, 2, 3, 4>(each, rows, args, stream);
      else return launch_pieces<F, T, VEC, 16, 1, 2, 3, 4, 5, 6, 8>(each, rows, args, stream);
  }
}

}  // namespace
}  // namespace re
