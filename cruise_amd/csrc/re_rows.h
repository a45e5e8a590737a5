// Whole rows in registers: what re_block_norms.hip and re_int8.hip share.
//
// A row of n elements lies over WAVES waves, P pieces of 16 bytes to a lane.  VEC:
// a piece is 16 consecutive bytes (rows start at multiples of 16 bytes and hold
// whole pieces); otherwise its elements are LANES apart, so that a load takes
// neighbouring elements wherever a row starts.
#pragma once

#include "re_ops.h"

namespace re {
namespace {

// Threads of a workgroup: four waves with a row each, or the waves of one row.
constexpr int row_threads(int waves) { return waves == 1 ? 256 : waves * 64; }

template <typename T, int WAVES, int P, bool VEC>
struct RowTile {
  static constexpr int E = Piece<T>::kElems, kLanes = WAVES * 64, kElems = P * E;
  static constexpr int kThreads = row_threads(WAVES);
  static constexpr int kRows = kThreads / kLanes;  // of a workgroup
  int lane;  // of the row

  __device__ __forceinline__ explicit RowTile(int tid) : lane(tid % kLanes) {}
  // Element e of piece p, in the row.
  __device__ __forceinline__ int at(int p, int e) const {
    return VEC ? (p * kLanes + lane) * E + e : (p * E + e) * kLanes + lane;
  }
  // The lane's elements of a row of n at `row`, 0 behind it.
  __device__ __forceinline__ void load(const T* row, int n, re_u32x4 (&v)[P]) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if constexpr (VEC) {
        v[p] = at(p, 0) < n ? *reinterpret_cast<const re_u32x4*>(row + at(p, 0)) : re_u32x4{};
      } else {
        uint32_t w[4] = {};
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (at(p, e) >= n) continue;
          if constexpr (sizeof(T) == 2) w[e / 2] |= static_cast<uint32_t>(row[at(p, e)]) << (16 * (e % 2));
          else w[e] = __float_as_uint(row[at(p, e)]);
        }
        v[p] = re_u32x4{w[0], w[1], w[2], w[3]};
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int n, const float (&f)[P][E]) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if constexpr (VEC) {
        if (at(p, 0) < n) __builtin_nontemporal_store(Piece<T>::pack(f[p]), reinterpret_cast<re_u32x4*>(row + at(p, 0)));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at(p, e) < n) row[at(p, e)] = Elt<T>::t(f[p][e]);
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
      if constexpr (VEC) {
        if (at(p, 0) >= n) continue;
        uint32_t w[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          const uint32_t lo = __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0c0c0400u);
          w[i] = lo | hi << 16;
        }
        if constexpr (E == 8) *reinterpret_cast<uint2*>(row + at(p, 0)) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(row + at(p, 0)) = w[0];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at(p, e) < n) row[at(p, e)] = static_cast<int8_t>(q[e]);
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
