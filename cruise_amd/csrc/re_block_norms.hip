// The norm after a block, its gate and residual scale, the residual sum and the
// norm before the next block, in one pass.
#include "re_rows.h"

namespace re {
namespace {

// Whole rows stay in registers from their load to both stores, so each input is
// read and each output written once, and HBM bounds it: 64,000 rows of 3,584 bf16 with a
// gate for each element 395 us (5.8 TB/s), 4,096 of 18,944 162 us (4.8), 4,097 of 1,001 fp32
// 13 us (5.1); 4 of 3,584 4 us, two sums over the row and three round trips.  The residual
// that the second norm is made of is the fp32 sum, not what is stored: one rounding less,
// and the row is not read again.
template <typename T, int WAVES, int P, bool VEC>
__global__ void __launch_bounds__(row_threads(WAVES)) k_block_norms(ResidentBlockNorms a) {
  using Tile = RowTile<T, WAVES, P, VEC>;
  constexpr int E = Tile::E;
  __shared__ float sums[2][WAVES];
  __shared__ uint32_t tops[WAVES];
  const Tile tile(threadIdx.x);
  const int n = a.hidden;
  const float per = 1.f / n;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * Tile::kRows + threadIdx.x / Tile::kLanes; t < a.tokens;
       t += static_cast<int64_t>(gridDim.x) * Tile::kRows) {
    re_u32x4 raw_x[P], raw_r[P], raw_g[P];
    float gate = 1.f;
    const bool whole_gate = a.gate != nullptr && a.gate_strides[1] != 0;
    tile.load(static_cast<const T*>(a.residual) + t * a.residual_stride, n, raw_r);
    if (a.x != nullptr) tile.load(static_cast<const T*>(a.x) + t * a.x_stride, n, raw_x);
    if (whole_gate) tile.load(static_cast<const T*>(a.gate) + t * a.gate_strides[0], n, raw_g);
    else if (a.gate != nullptr) gate = Elt<T>::f(static_cast<const T*>(a.gate)[t * a.gate_strides[0]]);
    float r[P][E], w[P][E];
#pragma unroll
    for (int p = 0; p < P; ++p) Piece<T>::unpack(raw_r[p], r[p]);
    if (a.x != nullptr) {
      float x[P][E];
#pragma unroll
      for (int p = 0; p < P; ++p) Piece<T>::unpack(raw_x[p], x[p]);
      if (a.post_norm != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int e = 0; e < E; ++e) sum += x[p][e] * x[p][e];
        const float by = rsqrtf(tile.sum(sum, sums[0]) * per + a.eps);
        tile.load(static_cast<const T*>(a.post_norm), n, raw_x);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          Piece<T>::unpack(raw_x[p], w[p]);
#pragma unroll
          for (int e = 0; e < E; ++e) x[p][e] *= by * w[p][e];
        }
      }
      const float by = a.scale * gate;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (whole_gate) Piece<T>::unpack(raw_g[p], w[p]);
#pragma unroll
        for (int e = 0; e < E; ++e) r[p][e] += whole_gate ? by * w[p][e] * x[p][e] : by * x[p][e];
      }
      tile.store(static_cast<T*>(a.residual_out) + t * a.residual_out_stride, n, r);
    }
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < E; ++e) sum += r[p][e] * r[p][e];
    const float by = rsqrtf(tile.sum(sum, sums[1]) * per + a.eps);
    tile.load(static_cast<const T*>(a.pre_norm), n, raw_r);
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      Piece<T>::unpack(raw_r[p], w[p]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        r[p][e] *= by * w[p][e];
        top = max(top, __float_as_uint(r[p][e]) & 0x7fffffffu);
      }
    }
    if (a.out_scales == nullptr) {
      tile.store(static_cast<T*>(a.out) + t * a.out_stride, n, r);
    } else {
      const float step = step_of(tile.max(top, tops));
      if (tile.lane == 0) a.out_scales[t] = step;
      tile.store_bytes(static_cast<int8_t*>(a.out) + t * a.out_stride, n, r, step);
    }
    if constexpr (WAVES > 1) __syncthreads();  // the sums are read
  }
}

template <typename T, int WAVES, int P, bool VEC>
struct Norms {
  static hipError_t go(int64_t rows, const ResidentBlockNorms& a, hipStream_t stream) {
    using Tile = RowTile<T, WAVES, P, VEC>;
    return launch(k_block_norms<T, WAVES, P, VEC>, std::min(ceil_div(rows, Tile::kRows), kRowMaxBlocks), Tile::kThreads, 0, stream, a);
  }
};

// Every row that the kernel loads or stores as pieces starts at a multiple of 16 bytes.
template <typename T>
hipError_t launch_norms(const ResidentBlockNorms& a, hipStream_t stream) {
  constexpr int E = Piece<T>::kElems;
  const auto fits = [&](const void* p, int64_t stride, int bytes = 16) {
    return p == nullptr || (aligned(p, bytes) && (a.tokens == 1 || stride % E == 0));
  };
  const bool whole_gate = a.gate != nullptr && a.gate_strides[1] != 0;
  const bool vec = a.hidden % E == 0 && fits(a.x, a.x_stride) && fits(a.residual, a.residual_stride) &&
                   fits(a.residual_out, a.residual_out_stride) && fits(a.post_norm, 0) && fits(a.pre_norm, 0) &&
                   fits(a.out, a.out_stride, a.out_scales != nullptr ? E : 16) && (!whole_gate || fits(a.gate, a.gate_strides[0]));
  const int64_t pieces = ceil_div(a.hidden, E);
  return vec ? launch_rows<Norms, T, true>(pieces, a.tokens, a, stream) : launch_rows<Norms, T, false>(pieces, a.tokens, a, stream);
}

HeadRows rows_of(const void* p, int64_t stride, int64_t rows, int columns, int bytes) {
  const int64_t strides[2] = {stride, 0};
  return HeadRows(p, strides, rows, 1, columns, bytes);
}

bool norms_ok(const ResidentBlockNorms& a) {
  const int T = a.dtype_bytes;
  if (T != 2 && T != 4) return false;
  if (a.tokens < 0 || a.hidden <= 0 || a.hidden > kRowElems || !(a.eps >= 0.f) || a.scale != a.scale) return false;
  if (a.x_stride < 0 || a.residual_stride < 0 || a.residual_out_stride < 0 || a.out_stride < 0 || a.gate_strides[0] < 0) return false;
  if (a.gate_strides[1] != 0 && a.gate_strides[1] != 1) return false;
  if (a.tokens == 0) return true;
  if (a.residual == nullptr || a.pre_norm == nullptr || a.out == nullptr) return false;
  if (a.x == nullptr ? a.post_norm != nullptr || a.gate != nullptr || a.residual_out != nullptr : a.residual_out == nullptr) return false;
  const bool bytes = a.out_scales != nullptr;
  for (const void* p : {a.x, a.residual, a.post_norm, a.gate, a.pre_norm, static_cast<const void*>(a.residual_out)})
    if (!aligned(p, T)) return false;
  if (!aligned(a.out_scales, 4) || (!bytes && !aligned(a.out, T))) return false;
  // An output may take the place of an input, row by row; otherwise it lies apart from all else.  (Without x the
  // residual is the new residual too, so out lies apart from it.)
  const HeadRows out = rows_of(a.out, a.out_stride, a.tokens, a.hidden, bytes ? 1 : T);
  const HeadRows sum = rows_of(a.residual_out, a.residual_out_stride, a.tokens, a.hidden, T);
  const HeadRows steps = rows_of(a.out_scales, 1, a.tokens, 1, 4);
  if (!out.distinct() || (a.x != nullptr && (!sum.distinct() || !apart(sum, out)))) return false;
  if (bytes && (!apart(steps, out) || (a.x != nullptr && !apart(steps, sum)))) return false;
  const auto fits = [&](const void* p, int64_t stride, int64_t rows, int columns, bool same) {
    if (p == nullptr) return true;
    const HeadRows in = rows_of(p, stride, rows, columns, T);
    return (apart(out, in) || (same && !bytes && out.same(in))) && (a.x == nullptr || apart(sum, in) || (same && sum.same(in))) &&
           (!bytes || apart(steps, in));
  };
  const bool element_gate = a.gate_strides[0] != 0 && a.gate_strides[1] != 0;
  return fits(a.x, a.x_stride, a.tokens, a.hidden, true) && fits(a.residual, a.residual_stride, a.tokens, a.hidden, a.x != nullptr) &&
         fits(a.post_norm, 0, 1, a.hidden, false) && fits(a.pre_norm, 0, 1, a.hidden, false) &&
         fits(a.gate, a.gate_strides[0], a.gate_strides[0] != 0 ? a.tokens : 1, a.gate_strides[1] != 0 ? a.hidden : 1, element_gate);
}

}  // namespace
}  // namespace re

extern "C" int32_t resident_block_norms(const ResidentBlockNorms* args, void* stream) {
  using namespace re;
  if (args == nullptr || !norms_ok(*args)) return -1;
  if (args->tokens == 0) return 0;
  const DeviceScope device(args->device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->dtype_bytes == 2 ? launch_norms<bf16_t>(*args, s) : launch_norms<float>(*args, s);
  return e == hipSuccess ? 0 : -2;
}
