// Rows to 8-bit integers with a step of their own, and the product of such rows
// with 8-bit weights.
#include "re_rows.h"

namespace re {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// ---- rows to 8 bits ----

template <typename T, int WAVES, int P, bool VEC>
__global__ void __launch_bounds__(row_threads(WAVES)) k_quantize_rows(ResidentQuantizeRows a) {
  using Tile = RowTile<T, WAVES, P, VEC>;
  constexpr int E = Tile::E, kSpan = Tile::kLanes * P * E;
  __shared__ uint32_t tops[WAVES];
  const Tile tile(threadIdx.x);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * Tile::kRows + threadIdx.x / Tile::kLanes; t < a.rows;
       t += static_cast<int64_t>(gridDim.x) * Tile::kRows) {
    const T* row = static_cast<const T*>(a.x) + t * a.x_stride;
    re_u32x4 raw[P];
    float x[P][E];
    uint32_t top = 0;
    // Rows beyond the registers (of 65,536 bf16 or 32,768 fp32) are read twice.
    for (int at = 0; at < a.columns; at += kSpan) {
      tile.load(row + at, a.columns - at, raw);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        Piece<T>::unpack(raw[p], x[p]);
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(x[p][e]) & 0x7fffffffu);
      }
    }
    const float step = step_of(tile.max(top, tops));
    if (tile.lane == 0) a.scales[t] = step;
    int8_t* out = a.out + t * a.out_stride;
    if (a.columns <= kSpan) {
      tile.store_bytes(out, a.columns, x, step);
    } else {
      for (int at = 0; at < a.columns; at += kSpan) {
        tile.load(row + at, a.columns - at, raw);
#pragma unroll
        for (int p = 0; p < P; ++p) Piece<T>::unpack(raw[p], x[p]);
        tile.store_bytes(out + at, a.columns - at, x, step);
      }
    }
    if constexpr (WAVES > 1) __syncthreads();  // the maxima are read
  }
}

template <typename T, int WAVES, int P, bool VEC>
struct Quantize {
  static hipError_t go(int64_t rows, const ResidentQuantizeRows& a, hipStream_t stream) {
    using Tile = RowTile<T, WAVES, P, VEC>;
    return launch(k_quantize_rows<T, WAVES, P, VEC>, std::min(ceil_div(rows, Tile::kRows), kRowMaxBlocks), Tile::kThreads, 0, stream, a);
  }
};

template <typename T>
hipError_t launch_quantize(const ResidentQuantizeRows& a, hipStream_t stream) {
  constexpr int E = Piece<T>::kElems;
  const bool one = a.rows == 1;
  const bool vec = a.columns % E == 0 && aligned(a.x, 16) && (one || a.x_stride % E == 0) && aligned(a.out, E) && (one || a.out_stride % E == 0);
  const int64_t pieces = std::min<int64_t>(ceil_div(a.columns, E), 16 * 64 * kRowPieces);
  return vec ? launch_rows<Quantize, T, true>(pieces, a.rows, a, stream) : launch_rows<Quantize, T, false>(pieces, a.rows, a, stream);
}

hipError_t launch_quantize(const ResidentQuantizeRows& a, hipStream_t stream) {
  return a.dtype_bytes == 2 ? launch_quantize<bf16_t>(a, stream) : launch_quantize<float>(a, stream);
}

HeadRows rows_of(const void* p, int64_t stride, int64_t rows, int columns, int bytes) {
  const int64_t strides[2] = {stride, 0};
  return HeadRows(p, strides, rows, 1, columns, bytes);
}

bool quantize_ok(const ResidentQuantizeRows& a) {
  const int T = a.dtype_bytes;
  if ((T != 2 && T != 4) || a.rows < 0 || a.columns <= 0 || a.columns > (1 << 30) || a.x_stride < 0 || a.out_stride < 0) return false;
  if (a.rows == 0) return true;
  if (a.x == nullptr || a.out == nullptr || a.scales == nullptr || !aligned(a.x, T) || !aligned(a.scales, 4)) return false;
  const HeadRows in = rows_of(a.x, a.x_stride, a.rows, a.columns, T), out = rows_of(a.out, a.out_stride, a.rows, a.columns, 1);
  const HeadRows steps = rows_of(a.scales, 1, a.rows, 1, 4);
  return out.distinct() && apart(out, in) && apart(steps, in) && apart(steps, out);
}

// ---- the product ----

struct ProductArgs {
  ResidentInt8Linear a;
  const int8_t* x;       // the tokens in 8 bits: the caller's, or the workspace's
  const float* x_scales;
  int64_t x_stride;
};

__device__ __forceinline__ float bias_of(const void* bias, int64_t n, int bytes) {
  return bias == nullptr ? 0.f : bytes == 2 ? bf16_to_f(static_cast<const bf16_t*>(bias)[n]) : static_cast<const float*>(bias)[n];
}

constexpr int kProductThreads = 256, kProductTile = 64;

// A workgroup: 64 tokens x 64 channels, a wave 16 of the channels.  Operands of
// v_mfma_i32_16x16x64_i8 straight from memory: lane (x = lane % 16, y = lane / 16)
// holds 16 bytes of row x at 16 y; the result holds column x (a token), rows 4 y ..
// 4 y + 3 (channels).
__global__ void __launch_bounds__(kProductThreads) k_int8_linear(ProductArgs args) {
  const ResidentInt8Linear& a = args.a;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_index(tid), x = lane & 15, y = lane >> 4;
  const int tiles = (a.outer + kProductTile - 1) / kProductTile;
  const int n0 = blockIdx.x % tiles * kProductTile + 16 * w;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / tiles) * kProductTile;
  i32x4 sum[4] = {};
  for (int k = 0; k < a.inner; k += 64) {
    const int at = k + 16 * y;
    const bool there = at < a.inner;
    const i32x4 rows = there && n0 + x < a.outer ? *reinterpret_cast<const i32x4*>(a.weight + (n0 + x) * a.weight_stride + at) : i32x4{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + 16 * i + x;
      const i32x4 col = there && m < a.tokens ? *reinterpret_cast<const i32x4*>(args.x + m * args.x_stride + at) : i32x4{};
      sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(rows, col, sum[i], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 16 * i + x;
    if (m >= a.tokens) continue;
    const float step = args.x_scales[m];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + 4 * y + e;
      if (n >= a.outer) continue;
      const float v = static_cast<float>(sum[i][e]) * (step * a.weight_scales[n]) + bias_of(a.bias, n, a.out_bytes);
      if (a.out_bytes == 2) static_cast<bf16_t*>(a.out)[m * a.out_stride + n] = f_to_bf16(v);
      else static_cast<float*>(a.out)[m * a.out_stride + n] = v;
    }
  }
}

// The workspace of a call whose tokens are not in 8 bits: their bytes, then their steps.
struct LinearBytes {
  int64_t rows, steps;
};
LinearBytes linear_bytes(const ResidentInt8Linear& a) {
  if (a.x_bytes == 1) return {0, 0};
  return {round_up(static_cast<int64_t>(a.tokens) * a.inner, 16), static_cast<int64_t>(a.tokens) * 4};
}

bool linear_ok(const ResidentInt8Linear& a) {
  if ((a.x_bytes != 1 && a.x_bytes != 2 && a.x_bytes != 4) || (a.out_bytes != 2 && a.out_bytes != 4)) return false;
  // Sums of products of bytes fit 32 bits up to here.
  if (a.tokens < 0 || a.outer <= 0 || a.inner <= 0 || a.inner % 16 != 0 || a.inner >= 1 << 17) return false;
  if (a.x_stride < 0 || a.weight_stride < 0 || a.out_stride < 0 || a.workspace_bytes < 0) return false;
  if (ceil_div(a.tokens, kProductTile) * ceil_div(a.outer, kProductTile) >= 1 << 24) return false;
  if (a.tokens == 0) return true;
  if (a.x == nullptr || a.weight == nullptr || a.weight_scales == nullptr || a.out == nullptr || (a.x_bytes == 1 && a.x_scales == nullptr))
    return false;
  if (!aligned(a.x, a.x_bytes == 1 ? 16 : a.x_bytes) || (a.x_bytes == 1 && a.tokens > 1 && a.x_stride % 16 != 0)) return false;
  if (!aligned(a.weight, 16) || (a.outer > 1 && a.weight_stride % 16 != 0)) return false;
  if (!aligned(a.out, a.out_bytes) || !aligned(a.bias, a.out_bytes) || !aligned(a.x_scales, 4) || !aligned(a.weight_scales, 4) ||
      !aligned(a.workspace, 16))
    return false;
  const HeadRows out = rows_of(a.out, a.out_stride, a.tokens, a.outer, a.out_bytes);
  return out.distinct() && apart(out, rows_of(a.x, a.x_stride, a.tokens, a.inner, a.x_bytes)) &&
         apart(out, rows_of(a.weight, a.weight_stride, a.outer, a.inner, 1)) && apart(out, rows_of(a.weight_scales, 0, 1, a.outer, 4)) &&
         (a.bias == nullptr || apart(out, rows_of(a.bias, 0, 1, a.outer, a.out_bytes))) &&
         (a.x_bytes != 1 || apart(out, rows_of(a.x_scales, 0, 1, a.tokens, 4)));
}

}  // namespace
}  // namespace re

extern "C" int32_t resident_quantize_rows(const ResidentQuantizeRows* args, void* stream) {
  using namespace re;
  if (args == nullptr || !quantize_ok(*args)) return -1;
  if (args->rows == 0) return 0;
  const DeviceScope device(args->device);
  if (!device.ok()) return -2;
  return launch_quantize(*args, static_cast<hipStream_t>(stream)) == hipSuccess ? 0 : -2;
}

extern "C" int64_t resident_int8_linear_workspace(const ResidentInt8Linear* args) {
  using namespace re;
  if (args == nullptr || !linear_ok(*args)) return -1;
  if (args->tokens == 0) return 0;
  const LinearBytes b = linear_bytes(*args);
  return b.rows + b.steps;
}

extern "C" int32_t resident_int8_linear(const ResidentInt8Linear* args, void* stream) {
  using namespace re;
  if (args == nullptr || !linear_ok(*args)) return -1;
  if (args->tokens == 0) return 0;
  const LinearBytes b = linear_bytes(*args);
  if (b.rows + b.steps > 0 && (args->workspace == nullptr || args->workspace_bytes < b.rows + b.steps)) return -1;
  const DeviceScope device(args->device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  ProductArgs p{*args, static_cast<const int8_t*>(args->x), args->x_scales, args->x_stride};
  if (args->x_bytes != 1) {
    int8_t* rows = static_cast<int8_t*>(args->workspace);
    float* steps = reinterpret_cast<float*>(rows + b.rows);
    p.x = rows;
    p.x_scales = steps;
    p.x_stride = args->inner;
    const ResidentQuantizeRows q{args->x, rows, steps, args->x_stride, args->inner, args->tokens, args->inner, args->x_bytes, args->device};
    if (launch_quantize(q, s) != hipSuccess) return -2;
  }
  const int64_t blocks = ceil_div(args->tokens, kProductTile) * ceil_div(args->outer, kProductTile);
  return launch(k_int8_linear, blocks, kProductThreads, 0, s, p) == hipSuccess ? 0 : -2;
}
