// New tokens into a paged cache: the norm of each query and key head, the
// rotation by the token's position, and the write of keys and values.
#include "re_ops.h"

namespace re {
namespace {

constexpr int kWriteThreads = 256;
constexpr int kWriteTokens = 8;               // tokens of one workgroup at most
constexpr int64_t kWriteMaxBlocks = 1 << 20;  // the kernel strides over the rest

struct WriteArgs {
  ResidentKvWrite a;
  int group;  // tokens of one workgroup
};

// v summed over LANES neighbouring lanes (a power of two).
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v, int lane) {
  v = xor_add<1>(v, lane);
  v = xor_add<2>(v, lane);
  if constexpr (LANES > 4) v = xor_add<4>(v, lane);
  if constexpr (LANES > 8) v = xor_add<8>(v, lane);
  if constexpr (LANES > 16) v = xor_add<16>(v, lane);
  return v;
}

// Sine and cosine of an angle in turns, in 64 bits and rounded once: the angle less
// its nearest quarter turn, both by their Taylor series on the eighth of a turn that
// is left (x^13 / 13! and x^14 / 14! are below 2^-36 of what they end), swapped and
// negated by the quarter.  It costs what fp32 sines of the rounded turn do (64,000
// tokens 262 us); the library's in 64 bits, whose registers leave four waves on a
// SIMD and not five, 303.
__device__ __forceinline__ void sine_cosine(double turns, float& sine, float& cosine) {
  const double part = turns - rint(turns), quarters = rint(4.0 * part), x = (part - 0.25 * quarters) * 6.283185307179586477, z = x * x;
  double s = -1.0 / 39916800, c = 1.0 / 479001600;
  s = fma(s, z, 1.0 / 362880);
  c = fma(c, z, -1.0 / 3628800);
  s = fma(s, z, -1.0 / 5040);
  c = fma(c, z, 1.0 / 40320);
  s = fma(s, z, 1.0 / 120);
  c = fma(c, z, -1.0 / 720);
  s = fma(s, z, -1.0 / 6);
  c = fma(c, z, 1.0 / 24);
  s = fma(s, z, 1.0);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const float fs = static_cast<float>(s * x), fc = static_cast<float>(c);
  const int quarter = static_cast<int>(quarters);
  sine = quarter & 1 ? fc : fs;
  cosine = quarter & 1 ? fs : fc;
  if (quarter & 2) sine = -sine;
  if ((quarter + 1) & 2) cosine = -cosine;
}

// Every value is read and written once, with a few operations on each, so HBM
// bounds this: 64,000 tokens of 28 + 2 x 4 heads of 128 in bf16 (1.18 GB in and
// out) take 262 us, 4.5 TB/s, where a large copy reaches 4.8.  Stores go past the
// caches (8,000 tokens: 28 us, 41 through them).  A lane holds 16 bytes of a head's first half and the 16 of its
// second half that rotate with them, so a head is d / 16 lanes (bf16; d / 8
// fp32), its norm a sum over those, and a workgroup works on 256 / lanes heads
// at a time.  A token's angles, sines and cosines are computed in 64 bits once for
// all of its heads and kept in LDS, rounded once.
template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) k_kv_write(WriteArgs args) {
  constexpr int E = Piece<T>::kElems, kLanes = D / 2 / E, kHeads = kWriteThreads / kLanes;
  const ResidentKvWrite& a = args.a;
  const ResidentKvCache& c = a.cache;
  __shared__ __align__(16) float cos_s[kWriteTokens][D / 2], sin_s[kWriteTokens][D / 2];
  const int tid = threadIdx.x, lane = tid & 63, e = tid % kLanes * E;
  const int per_token = a.heads + 2 * c.kv_heads, slot_count = c.pages * c.block_size;
  re_u32x4 norms[2][2] = {};  // of the lane's elements: queries' and keys', first and second half
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const T* norm = static_cast<const T*>(i == 0 ? a.q_norm : a.k_norm);
    if (norm == nullptr) continue;
    norms[i][0] = *reinterpret_cast<const re_u32x4*>(norm + e);
    norms[i][1] = *reinterpret_cast<const re_u32x4*>(norm + D / 2 + e);
  }
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * args.group; t0 < a.tokens; t0 += static_cast<int64_t>(gridDim.x) * args.group) {
    const int tokens = static_cast<int>(min(static_cast<int64_t>(args.group), a.tokens - t0));
    const int units = tokens * per_token;
    // The head of this lane's unit: its token in the group and its part
    // (queries, then keys, then values).
    int t = 0, part = tid / kLanes;
    auto wrap = [&] {
      while (part >= per_token) {
        part -= per_token;
        ++t;
      }
    };
    auto source = [&]() -> const T* {
      const int64_t at = t0 + t;
      if (part < a.heads) return static_cast<const T*>(a.q) + at * a.q_strides[0] + part * a.q_strides[1];
      const int h = part - a.heads;
      if (h < c.kv_heads) return static_cast<const T*>(a.k) + at * a.k_strides[0] + h * a.k_strides[1];
      return static_cast<const T*>(a.v) + at * a.v_strides[0] + (h - c.kv_heads) * a.v_strides[1];
    };
    re_u32x4 lo = {}, hi = {};
    wrap();
    if (tid / kLanes < units) {
      const T* src = source();
      lo = *reinterpret_cast<const re_u32x4*>(src + e);
      hi = *reinterpret_cast<const re_u32x4*>(src + D / 2 + e);
    }
    __syncthreads();  // the angles before are no longer read
    for (int i = tid; i < tokens * (D / 2); i += kWriteThreads) {
      const double turns = static_cast<double>(a.positions[t0 + i / (D / 2)]) * a.inv_freq[i % (D / 2)] * 0.15915494309189533577;  // / 2 pi
      sine_cosine(turns, sin_s[0][i], cos_s[0][i]);
    }
    __syncthreads();
    for (int u = tid / kLanes; u < units; u += kHeads) {
      const int now_t = t, now_part = part;
      const re_u32x4 now_lo = lo, now_hi = hi;
      part += kHeads;
      wrap();
      if (u + kHeads < units) {
        const T* src = source();
        lo = *reinterpret_cast<const re_u32x4*>(src + e);
        hi = *reinterpret_cast<const re_u32x4*>(src + D / 2 + e);
      }
      const bool is_q = now_part < a.heads, is_v = now_part >= a.heads + c.kv_heads;
      const int h = now_part - (is_q ? 0 : is_v ? a.heads + c.kv_heads : a.heads);
      re_u32x4 out_lo = now_lo, out_hi = now_hi;
      if (!is_v) {
        float x[E], y[E];
        Piece<T>::unpack(now_lo, x);
        Piece<T>::unpack(now_hi, y);
        if ((is_q ? a.q_norm : a.k_norm) != nullptr) {
          float sum = 0.f, nx[E], ny[E];
#pragma unroll
          for (int i = 0; i < E; ++i) sum += x[i] * x[i] + y[i] * y[i];
          const float r = rsqrtf(lanes_sum<kLanes>(sum, lane) * (1.f / D) + a.eps);
          Piece<T>::unpack(is_q ? norms[0][0] : norms[1][0], nx);
          Piece<T>::unpack(is_q ? norms[0][1] : norms[1][1], ny);
#pragma unroll
          for (int i = 0; i < E; ++i) {
            x[i] *= r * nx[i];
            y[i] *= r * ny[i];
          }
        }
        float co[E], si[E];
#pragma unroll
        for (int i = 0; i < E; i += 4) {
          const re_f32x4 cv = *reinterpret_cast<const re_f32x4*>(&cos_s[0][now_t * (D / 2) + e + i]);
          const re_f32x4 sv = *reinterpret_cast<const re_f32x4*>(&sin_s[0][now_t * (D / 2) + e + i]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            co[i + q] = cv[q];
            si[i + q] = sv[q];
          }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float n = x[i];
          x[i] = n * co[i] - y[i] * si[i];
          y[i] = y[i] * co[i] + n * si[i];
        }
        out_lo = Piece<T>::pack(x);
        out_hi = Piece<T>::pack(y);
      }
      T* dst;
      if (is_q) {
        dst = static_cast<T*>(a.q_out) + (t0 + now_t) * a.q_out_strides[0] + h * a.q_out_strides[1];
      } else {
        const int slot = a.slots[t0 + now_t];
        if (slot < 0 || slot >= slot_count) continue;
        const int page = slot / c.block_size, at = slot - page * c.block_size;
        dst = is_v ? static_cast<T*>(c.values) + page * c.value_strides[0] + at * c.value_strides[1] + h * c.value_strides[2]
                   : static_cast<T*>(c.keys) + page * c.key_strides[0] + at * c.key_strides[1] + h * c.key_strides[2];
        if (!is_v && e == 0) {
          if (c.weights != nullptr) c.weights[page * c.weight_strides[0] + h * c.weight_strides[1] + at] = 0.f;
          if (c.positions != nullptr)
            c.positions[page * c.position_strides[0] + h * c.position_strides[1] + at] = static_cast<int32_t>(a.positions[t0 + now_t]);
        }
      }
      __builtin_nontemporal_store(out_lo, reinterpret_cast<re_u32x4*>(dst + e));
      __builtin_nontemporal_store(out_hi, reinterpret_cast<re_u32x4*>(dst + D / 2 + e));
    }
  }
}

// Tokens of a workgroup: as few as give every lane a head, so that few tokens
// spread over the chip; where there are many, as many as give every lane an angle
// (28 + 2 x 4 heads of 128, one against four tokens: 11.6 and 13.1 us for 2,000
// of them, 18.7 and 16.3 for 4,000, 327 and 265 for 64,000; 4 + 2 x 2 heads of 64,
// one against eight: 4.2 and 4.4 us for 64, 6.5 and 4.8 for 2,000).
template <typename T, int D>
hipError_t launch_write(const ResidentKvWrite& a, hipStream_t stream) {
  constexpr int kHeads = kWriteThreads / (D / 2 / Piece<T>::kElems);
  const int full = std::min(kWriteTokens, kWriteThreads / (D / 2));
  const int fill = static_cast<int>(std::min<int64_t>(full, ceil_div(kHeads, a.heads + 2 * static_cast<int64_t>(a.cache.kv_heads))));
  const WriteArgs args{a, a.tokens >= 768 * full ? full : fill};
  return launch(k_kv_write<T, D>, std::min(ceil_div(a.tokens, args.group), kWriteMaxBlocks), kWriteThreads, 0, stream, args);
}

template <typename T>
hipError_t launch_write(const ResidentKvWrite& a, hipStream_t stream) {
  const int d = a.cache.head_dim;
  return d == 64 ? launch_write<T, 64>(a, stream) : d == 128 ? launch_write<T, 128>(a, stream) : launch_write<T, 256>(a, stream);
}

bool write_ok(const ResidentKvWrite& a) {
  if (!cache_ok(a.cache) || a.tokens < 0 || a.heads <= 0 || a.heads > (1 << 20) || a.cache.kv_heads > (1 << 20) || a.reserved != 0)
    return false;
  if (!(a.eps >= 0.f) || a.inv_freq == nullptr) return false;
  if (a.tokens == 0) return true;
  const int T = a.cache.dtype_bytes;
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.q_out == nullptr || a.positions == nullptr || a.slots == nullptr)
    return false;
  const int d = a.cache.head_dim, kv_heads = a.cache.kv_heads;
  const HeadRows out(a.q_out, a.q_out_strides, a.tokens, a.heads, d, T);
  return aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.q_out, 16) && aligned(a.q_norm, 16) &&
         aligned(a.k_norm, 16) && aligned(a.inv_freq, 4) && aligned(a.positions, 8) && aligned(a.slots, 4) &&
         row_strides_ok(a.q_strides, {a.tokens, a.heads}, T) && row_strides_ok(a.q_out_strides, {a.tokens, a.heads}, T) &&
         row_strides_ok(a.k_strides, {a.tokens, a.cache.kv_heads}, T) &&
         row_strides_ok(a.v_strides, {a.tokens, a.cache.kv_heads}, T) &&
         output_ok(out, HeadRows(a.q, a.q_strides, a.tokens, a.heads, d, T)) &&
         apart(out, HeadRows(a.k, a.k_strides, a.tokens, kv_heads, d, T)) &&
         apart(out, HeadRows(a.v, a.v_strides, a.tokens, kv_heads, d, T));
}

}  // namespace
}  // namespace re

extern "C" int32_t resident_kv_write(const ResidentKvWrite* args, void* stream) {
  using namespace re;
  if (args == nullptr || !write_ok(*args)) return -1;
  if (args->tokens == 0) return 0;
  const DeviceScope device(args->cache.device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = args->cache.dtype_bytes == 2 ? launch_write<bf16_t>(*args, s) : launch_write<float>(*args, s);
  return e == hipSuccess ? 0 : -2;
}
