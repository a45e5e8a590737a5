// Rows to 8-bit integers with a step of their own, and the product of such rows
// with 8-bit weights: out = T((sum_k x_k w_k) (s_x s_w) + bias).  The sum is exact in 32
// bits (inner is below 2^17), so ranges of K and waves are added in any order; the
// scales and the bias are applied in fp32 once, in the epilogue.
//
// Up to 64 tokens the weights' bytes are the work and k_int8_few streams them; above,
// k_int8_tiles is a matrix product on v_mfma_i32_16x16x64_i8.
#include "re_gemm_tiles.h"
#include "re_int8_plan.h"
#include "re_rows.h"

namespace re {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// ---- rows to 8 bits ----

// One pass: a row stays in registers between its maximum and its bytes.  4,096 rows of
// 18,944 bf16 37 us (6.3 TB/s), 64,000 of 3,584 117 us (5.9); 4 of 3,584 3 us, the
// latency of one load, the maximum and the store.
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
    // Rows beyond the registers (32,768) are read twice.
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
  const int64_t pieces = std::min<int64_t>(ceil_div(a.columns, E), kRowElems / E);
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
  int vec;               // 1: the output's rows start at multiples of 16 bytes
  int ranges;            // of K; more than one: their sums go to part, [ranges][tokens][part_stride]
  int32_t* part;
  int64_t part_stride;
  int m_tiles, n_tiles;
  int few_rows;  // channels of a workgroup of k_int8_few
};

__device__ __forceinline__ float bias_of(const void* bias, int64_t n, int bytes) {
  return bias == nullptr ? 0.f : bytes == 2 ? bf16_to_f(static_cast<const bf16_t*>(bias)[n]) : static_cast<const float*>(bias)[n];
}

// 64 MJ tokens x GN channels (64 to 256) per workgroup of 8 waves, K in steps of 128 bytes,
// over all of K or over one of its ranges: the stages, their swizzle and their
// barrier are the bf16 product's (a row of a stage is 128 bytes there too), with
// v_mfma_i32_16x16x64_i8 for its products, so a byte that passes through LDS does
// twice the work.  The last step of K is filled up with zeros.  What bounds it is what
// bounds that one, the loop that feeds the matrix cores from LDS: 4,096 x 3,584 x 18,944
// 276-287 us in a run of calls (1.94 to 2.01 POP/s; under the profiler 284 to 343, the median
// 308), 4,096 x 18,944 x 3,584 232-245 us (2.3 to 2.4), 1,000 x 3,584 x 4,608 27 us, 192
// workgroups on 256 CUs.
__device__ const uint4 kZeros = {0, 0, 0, 0};

constexpr int tile_lds_bytes(int mj, int st, int gn) {
  return std::max(gemm_tile_m(mj) * gemm_out_ld(gn) * 2, st * gemm_stage_bytes(mj, gn));
}

template <int MJ, int ST, int GN, bool PART>
__global__ void __launch_bounds__(kGthreads, 1) k_int8_tiles(ProductArgs args) {
  extern __shared__ __align__(16) unsigned char gsm[];
  const ResidentInt8Linear& a = args.a;
  constexpr int kTm = gemm_tile_m(MJ), kStage = gemm_stage_bytes(MJ, GN), kOutLd = gemm_out_ld(GN);
  constexpr int kWInsts = GN / 64, kInsts = kWInsts + MJ;  // 1 KB loads (8 rows) of each wave and stage
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(tid);
  int mt, nt, ks;
  gemm_tile_of(blockIdx.x, args.m_tiles, args.n_tiles, args.ranges, mt, nt, ks);
  const int m0 = mt * kTm, n0 = nt * GN;
  const int steps = (a.inner + kGrowBytes - 1) / kGrowBytes;
  const int k_begin = PART ? static_cast<int>(static_cast<int64_t>(ks) * steps / args.ranges) : 0;
  const int nk = (PART ? static_cast<int>(static_cast<int64_t>(ks + 1) * steps / args.ranges) : steps) - k_begin;
  // The step that K ends in, of this range's; -1: none does.
  const int rest = a.inner % kGrowBytes, tail = rest != 0 && k_begin + nk == steps ? nk - 1 : -1;
  // Loads: every wave GN / 8 rows of weights and 8 MJ tokens.  Rows past the end
  // read a valid row (clamped) whose results are never stored.
  const char* wbase = reinterpret_cast<const char*>(a.weight) + n0 * a.weight_stride + static_cast<int64_t>(k_begin) * kGrowBytes;
  const char* xbase = reinterpret_cast<const char*>(args.x) + m0 * args.x_stride + static_cast<int64_t>(k_begin) * kGrowBytes;
  const int wrow = wave * (GN / 8), xrow = GN + wave * 8 * MJ;
  uint32_t goff[kInsts];
#pragma unroll
  for (int i = 0; i < kInsts; ++i) {
    const int row = (i < kWInsts ? wrow + i * 8 : xrow + (i - kWInsts) * 8) + (lane >> 3);
    const int chunk = (lane & 7) ^ gemm_swz(row);
    goff[i] = i < kWInsts ? static_cast<uint32_t>(min(row, a.outer - n0 - 1) * static_cast<int>(a.weight_stride) + chunk * 16)
                          : static_cast<uint32_t>(min(row - GN, a.tokens - m0 - 1) * static_cast<int>(args.x_stride) + chunk * 16);
  }
  auto issue = [&](int kt, int buf) {
    const int64_t kb = static_cast<int64_t>(kt) * kGrowBytes;
    unsigned char* l = gsm + buf * kStage;
    auto at = [&](int i) { return l + (i < kWInsts ? wrow * kGrowBytes + i * 1024 : xrow * kGrowBytes + (i - kWInsts) * 1024); };
    if (kt != tail) {
#pragma unroll
      for (int i = 0; i < kInsts; ++i)
        __builtin_amdgcn_global_load_lds((gemm_gptr)((i < kWInsts ? wbase : xbase) + kb + goff[i]), (gemm_lptr)at(i), 16, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kInsts; ++i) {
        const int row = (i < kWInsts ? wrow + i * 8 : xrow + (i - kWInsts) * 8) + (lane >> 3);
        const bool there = ((lane & 7) ^ gemm_swz(row)) * 16 < rest;
        const char* p = (i < kWInsts ? wbase : xbase) + kb + goff[i];
        __builtin_amdgcn_global_load_lds((gemm_gptr)(there ? p : reinterpret_cast<const char*>(&kZeros)), (gemm_lptr)at(i), 16, 0, 0);
      }
    }
  };
  constexpr int kWn = gemm_waves_n(MJ), NI = GN / 16 / kWn, MI = 4 * MJ / (kGwaves / kWn);
  const int wn = wave % kWn, wm = wave / kWn;
  i32x4 acc[NI][MI] = {};
  const int fr = lane & 15, fq = lane >> 4;
  const int frag_off[2] = {fr * kGrowBytes + ((fq ^ gemm_swz(fr)) * 16), fr * kGrowBytes + (((4 + fq) ^ gemm_swz(fr)) * 16)};
  // fragment sets: [set][0 .. NI - 1] weights (n), [set][NI ..] tokens (m)
  constexpr int kFrags = NI + MI, kProds = NI * MI;
  i32x4 f[2][kFrags];
  auto read_frag = [&](int set, int idx, int st, int ks2) {
    const int row0 = idx < NI ? (wn * NI + idx) * 16 : GN + (wm * MI + idx - NI) * 16;
    f[set][idx] = *reinterpret_cast<const i32x4*>(gsm + st * kStage + row0 * kGrowBytes + frag_off[ks2]);
  };
  auto read_set = [&](int set, int st, int ks2) {
#pragma unroll
    for (int i = 0; i < kFrags; ++i) read_frag(set, i, st, ks2);
  };
  const int first = min(ST, nk);
  for (int s = 0; s < first; ++s) issue(s, s);
  if (first == ST)
    __builtin_amdgcn_s_waitcnt(gemm_wait_vm((ST - 1) * kInsts));  // this wave's stage 0
  else
    __builtin_amdgcn_s_waitcnt(gemm_wait_vm(0));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  read_set(0, 0, 0);
  __builtin_amdgcn_sched_barrier(0);
  int ring = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const int st = ST == 2 ? kt & 1 : ring, nst = ST == 2 ? st ^ 1 : ring + 1 == ST ? 0 : ring + 1;
    read_set(1, st, 1);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[0][i], f[0][NI + j], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int r = 0; r < kFrags; ++r) {  // fragment reads spread over the products
      __builtin_amdgcn_sched_group_barrier(0x008, kProds / kFrags > 0 ? kProds / kFrags : 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    // stage kt + 1 complete (stages kt + 2 .. kt + ST - 1 may be in flight), stage kt's buffer free
    if (ST > 2 && kt + ST - 1 < nk)
      gemm_stage_barrier<(ST - 2) * kInsts>();
    else
      gemm_stage_barrier();
    const bool more = kt + ST < nk;
#pragma unroll
    for (int p = 0; p < kProds; ++p) {
      const int i = p / MI, j = p % MI;
      if (p == 0 && wave < 4 && more) issue(kt + ST, st);
      if (p == kProds * 3 / 8 && wave >= 4 && more) issue(kt + ST, st);
      if (j == 0) __builtin_amdgcn_sched_barrier(0);
      acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[1][i], f[1][NI + j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int r = gemm_reads_by(kFrags, kProds, p); r < gemm_reads_by(kFrags, kProds, p + 1); ++r) read_frag(0, r, nst, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    ring = nst;
  }
  // acc[i][j] value v of lane l: n = 16 i + 4 (l / 16) + v, m = 16 j + l % 16 within the wave's block
  if constexpr (PART) {
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int m = m0 + (wm * MI + j) * 16 + fr, n = n0 + (wn * NI + i) * 16 + 4 * fq;
        if (m < a.tokens && n < a.outer)
          *reinterpret_cast<i32x4*>(args.part + (static_cast<int64_t>(ks) * a.tokens + m) * args.part_stride + n) = acc[i][j];
      }
    return;
  }
  gemm_stage_barrier();
  bf16_t* T = reinterpret_cast<bf16_t*>(gsm);
  float step[MI];
#pragma unroll
  for (int j = 0; j < MI; ++j) step[j] = args.x_scales[min(m0 + (wm * MI + j) * 16 + fr, a.tokens - 1)];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int nl = (wn * NI + i) * 16 + 4 * fq;
    float by[4], add[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      by[e] = a.weight_scales[min(n0 + nl + e, a.outer - 1)];
      add[e] = bias_of(a.bias, min(n0 + nl + e, a.outer - 1), a.out_bytes);
    }
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int ml = (wm * MI + j) * 16 + fr;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(acc[i][j][e]) * (step[j] * by[e]) + add[e];
      if (a.out_bytes == 2) {
        *reinterpret_cast<uint2*>(T + ml * kOutLd + nl) = make_uint2(f2_to_bf16x2(y[0], y[1]), f2_to_bf16x2(y[2], y[3]));
      } else if (m0 + ml < a.tokens) {
        float* to = static_cast<float*>(a.out) + (m0 + ml) * a.out_stride + n0 + nl;
        if (args.vec && n0 + nl + 4 <= a.outer) {
          *reinterpret_cast<re_f32x4*>(to) = re_f32x4{y[0], y[1], y[2], y[3]};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + nl + e < a.outer) to[e] = y[e];
        }
      }
    }
  }
  if (a.out_bytes != 2) return;
  gemm_stage_barrier();
#pragma unroll 4
  for (int idx = tid; idx < kTm * GN / 8; idx += kGthreads) {
    const int r = idx / (GN / 8), c = idx % (GN / 8) * 8;
    if (m0 + r >= a.tokens || n0 + c >= a.outer) continue;
    const re_u32x4 t = *reinterpret_cast<const re_u32x4*>(T + r * kOutLd + c);
    bf16_t* to = static_cast<bf16_t*>(a.out) + (m0 + r) * a.out_stride + n0 + c;
    if (args.vec && n0 + c + 8 <= a.outer) {
      *reinterpret_cast<re_u32x4*>(to) = t;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n0 + c + e < a.outer) to[e] = static_cast<bf16_t>(t[e / 2] >> (16 * (e % 2)));
    }
  }
}

// Few tokens (up to 64): the weights' bytes are all the work, and every CU streams
// its share of them.  A workgroup has `few_rows` channels (NT tiles of 16 at most) and
// all tokens (MT tiles), its 8 waves every eighth 128-byte step of its K range, all
// tiles of each.  What a wave reads passes through a ring of its own in LDS, D places
// of 16 rows x 128 bytes (two 1 KB loads, full lines), so that nothing waits for
// another wave until the sums are added at the end, in whole numbers and therefore
// in any order.  4 tokens, weights cold: 3,584 x 18,944 13.2 us (5.2 TB/s; a plain read of
// as many bytes takes 11.2, the same loads without the products 12.4), x 37,888 24.8;
// 18,944 x 3,584 16 us, where 14 channels a workgroup come with as many tokens' bytes; 64
// tokens 3,584 x 18,944 18.6 us, a third of it the tokens, which every CU reads.  The same
// with each tile's scales requested after its sums took 18.6 us for 4 tokens, through the
// caches 2 us longer.
constexpr int kFewPlaces = 9;  // 8 waves x 9 x 2 KB: 144 of 160 KB
constexpr int kPlaceBytes = 16 * kGrowBytes;
constexpr int kStream = 2;  // a load's non-temporal bit

// MH: halves of the token tiles.  The second half of a single tile is not loaded for
// up to 8 tokens: what lies in its place gives products that are not stored.
template <int MH, int NT, bool PART>
__global__ void __launch_bounds__(kGthreads, 1) k_int8_few(ProductArgs args) {
  extern __shared__ __align__(16) unsigned char gsm[];
  constexpr int D = kFewPlaces, MT = (MH + 1) / 2, kItems = MT + NT;
  const ResidentInt8Linear& a = args.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(tid);
  const int nt = blockIdx.x % args.n_tiles, ks = blockIdx.x / args.n_tiles;
  const int n0 = nt * args.few_rows, rows = min(args.few_rows, a.outer - n0);
  const int steps = (a.inner + kGrowBytes - 1) / kGrowBytes;
  const int k_begin = PART ? static_cast<int>(static_cast<int64_t>(ks) * steps / args.ranges) : 0;
  const int k_end = PART ? static_cast<int>(static_cast<int64_t>(ks + 1) * steps / args.ranges) : steps;
  const int nk = (k_end - k_begin - wave + kGwaves - 1) / kGwaves;  // steps of this wave
  const int rest = a.inner % kGrowBytes;
  const char* wbase = reinterpret_cast<const char*>(a.weight) + n0 * a.weight_stride;
  const char* xbase = reinterpret_cast<const char*>(args.x);
  // Lane l of a load writes slot l % 8 of row l / 8 (and + 8).  Items 0 .. MT - 1 of a
  // step are token tiles, the others channel tiles; rows past the end read a valid one.
  uint32_t goff[kItems][2];
#pragma unroll
  for (int t = 0; t < kItems; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 8 * i + (lane >> 3), chunk = (lane & 7) ^ gemm_swz(row);
      goff[t][i] = (t < MT ? min(16 * t + row, a.tokens - 1) * static_cast<int>(args.x_stride)
                           : min(16 * (t - MT) + row, rows - 1) * static_cast<int>(a.weight_stride)) + chunk * 16;
    }
  unsigned char* ring = gsm + wave * (D * kPlaceBytes);
  auto issue = [&](int kt, int t, int place) {
    const int step = k_begin + wave + kt * kGwaves;
    const char* from = (t < MT ? xbase : wbase) + static_cast<int64_t>(step) * kGrowBytes;
    unsigned char* to = ring + place * kPlaceBytes;
    if (rest == 0 || step != steps - 1) {
#pragma unroll
      for (int i = 0; i < (MH == 1 && t == 0 ? 1 : 2); ++i) {  // the weights past the caches: every workgroup reads others
        if (t < MT) __builtin_amdgcn_global_load_lds((gemm_gptr)(from + goff[t][i]), (gemm_lptr)(to + 1024 * i), 16, 0, 0);
        else __builtin_amdgcn_global_load_lds((gemm_gptr)(from + goff[t][i]), (gemm_lptr)(to + 1024 * i), 16, 0, kStream);
      }
    } else {
#pragma unroll
      for (int i = 0; i < (MH == 1 && t == 0 ? 1 : 2); ++i) {
        const bool there = ((lane & 7) ^ gemm_swz(8 * i + (lane >> 3))) * 16 < rest;
        const char* p = there ? from + goff[t][i] : reinterpret_cast<const char*>(&kZeros);
        __builtin_amdgcn_global_load_lds((gemm_gptr)p, (gemm_lptr)(to + 1024 * i), 16, 0, 0);
      }
    }
  };
  const int fr = lane & 15, fq = lane >> 4;
  const int frag_off[2] = {fr * kGrowBytes + ((fq ^ gemm_swz(fr)) * 16), fr * kGrowBytes + (((4 + fq) ^ gemm_swz(fr)) * 16)};
  i32x4 acc[NT][MT] = {};
#pragma unroll
  for (int i = 0; i < D; ++i)
    if (i / kItems < nk) issue(i / kItems, i % kItems, i);
  // What a thread finishes at the end: four channels of a token, of the tiles wave,
  // wave + 8, ...  Their scales are requested now, behind the first places.
  constexpr int kTiles = NT * MT, kQuads = (kTiles + kGwaves - 1) / kGwaves, kOnce = std::min(kTiles, D * kPlaceBytes / 1024);
  auto quad_tile = [&](int q) { return q * kGwaves + wave; };
  auto quad_token = [&](int i) { return i % MT * 16 + fr; };
  auto quad_channel = [&](int i) { return i / MT * 16 + 4 * fq; };
  float step[kQuads], by[kQuads][4], add[kQuads][4];
  if constexpr (!PART) {
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const int i = min(quad_tile(q), kTiles - 1);
      step[q] = args.x_scales[min(quad_token(i), a.tokens - 1)];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = min(n0 + quad_channel(i) + e, a.outer - 1);
        by[q][e] = a.weight_scales[n];
        add[q][e] = bias_of(a.bias, n, a.out_bytes);
      }
    }
  }
  int place = 0;
  for (int kt = 0; kt < nk; ++kt) {
    i32x4 x[MT][2];
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
      // The item's own loads are done; those of the D - 1 items behind it may be in flight.
      constexpr int kSingle = MH == 1 ? (D - 1 + kItems - 1) / kItems : 0;  // items of one load among those, at most
      constexpr int kNone = gemm_wait_vm(0), kMost = gemm_wait_vm(2 * (D - 1) - kSingle);
      const int next_kt = kt + (t + D) / kItems;
      const bool more = next_kt < nk;
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      if (kt + (t + D - 1) / kItems < nk) __builtin_amdgcn_s_waitcnt(kMost);
      else __builtin_amdgcn_s_waitcnt(kNone);
      asm volatile("" ::: "memory");
      const unsigned char* from = ring + place * kPlaceBytes;
      i32x4 f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) f[h] = *reinterpret_cast<const i32x4*>(from + frag_off[h]);
      if (t < MT) {
        x[t][0] = f[0];
        x[t][1] = f[1];
      }
      // The place is free once it is read.
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      __builtin_amdgcn_sched_barrier(0);
      if (more) issue(next_kt, (t + D) % kItems, place);
      place = place + 1 == D ? 0 : place + 1;
      if (t >= MT) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[t - MT][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h], x[j][h], acc[t - MT][j], 0, 0, 0);
      }
    }
  }
  // Add the waves' sums, as many tiles at a time as LDS holds.
  i32x4* sums = reinterpret_cast<i32x4*>(gsm);  // [waves][kOnce tiles][64]
#pragma unroll
  for (int first = 0; first < kTiles; first += kOnce) {
    __syncthreads();  // the rings, or the sums before, are no longer read
#pragma unroll
    for (int i = first; i < kTiles && i < first + kOnce; ++i) sums[(wave * kOnce + i - first) * 64 + lane] = acc[i / MT][i % MT];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const int i = quad_tile(q);
      if (i < first || i >= min(first + kOnce, kTiles)) continue;
      i32x4 sum = sums[(i - first) * 64 + lane];
#pragma unroll
      for (int o = 1; o < kGwaves; ++o) sum += sums[(o * kOnce + i - first) * 64 + lane];
      const int m = quad_token(i), local = quad_channel(i);
      if (m >= a.tokens) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (local + e >= rows) continue;
        const int n = n0 + local + e;
        if constexpr (PART) {
          args.part[(static_cast<int64_t>(ks) * a.tokens + m) * args.part_stride + n] = sum[e];
        } else {
          const float y = static_cast<float>(sum[e]) * (step[q] * by[q][e]) + add[q][e];
          if (a.out_bytes == 2) static_cast<bf16_t*>(a.out)[m * a.out_stride + n] = f_to_bf16(y);
          else static_cast<float*>(a.out)[m * a.out_stride + n] = y;
        }
      }
    }
  }
}

// The ranges' sums of four channels of a token, and the scales.
constexpr int kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads) k_int8_sum(ProductArgs args) {
  const ResidentInt8Linear& a = args.a;
  const int quads = static_cast<int>(args.part_stride / 4);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kSumThreads + threadIdx.x;
  if (at >= static_cast<int64_t>(a.tokens) * quads) return;
  const int m = static_cast<int>(at / quads), n = static_cast<int>(at - static_cast<int64_t>(m) * quads) * 4;
  const int64_t range = static_cast<int64_t>(a.tokens) * args.part_stride;
  const int32_t* from = args.part + m * args.part_stride + n;
  i32x4 sum = *reinterpret_cast<const i32x4*>(from);
  for (int s = 1; s < args.ranges; ++s) sum += *reinterpret_cast<const i32x4*>(from + s * range);
  const float step = args.x_scales[m];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= a.outer) continue;
    const float y = static_cast<float>(sum[e]) * (step * a.weight_scales[n + e]) + bias_of(a.bias, n + e, a.out_bytes);
    if (a.out_bytes == 2) static_cast<bf16_t*>(a.out)[m * a.out_stride + n + e] = f_to_bf16(y);
    else static_cast<float*>(a.out)[m * a.out_stride + n + e] = y;
  }
}

static_assert(kGrowBytes == kInt8StepBytes && kGwaves == kInt8Waves && kGn == 256 && gemm_tile_m(1) == 64);
LinearPlan plan_of(const ResidentInt8Linear& a) { return linear_plan(a.tokens, a.inner, a.outer); }

// The workspace: of a call whose tokens are not in 8 bits their bytes and their
// steps, of one whose K is cut into ranges their sums.
struct LinearBytes {
  int64_t rows, steps, part;
  int64_t all() const { return rows + steps + part; }
};
LinearBytes linear_bytes(const ResidentInt8Linear& a, const LinearPlan& p) {
  LinearBytes b{};
  if (a.x_bytes != 1) {
    b.rows = round_up(static_cast<int64_t>(a.tokens) * a.inner, 16);
    b.steps = round_up(static_cast<int64_t>(a.tokens) * 4, 16);
  }
  if (p.ranges > 1) b.part = p.ranges * (static_cast<int64_t>(a.tokens) * round_up(a.outer, 4) * 4);
  return b;
}

template <int MJ, int GN, bool PART>
hipError_t launch_tiles(const ProductArgs& p, hipStream_t stream) {
  constexpr int ST = gemm_stages(MJ), kLds = tile_lds_bytes(MJ, ST, GN);
  void (*const kernel)(ProductArgs) = k_int8_tiles<MJ, ST, GN, PART>;
  static std::atomic<uint64_t> allowed{0};
  const hipError_t attr = allow_lds(kernel, kLds, allowed);
  if (attr != hipSuccess) return attr;
  ProductArgs args = p;
  args.m_tiles = static_cast<int>(ceil_div(p.a.tokens, gemm_tile_m(MJ)));
  args.n_tiles = static_cast<int>(ceil_div(p.a.outer, GN));
  return launch(kernel, static_cast<int64_t>(args.m_tiles) * args.n_tiles * args.ranges, kGthreads, kLds, stream, args);
}

template <int MH, int NT, bool PART>
hipError_t launch_few(const ProductArgs& p, hipStream_t stream) {
  constexpr int kLds = kGwaves * kFewPlaces * kPlaceBytes;
  void (*const kernel)(ProductArgs) = k_int8_few<MH, NT, PART>;
  static std::atomic<uint64_t> allowed{0};
  const hipError_t attr = allow_lds(kernel, kLds, allowed);
  if (attr != hipSuccess) return attr;
  ProductArgs args = p;
  args.n_tiles = static_cast<int>(ceil_div(p.a.outer, p.few_rows));
  return launch(kernel, static_cast<int64_t>(args.n_tiles) * args.ranges, kGthreads, kLds, stream, args);
}

template <int MH, bool PART>
hipError_t launch_few(const ProductArgs& p, hipStream_t stream) {
  switch ((p.few_rows + 15) / 16) {
    case 1: return launch_few<MH, 1, PART>(p, stream);
    case 2: return launch_few<MH, 2, PART>(p, stream);
    case 3: return launch_few<MH, 3, PART>(p, stream);
    case 4: return launch_few<MH, 4, PART>(p, stream);
    case 5: return launch_few<MH, 5, PART>(p, stream);
    case 6: return launch_few<MH, 6, PART>(p, stream);
  }
  return hipErrorInvalidValue;
}

template <bool PART>
hipError_t launch_product(const ProductArgs& p, const LinearPlan& plan, hipStream_t stream) {
  if (p.few_rows != 0) {
    const int tokens = p.a.tokens;
    if (tokens <= 8) return launch_few<1, PART>(p, stream);
    return tokens <= 16 ? launch_few<2, PART>(p, stream) : tokens <= 32 ? launch_few<4, PART>(p, stream) : launch_few<8, PART>(p, stream);
  }
  if constexpr (!PART) {
    if (plan.gn == 64) return plan.mj == 1 ? launch_tiles<1, 64, false>(p, stream) : launch_tiles<2, 64, false>(p, stream);
    if (plan.gn == 128) return plan.mj == 1 ? launch_tiles<1, 128, false>(p, stream) : launch_tiles<2, 128, false>(p, stream);
    if (plan.gn == 192) return plan.mj == 1 ? launch_tiles<1, 192, false>(p, stream) : plan.mj == 2 ? launch_tiles<2, 192, false>(p, stream) : launch_tiles<3, 192, false>(p, stream);
  }
  switch (plan.mj) {
    case 1: return launch_tiles<1, kGn, PART>(p, stream);
    case 2: return launch_tiles<2, kGn, PART>(p, stream);
    case 3: return launch_tiles<3, kGn, PART>(p, stream);
    case 4: return launch_tiles<4, kGn, PART>(p, stream);
  }
  return hipErrorInvalidValue;
}

constexpr int64_t kMostByteStride = 1 << 22;

bool linear_ok(const ResidentInt8Linear& a) {
  if ((a.x_bytes != 1 && a.x_bytes != 2 && a.x_bytes != 4) || (a.out_bytes != 2 && a.out_bytes != 4)) return false;
  // Sums of products of bytes fit 32 bits up to here.
  if (a.tokens < 0 || a.outer <= 0 || a.inner <= 0 || a.inner % 16 != 0 || a.inner >= 1 << 17) return false;
  if (a.x_stride < 0 || a.weight_stride < 0 || a.out_stride < 0 || a.workspace_bytes < 0) return false;
  // A tile's rows are reached by 32-bit offsets.
  if ((a.outer > 1 && a.weight_stride > kMostByteStride) || (a.x_bytes == 1 && a.tokens > 1 && a.x_stride > kMostByteStride)) return false;
  if (ceil_div(a.tokens, 64) * ceil_div(a.outer, kGn) >= 1 << 21) return false;  // launches stay below 2^32 threads
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
  return linear_bytes(*args, plan_of(*args)).all();
}

extern "C" int32_t resident_int8_linear(const ResidentInt8Linear* args, void* stream) {
  using namespace re;
  if (args == nullptr || !linear_ok(*args)) return -1;
  if (args->tokens == 0) return 0;
  const ResidentInt8Linear& a = *args;
  const LinearPlan plan = plan_of(a);
  if (!has_kernel(plan)) return -2;
  const LinearBytes b = linear_bytes(a, plan);
  if (b.all() > 0 && (a.workspace == nullptr || a.workspace_bytes < b.all())) return -1;
  const DeviceScope device(a.device);
  if (!device.ok()) return -2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  int8_t* rows = static_cast<int8_t*>(a.workspace);
  const int64_t per = 16 / a.out_bytes;
  ProductArgs p{a, static_cast<const int8_t*>(a.x), a.x_scales, a.x_stride, aligned(a.out, 16) && (a.tokens == 1 || a.out_stride % per == 0),
                plan.ranges, reinterpret_cast<int32_t*>(rows + b.rows + b.steps), round_up(a.outer, 4), 0, 0, plan.few_rows};
  if (a.tokens == 1) p.x_stride = 0;
  if (a.outer == 1) p.a.weight_stride = 0;
  if (a.x_bytes != 1) {
    float* steps = reinterpret_cast<float*>(rows + b.rows);
    p.x = rows;
    p.x_scales = steps;
    p.x_stride = a.inner;
    const ResidentQuantizeRows q{a.x, rows, steps, a.x_stride, a.inner, a.tokens, a.inner, a.x_bytes, a.device};
    if (launch_quantize(q, s) != hipSuccess) return -2;
  }
  if (plan.ranges == 1) return launch_product<false>(p, plan, s) == hipSuccess ? 0 : -2;
  if (launch_product<true>(p, plan, s) != hipSuccess) return -2;
  return launch(k_int8_sum, ceil_div(a.tokens * (p.part_stride / 4), kSumThreads), kSumThreads, 0, s, p) == hipSuccess ? 0 : -2;
}
