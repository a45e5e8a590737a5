// What the tiled products through LDS share (the bf16 one of re_prefill.hip, where
// it is described, and the 8-bit one of re_int8.hip): the stages' layout and
// barrier, the order of the tiles.
#pragma once

#include "re_device.h"

namespace re {
namespace {

constexpr int kGn = 256;
constexpr int kGrowBytes = 128;  // one K step of one row
constexpr int kGwaves = 8, kGthreads = kGwaves * 64;
constexpr int kGgroupM = 4;
constexpr int gemm_tile_m(int mj) { return 64 * mj; }
constexpr int gemm_stage_bytes(int mj, int gn) { return (gn + gemm_tile_m(mj)) * kGrowBytes; }
constexpr int gemm_stages(int mj) { return mj <= 2 ? 3 : 2; }
constexpr int gemm_out_ld(int gn) { return gn + 8; }  // epilogue row stride (elements)

typedef const __attribute__((address_space(1))) void* gemm_gptr;
typedef __attribute__((address_space(3))) void* gemm_lptr;

__device__ __forceinline__ int gemm_swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// s_waitcnt immediate: vmcnt <= vm (6 bits), lgkmcnt 0, expcnt untouched.
constexpr int gemm_wait_vm(int vm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4); }

// End of a stage: this wave's LDS reads and all but the last VM of its loads
// are done, then the barrier.  The empty asm statements keep the compiler
// from moving memory accesses across; the wait is a real instruction the
// wait-count pass accounts for.
template <int VM = 0>
__device__ __forceinline__ void gemm_stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(gemm_wait_vm(VM));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// Tile and K range of workgroup b (see k_gemm_bf16): K ranges outermost.
__device__ __forceinline__ void gemm_tile_of(int b, int nM, int nN, int nS, int& mt, int& nt, int& ks) {
  const int tiles = nM * nN, total = tiles * nS, x = b & 7, local = b >> 3, q = total >> 3, r = total & 7;
  int t = x < r ? x * (q + 1) + local : r * (q + 1) + (x - r) * q + local;
  ks = t / tiles;
  t -= ks * tiles;
  const int group_m = nM <= 2 * kGgroupM ? nM : kGgroupM;
  const int per_group = group_m * nN, g = t / per_group, first = g * group_m;
  const int gm = min(group_m, nM - first), w = t - g * per_group;
  mt = first + w % gm;
  nt = w / gm;
}

// Waves along n: a wave's block of 16 x 16 tiles is 8 x 4 (n x m) of a 256-row
// tile and 4 x 6, 4 x 4 and 4 x 2 of the lower ones, the fewest fragment reads
// per product (two waves along n throughout: 11 reads for 24 products, 10 for
// 16 and 9 for 8 instead of 10, 8 and 6).  Gate/up at 570 tokens, 128-row tiles:
// 181 -> 171 us; 400 tokens 170 -> 161; 2,000 tokens, 64-row tiles 811 -> 774;
// 192-row tiles the same within 1 %.
constexpr int gemm_waves_n(int mj) { return mj == 4 ? 2 : 4; }

// Fragments of the next stage read before product p of the second sub-step:
// one per two products where that covers them, else spread over the first 7/8
// of the products.
constexpr int gemm_reads_by(int frags, int prods, int p) {
  const int span = prods - prods / 8;
  const int n = 2 * frags <= prods ? p / 2 : (p * frags + span - 1) / span;
  return n < frags ? n : frags;
}

}  // namespace
}  // namespace re
