// Pieces shared by the attention kernels that read a paged 8-bit cache: a page on its way to a wave's LDS, and
// the merge of partial rows.
#pragma once

#include "attn_tile.h"
#include "paged.h"

namespace lq {
namespace attn {

// A page on its way: rows 8 i + lane / 8 of K and V, the words of row `lane`. Read once: non-temporal (8
// sessions of 42,771 to 82,671 rows 244 -> 229 us), in whole lines (K as MFMA operands straight from memory
// takes half lines: 220 -> 238).
struct PageRegs {
  u4_t k[8], v[8];
  uint32_t w[4];
};

__device__ __forceinline__ void load_page(const PagedBufs& buf, int64_t row, int lane, PageRegs& p) {
  const u4_t* k = reinterpret_cast<const u4_t*>(buf.kc + row * D) + lane;
  const u4_t* v = reinterpret_cast<const u4_t*>(buf.vc + row * D) + lane;
#pragma unroll
  for (int i = 0; i < 8; ++i) p.k[i] = __builtin_nontemporal_load(k + 64 * i);
  p.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(buf.ks) + row + lane);
  p.w[1] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(buf.kb) + row + lane);
#pragma unroll
  for (int i = 0; i < 8; ++i) p.v[i] = __builtin_nontemporal_load(v + 64 * i);
  p.w[2] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(buf.vs) + row + lane);
  p.w[3] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(buf.vb) + row + lane);
}

__device__ __forceinline__ int kswz(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int vswz(int r) { return (r & 3) | ((r >> 2) & 4); }

__device__ __forceinline__ void wave_fence() {  // LDS of the wave's own: order across its lanes
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Adds a partial (maximum m, sum l, values x) to another; one without keys (m = -infinity) has x = 0.
__device__ __forceinline__ void merge_into(float& M, float& den, f4_t& acc, float m, float l, f4_t x) {
  const float mn = max_ieee(M, m);
  const float mr = mn == -INFINITY ? 0.0f : mn;
  const float e0 = exp2_nonpos(M - mr), e1 = exp2_nonpos(m - mr);
  acc = acc * e0 + x * e1;
  den = den * e0 + l * e1;
  M = mn;
}

}  // namespace attn
}  // namespace lq
