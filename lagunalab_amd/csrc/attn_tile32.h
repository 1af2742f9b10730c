// Attention of 32 query rows per wave over one 64-key tile of bf16 K and V in LDS: attn_tile.h's step on
// v_mfma_f32_32x32x16_bf16 (M = 32 keys, N = 32 rows, K = 16 dims), for kernels whose vector phase is the longer
// one: VALU instructions of another wave of the SIMD issue every 6 cycles beside it, 8.2 beside 16x16x32.
//
// S = K Q^T: lane (ln = lane % 32, h = lane / 32) ends with the scores of row ln alone, register i of key tile mt
// those of key 32 mt + 8 (i / 4) + 4 h + i % 4; a row's maximum meets one other lane. P of registers 8 e .. 8 e + 7
// is, as it lies, the B operand of 16 keys of O^T = V^T P^T: slot 8 h + j is key 16 (2 mt + e) + 8 (j / 4) + 4 h +
// j % 4, and V^T's A operand takes the keys in that order with two transposed LDS reads (ds_read_b64_tr_b16).
//
// Softmax as in attn_tile.h: fp32, a running maximum that moves only when exceeded by 2^8, P rounded to bf16 in the
// values and in the row sums alike (v_dot2 with ones).
#pragma once

#include "attn_tile.h"

namespace lq {
namespace attn {

typedef float f16v_t __attribute__((ext_vector_type(16)));

// A tile in LDS. K: 16-byte chunk j of key r at chunk j ^ (r & 15), as in attn_tile.h. V: 32-byte window w of key r
// at window w ^ vswz32(r), so that the four keys and two windows that half a wave reads lie in different banks.
__device__ __forceinline__ int vswz32(int r) { return 2 * (r & 3) | ((r >> 2) & 1); }
__device__ __forceinline__ uint4* v_chunk32(KvTile& t, int key, int chunk) {
  return reinterpret_cast<uint4*>(t.v) + 16 * key + (chunk ^ (2 * vswz32(key)));
}

// State of a wave's rows: row ln.
struct Rows32 {
  bf16x8_t q[8];  // B operands: dims 16 kk + 8 h .. + 7
  f16v_t o[4];    // O^T: dims 32 w + 8 (i / 4) + 4 h + i % 4
  float l, m;     // sum of this lane's P (the row's other keys are lane ln + 32's), running maximum in log2 units
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[w][i] = 0.0f;
    l = 0.0f;
    m = -INFINITY;
  }
};

// As settle_huge of attn_tile.h.
template <int MT>
__device__ __forceinline__ void settle_huge32(f16v_t (&c)[MT], float& off, float scale) {
#pragma clang fp contract(off)
  const bool huge = is_huge(off);
  const float inv = 1.0f / scale;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = c[mt][i] * scale;  // rounded as the maximum was
      c[mt][i] = huge ? (x + off) * inv : c[mt][i];
    }
  off = huge ? 0.0f : off;
}

// Scores of keys that the lane's row does not see to -infinity: it sees the `window` keys up to key `rel` of those
// from 4 h on. By bits: a key's bit spread over a word chooses between the score and -infinity.
template <int MT>
__device__ __forceinline__ void mask32(f16v_t (&c)[MT], int rel, int window) {
  uint64_t seen = rel < 0 ? 0 : ~0ull >> (63 - min(rel, 63));
  const int out = rel - window;  // the last key before the window
  if (out >= 0) seen = out >= 63 ? 0 : seen >> (out + 1) << (out + 1);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int w = (int)(seen >> (32 * mt));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t on = (uint32_t)((w << (31 - 8 * (i >> 2) - (i & 3))) >> 31);
      c[mt][i] = __uint_as_float((__float_as_uint(c[mt][i]) & on) | (0xff800000u & ~on));
    }
  }
}

// Scores of MT key tiles to weights: raises the running maximum where needed (and rescales the row), P in bf16 as the
// B operands of the 16-key steps. work(): done when half of the scores are weights and their registers free.
template <int MT, typename Work>
__device__ __forceinline__ void softmax32(f16v_t (&c)[MT], Rows32& st, float scale, bf16x8_t (&p)[2 * MT], Work work) {
  float x[2 * MT];
#pragma unroll
  for (int j = 0; j < 2 * MT; ++j) {  // chains
    const f16v_t& s = c[j >> 1];
    const int i = 8 * (j & 1);
    x[j] = max_ieee(max_ieee(s[i], s[i + 1]), s[i + 2]);
#pragma unroll
    for (int k = 3; k < 7; k += 2) x[j] = max_ieee(max_ieee(x[j], s[i + k]), s[i + k + 1]);
    x[j] = max_ieee(x[j], s[i + 7]);
  }
  float top = max_ieee(x[0], x[1]);
  if constexpr (MT == 2) top = max_ieee(top, max_ieee(x[2], x[3]));
  const float t = max_xor32(top) * scale;
  const bool bump = t > (st.m == -INFINITY ? -INFINITY : st.m + RESCALE_LOG2);
  float off = st.m == -INFINITY ? 0.0f : -st.m;
  if (__builtin_amdgcn_ballot_w64(bump | is_huge(off))) {
    const float mn = bump ? t : st.m;
    const float alpha = st.m == -INFINITY ? 0.0f : exp2_nonpos(st.m - mn);
    st.m = mn;
    st.l *= alpha;
#pragma unroll
    for (int w = 0; w < 4; ++w) st.o[w] *= alpha;
    off = mn == -INFINITY ? 0.0f : -mn;
    if (__builtin_amdgcn_ballot_w64(is_huge(off))) settle_huge32(c, off, scale);
  }
#pragma unroll
  for (int e = 0; e < 2 * MT; ++e) {
    if (e == MT) work();
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 8 * (e & 1) + 2 * j;
      w[j] = pack_bf2(__builtin_amdgcn_exp2f(fmaf(c[e >> 1][i], scale, off)),
                      __builtin_amdgcn_exp2f(fmaf(c[e >> 1][i + 1], scale, off)));
    }
    // made here, not sunk into the product's phase
    asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
    p[e] = words_as_bf8(w[0], w[1], w[2], w[3]);
  }
}

template <int MT>
__device__ __forceinline__ void softmax32(f16v_t (&c)[MT], Rows32& st, float scale, bf16x8_t (&p)[2 * MT]) {
  softmax32(c, st, scale, p, []() {});
}

// Adds the rounded weights to the row sums.
template <int E>
__device__ __forceinline__ void sums32(Rows32& st, const bf16x8_t (&p)[E]) {
  typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
  const bf2_t ones = __builtin_bit_cast(bf2_t, 0x3f803f80u);
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const u4_t w = __builtin_bit_cast(u4_t, p[e]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = w[j];
      float& l = j & 1 ? sum : st.l;
      l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2_t, x), ones, l, false);
    }
  }
  st.l += sum;
}

// A wave's place in a tile: byte addresses of its operands' first fragments. The tile is 256-byte aligned, so that
// the bits that choose among a row's chunks and windows are the lane's alone.
__device__ __forceinline__ uint32_t k_lane32(const KvTile& t, int lane) {
  const int ln = lane & 31, h = lane >> 5;
  return lds_addr(t.k) + 256u * ln + 16u * (h ^ (ln & 15));
}
__device__ __forceinline__ uint32_t v_lane32(const KvTile& t, int lane) {
  const int h = lane >> 5, r = (lane >> 2) & 3;
  return lds_addr(t.v) + 256u * (4 * h + r) + 32u * (((lane >> 4) & 1) ^ vswz32(4 * h + r)) + 8u * (lane & 3);
}
typedef __attribute__((address_space(3))) bf16x8_t lds_bf8_t;
// K of key tile mt, dims 16 kk ...
__device__ __forceinline__ bf16x8_t k_operand32(uint32_t k, int mt, int kk) {
  return *(const lds_bf8_t*)(uintptr_t)((k ^ (32u * kk)) + 8192u * mt);
}
// V^T of dims 32 w .., keys 16 e ...
__device__ __forceinline__ bf16x8_t v_operand32(uint32_t v, int w, int e) {
  const uint32_t a = (v ^ (64u * w)) + 4096u * e;
  const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)a);
  const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)(a + 2048u));
  typedef short s8_t __attribute__((ext_vector_type(8)));
  const s8_t u = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8_t, u);
}

// Q.K^T of one tile, then P.V of another: 32 MFMAs in 16 steps of two, whose fragments are read three steps ahead
// (ahead32: the first three steps', which may lie in the phase before). k, v: the lane's place
// in the tiles.
// work(n): what else there is to do behind MFMA n. It and one fragment's read fit beside the MFMA that runs; all of a
// step's behind its second MFMA did not (a phase 1,870 cycles instead of 1,640).
constexpr int AHEAD = 3;
struct Ahead32 {
  bf16x8_t f[AHEAD + 1][2];
};
__device__ __forceinline__ void fetch32(uint32_t k, uint32_t v, int step, int j, Ahead32& a) {
  a.f[step % (AHEAD + 1)][j] =
      step < 8 ? k_operand32(k, j, step) : v_operand32(v, 2 * (step & 1) + j, (step - 8) >> 1);
}
__device__ __forceinline__ void ahead32(uint32_t k, Ahead32& a) {
#pragma unroll
  for (int u = 0; u < AHEAD; ++u)
#pragma unroll
    for (int j = 0; j < 2; ++j) fetch32(k, 0, u, j, a);
}
template <typename Work>
__device__ __forceinline__ void matrix32(uint32_t k, uint32_t v, Rows32& st, f16v_t (&c)[2],
                                         const bf16x8_t (&p)[4], Ahead32& a, Work work) {
#pragma unroll
  for (int u = 0; u < 16; ++u) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (u < 8) {
        f16v_t z;
        if (u == 0) {
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = 0.0f;
        }
        c[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f[u % (AHEAD + 1)][j], st.q[u], u == 0 ? z : c[j], 0, 0, 0);
      } else {
        const int w = 2 * (u & 1) + j;
        st.o[w] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f[u % (AHEAD + 1)][j], p[(u - 8) >> 1], st.o[w], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (u + AHEAD < 16) fetch32(k, v, u + AHEAD, j, a);
      work(2 * u + j);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // behind the last MFMA: beside MFMAs, of either wave of the SIMD, v_dot2 stalls both (2,048 rows behind 32,771
  // positions, 32/8 heads: 1,113 us here, 1,212 between the steps, 1,135 in the softmax)
  sums32(st, p);
}
// Raw scores of one tile.
__device__ __forceinline__ void scores32(uint32_t k, const Rows32& st, f16v_t (&c)[2]) {
  Ahead32 a;
  ahead32(k, a);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    if (u + AHEAD < 8) {
      fetch32(k, 0, u + AHEAD, 0, a);
      fetch32(k, 0, u + AHEAD, 1, a);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f16v_t z;
      if (u == 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.0f;
      }
      c[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f[u % (AHEAD + 1)][j], st.q[u], u == 0 ? z : c[j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The weight of key `key` (of the tile) for the lane's row.
template <int E>
__device__ __forceinline__ float weight32(const bf16x8_t (&p)[E], int key, int lane) {
  const int word = 2 * ((key >> 3) & 1) + ((key & 3) >> 1);
  uint32_t mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const u4_t w = __builtin_bit_cast(u4_t, p[e]);
#pragma unroll
    for (int j = 0; j < 4; ++j) mine = e == (key >> 4) && j == word ? w[j] : mine;
  }
  const uint32_t w = __shfl(mine, 32 * ((key >> 2) & 1) + (lane & 31), 64);
  return key & 1 ? bf16_hi(w) : bf16_lo(w);
}

}  // namespace attn
}  // namespace lq
