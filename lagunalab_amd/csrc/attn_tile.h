// Attention of 16 NT query rows per wave over one 64-key tile of bf16 K and V in LDS, on the matrix
// cores: the inner step of the paged prefix and the packed prompt kernels.
//
// S = K Q^T as v_mfma_f32_16x16x32_bf16 (M = 16 keys, N = 16 rows, K = 32 dims): lane (lc = lane % 16,
// lq4 = lane / 16) ends with the scores of keys 16 mt + 4 lq4 + r of row lc. P of key tiles 2 e and
// 2 e + 1 is then, as it lies in the lane's registers, the B operand of k-step e of O^T = V^T P^T: slot
// 4 h + r of lane group lq4 is key 32 e + 16 h + 4 lq4 + r. V^T's A operand takes the keys in that order
// with two transposed LDS reads (ds_read_b64_tr_b16: of 4 keys x 16 dims per 16 lanes, lane i gets dim
// i of the four keys), so neither P nor V is moved between lanes.
//
// Softmax in fp32 with a running maximum that moves only when a tile's exceeds it by 2^8; P rounded to
// bf16 for its product (2^-8 relative at most per key, of either sign, against an output of the same
// type; bf16 keeps the range of V). The row sums are those of the rounded P, one more product with ones.
#pragma once

#include "attn_dev.h"

namespace lq {
namespace attn {

constexpr int TKEYS = 64;  // keys of a tile, positions of a page

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4_t;
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

// A tile in LDS. K: 16-byte chunk j of key r at chunk j ^ (r & 15); V: 32-byte window w of key r at
// window w ^ (r & 7): operand reads touch every bank equally.
struct alignas(256) KvTile {
  uint16_t k[TKEYS * D];
  uint16_t v[TKEYS * D];
};
__device__ __forceinline__ uint4* k_chunk(KvTile& t, int key, int chunk) {
  return reinterpret_cast<uint4*>(t.k) + 16 * key + (chunk ^ (key & 15));
}
__device__ __forceinline__ uint4* v_chunk(KvTile& t, int key, int chunk) {
  return reinterpret_cast<uint4*>(t.v) + 16 * key + (chunk ^ (2 * (key & 7)));
}

// Two floats as one dword of bf16, round to nearest even, x in the low half (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack_bf2(float x, float y) {
  typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
  const bf2_t p = {(__bf16)x, (__bf16)y};
  return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ bf16x8_t words_as_bf8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const u4_t u = {a, b, c, d};
  return __builtin_bit_cast(bf16x8_t, u);
}
__device__ __forceinline__ bf16x8_t u4_as_bf8(uint4 u) { return words_as_bf8(u.x, u.y, u.z, u.w); }

// Codes 0..3 of a word as scale * code + bias in bf16: the product is exact in fp32, so the fused
// multiply-add rounds as the two operations of the dequantizer do.
__device__ __forceinline__ uint2 dequant4(uint32_t w, float s, float b) {
  return make_uint2(pack_bf2(fmaf(s, (float)(w & 0xffu), b), fmaf(s, (float)((w >> 8) & 0xffu), b)),
                    pack_bf2(fmaf(s, (float)((w >> 16) & 0xffu), b), fmaf(s, (float)(w >> 24), b)));
}

__device__ __forceinline__ bf16x8_t bf16_ones() {
  return words_as_bf8(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
}

// The softmax scale in log2 units, as its magnitude (the sign goes into q): never 0, so that a masked
// score of -infinity stays one.
__device__ __forceinline__ float abs_scale(float sl2) { return fmaxf(fabsf(sl2), 1e-37f); }
// A q row's 16 bytes with the scale's sign.
__device__ __forceinline__ uint4 signed_q(uint4 u, float sl2) {
  const uint32_t x = sl2 < 0.0f ? 0x80008000u : 0u;
  return make_uint4(u.x ^ x, u.y ^ x, u.z ^ x, u.w ^ x);
}

// A weight is exp2(fma(score, scale, off)) with off = -m, the running maximum rounded to fp32; the product
// is not rounded, so that the largest key's exponent is not 0 but off's rounding, up to 2^-24 of it: a
// common factor of the row as long as it is small, 2^128 and beyond fp32 at a maximum of 2^31. From
// HUGE_LOG2 on, where it is up to 2^(1/2), the scores of a row are made differences to the maximum first,
// of rounded products, in raw units, and off 0. The test costs 0 to 1% (7 prompts of 1 to 4,099 rows 545
// -> 551 us, 2,048 rows 51.7 -> 51.9, 16,384 rows 1,870 -> 1,865, 48 sessions behind 16,384 64.8 -> 64.7).
constexpr float HUGE_LOG2 = 8388608.0f;  // 2^23
__device__ __forceinline__ bool is_huge(float off) { return fabsf(off) >= HUGE_LOG2; }
template <int MT>
__device__ __forceinline__ void settle_huge(f4_t (&c)[MT], float& off, float scale) {
#pragma clang fp contract(off)
  const bool huge = is_huge(off);
  const float inv = 1.0f / scale;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = c[mt][r] * scale;  // rounded as the maximum was
      c[mt][r] = huge ? (x + off) * inv : c[mt][r];
    }
  off = huge ? 0.0f : off;
}

// State of a wave's rows: row 16 nt + lc in column lc of N tile nt.
template <int NT>
struct TileRows {
  bf16x8_t q[NT][4];  // B operands: dims 32 kk + 8 lq4 .. + 7
  f4_t o[NT][8];      // O^T: dims 16 w + 4 lq4 + r
  f4_t l[NT];         // row sums of P, the same in all four
  float m[NT];        // running maximum, log2 units
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int w = 0; w < 8; ++w) o[nt][w] = f4_t{0.f, 0.f, 0.f, 0.f};
      l[nt] = f4_t{0.f, 0.f, 0.f, 0.f};
      m[nt] = -INFINITY;
    }
  }
};

// Raw scores of the tile's keys. K fragments are read one key tile ahead of the MFMAs that use them (the
// scheduling barriers keep it so).
template <int NT, int MT>
__device__ __forceinline__ void tile_scores(const uint16_t* kt, const TileRows<NT>& st, int lane,
                                            f4_t (&c)[NT][MT]) {
  const int lc = lane & 15, lq4 = lane >> 4;
  const bf16x8_t* k = reinterpret_cast<const bf16x8_t*>(kt) + 16 * lc;
  bf16x8_t f[2][4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) f[0][kk] = k[(4 * kk + lq4) ^ lc];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt + 1 < MT) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) f[(mt + 1) & 1][kk] = k[256 * (mt + 1) + ((4 * kk + lq4) ^ lc)];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        c[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            f[mt & 1][kk], st.q[nt][kk], kk == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : c[nt][mt], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Scores to weights: raises the running maximum where needed (and rescales the row), P in bf16 as the
// B operands of the two k-steps.
template <int NT, int MT>
__device__ __forceinline__ void tile_softmax(f4_t (&c)[NT][MT], TileRows<NT>& st, float scale,
                                             bf16x8_t (&p)[NT][MT / 2]) {
  float t[NT], off[NT];
  bool bump[NT], any = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // four chains
    float x[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      x[mt] = max_ieee(max_ieee(max_ieee(c[nt][mt][0], c[nt][mt][1]), c[nt][mt][2]), c[nt][mt][3]);
    t[nt] = max_ieee(x[0], x[1]);
    if constexpr (MT == 4) t[nt] = max_ieee(t[nt], max_ieee(x[2], x[3]));
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) t[nt] = max_xor16(t[nt]);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    t[nt] = max_xor32(t[nt]) * scale;
    bump[nt] = t[nt] > (st.m[nt] == -INFINITY ? -INFINITY : st.m[nt] + RESCALE_LOG2);
    off[nt] = st.m[nt] == -INFINITY ? 0.0f : -st.m[nt];
    any |= bump[nt] | is_huge(off[nt]);
  }
  if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mn = bump[nt] ? t[nt] : st.m[nt];
      const float alpha = st.m[nt] == -INFINITY ? 0.0f : exp2_nonpos(st.m[nt] - mn);
      st.m[nt] = mn;
      st.l[nt] *= alpha;
#pragma unroll
      for (int w = 0; w < 8; ++w) st.o[nt][w] *= alpha;
      off[nt] = mn == -INFINITY ? 0.0f : -mn;
      if (__builtin_amdgcn_ballot_w64(is_huge(off[nt]))) settle_huge(c[nt], off[nt], scale);
    }
  }
  uint32_t w[NT][2 * MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[nt][2 * mt + h] = pack_bf2(__builtin_amdgcn_exp2f(fmaf(c[nt][mt][2 * h], scale, off[nt])),
                                     __builtin_amdgcn_exp2f(fmaf(c[nt][mt][2 * h + 1], scale, off[nt])));
    }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // made here, not sunk into the product's phase
#pragma unroll
    for (int e = 0; e < MT / 2; ++e) {
      asm volatile("" : "+v"(w[nt][4 * e]), "+v"(w[nt][4 * e + 1]), "+v"(w[nt][4 * e + 2]), "+v"(w[nt][4 * e + 3]));
      p[nt][e] = words_as_bf8(w[nt][4 * e], w[nt][4 * e + 1], w[nt][4 * e + 2], w[nt][4 * e + 3]);
    }
  }
}

// A operand of dims 16 w .. 16 w + 15 and k-step e of a tile's V^T (v 256-byte aligned).
__device__ __forceinline__ uint32_t v_lane(const uint16_t* v, int lane) {
  const int rk = 4 * (lane >> 4) + ((lane >> 2) & 3);  // key of this lane's source within 16
  return lds_addr(v) + (uint32_t)(256 * rk + 8 * (lane & 3) + 32 * (rk & 7));
}
__device__ __forceinline__ bf16x8_t v_operand(uint32_t vl, int w, int e) {
  const uint32_t a = (vl ^ (uint32_t)(32 * w)) + 8192u * e;
  const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)a);
  const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)(a + 4096u));
  typedef short s8_t __attribute__((ext_vector_type(8)));
  const s8_t u = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8_t, u);
}

// A bf16 pair with infinities and NaN as 0.
__device__ __forceinline__ uint32_t finite_bf2(uint32_t u) {
  if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
  if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
  return u;
}

// O^T += V^T P^T. Fragments of half a k-step (four windows of 16 dims) are read ahead of the MFMAs, as in
// tile_scores.
template <int NT, int E>
__device__ __forceinline__ void tile_values(const uint16_t* v, TileRows<NT>& st, int lane,
                                            const bf16x8_t (&p)[NT][E]) {
  const uint32_t vl = v_lane(v, lane);
  bf16x8_t f[2][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) f[0][j] = v_operand(vl, j, 0);
#pragma unroll
  for (int u = 0; u < 2 * E; ++u) {  // k-step u / 2, windows 4 (u % 2) ..
    if (u + 1 < 2 * E) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[(u + 1) & 1][j] = v_operand(vl, 4 * ((u + 1) & 1) + j, (u + 1) >> 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int e = u >> 1, w0 = 4 * (u & 1);
    if (u & 1) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        st.l[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_ones(), p[nt][e], st.l[nt], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        st.o[nt][w0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[u & 1][j], p[nt][e],
                                                                 st.o[nt][w0 + j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Q.K^T of one tile, then P.V of another, in eight steps of 4 NT MFMAs: two key tiles of K by half the
// dims (so that an MFMA's accumulator was last written 2 NT MFMAs before), then half a k-step of V. A step's
// four fragments are read two steps ahead (tile_ahead: the first two, which may lie in the phase before), so
// that no MFMA waits for LDS.
struct Ahead {
  bf16x8_t f[3][4];
};
__device__ __forceinline__ void tile_fetch(const bf16x8_t* k, uint32_t vl, int lane, int step, bf16x8_t (&f)[4]) {
  const int lc = lane & 15, lq4 = lane >> 4;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    f[j] = step < 4 ? k[256 * (2 * (step >> 1) + (j >> 1)) + ((4 * (2 * (step & 1) + (j & 1)) + lq4) ^ lc)]
                    : v_operand(vl, 4 * (step & 1) + j, (step - 4) >> 1);
}
__device__ __forceinline__ void tile_ahead(const uint16_t* kt, int lane, Ahead& a) {
  const bf16x8_t* k = reinterpret_cast<const bf16x8_t*>(kt) + 16 * (lane & 15);
  tile_fetch(k, 0, lane, 0, a.f[0]);
  tile_fetch(k, 0, lane, 1, a.f[1]);
}
template <int NT>
__device__ __forceinline__ void tile_matrix(const uint16_t* kt, const uint16_t* vt, TileRows<NT>& st, int lane,
                                            f4_t (&c)[NT][4], const bf16x8_t (&p)[NT][2], Ahead& a) {
  const bf16x8_t* k = reinterpret_cast<const bf16x8_t*>(kt) + 16 * (lane & 15);
  const uint32_t vl = v_lane(vt, lane);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    if (u + 2 < 8) tile_fetch(k, vl, lane, u + 2, a.f[(u + 2) % 3]);
    __builtin_amdgcn_sched_barrier(0);
    if (u < 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int mt = 2 * (u >> 1) + (i & 1), kk = 2 * (u & 1) + (i >> 1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          c[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a.f[u % 3][2 * (i & 1) + (i >> 1)], st.q[nt][kk],
              kk == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : c[nt][mt], 0, 0, 0);
      }
    } else {
      const int e = (u - 4) >> 1, w0 = 4 * (u & 1);
      if (u & 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          st.l[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_ones(), p[nt][e], st.l[nt], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          st.o[nt][w0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.f[u % 3][j], p[nt][e],
                                                                     st.o[nt][w0 + j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The infinities and NaN of one V row (key `key` of a tile whose P is p, position `at`), for the rows that see
// it: O^T took 0 in their place, since 0 times one of them is no 0.
template <int NT>
__device__ __forceinline__ void tile_nonfinite(const uint8_t* vrow, int key, int at, TileRows<NT>& st, int lane,
                                               const bf16x8_t (&p)[NT][2], const int (&lim)[NT]) {
  const int lc = lane & 15, lq4 = lane >> 4;
  const int word = 2 * ((key >> 4) & 1) + ((key >> 1) & 1);
  float pk[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const u4_t p0 = __builtin_bit_cast(u4_t, p[nt][0]), p1 = __builtin_bit_cast(u4_t, p[nt][1]);
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mine = j == word ? (key < 32 ? p0[j] : p1[j]) : mine;
    const uint32_t w = __shfl(mine, 16 * ((key >> 2) & 3) + lc, 64);
    pk[nt] = key & 1 ? bf16_hi(w) : bf16_lo(w);
  }
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint2 v2 = *reinterpret_cast<const uint2*>(vrow + 2 * (16 * w + 4 * lq4));
    const float v[4] = {bf16_lo(v2.x), bf16_hi(v2.x), bf16_lo(v2.y), bf16_hi(v2.y)};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (at <= lim[nt] && !(fabsf(v[r]) < INFINITY)) st.o[nt][w][r] = fmaf(pk[nt], v[r], st.o[nt][w][r]);
  }
}

}  // namespace attn
}  // namespace lq
