// Rows into and out of a paged 8-bit cache, and pages copied within it.
//
// lq_paged_append quantizes K/V rows (bf16, any token and head strides) into the pages of several
// sequences, with the arithmetic of the contiguous cache's append; lq_paged_append_rotated norms and rotates
// queries and keys on the way; lq_paged_gather reads positions back
// as bf16 rows, packed one sequence behind the other, as the contiguous cache's dequantize; lq_copy_pages
// copies pages of all heads. All are bound by their traffic (append 512 B read and 272 B written
// per row and head, gather 272 and 512, copy 17,408 each way per page and head).
#include <algorithm>
#include <vector>

#include "attn_tile.h"
#include "paged.h"

namespace lq {
namespace {

using namespace attn;

// The rows of a call, packed one sequence behind the other: sequence b has rows [begin[b], begin[b + 1]).
struct PackedRows {
  int nseq;
  int begin[LQ_MAX_SEQS + 1];
};

// The sequence whose range in `begin` holds x: a lane per sequence. x wave-uniform, below the last end.
__device__ __forceinline__ int find_packed(int end_of_lane, int x) {
  return (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(end_of_lane <= x));
}

// ---- append: 16 lanes per row (8 values each), 4 rows per wave; blockIdx.y: K or V. A lane's 8 codes
// are one 8-byte store; the group's minimum and maximum meet over its 8 lanes by DPP.
__device__ __forceinline__ float min8(float x) {
  x = fminf(x, dpp<DPP_QUAD_XOR1>(x));
  x = fminf(x, dpp<DPP_QUAD_XOR2>(x));
  return fminf(x, dpp<DPP_ROW_HALF_MIRROR>(x));
}
__device__ __forceinline__ float max8(float x) {
  x = fmaxf(x, dpp<DPP_QUAD_XOR1>(x));
  x = fmaxf(x, dpp<DPP_QUAD_XOR2>(x));
  return fmaxf(x, dpp<DPP_ROW_HALF_MIRROR>(x));
}

// Codes of a lane's 8 values (8 lanes hold a group of 64) and the group's parameters.
__device__ __forceinline__ AffineParams quantize8(const float (&x)[8], uint2& codes) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) {
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
  }
  const AffineParams p = affine_params<8>(min8(lo), max8(hi));
  const float rs = __builtin_amdgcn_rcpf(p.scale);
  uint32_t c[8];
  bool any = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    bool slow;
    c[j] = fast_code<8>(x[j], p, rs, slow);
    any |= slow;
  }
  if (__builtin_amdgcn_ballot_w64(any)) {  // the rare lanes next to a border divide
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bool slow;
      (void)fast_code<8>(x[j], p, rs, slow);
      if (slow) c[j] = affine_code<8>(x[j], p);
    }
  }
  codes = make_uint2(c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24),
                     c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24));
  return p;
}
__device__ __forceinline__ void unpack8(uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = bf16_lo(w[j]);
    x[2 * j + 1] = bf16_hi(w[j]);
  }
}

__global__ __launch_bounds__(256) void paged_append_kernel(
    const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int64_t k_tok, int64_t k_head,
    int64_t v_tok, int64_t v_head, PagedBufs buf, PageTable tab, const int32_t* __restrict__ starts,
    PackedRows rows, uint32_t units, FastDiv per_tok, int Hkv) {
  const int lane = threadIdx.x & 63;
  const int sub = lane & 15;
  const uint32_t u = blockIdx.x * 16 + (threadIdx.x >> 4);  // (token, head)
  const bool is_v = blockIdx.y != 0;
  const uint32_t uc = min(u, units - 1);
  const int t = (int)fdiv_u(uc, per_tok);
  const int h = (int)(uc - (uint32_t)t * (uint32_t)Hkv);
  const int end = lane < rows.nseq ? rows.begin[lane + 1] : INT32_MAX;
  int b = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {  // the four rows of the wave
    const int bs = find_packed(end, __builtin_amdgcn_readlane(t, 16 * r));
    b = (lane >> 4) == r ? bs : b;
  }
  const int64_t pos = (int64_t)starts[b] + (t - rows.begin[b]);
  const bool inside = u < units && pos >= 0 && pos < (int64_t)tab.width * PAGE;
  const int id = inside ? tab.ids[b * tab.stride + (pos >> 6)] : -1;
  const uint16_t* src = is_v ? v + t * v_tok + h * v_head : k + t * k_tok + h * k_head;
  float x[8];
  unpack8(*reinterpret_cast<const uint4*>(src + 8 * sub), x);
  uint2 c;
  const AffineParams p = quantize8(x, c);
  if (id < 0 || id >= tab.pages) return;
  const int64_t row = ((int64_t)id * Hkv + h) * PAGE + (pos & (PAGE - 1));
  uint8_t* codes = is_v ? buf.vc : buf.kc;
  *reinterpret_cast<uint2*>(codes + row * D + 8 * sub) = c;
  if ((sub & 7) == 0) {
    (is_v ? buf.vs : buf.ks)[2 * row + (sub >> 3)] = f32_to_bf16(p.scale);
    (is_v ? buf.vb : buf.kb)[2 * row + (sub >> 3)] = f32_to_bf16(p.bias);
  }
}

// ---- append with the norm and the rotation on the way: the heads of a token are its queries', keys' and values',
// 16 lanes per head (8 dims each), 4 heads per wave at a time and RT times that many in turn. A wave finds its
// token's angles, one per lane, and hands them round through LDS (8 per lane in registers, as the lanes need them:
// 2,048 rows of 48/8 heads 27.6 us, VALU-bound). A rotated dim's partner (half layout) comes by a load of its own,
// out with the lane's own values, rather than from another lane behind them.
struct RotateArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const uint16_t* q_w;  // norm weights; null: no norm
  const uint16_t* k_w;
  float eps;
  const float* freq;  // radians per position [dims / 2]
  int dims;           // rotated dims of a head
  float mscale;       // factor on rotated dims
  PagedBufs buf;
  PageTable tab;
  const int32_t* starts;
  uint16_t* q_out;  // [T, Hq, 128]
  uint16_t* k_out;  // the stored rows as they read, [T, Hkv, 128]; null: not asked for
  uint16_t* v_out;
  int T, Hq, Hkv;
  int per_tok;  // waves of a token
  FastDiv tok;
};

// cos and sin (times mscale) of a pair's angle at a position. The angle is a product in 64 bits, reduced to a turn
// there: in 32 it would be off by 0.004 radians at position 82,671, two steps of a bf16 sine.
__device__ __forceinline__ float2 rotation(const RotateArgs& a, int64_t pos, int pair) {
  const double turns = (double)pos * (double)a.freq[pair] * 0.15915494309189535;
  float sn, cs;
  sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
  return make_float2(cs * a.mscale, sn * a.mscale);
}
// Those of a lane's 8 dims, the sine with the sign that its partner takes; 1 and 0 of dims that stay.
template <bool PAIRS>
__device__ __forceinline__ void rotation8(const float2* pairs, int d0, int dims, float (&c)[8], float (&s)[8]) {
  const int half = dims >> 1;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const int d = d0 + j;
    if (PAIRS) {
      const float2 p = d < dims ? pairs[d >> 1] : make_float2(1.0f, 0.0f);
      c[j] = c[j + 1] = p.x;
      s[j] = -p.y;
      s[j + 1] = p.y;
    } else {  // half is even: two dims are of one side
      const int at = d < half ? d : d - half;
      const float4 p = d < dims ? *reinterpret_cast<const float4*>(pairs + at) : make_float4(1.0f, 0.0f, 1.0f, 0.0f);
      c[j] = p.x;
      s[j] = d < half ? -p.y : p.y;
      c[j + 1] = p.z;
      s[j + 1] = d < half ? -p.w : p.w;
    }
  }
}
// The 8 values at a lane's partner dims (half layout), 0 for dims that stay. WIDE: dims / 2 is a multiple of 8, they
// lie together.
template <bool WIDE>
__device__ __forceinline__ uint4 partner8(const uint16_t* row, int d0, int dims) {
  const int half = dims >> 1;
  if constexpr (WIDE) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + (d0 < half ? d0 + half : d0 < dims ? d0 - half : d0));
    return d0 < dims ? u : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // half is even
      const int d = d0 + 2 * j;
      const uint32_t u = *reinterpret_cast<const uint32_t*>(row + (d < half ? d + half : d < dims ? d - half : d));
      w[j] = d < dims ? u : 0;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// Sum over the 16 lanes of a head.
__device__ __forceinline__ float sum16(float x) {
  x += dpp<DPP_QUAD_XOR1>(x);
  x += dpp<DPP_QUAD_XOR2>(x);
  x += dpp<DPP_ROW_ROR4>(x);
  return x + dpp<DPP_ROW_ROR8>(x);
}

// Turns of a wave where the heads of all tokens fill this many waves per CU: its norm weights and angles are loaded once.
// us, of 2, 4 and 8: 2,048 rows of 48/8 heads 21.1, 20.6, 20.0; 7 packed prompts of up to 4,099 78.5, 82.4, 96.4.
constexpr int ROTATE_TURNS = 4, ROTATE_MANY = 32;

template <bool PAIRS, bool WIDE, int RT>
__global__ __launch_bounds__(256) void paged_rotate_kernel(const RotateArgs a, const PackedRows rows) {
  __shared__ alignas(16) float2 sh_pairs[4][D / 2];
  const int lane = threadIdx.x & 63, sub = lane & 15, d0 = 8 * sub;
  const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int t = (int)fdiv_u((uint32_t)wave, a.tok);
  if (t >= a.T) return;
  const int h0 = 4 * RT * (wave - t * a.per_tok) + (lane >> 4);
  const int heads = a.Hq + 2 * a.Hkv;
  // a head's row; past the last head the last one's, not stored
  auto row_of = [&](int h) {
    h = min(h, heads - 1);
    return h < a.Hq             ? a.q + t * a.q_tok + h * a.q_head
           : h < a.Hq + a.Hkv ? a.k + t * a.k_tok + (h - a.Hq) * a.k_head
                              : a.v + t * a.v_tok + (h - a.Hq - a.Hkv) * a.v_head;
  };
  uint4 own[RT], other[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const uint16_t* row = row_of(h0 + 4 * i);
    own[i] = *reinterpret_cast<const uint4*>(row + d0);
    if constexpr (!PAIRS) other[i] = partner8<WIDE>(row, d0, a.dims);
  }
  const int end = lane < rows.nseq ? rows.begin[lane + 1] : INT32_MAX;
  const int b = __builtin_amdgcn_readfirstlane(find_packed(end, t));
  const int64_t pos = (int64_t)a.starts[b] + (t - rows.begin[b]);
  const bool inside = pos >= 0 && pos < (int64_t)a.tab.width * PAGE;
  const int id = inside ? a.tab.ids[b * a.tab.stride + (pos >> 6)] : -1;
  const bool stored = id >= 0 && id < a.tab.pages;
  float2* pairs = sh_pairs[threadIdx.x >> 6];
  if (2 * lane < a.dims) pairs[lane] = rotation(a, pos, lane);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float c[8], s[8];
  rotation8<PAIRS>(pairs, d0, a.dims, c, s);
  // a dim's partner among neighbours; of dims that stay 0, as partner8's: 0 times an infinite one is no 0
  auto neighbour = [&](const float (&v)[8], int j) { return d0 + j < a.dims ? v[j ^ 1] : 0.0f; };
  float cw[8], sw[8];  // with the norm weights of the dim and of its partner
  const uint16_t* of = nullptr;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    cw[j] = c[j];
    sw[j] = s[j];
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int h = h0 + 4 * i;
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    const uint16_t* w = is_v ? of : is_q ? a.q_w : a.k_w;
    if (w != of) {  // a lane's first head, and where its queries end
      of = w;
      float g[8], o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = o[j] = 1.0f;
      if (w) {
        unpack8(*reinterpret_cast<const uint4*>(w + d0), g);
        if constexpr (!PAIRS) unpack8(partner8<WIDE>(w, d0, a.dims), o);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cw[j] = c[j] * g[j];
        sw[j] = s[j] * (PAIRS ? neighbour(g, j) : o[j]);
      }
    }
    float x[8], y[8];
    unpack8(own[i], x);
    if constexpr (PAIRS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = neighbour(x, j);
    } else {
      unpack8(other[i], y);
    }
    if (!is_v) {
      float inv = 1.0f;
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
        inv = rsqrtf(sum16(ss) * (1.0f / D) + a.eps);
      }
      float r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = fmaf(y[j], sw[j], x[j] * cw[j]) * inv;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = r[j];
    }
    if (is_q)  // rounded here and nowhere before
      *reinterpret_cast<uint4*>(a.q_out + ((int64_t)t * a.Hq + h) * D + d0) =
          make_uint4(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7]));
    if (!__builtin_amdgcn_ballot_w64(!is_q)) continue;  // queries alone
    uint2 codes;
    const AffineParams p = quantize8(x, codes);
    if (is_q || h >= heads) continue;
    const int hk = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
    const uint16_t sb = f32_to_bf16(p.scale), zb = f32_to_bf16(p.bias);
    if (stored) {
      const int64_t row = ((int64_t)id * a.Hkv + hk) * PAGE + (pos & (PAGE - 1));
      *reinterpret_cast<uint2*>((is_v ? a.buf.vc : a.buf.kc) + row * D + d0) = codes;
      if ((sub & 7) == 0) {
        (is_v ? a.buf.vs : a.buf.ks)[2 * row + (sub >> 3)] = sb;
        (is_v ? a.buf.vb : a.buf.kb)[2 * row + (sub >> 3)] = zb;
      }
    }
    if (a.k_out) {
      const uint2 lo = dequant4(codes.x, bf16_to_f32(sb), bf16_to_f32(zb));
      const uint2 hi = dequant4(codes.y, bf16_to_f32(sb), bf16_to_f32(zb));
      *reinterpret_cast<uint4*>((is_v ? a.v_out : a.k_out) + ((int64_t)t * a.Hkv + hk) * D + d0) =
          make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
}

// ---- gather: a workgroup per (page of a sequence, head, K or V): 16 codes of two rows per thread. A
// sequence of n rows touches at most (n + 62) / 64 + 1 pages, whatever its start.
struct GatherUnits {
  int begin[LQ_MAX_SEQS + 1];
};

__global__ __launch_bounds__(256) void paged_gather_kernel(PagedBufs buf, PageTable tab,
                                                           const int32_t* __restrict__ starts,
                                                           PackedRows rows, GatherUnits units, int Hkv,
                                                           uint16_t* __restrict__ k_out,
                                                           uint16_t* __restrict__ v_out) {
  const int tid = threadIdx.x, lane = tid & 63;
  const bool is_v = blockIdx.y != 0;
  const int x = blockIdx.x / Hkv, h = blockIdx.x - x * Hkv;
  const int end = lane < rows.nseq ? units.begin[lane + 1] : INT32_MAX;
  const int b = __builtin_amdgcn_readfirstlane(find_packed(end, x));
  const int64_t first = starts[b];
  const int64_t page = (first >> 6) + (x - units.begin[b]);  // of the sequence
  const int n = rows.begin[b + 1] - rows.begin[b];
  const int id = page >= 0 && page < tab.width ? tab.ids[b * tab.stride + page] : -1;
  const bool good = id >= 0 && id < tab.pages;
  const int64_t base = ((int64_t)(good ? id : 0) * Hkv + h) * PAGE;
  const uint8_t* codes = is_v ? buf.vc : buf.kc;
  const uint16_t* sc = is_v ? buf.vs : buf.ks;
  const uint16_t* bi = is_v ? buf.vb : buf.kb;
  uint16_t* out = is_v ? v_out : k_out;
  const int chunk = tid & 7;
  uint4 c[2];
  float s[2], z[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = base + (tid >> 3) + 32 * i;
    c[i] = __builtin_bit_cast(
        uint4, __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(codes + row * D + 16 * chunk)));
    s[i] = bf16_to_f32(sc[2 * row + (chunk >> 2)]);
    z[i] = bf16_to_f32(bi[2 * row + (chunk >> 2)]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = PAGE * page + (tid >> 3) + 32 * i - first;  // row of the sequence's range
    if (r < 0 || r >= n) continue;
    uint2 o[4] = {dequant4(c[i].x, s[i], z[i]), dequant4(c[i].y, s[i], z[i]),
                  dequant4(c[i].z, s[i], z[i]), dequant4(c[i].w, s[i], z[i])};
    if (!good) {  // no such page: not a number
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
    }
    uint4* dst = reinterpret_cast<uint4*>(out + ((rows.begin[b] + r) * Hkv + h) * D + 16 * chunk);
    dst[0] = make_uint4(o[0].x, o[0].y, o[1].x, o[1].y);
    dst[1] = make_uint4(o[2].x, o[2].y, o[3].x, o[3].y);
  }
}

// ---- page copies: a workgroup per (pair, head), all loads before the first store, non-temporal (1,500
// pages of 8 heads 94 -> 80 us, 5.2 TB/s; the loads alone 94).
constexpr int COPY_PAIRS = 480;  // of one launch: kernel arguments are limited to 4 KB
struct CopyPairs {
  int src[COPY_PAIRS], dst[COPY_PAIRS];
};

__global__ __launch_bounds__(256) void copy_pages_kernel(PagedBufs buf, CopyPairs pairs, int Hkv) {
  const int tid = threadIdx.x;
  const int x = blockIdx.x / Hkv, h = blockIdx.x - x * Hkv;
  const int64_t from = ((int64_t)pairs.src[x] * Hkv + h) * PAGE;
  const int64_t to = ((int64_t)pairs.dst[x] * Hkv + h) * PAGE;
  const u4_t* kf = reinterpret_cast<const u4_t*>(buf.kc + from * D) + tid;
  const u4_t* vf = reinterpret_cast<const u4_t*>(buf.vc + from * D) + tid;
  u4_t* kt = reinterpret_cast<u4_t*>(buf.kc + to * D) + tid;
  u4_t* vt = reinterpret_cast<u4_t*>(buf.vc + to * D) + tid;
  const u4_t a0 = __builtin_nontemporal_load(kf), a1 = __builtin_nontemporal_load(kf + 256);
  const u4_t b0 = __builtin_nontemporal_load(vf), b1 = __builtin_nontemporal_load(vf + 256);
  // scales and biases: 4 arrays of 256 bytes, 16 threads each
  const int arr = tid >> 4;
  uint16_t* w = arr == 0 ? buf.ks : arr == 1 ? buf.kb : arr == 2 ? buf.vs : buf.vb;
  uint4 c = make_uint4(0, 0, 0, 0);
  if (arr < 4) c = reinterpret_cast<const uint4*>(w + 2 * from)[tid & 15];
  __builtin_nontemporal_store(a0, kt);
  __builtin_nontemporal_store(a1, kt + 256);
  __builtin_nontemporal_store(b0, vt);
  __builtin_nontemporal_store(b1, vt + 256);
  if (arr < 4) reinterpret_cast<uint4*>(w + 2 * to)[tid & 15] = c;
}

// Row ranges of up to LQ_MAX_SEQS sequences from their host counts; -1 with the error set if they are bad.
int64_t pack_rows(const int32_t* counts, int64_t nseq, PackedRows* r) {
  if (nseq < 1 || nseq > LQ_MAX_SEQS || !counts) {
    set_error("%lld sequences are not in [1, %d], or no counts", (long long)nseq, LQ_MAX_SEQS);
    return -1;
  }
  int64_t at = 0;
  r->nseq = (int)nseq;
  r->begin[0] = 0;
  for (int i = 0; i < nseq; ++i) {
    if (counts[i] < 0 || (at += counts[i]) >= (1 << 30)) {
      set_error("row count %d of sequence %d", (int)counts[i], i);
      return -1;
    }
    r->begin[i + 1] = (int)at;
  }
  return at;
}

}  // namespace
}  // namespace lq

extern "C" int lq_paged_append(const uint16_t* k, const uint16_t* v, int64_t k_tok, int64_t k_head,
                               int64_t v_tok, int64_t v_head, uint8_t* kc, uint16_t* ks, uint16_t* kb,
                               uint8_t* vc, uint16_t* vs, uint16_t* vb, int64_t pages, int64_t Hkv,
                               int64_t D, const int32_t* table, int64_t table_stride,
                               int64_t table_width, const int32_t* starts, const int32_t* counts_host,
                               int64_t nseq, void* stream) {
  using namespace lq;
  clear_error();
  const PagedBufs buf{kc, ks, kb, vc, vs, vb};
  const PageTable tab{table, table_stride, (int)table_width, (int)pages};
  if (const int st = check_pool(buf, tab, table_stride, table_width, pages, Hkv, D)) return st;
  PackedRows rows;
  const int64_t T = pack_rows(counts_host, nseq, &rows);
  if (T < 0) return LQ_EINVAL;
  if (T == 0) return LQ_OK;
  LQ_CHECK_ARG(k && v && starts, "null pointer");
  LQ_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0 &&
                   ((k_tok | k_head | v_tok | v_head) & 7) == 0,
               "rows must be 16-byte aligned (strides a multiple of 8)");
  const int64_t units = T * Hkv;
  LQ_CHECK_ARG((units + 15) / 16 < 1 << 24, "an append of %lld rows is too large for one call",
               (long long)T);
  paged_append_kernel<<<dim3((unsigned)((units + 15) / 16), 2), dim3(256), 0, (hipStream_t)stream>>>(
      k, v, k_tok, k_head, v_tok, v_head, buf, tab, starts, rows, (uint32_t)units,
      make_fastdiv((uint32_t)Hkv), (int)Hkv);
  LQ_CHECK_LAUNCH("paged_append_kernel");
  return LQ_OK;
}

extern "C" int lq_paged_append_rotated(
    const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t q_tok, int64_t q_head, int64_t k_tok,
    int64_t k_head, int64_t v_tok, int64_t v_head, const uint16_t* q_norm_w, const uint16_t* k_norm_w, float eps,
    const float* inv_freq, int64_t rot_dims, float mscale, int interleaved, uint8_t* kc, uint16_t* ks, uint16_t* kb,
    uint8_t* vc, uint16_t* vs, uint16_t* vb, int64_t pages, int64_t Hq, int64_t Hkv, int64_t D,
    const int32_t* table, int64_t table_stride, int64_t table_width, const int32_t* starts,
    const int32_t* counts_host, int64_t nseq, uint16_t* q_out, uint16_t* k_out, uint16_t* v_out, void* stream) {
  using namespace lq;
  clear_error();
  const PagedBufs buf{kc, ks, kb, vc, vs, vb};
  const PageTable tab{table, table_stride, (int)table_width, (int)pages};
  if (const int st = check_pool(buf, tab, table_stride, table_width, pages, Hkv, D)) return st;
  LQ_CHECK_ARG(Hq >= 0 && Hq <= (1 << 16), "%lld query heads are not in [0, 2^16]", (long long)Hq);
  LQ_CHECK_ARG(rot_dims >= 0 && rot_dims <= D && rot_dims % (interleaved ? 2 : 4) == 0,
               "%lld rotated dims are not a multiple of %d in [0, %lld]", (long long)rot_dims, interleaved ? 2 : 4,
               (long long)D);
  LQ_CHECK_ARG(rot_dims == 0 || inv_freq, "no frequencies for %lld rotated dims", (long long)rot_dims);
  LQ_CHECK_ARG(std::isfinite(mscale) && eps >= 0.0f && std::isfinite(eps), "mscale or eps out of range");
  PackedRows rows;
  const int64_t T = pack_rows(counts_host, nseq, &rows);
  if (T < 0) return LQ_EINVAL;
  if (T == 0) return LQ_OK;
  LQ_CHECK_ARG((Hq == 0 || (q && q_out)) && k && v && starts, "null pointer");
  LQ_CHECK_ARG((k_out == nullptr) == (v_out == nullptr), "one of k_out and v_out alone");
  LQ_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_out |
                 (uintptr_t)v_out | (uintptr_t)q_norm_w | (uintptr_t)k_norm_w) & 15) == 0 &&
                   ((q_tok | q_head | k_tok | k_head | v_tok | v_head) & 7) == 0,
               "rows and norm weights must be 16-byte aligned (strides a multiple of 8)");
  RotateArgs a{q, k, v, q_tok, q_head, k_tok, k_head, v_tok, v_head, q_norm_w, k_norm_w, eps, inv_freq, (int)rot_dims,
               mscale, buf, tab, starts, q_out, k_out, v_out, (int)T, (int)Hq, (int)Hkv, 0, {}};
  const int64_t heads = Hq + 2 * Hkv;
  const bool wide = rot_dims % 16 == 0, many = T * ((heads + 3) / 4) >= ROTATE_MANY * (int64_t)device_cu_count();
  a.per_tok = (int)((heads + 3) / 4);
  if (many) a.per_tok = (a.per_tok + ROTATE_TURNS - 1) / ROTATE_TURNS;
  a.tok = make_fastdiv((uint32_t)a.per_tok);
  const int64_t waves = T * a.per_tok;
  LQ_CHECK_ARG(waves < (int64_t)1 << 26, "an append of %lld rows is too large for one call", (long long)T);
  auto* kern = interleaved ? (many ? paged_rotate_kernel<true, true, ROTATE_TURNS> : paged_rotate_kernel<true, true, 1>)
               : wide      ? (many ? paged_rotate_kernel<false, true, ROTATE_TURNS> : paged_rotate_kernel<false, true, 1>)
                      : (many ? paged_rotate_kernel<false, false, ROTATE_TURNS> : paged_rotate_kernel<false, false, 1>);
  kern<<<dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, (hipStream_t)stream>>>(a, rows);
  LQ_CHECK_LAUNCH("paged_rotate_kernel");
  return LQ_OK;
}

extern "C" int lq_paged_gather(const uint8_t* kc, const uint16_t* ks, const uint16_t* kb,
                               const uint8_t* vc, const uint16_t* vs, const uint16_t* vb, int64_t pages,
                               int64_t Hkv, int64_t D, const int32_t* table, int64_t table_stride,
                               int64_t table_width, const int32_t* starts, const int32_t* counts_host,
                               int64_t nseq, uint16_t* k_out, uint16_t* v_out, void* stream) {
  using namespace lq;
  clear_error();
  const PagedBufs buf{const_cast<uint8_t*>(kc),  const_cast<uint16_t*>(ks), const_cast<uint16_t*>(kb),
                      const_cast<uint8_t*>(vc),  const_cast<uint16_t*>(vs), const_cast<uint16_t*>(vb)};
  const PageTable tab{table, table_stride, (int)table_width, (int)pages};
  if (const int st = check_pool(buf, tab, table_stride, table_width, pages, Hkv, D)) return st;
  PackedRows rows;
  const int64_t T = pack_rows(counts_host, nseq, &rows);
  if (T < 0) return LQ_EINVAL;
  if (T == 0) return LQ_OK;
  LQ_CHECK_ARG(k_out && v_out && starts, "null pointer");
  LQ_CHECK_ARG((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "outputs must be 16-byte aligned");
  GatherUnits units;
  units.begin[0] = 0;
  for (int i = 0; i < nseq; ++i)
    units.begin[i + 1] = units.begin[i] + (counts_host[i] ? (counts_host[i] + 62) / PAGE + 1 : 0);
  const int64_t wgs = (int64_t)units.begin[nseq] * Hkv;
  LQ_CHECK_ARG(wgs < (int64_t)1 << 24, "a gather of %lld rows is too large for one call", (long long)T);
  paged_gather_kernel<<<dim3((unsigned)wgs, 2), dim3(256), 0, (hipStream_t)stream>>>(
      buf, tab, starts, rows, units, (int)Hkv, k_out, v_out);
  LQ_CHECK_LAUNCH("paged_gather_kernel");
  return LQ_OK;
}

extern "C" int lq_copy_pages(uint8_t* kc, uint16_t* ks, uint16_t* kb, uint8_t* vc, uint16_t* vs,
                             uint16_t* vb, int64_t pages, int64_t Hkv, int64_t D,
                             const int32_t* src_host, const int32_t* dst_host, int64_t n, void* stream) {
  using namespace lq;
  clear_error();
  const PagedBufs buf{kc, ks, kb, vc, vs, vb};
  const PageTable tab{src_host, 0, 1, (int)pages};
  LQ_CHECK_ARG(n >= 0, "%lld pages to copy", (long long)n);
  if (n == 0) return LQ_OK;
  LQ_CHECK_ARG(dst_host, "null pointer");
  if (const int st = check_pool(buf, tab, 0, 1, pages, Hkv, D)) return st;
  LQ_CHECK_ARG(n <= pages, "%lld pages to copy in a pool of %lld", (long long)n, (long long)pages);
  // every destination once, and no page that is also a source: the copies run in any order
  std::vector<uint8_t> role;
  try {
    role.resize((size_t)pages);
  } catch (...) {
    set_error("no host memory for a pool of %lld pages", (long long)pages);
    return LQ_EHIP;
  }
  for (int64_t i = 0; i < n; ++i) {
    LQ_CHECK_ARG(src_host[i] >= 0 && src_host[i] < pages && dst_host[i] >= 0 && dst_host[i] < pages,
                 "pair %lld: page %d to %d of a pool of %lld", (long long)i, (int)src_host[i],
                 (int)dst_host[i], (long long)pages);
    role[src_host[i]] = 1;
  }
  for (int64_t i = 0; i < n; ++i) {
    LQ_CHECK_ARG(role[dst_host[i]] == 0, "page %d is written twice, or is both read and written",
                 (int)dst_host[i]);
    role[dst_host[i]] = 2;
  }
  for (int64_t at = 0; at < n; at += COPY_PAIRS) {
    CopyPairs pairs;
    const int m = (int)std::min<int64_t>(COPY_PAIRS, n - at);
    for (int i = 0; i < m; ++i) {
      pairs.src[i] = src_host[at + i];
      pairs.dst[i] = dst_host[at + i];
    }
    for (int i = m; i < COPY_PAIRS; ++i) pairs.src[i] = pairs.dst[i] = 0;
    copy_pages_kernel<<<dim3((unsigned)(m * Hkv)), dim3(256), 0, (hipStream_t)stream>>>(buf, pairs,
                                                                                      (int)Hkv);
    LQ_CHECK_LAUNCH("copy_pages_kernel");
  }
  return LQ_OK;
}
