// Rows into and out of a paged 8-bit cache, and pages copied within it.
//
// lq_paged_append quantizes K/V rows (bf16, any token and head strides) into the pages of several
// sequences, with the arithmetic of the contiguous cache's append; lq_paged_gather reads positions back
// as bf16 rows, packed one sequence behind the other, as the contiguous cache's dequantize; lq_copy_pages
// copies pages of all heads. All three are bound by their traffic (append 512 B read and 272 B written
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
  const uint4 x4 = *reinterpret_cast<const uint4*>(src + 8 * sub);
  const uint32_t xw[4] = {x4.x, x4.y, x4.z, x4.w};
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = bf16_lo(xw[j]);
    x[2 * j + 1] = bf16_hi(xw[j]);
  }
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
  if (id < 0 || id >= tab.pages) return;
  const int64_t row = ((int64_t)id * Hkv + h) * PAGE + (pos & (PAGE - 1));
  uint8_t* codes = is_v ? buf.vc : buf.kc;
  *reinterpret_cast<uint2*>(codes + row * D + 8 * sub) =
      make_uint2(c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24),
                 c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24));
  if ((sub & 7) == 0) {
    (is_v ? buf.vs : buf.ks)[2 * row + (sub >> 3)] = f32_to_bf16(p.scale);
    (is_v ? buf.vb : buf.kb)[2 * row + (sub >> 3)] = f32_to_bf16(p.bias);
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
