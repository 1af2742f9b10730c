// Attention of one new token per sequence over a paged 8-bit cache, the pages that all sequences share
// read once for the batch (a prompt and the answers sampled from it, a long system prompt).
//
// Work. A KV head's shared pages are cut into np parts; a workgroup takes one part for a block of 32, 64 or
// 128 query rows (the G rows of each sequence, one sequence behind the other), dequantizes each page
// once into LDS and runs the matrix-core tile of attn_tile.h on it; of long parts the workgroup of own pages
// beside it takes the last pages (late_pages). The sequences' own pages, one sequence
// behind the other, are dealt out to the workgroups in equal shares; a workgroup runs its pages of a sequence
// for the G <= 16 rows, one page per wave at a time, through the wave's own LDS (no barriers), the next
// page's loads out while it computes. With up to 16 query rows in the batch the shared pages are dealt out
// with the own ones, in front of them, as those of one sequence with all the rows. Both kinds write
// partial rows (max, sum, weighted values), which a second launch merges. Where table rows list few pages a
// workgroup takes a whole sequence instead, and writes its output rows (short_waves has the rule).
//
// Lengths are read on the device, so one recorded launch serves every step of a growing batch: every
// workgroup adds up the sequences' own pages and finds its share of them. Workgroups without one leave at
// once.
//
// Values: an attended K or V is bf16(scale * code + bias), what dequantizing the page gives; products on
// bf16 operands with fp32 sums, P rounded to bf16 (in the values and in its sum alike, so that a row that
// one key rules keeps that key's V). Positions past a length are not attended whatever their slots hold:
// their scores are -infinity and their V terms 0. A length outside [0, 64 width] or a page outside the
// pool makes the sequence's rows NaN; length 0 makes them 0. A sequence shorter than the shared part takes
// no part in it: its own parts cover it whole.
#include "paged_tile.h"

namespace lq {
namespace {

using namespace attn;

constexpr int DW = 4;         // waves per workgroup
constexpr int SHARE_MIN = 4;  // pages of a share: one per wave
// Cost of starting on a sequence, in pages: shares of many short ones would end last. us at 0 / 2 / 4 / 8: 64
// sessions of 10 to 500 positions (in wider tables than those of short_waves), 32/8 heads 26.9 / 21.7 / 20.8 /
// 20.8, 8 of 100 to 4,000 21.8 / 19.2 / 17.8 / 19.6, 4 of 100 to 300 behind 65,536 50.2 / 42.0 / 40.2 / 39.8.
constexpr int SEQ_COST = 4;

struct PagedArgs {
  const uint16_t* q;
  PagedBufs buf;
  PageTable tab;
  const int32_t* lens;
  float* part_acc;    // [Hkv][slots][128], slots: (share + sequence) x G, then np x rows of all
  float2* part_ml;
  uint16_t* out;
  int B, Hkv, G;
  int shared;         // pages that all sequences share
  int np, rb;         // their parts, blocks of query rows; 0: dealt out with the own pages
  bool late;          // parts long enough for late_pages
  int shares;         // workgroups for the own pages of a KV head
  float sl2;          // softmax scale, log2 units
};

__device__ __forceinline__ bool len_ok(const PagedArgs& a, int len) {
  return len >= 0 && len <= (int64_t)a.tab.width * PAGE;
}
// First own page of a sequence, and how many.
__device__ __forceinline__ int own_first(const PagedArgs& a, int len) {
  return len >= a.shared * PAGE ? a.shared : 0;
}
__device__ __forceinline__ int own_pages(const PagedArgs& a, int len) {
  return len_ok(a, len) ? (len + PAGE - 1) / PAGE - own_first(a, len) : 0;
}

// What a sequence's own pages cost: one each, and a constant in front.
__device__ __forceinline__ int own_cost(const PagedArgs& a, int len) {
  const int n = own_pages(a, len);
  return n ? n + SEQ_COST : 0;
}

// What the call deals out, in pages, the shared ones in front (0: no sequence is long enough, or the shared
// part is not dealt out), and a share. The same in every workgroup of a call.
struct Deal {
  int lead, total, share;
};
__device__ __forceinline__ Deal deal_out(const PagedArgs& a, int lane) {
  int total = 0;
  bool joins = false;
  for (int i = lane; i < a.B; i += 64) {
    const int len = a.lens[i];
    total += own_cost(a, len);
    joins |= len_ok(a, len) && len >= a.shared * PAGE;
  }
  const int lead = a.np == 0 && __builtin_amdgcn_ballot_w64(joins) ? a.shared : 0;
  total = wave_sum_i(total) + lead;
  return {lead, total, max(SHARE_MIN, (total + a.shares - 1) / a.shares)};
}
// Pages of each shared part that are left to the workgroup of own pages beside it on the CU, so that both end
// together: a share takes about OWN_START and 2/3 per page in times of a shared page, with the start on the part.
// LATE_MIN: fewer do not pay for the partials. us without and with, 8 KV heads, own pages of 1 to 64 / 1,500 to
// 2,500 positions: 82,688 shared positions of 5 sequences, 32 heads 64.1 / 65.9 -> 44.7 / 48.6, of 16 66.5 / 71.6 ->
// 54.2 / 65.3, of 48, 48 heads 232 / 242 -> 176 / 200 (together with SPLIT); 16,384 of 48, which leave none, alike.
constexpr int OWN_START = 10, LATE_MIN = 8;
__device__ __forceinline__ int late_pages(const PagedArgs& a, const Deal& deal) {
  const int own = deal.total ? OWN_START + 2 * deal.share / 3 : 0;
  const int left = (a.shared / a.np - own) / 2;
  return left < LATE_MIN ? 0 : left;
}
// The table row that lists the shared pages: of the first sequence that is long enough (a shorter one's may
// end before them); null: there is none.
__device__ __forceinline__ const int32_t* shared_ids(const PagedArgs& a, int lane) {
  for (int i = 0; i < a.B; i += 64) {
    const int len = i + lane < a.B ? a.lens[i + lane] : -1;
    const uint64_t joins = __builtin_amdgcn_ballot_w64(len_ok(a, len) && len >= a.shared * PAGE);
    if (joins) return a.tab.ids + (i + __builtin_ctzll(joins)) * a.tab.stride;
  }
  return nullptr;
}

template <int WV>  // waves
struct OwnSmem {
  // a page's codes, per wave: 16-byte chunk c of row r of K at c ^ kswz(r), of V at c ^ vswz(r)
  alignas(16) uint8_t k[WV][PAGE * D], v[WV][PAGE * D];
  uint32_t w[WV][4][PAGE];  // its K scale, K bias, V scale, V bias words
  float2 ml[WV][16];
};
// Pages [p0, p1) listed at ids, of a sequence of len positions, for R <= 16 query rows (row lane % 16 of them
// at qrow): partial rows to slot .., or with WHOLE output rows from slot on.
template <int WV, bool WHOLE>
__device__ __forceinline__ void own_part(const PagedArgs& a, OwnSmem<WV>& sm, const int32_t* ids, int R,
                                         int64_t qrow, int hk, int p0, int p1, int len, int64_t slot) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 15, lq4 = lane >> 4;
  __syncthreads();  // the sequence before is written
  const float scale = abs_scale(a.sl2);
  // q as B operands in K's order of dims: k-step 2 h + j holds dims 64 h + 16 lq4 + 8 j .. + 7
  bf16x8_t qf[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (lc < R)
      u = *reinterpret_cast<const uint4*>(a.q + qrow * D + 64 * (kk >> 1) + 16 * lq4 + 8 * (kk & 1));
    qf[kk] = u4_as_bf8(signed_q(u, a.sl2));
  }
  f4_t o[8];
#pragma unroll
  for (int w = 0; w < 8; ++w) o[w] = f4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY;
  f4_t l = {0.f, 0.f, 0.f, 0.f};  // sums of the rounded weights, the same in all four (a product with ones)
  bool bad = false;

  auto page_row = [&](int p) {
    const int id = __builtin_amdgcn_readfirstlane(ids[p]);
    const bool ok = id >= 0 && id < a.tab.pages;
    bad |= !ok;
    return ((int64_t)(ok ? id : 0) * a.Hkv + hk) * PAGE;
  };

  PageRegs cur;
  int p = p0 + wv;
  if (p < p1) load_page(a.buf, page_row(p), lane, cur);
  for (; p < p1; p += WV) {
    const int limit = min(PAGE, len - p * PAGE);  // keys of the page that are the sequence's
    // to LDS, and the next page's loads out at once; V words of keys past the length 0, so that their
    // slots' contents reach nothing
    wave_fence();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 8 * i + (lane >> 3), c = lane & 7;
      reinterpret_cast<u4_t*>(sm.k[wv])[8 * r + (c ^ kswz(r))] = cur.k[i];
      reinterpret_cast<u4_t*>(sm.v[wv])[8 * r + (c ^ vswz(r))] = cur.v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sm.w[wv][i][lane] = i < 2 || lane < limit ? cur.w[i] : 0u;
    if (p + WV < p1) load_page(a.buf, page_row(p + WV), lane, cur);
    wave_fence();
    // scores
    f4_t c[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      c[mt] = f4_t{0.f, 0.f, 0.f, 0.f};
      const int key = 16 * mt + lc;
      const uint32_t sw = sm.w[wv][0][key], zw = sm.w[wv][1][key];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float s = h ? bf16_hi(sw) : bf16_lo(sw), z = h ? bf16_hi(zw) : bf16_lo(zw);
        const u4_t w = reinterpret_cast<const u4_t*>(sm.k[wv])[8 * key + ((lq4 + 4 * h) ^ kswz(lc))];
        const uint2 d0 = dequant4(w[0], s, z), d1 = dequant4(w[1], s, z);
        const uint2 d2 = dequant4(w[2], s, z), d3 = dequant4(w[3], s, z);
        c[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(words_as_bf8(d0.x, d0.y, d1.x, d1.y), qf[2 * h],
                                                        c[mt], 0, 0, 0);
        c[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(words_as_bf8(d2.x, d2.y, d3.x, d3.y),
                                                        qf[2 * h + 1], c[mt], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (limit < PAGE) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          c[mt][r] = 16 * mt + 4 * lq4 + r < limit ? c[mt][r] : -INFINITY;
    }
    float t = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) t = max_ieee(t, c[mt][r]);
    t = max_xor32(max_xor16(t)) * scale;
    const bool bump = t > (m == -INFINITY ? -INFINITY : m + RESCALE_LOG2);
    if (__builtin_amdgcn_ballot_w64(bump)) {
      const float mn = bump ? t : m;
      const float alpha = m == -INFINITY ? 0.0f : exp2_nonpos(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int w = 0; w < 8; ++w) o[w] *= alpha;
    }
    float off = m == -INFINITY ? 0.0f : -m;
    if (__builtin_amdgcn_ballot_w64(is_huge(off))) settle_huge(c, off, scale);
    uint32_t pw[8];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(c[mt][r], scale, off));
      pw[2 * mt] = pack_bf2(e[0], e[1]);
      pw[2 * mt + 1] = pack_bf2(e[2], e[3]);
    }
    // values: lane (lq4, lc) gets the codes of keys 32 e + 16 h + 4 lq4 + r at dim 16 w + lc
    const int skey = 4 * lq4 + 16 * (lc >> 3) + ((lc >> 1) & 3);  // this lane's source key
    const uint8_t* src = sm.v[wv] + skey * D + 8 * (lc & 1);
    const int ssw = vswz(skey);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bf16x8_t pe = words_as_bf8(pw[4 * e], pw[4 * e + 1], pw[4 * e + 2], pw[4 * e + 3]);
      l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_ones(), pe, l, 0, 0, 0);
      const uint4 s0 = *reinterpret_cast<const uint4*>(&sm.w[wv][2][32 * e + 4 * lq4]);
      const uint4 s1 = *reinterpret_cast<const uint4*>(&sm.w[wv][2][32 * e + 4 * lq4 + 16]);
      const uint4 z0 = *reinterpret_cast<const uint4*>(&sm.w[wv][3][32 * e + 4 * lq4]);
      const uint4 z1 = *reinterpret_cast<const uint4*>(&sm.w[wv][3][32 * e + 4 * lq4 + 16]);
      const uint32_t sw[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
      const uint32_t zw[8] = {z0.x, z0.y, z0.z, z0.w, z1.x, z1.y, z1.z, z1.w};
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const v2i_t raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_v2i_t*)(src + 32 * e * D + 16 * (w ^ ssw)));
        const uint32_t r0 = (uint32_t)raw.x, r1 = (uint32_t)raw.y;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float s = w < 4 ? bf16_lo(sw[j]) : bf16_hi(sw[j]);
          const float z = w < 4 ? bf16_lo(zw[j]) : bf16_hi(zw[j]);
          v[j] = fmaf(s, (float)(((j < 4 ? r0 : r1) >> (8 * (j & 3))) & 0xffu), z);
        }
        o[w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            words_as_bf8(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]),
                         pack_bf2(v[6], v[7])),
            pe, o[w], 0, 0, 0);
        if (w & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // ---- the waves' rows meet in LDS (wave wv's in its own V area: 16 rows of 128 floats)
  wave_fence();
  float* acc = reinterpret_cast<float*>(sm.v[wv]);
  if (lc < R) {
#pragma unroll
    for (int w = 0; w < 8; ++w)
      *reinterpret_cast<float4*>(acc + lc * D + 16 * w + 4 * lq4) =
          make_float4(o[w][0], o[w][1], o[w][2], o[w][3]);
    if (lq4 == 0) sm.ml[wv][lc] = make_float2(m, bad ? NAN : l[0]);
  }
  __syncthreads();
  for (int i = tid; i < R * (D / 4); i += 64 * WV) {
    const int row = i >> 5, d = 4 * (i & 31);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WV; ++w) M = max_ieee(M, sm.ml[w][row].x);
    const float Mr = M == -INFINITY ? 0.0f : M;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < WV; ++w) {
      const float2 ml = sm.ml[w][row];
      const float e = ml.x == -INFINITY ? 0.0f : exp2_nonpos(ml.x - Mr);
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.v[w]) + row * D + d);
      s.x = fmaf(e, x.x, s.x);
      s.y = fmaf(e, x.y, s.y);
      s.z = fmaf(e, x.z, s.z);
      s.w = fmaf(e, x.w, s.w);
      L = fmaf(ml.x == -INFINITY ? 1.0f : e, ml.y, L);
    }
    if constexpr (WHOLE) {
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // no keys: 0; a sum that is NaN stays
      *reinterpret_cast<uint2*>(a.out + (slot + row) * D + d) =
          make_uint2(pack_bf2(s.x * inv, s.y * inv), pack_bf2(s.z * inv, s.w * inv));
      continue;
    }
    *reinterpret_cast<float4*>(a.part_acc + (slot + row) * D + d) = s;
    if (d == 0) a.part_ml[slot + row] = make_float2(M, L);
  }
}

// Shared pages [p0, p1) (listed in the table at ids) for the query rows of block `block` of a KV head. Each page
// is dequantized once into one of two tiles, the next one's codes on their way. With SPLIT (up to 32 rows) the two
// halves of the waves take the same rows, and half of a page's keys each, and meet in LDS at the end.
constexpr int CH = 8 / DW;  // chunks of a thread
template <int NT, bool SPLIT>
constexpr int block_rows() {
  return 16 * NT * (SPLIT ? DW / 2 : DW);
}
struct RawPage {  // key tid / 8 + 8 DW i, codes 16 (tid % 8) ..
  uint4 k[CH], v[CH];
  uint32_t ks[CH], kb[CH], vs[CH], vb[CH];
};
struct SharedSmem {
  KvTile tile[2];
};

template <int NT, bool SPLIT>
__device__ __forceinline__ void shared_part(const PagedArgs& a, SharedSmem& sm, const int32_t* ids, int hk,
                                            int p0, int p1, int block, int64_t slot) {
  constexpr int MT = SPLIT ? 2 : 4;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool upper = wv >= DW / 2;
  const int lc = lane & 15, lq4 = lane >> 4;
  const int rows = a.B * a.G;
  const int f0 = block * block_rows<NT, SPLIT>() + 16 * NT * (SPLIT ? wv % (DW / 2) : wv);
  const float scale = abs_scale(a.sl2);
  const int key0 = tid >> 3, chunk = tid & 7;
  bool bad = false;
  RawPage pre[2];  // pages p + 1 and p + 2
  auto load = [&](int p, RawPage& raw) {
    const int id = __builtin_amdgcn_readfirstlane(ids[min(p, p1 - 1)]);
    const bool ok = id >= 0 && id < a.tab.pages;
    bad |= !ok;
    const int64_t row = ((int64_t)(ok ? id : 0) * a.Hkv + hk) * PAGE;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      raw.k[i] = *reinterpret_cast<const uint4*>(a.buf.kc + row * D + 1024 * DW * i + 16 * tid);
      raw.v[i] = *reinterpret_cast<const uint4*>(a.buf.vc + row * D + 1024 * DW * i + 16 * tid);
      const int64_t r = row + key0 + 8 * DW * i;
      raw.ks[i] = reinterpret_cast<const uint32_t*>(a.buf.ks)[r];
      raw.kb[i] = reinterpret_cast<const uint32_t*>(a.buf.kb)[r];
      raw.vs[i] = reinterpret_cast<const uint32_t*>(a.buf.vs)[r];
      raw.vb[i] = reinterpret_cast<const uint32_t*>(a.buf.vb)[r];
    }
  };
  auto pick = [&](uint32_t w) { return chunk < 4 ? bf16_lo(w) : bf16_hi(w); };
  auto stage = [&](KvTile& t, const RawPage& raw) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int key = key0 + 8 * DW * i;
      const float s = pick(raw.ks[i]), z = pick(raw.kb[i]);
      const uint2 k0 = dequant4(raw.k[i].x, s, z), k1 = dequant4(raw.k[i].y, s, z);
      const uint2 k2 = dequant4(raw.k[i].z, s, z), k3 = dequant4(raw.k[i].w, s, z);
      *k_chunk(t, key, 2 * chunk) = make_uint4(k0.x, k0.y, k1.x, k1.y);
      *k_chunk(t, key, 2 * chunk + 1) = make_uint4(k2.x, k2.y, k3.x, k3.y);
      const float vs = pick(raw.vs[i]), vz = pick(raw.vb[i]);
      const uint2 v0 = dequant4(raw.v[i].x, vs, vz), v1 = dequant4(raw.v[i].y, vs, vz);
      const uint2 v2 = dequant4(raw.v[i].z, vs, vz), v3 = dequant4(raw.v[i].w, vs, vz);
      *v_chunk(t, key, 2 * chunk) = make_uint4(v0.x, v0.y, v1.x, v1.y);
      *v_chunk(t, key, 2 * chunk + 1) = make_uint4(v2.x, v2.y, v3.x, v3.y);
    }
  };
  load(p0, pre[0]);
  load(p0 + 1, pre[1]);
  TileRows<NT> st;
  st.clear();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int f = f0 + 16 * nt + lc;
    const int b = f / a.G;
    const int64_t row = ((int64_t)b * a.Hkv + hk) * a.G + (f - b * a.G);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (f < rows) u = *reinterpret_cast<const uint4*>(a.q + row * D + 32 * kk + 8 * lq4);
      st.q[nt][kk] = u4_as_bf8(signed_q(u, a.sl2));
    }
  }
  stage(sm.tile[0], pre[0]);
  load(p0 + 2, pre[0]);
  __syncthreads();
  const int part = SPLIT && upper ? 32 * D : 0;  // the wave's keys of a tile
  for (int p = p0; p < p1; p += 2) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {  // page p + s in tile s
      if (p + s >= p1) break;
      f4_t c[NT][MT];
      bf16x8_t pr[NT][MT / 2];
      tile_scores<NT>(sm.tile[s].k + part, st, lane, c);
      tile_softmax<NT>(c, st, scale, pr);
      tile_values<NT>(sm.tile[s].v + part, st, lane, pr);
      if (p + s + 1 < p1) {
        stage(sm.tile[s ^ 1], pre[s ^ 1]);
        load(p + s + 3, pre[s ^ 1]);
      }
      __syncthreads();
    }
  }
  if constexpr (SPLIT) {  // the upper half's rows to the lower's: a row of 132 floats, its maximum and sum
    float* at = reinterpret_cast<float*>(&sm) + (16 * (wv % (DW / 2)) + lc) * 132;
    if (upper) {
#pragma unroll
      for (int w = 0; w < 8; ++w) *reinterpret_cast<f4_t*>(at + 16 * w + 4 * lq4) = st.o[0][w];
      if (lq4 == 0) *reinterpret_cast<float2*>(at + 128) = make_float2(st.m[0], st.l[0][0]);
    }
    __syncthreads();
    if (upper) return;
    const float2 ml = *reinterpret_cast<const float2*>(at + 128);
    const float m = max_ieee(st.m[0], ml.x), mr = m == -INFINITY ? 0.0f : m;
    const float e0 = exp2_nonpos(st.m[0] - mr), e1 = exp2_nonpos(ml.x - mr);
#pragma unroll
    for (int w = 0; w < 8; ++w)
      st.o[0][w] = st.o[0][w] * e0 + *reinterpret_cast<const f4_t*>(at + 16 * w + 4 * lq4) * e1;
    st.l[0] = st.l[0] * e0 + ml.y * e1;
    st.m[0] = m;
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int f = f0 + 16 * nt + lc;
    if (f >= rows) continue;
#pragma unroll
    for (int w = 0; w < 8; ++w)
      *reinterpret_cast<float4*>(a.part_acc + (slot + f) * D + 16 * w + 4 * lq4) =
          make_float4(st.o[nt][w][0], st.o[nt][w][1], st.o[nt][w][2], st.o[nt][w][3]);
    if (lq4 == 0) a.part_ml[slot + f] = make_float2(st.m[nt], bad ? NAN : st.l[nt][0]);
  }
}

// Partial rows of one KV head: own parts first (along the shares and sequences each part adds one to their
// sum), then those of the shared pages, by part or by share.
__device__ __forceinline__ int64_t shared_slots(const PagedArgs& a) { return (int64_t)(a.shares + a.B) * a.G; }
__device__ __forceinline__ int64_t head_slots(const PagedArgs& a) {
  return shared_slots(a) + (int64_t)(a.np ? a.np << a.late : a.shared ? a.shares : 0) * a.B * a.G;
}

// Share x of the pages that are dealt out for a KV head.
template <int WV>
__device__ __forceinline__ void own_share(const PagedArgs& a, const Deal& deal, OwnSmem<WV>& sm, int hk, int x,
                                          int64_t slot0) {
  const int lane = threadIdx.x & 63;
  const int u0 = x * deal.share, u1 = min(u0 + deal.share, deal.total);
  if (u0 >= u1) return;
  const int lc = lane & 15;
  int u = u0;
  if (u < deal.lead) {  // shared pages, for all rows of the batch
    const int e = min(u1, deal.lead), b = lc / a.G;
    own_part<WV, false>(a, sm, shared_ids(a, lane), a.B * a.G, ((int64_t)b * a.Hkv + hk) * a.G + (lc - b * a.G), hk,
                        u, e, a.shared * PAGE, slot0 + shared_slots(a) + (int64_t)x * a.B * a.G);
    u = e;
  }
  if (u == u1) return;
  int b = 0, begin = deal.lead;  // the sequence that holds u, and the cost before it
  for (int i = 0;; i += 64) {
    const int n = i + lane < a.B ? own_cost(a, a.lens[i + lane]) : 0;
    const int upto = begin + wave_scan_i(n);
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > u);
    if (past || i + 64 >= a.B) {
      const int src = past ? __builtin_ctzll(past) : 0;
      b = i + src;
      begin = __builtin_amdgcn_readlane(upto - n, src);
      break;
    }
    begin = __builtin_amdgcn_readlane(upto, 63);
  }
  for (; u < u1; ++b) {
    const int len = a.lens[b], n = own_pages(a, len);
    if (n == 0) continue;
    begin += SEQ_COST;
    const int p0 = max(u - begin, 0), p1 = min(u1 - begin, n), first = own_first(a, len);
    if (p0 < p1)
      own_part<WV, false>(a, sm, a.tab.ids + b * a.tab.stride, a.G, ((int64_t)b * a.Hkv + hk) * a.G + lc, hk,
                          first + p0, first + p1, len, slot0 + (int64_t)(x + b) * a.G);
    begin += n;
    u = begin;
  }
}

__global__ __launch_bounds__(64 * DW, 2) void paged_decode_kernel(PagedArgs a) {
  __shared__ OwnSmem<DW> sm;
  const int hk = blockIdx.x % a.Hkv;
  own_share<DW>(a, deal_out(a, threadIdx.x & 63), sm, hk, blockIdx.x / a.Hkv, hk * head_slots(a));
}

// Two workgroups per CU: one takes a shared part for a block of rows, the other a share of the own pages, then, of
// a long part, the last pages.
template <int NT, bool SPLIT>
__global__ __launch_bounds__(64 * DW, 2) void paged_shared_kernel(PagedArgs a) {
  __shared__ union Smem {
    OwnSmem<DW> own;
    SharedSmem shared;
    __device__ Smem() {}
  } sm;
  const int hk = blockIdx.x % a.Hkv, n = a.np * a.rb;
  int x = blockIdx.x / a.Hkv;
  const bool late = x >= n;
  if (late) x -= n;
  const int64_t slot0 = hk * head_slots(a);
  const int lane = threadIdx.x & 63;
  if (late && x < a.shares) own_share<DW>(a, deal_out(a, lane), sm.own, hk, x, slot0);
  if (x >= n || (late && !a.late)) return;
  const int32_t* ids = shared_ids(a, lane);
  const int left = a.late ? late_pages(a, deal_out(a, lane)) : 0;
  if (!ids || (late && left == 0)) return;
  const int part = x / a.rb, block = x - part * a.rb;
  const int p0 = (int)((int64_t)a.shared * part / a.np);
  const int p1 = (int)((int64_t)a.shared * (part + 1) / a.np);
  __syncthreads();  // the share is written
  shared_part<NT, SPLIT>(a, sm.shared, ids, hk, late ? p1 - left : p0, late ? p1 : p1 - left, block,
                         slot0 + shared_slots(a) + (int64_t)(late ? a.np + part : part) * a.B * a.G);
}

// A whole sequence per workgroup, by 4 or 8 waves: nothing to merge.
template <int WV>
__global__ __launch_bounds__(64 * WV, 2) void paged_short_kernel(PagedArgs a) {
  __shared__ OwnSmem<WV> sm;
  const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv;
  const int len = a.lens[b];
  const int64_t row = ((int64_t)b * a.Hkv + hk) * a.G;
  if (!len_ok(a, len)) {
    for (int i = threadIdx.x; i < a.G * D; i += 64 * WV) a.out[row * D + i] = 0x7fc0;
    return;
  }
  own_part<WV, true>(a, sm, a.tab.ids + b * a.tab.stride, a.G, row + (threadIdx.x & 15), hk, 0,
                     (len + PAGE - 1) / PAGE, len, row);
}

// An output row by GR groups of 32 lanes (4 dims each), 8 / GR rows per workgroup: group g takes every GR-th
// partial, four at a time, and the groups meet in LDS.
template <int GR>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  __shared__ float2 sh_ml[8];
  __shared__ f4_t sh_acc[8][32];
  const int lane = threadIdx.x & 63;
  // wave-uniform: a row has at least a wave
  const int r = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / (32 * GR)));
  const int row = min((int)(blockIdx.x * (8 / GR)) + r, a.B * a.Hkv * a.G - 1);  // past the last: that again
  const int b = row / (a.Hkv * a.G), h = row - b * a.Hkv * a.G, hk = h / a.G, g = h - hk * a.G;
  const Deal deal = deal_out(a, lane);
  int before = 0;
  for (int i = lane; i < b; i += 64) before += own_cost(a, a.lens[i]);
  before = wave_sum_i(before) + deal.lead + SEQ_COST;
  const int S = deal.share;
  const int len = a.lens[b];
  const int pages = own_pages(a, len);
  const int first = before / S;
  const int n = pages ? (before + pages - 1) / S - first + 1 : 0;  // shares that hold own pages
  const bool joins = len_ok(a, len) && a.shared > 0 && len >= a.shared * PAGE;
  const int64_t slot0 = hk * head_slots(a);
  const int64_t own0 = slot0 + (int64_t)(first + b) * a.G + g;
  const int64_t sh0 = slot0 + shared_slots(a) + (int64_t)b * a.G + g;
  const int parts = n + (!joins ? 0 : a.np ? a.np << (a.late && late_pages(a, deal)) : (deal.lead - 1) / S + 1);
  const int grp = (threadIdx.x >> 5) % GR, ln = threadIdx.x & 31;
  float M = -INFINITY, den = 0.0f;
  f4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = grp; i0 < parts; i0 += 4 * GR) {
    float2 ml[4];
    f4_t x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = min(i0 + GR * j, parts - 1);
      const int64_t s = i < n ? own0 + (int64_t)i * a.G : sh0 + (int64_t)(i - n) * a.B * a.G;
      ml[j] = a.part_ml[s];
      x[j] = *reinterpret_cast<const f4_t*>(a.part_acc + s * D + 4 * ln);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + GR * j < parts) merge_into(M, den, acc, ml[j].x, ml[j].y, x[j]);
  }
  const int at = threadIdx.x >> 5;
  sh_acc[at][ln] = acc;
  if (ln == 0) sh_ml[at] = make_float2(M, den);
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int j = 1; j < GR; ++j)
    merge_into(M, den, acc, sh_ml[at + j].x, sh_ml[at + j].y, sh_acc[at + j][ln]);
  float inv = den == 0.0f ? 0.0f : 1.0f / den;  // no keys: 0; a sum that is NaN stays
  if (!len_ok(a, len)) inv = NAN;
  const f4_t o = acc * inv;
  *reinterpret_cast<uint2*>(a.out + (int64_t)row * D + 4 * ln) =
      make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
}

struct DecodeShape {
  int np, rb, shares, nt, shared;
  bool split, late;
  int64_t slots;  // partial rows, all heads
};

// Reading the shared pages once saves B - 1 readings of them; where these are fewer than SHARED_MIN pages of
// a head, the sequences are attended on their own. (us, shared / each on its own, 8 KV heads: 4,096 positions
// of 3 sequences 18.7 / 17.3, of 6 17.6 / 21.9, 16,384 of 2 22.0 / 23.3.)
constexpr int64_t SHARED_MIN = 1024;
DecodeShape decode_shape(int64_t B, int64_t Hkv, int64_t G, int64_t shared, int cus) {
  DecodeShape s{0, 0, 1, 0, 0, false, false, 0};
  if ((B - 1) * shared * Hkv >= SHARED_MIN) s.shared = (int)shared;
  const bool blocks = s.shared > 0 && B * G > 16;
  if (blocks) {
    s.nt = B * G > 16 * DW ? 2 : 1;
    s.split = B * G <= 8 * DW;
    s.rb = (int)((B * G + 16 * DW * s.nt - 1) / (16 * DW * s.nt));
    s.np = (int)std::min<int64_t>((shared + 3) / 4, std::max<int64_t>(1, cus / (Hkv * s.rb)));
    s.late = shared / s.np >= 2 * LATE_MIN + OWN_START;
  }
  s.shares = (int)std::max<int64_t>(1, (blocks ? cus : 2 * cus) / Hkv);
  s.slots = Hkv * G * (s.shares + B + (s.np ? s.np << s.late : s.shared ? s.shares : 0) * B);
  return s;
}

// Waves of a workgroup that takes a whole sequence, 0: the work is dealt out. Sequences of few pages are
// taken whole, with one launch and nothing to merge; 8 waves where each has a CU of its own. us, dealt out /
// whole, with the launch of the host and on the GPU alone (the rule goes by the first: in a captured graph one
// sequence of 1,000 positions is the faster dealt out, and a table with room to grow is never taken whole):
//   1 sequence of 1,000 positions, 8 KV heads   14.3 / 12.2, 10.1 / 11.8 (of 500 9.9 / 7.6, 2,000 10.1 / 19.5)
//   16 of 1,000                                 16.0 / 13.8  64 of 1,000 32 / 29  256 of 300 53 / 42
//   64 of 10 to 500                             20.0 / 14.2 (with 8 waves 16.9)
//   64 of 100 to 2,000                          38.5 / 39.3
// A shared part that is nearly all there is is read once all the same where workgroups are many (512
// sequences that share 12 of 16 pages: 117 / 131; 64 of them: 20.4 / 20.6).
constexpr int64_t SHORT_PAGES = 16;
int short_waves(const DecodeShape& s, int64_t B, int64_t Hkv, int64_t width, int64_t cus) {
  if (width > SHORT_PAGES || (4 * s.shared >= 3 * width && B * Hkv >= 4 * cus)) return 0;
  return B * Hkv <= cus ? 8 : 4;
}

int64_t decode_bytes(const DecodeShape& s) { return s.slots * (int64_t)(D * sizeof(float) + sizeof(float2)); }

int check_decode(int64_t B, int64_t Hq, int64_t Hkv, int64_t shared_pages) {
  LQ_CHECK_ARG(Hkv >= 1 && Hkv <= 1024 && Hq >= Hkv && Hq % Hkv == 0 && Hq / Hkv <= 16,
               "Hq=%lld must be 1 to 16 times Hkv=%lld", (long long)Hq, (long long)Hkv);
  LQ_CHECK_ARG(B >= 1 && B <= 4096, "a batch of %lld is not in [1, 4096]", (long long)B);
  LQ_CHECK_ARG(B * Hq < (1 << 23), "%lld query rows are too many", (long long)(B * Hq));
  LQ_CHECK_ARG(shared_pages >= 0, "%lld shared pages", (long long)shared_pages);
  return LQ_OK;
}

}  // namespace
}  // namespace lq

extern "C" int64_t lq_paged_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv,
                                                   int64_t shared_pages) {
  using namespace lq;
  clear_error();
  if (check_decode(B, Hq, Hkv, shared_pages)) return -1;
  return decode_bytes(decode_shape(B, Hkv, Hq / Hkv, shared_pages, device_cu_count()));
}

extern "C" int lq_paged_decode_attn(const uint16_t* q, const uint8_t* kc, const uint16_t* ks,
                                    const uint16_t* kb, const uint8_t* vc, const uint16_t* vs,
                                    const uint16_t* vb, int64_t pages, int64_t B, int64_t Hq,
                                    int64_t Hkv, int64_t D, const int32_t* table, int64_t table_stride,
                                    int64_t table_width, const int32_t* lens, int64_t shared_pages,
                                    float scale, uint16_t* out, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  using namespace lq;
  clear_error();
  PagedArgs a{};
  a.q = q;
  a.buf = {const_cast<uint8_t*>(kc),  const_cast<uint16_t*>(ks), const_cast<uint16_t*>(kb),
           const_cast<uint8_t*>(vc),  const_cast<uint16_t*>(vs), const_cast<uint16_t*>(vb)};
  a.tab = {table, table_stride, (int)table_width, (int)pages};
  if (const int st = check_pool(a.buf, a.tab, table_stride, table_width, pages, Hkv, D)) return st;
  if (const int st = check_decode(B, Hq, Hkv, shared_pages)) return st;
  LQ_CHECK_ARG(shared_pages <= table_width, "%lld shared pages of table rows of %lld",
               (long long)shared_pages, (long long)table_width);
  LQ_CHECK_ARG(q && lens && out, "null pointer");
  LQ_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "q and out must be 16-byte aligned");
  LQ_CHECK_ARG(std::isfinite(scale), "the softmax scale is not finite");
  const int64_t G = Hq / Hkv;
  const DecodeShape s = decode_shape(B, Hkv, G, shared_pages, device_cu_count());
  if (!workspace || workspace_bytes < decode_bytes(s)) {
    set_error("workspace of %lld bytes is smaller than the %lld needed", (long long)workspace_bytes,
              (long long)decode_bytes(s));
    return LQ_EWORKSPACE;
  }
  LQ_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  const int64_t parts = (int64_t)s.np * s.rb;
  const int64_t wgs = Hkv * (parts + std::max<int64_t>(s.late ? parts : 0, s.shares));
  LQ_CHECK_ARG(wgs < (1 << 23), "too many workgroups");
  a.lens = lens;
  a.part_acc = (float*)workspace;
  a.part_ml = (float2*)(a.part_acc + s.slots * 128);
  a.out = out;
  a.B = (int)B;
  a.Hkv = (int)Hkv;
  a.G = (int)G;
  a.shared = s.shared;
  a.np = s.np;
  a.late = s.late;
  a.rb = s.rb;
  a.shares = s.shares;
  a.sl2 = scale * 1.4426950408889634f;
  if (const int waves = short_waves(s, B, Hkv, table_width, device_cu_count())) {
    auto* kern = waves == 8 ? paged_short_kernel<8> : paged_short_kernel<4>;
    kern<<<dim3((unsigned)(B * Hkv)), dim3(64 * waves), 0, (hipStream_t)stream>>>(a);
    LQ_CHECK_LAUNCH("paged_short_kernel");
    return LQ_OK;
  }
  auto* kern = s.nt == 2   ? paged_shared_kernel<2, false>
               : s.split   ? paged_shared_kernel<1, true>
               : s.nt == 1 ? paged_shared_kernel<1, false>
                           : paged_decode_kernel;
  kern<<<dim3((unsigned)wgs), dim3(64 * DW), 0, (hipStream_t)stream>>>(a);
  LQ_CHECK_LAUNCH("paged_decode_kernel");
  // a row's partials: the shared parts and its share of the own ones
  if ((s.np << s.late) + s.shares / std::min<int64_t>(B, 4) > 16)
    paged_merge_kernel<8><<<dim3((unsigned)(B * Hq)), dim3(256), 0, (hipStream_t)stream>>>(a);
  else
    paged_merge_kernel<2><<<dim3((unsigned)((B * Hq + 3) / 4)), dim3(256), 0, (hipStream_t)stream>>>(a);
  LQ_CHECK_LAUNCH("paged_merge_kernel");
  return LQ_OK;
}
