// Attention of the last rows of several sequences -- a token, a verified block, a chunk of a prompt -- over a
// paged 8-bit cache, causal, over everything before a row or within a window. Sequence b has counts[b] query
// rows (host), packed one sequence behind the other, which are its last positions: row i is position
// p = lens[b] - counts[b] + i and sees max(0, p - window + 1) .. p. lens is read on the device, so that a
// recorded call follows growing sequences.
//
// A workgroup takes a block of query rows of a KV head, numbered position-major (row f is position f / G of
// query head f % G), walks the pages that the block sees, dequantizes each once into LDS as bf16 -- one tile of
// 64 keys, what paged_gather reads -- and runs it through attn_tile.h. The pages' codes are loaded into registers
// a tile ahead and staged into one of two tiles; one barrier per tile.
//
// The work is dealt out in equal shares of tiles: the blocks of all sequences stand one behind the other, a
// block costing its tiles and BLOCK_COST for its start and end, and a workgroup takes one share, which may begin
// and end inside blocks. Parts of blocks go to the workspace and a second launch merges them. Every workgroup
// adds the costs up itself, from the lengths.
//
// Keys that a row does not see reach it in no way: masked scores are -infinity, pages that no row of a block
// sees are not read, and a V row with infinities or NaN in a tile that is masked for some row is taken out of
// the product and added for the rows that see it (0 times it would be NaN). A page outside the pool is NaN to
// the rows that see one of its positions, a length outside the table to all rows of the sequence.
#include <algorithm>

#include "paged_tile.h"

namespace lq {
namespace {

using namespace attn;

constexpr int BLOCK_COST = 4;  // of a block's start and end, in tiles
constexpr int MIN_PART = 2;    // tiles of a block's part: nearer cuts move to the block's end
constexpr int NO_WINDOW = 1 << 25;

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_tok, q_head;
  PagedBufs buf;
  PageTable tab;
  const int32_t* lens;
  uint16_t* out;       // [rows, Hq, 128]
  float* part_acc;     // [2 x shares x Hkv][block rows][128]: slot 0 of a share the block that began in an
  float2* part_ml;     // earlier one, slot 1 the block that goes on in a later one
  int Hkv, G;
  FastDiv g;
  float sl2;
  int window;          // positions a row sees, NO_WINDOW: all
  int shares;          // per KV head
  int nseq, lanes;     // sequences, log2 of the lanes that add up the blocks of one
  int seq[LQ_MAX_SEQS], row0[LQ_MAX_SEQS], rows[LQ_MAX_SEQS];  // table row, first row of q, rows (not 0)
};

// A sequence: query rows times heads, its length (-1: outside the table), the position of its first row.
struct Seq {
  int R, len, base;
};
__device__ __forceinline__ Seq seq_of(const ChunkArgs& a, int s) {
  const int n = a.rows[s], len = a.lens[a.seq[s]];
  const bool ok = len >= 0 && len <= (int64_t)a.tab.width * PAGE;
  return {n * a.G, ok ? len : -1, ok ? len - n : -(1 << 30)};
}

// The tiles that block blk (of ROWS rows) sees.
struct Span {
  int lo, n;
};
template <int ROWS>
__device__ __forceinline__ Span block_span(const ChunkArgs& a, const Seq& q, int blk) {
  const int first = q.base + (int)fdiv_u((uint32_t)(blk * ROWS), a.g);
  const int last = q.base + (int)fdiv_u((uint32_t)min(blk * ROWS + ROWS - 1, q.R - 1), a.g);
  const int lo = max(0, first - a.window + 1) / TKEYS;
  return {lo, last < 0 ? 0 : last / TKEYS + 1 - lo};
}

// A block, its tiles, its place among its sequence's blocks and where its cost begins.
struct Block {
  int seq, blk, lo, tiles, begin, place;
};
// The block at a place among nb: the last, the first, the last but one, .., so that two neighbours cost about
// the same and cuts are few.
__device__ __forceinline__ int block_at(int place, int nb) {
  return place & 1 ? place >> 1 : nb - 1 - (place >> 1);
}

// What the call deals out: a lane's inclusive sum of costs (2^lanes of them per sequence), the whole and a share.
struct Deal {
  int upto, total, share;
};
template <int ROWS>
__device__ __forceinline__ Deal deal_out(const ChunkArgs& a, int lane) {
  const int s = lane >> a.lanes;
  int cost = 0;
  if (s < a.nseq) {
    const Seq q = seq_of(a, s);
    for (int b = lane & ((1 << a.lanes) - 1); b * ROWS < q.R; b += 1 << a.lanes)
      cost += block_span<ROWS>(a, q, b).n + BLOCK_COST;
  }
  const int upto = wave_scan_i(cost);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  return {upto, total, max(BLOCK_COST + MIN_PART, (total + a.shares - 1) / a.shares)};
}
// The block that holds cost u (below the total).
template <int ROWS>
__device__ __forceinline__ Block find_block(const ChunkArgs& a, const Deal& d, int u, int lane) {
  const int last = (1 << a.lanes) - 1;  // a sequence's last lane has its end
  const int s = __builtin_popcountll(__builtin_amdgcn_ballot_w64((lane & last) == last && d.upto <= u));
  int before = s ? __builtin_amdgcn_readlane(d.upto, (s << a.lanes) - 1) : 0;
  const Seq q = seq_of(a, s);
  const int nb = (q.R + ROWS - 1) / ROWS;
  for (int i = 0;; i += 64) {
    Span sp{0, 0};
    int c = 0;
    if (i + lane < nb) {
      sp = block_span<ROWS>(a, q, block_at(i + lane, nb));
      c = sp.n + BLOCK_COST;
    }
    const int upto = wave_scan_i(c);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > u);
    if (past || i + 64 >= nb) {
      const int l = past ? __builtin_ctzll(past) : 0;
      return {s, block_at(i + l, nb), __builtin_amdgcn_readlane(sp.lo, l), __builtin_amdgcn_readlane(sp.n, l),
              before + __builtin_amdgcn_readlane(upto - c, l), i + l};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
}
// The tile of a block at which a cut at cost u (anywhere) lies: not within MIN_PART of its ends.
__device__ __forceinline__ int cut_tile(const Block& b, int u) {
  const int t = u - b.begin - BLOCK_COST;
  return t >= b.tiles ? b.tiles : t < MIN_PART ? 0 : t > b.tiles - MIN_PART ? b.tiles : t;
}

// Whether a V scale and bias may give something that is no finite bf16.
__device__ __forceinline__ bool wild(float s, float z) { return !(fabsf(s) * 255.0f + fabsf(z) < 3.3e38f); }

// The wild groups of one V row (key `key` of a tile whose P is p, position `at`, row `row` of the pool), for the
// rows that see it: O^T took 0 in their place.
template <int NT>
__device__ __forceinline__ void add_wild(const PagedBufs& buf, int64_t row, int key, int at, TileRows<NT>& st,
                                         int lane, const bf16x8_t (&p)[NT][2], const int (&lim)[NT], int window) {
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
  const uint32_t sw = reinterpret_cast<const uint32_t*>(buf.vs)[row], zw = reinterpret_cast<const uint32_t*>(buf.vb)[row];
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float s = w < 4 ? bf16_lo(sw) : bf16_hi(sw), z = w < 4 ? bf16_lo(zw) : bf16_hi(zw);
    const uint2 v2 = dequant4(*reinterpret_cast<const uint32_t*>(buf.vc + row * D + 16 * w + 4 * lq4), s, z);
    const float v[4] = {bf16_lo(v2.x), bf16_hi(v2.x), bf16_lo(v2.y), bf16_hi(v2.y)};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (wild(s, z) && at <= lim[nt] && at > lim[nt] - window) st.o[nt][w][r] = fmaf(pk[nt], v[r], st.o[nt][w][r]);
  }
}

struct ChunkSmem {
  KvTile tile[2];            // K of tile t in tile[t % 2], V likewise
  uint32_t wild[3][2];       // keys of tile t % 3, if masked, whose V is wild
};

template <int PW, int NT>  // waves, 16-row tiles of each
__global__ __launch_bounds__(64 * PW, 2) void chunk_kernel(const ChunkArgs a) {
  constexpr int ROWS = 16 * NT * PW;
  constexpr int C = 8 / PW;  // 16-byte chunks of K (of V) that a thread brings per tile
  __shared__ ChunkSmem sm;
  const int share = blockIdx.x / a.Hkv, hk = blockIdx.x - share * a.Hkv;
  const Deal deal = deal_out<ROWS>(a, threadIdx.x & 63);
  const int u0 = deal.share * share, u1 = min(u0 + deal.share, deal.total);
  if (u0 >= u1) return;
  Block b = find_block<ROWS>(a, deal, u0, threadIdx.x & 63);
  for (bool more = true; more;) {
    // re-read per block, so that no lane value made of it is kept across blocks
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lc = lane & 15, lq4 = lane >> 4;
    const Seq sq = seq_of(a, b.seq);
    const int q0 = a.row0[b.seq];
    const int c0 = cut_tile(b, u0), c1 = cut_tile(b, u1);
    const int t0 = b.lo + c0, t1 = b.lo + c1;
    // a block without a tile (rows without keys) belongs to the share that its begin lies in
    const bool mine = c0 < c1 || (b.tiles == 0 && b.begin >= u0 && b.begin < u1);
    if (mine) {
      const float scale = abs_scale(a.sl2);
      // tiles in [t_open, t_masked) are open to all rows of the block
      const int first = sq.base + (int)fdiv_u((uint32_t)(b.blk * ROWS), a.g);
      const int last = sq.base + (int)fdiv_u((uint32_t)min(b.blk * ROWS + ROWS - 1, sq.R - 1), a.g);
      const int t_masked = first < 0 ? 0 : (first + 1) / TKEYS;
      const int t_open = (max(0, last - a.window + 1) + TKEYS - 1) / TKEYS;

      // ---- a tile: thread tid brings 16 codes (chunk tid % 8) of key tid / 8 (and + 8 PW)
      const int32_t* ids = a.tab.ids + (int64_t)a.seq[b.seq] * a.tab.stride;
      const int key0 = tid >> 3, chunk = tid & 7;
      uint4 rk[C], rv[C];
      uint32_t ks[C], kb[C], vs[C], vb[C];
      bool k_ok = true, v_ok = true;
      int id_k = 0, id_next = t0 < t1 ? ids[t0] : 0;  // of the last K loaded, of the next
      auto pool_row = [&](int id, bool& ok) {
        ok = id >= 0 && id < a.tab.pages;
        return ((int64_t)(ok ? id : 0) * a.Hkv + hk) * PAGE;
      };
      auto load_k = [&](int t) {  // tile t, in order
        id_k = __builtin_amdgcn_readfirstlane(id_next);
        id_next = ids[min(t + 1, t1 - 1)];
        const int64_t row = pool_row(id_k, k_ok);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          rk[i] = *reinterpret_cast<const uint4*>(a.buf.kc + row * D + 1024 * PW * i + 16 * tid);
          ks[i] = reinterpret_cast<const uint32_t*>(a.buf.ks)[row + key0 + 8 * PW * i];
          kb[i] = reinterpret_cast<const uint32_t*>(a.buf.kb)[row + key0 + 8 * PW * i];
        }
      };
      auto load_v = [&](int id) {
        const int64_t row = pool_row(id, v_ok);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          rv[i] = *reinterpret_cast<const uint4*>(a.buf.vc + row * D + 1024 * PW * i + 16 * tid);
          vs[i] = reinterpret_cast<const uint32_t*>(a.buf.vs)[row + key0 + 8 * PW * i];
          vb[i] = reinterpret_cast<const uint32_t*>(a.buf.vb)[row + key0 + 8 * PW * i];
        }
      };
      auto pick = [&](uint32_t w) { return chunk < 4 ? bf16_lo(w) : bf16_hi(w); };
      auto put = [&](uint4* lo, uint4* hi, uint4 c, float s, float z) {
        const uint2 d0 = dequant4(c.x, s, z), d1 = dequant4(c.y, s, z);
        const uint2 d2 = dequant4(c.z, s, z), d3 = dequant4(c.w, s, z);
        *lo = make_uint4(d0.x, d0.y, d1.x, d1.y);
        *hi = make_uint4(d2.x, d2.y, d3.x, d3.y);
      };
      auto stage_k = [&](int t) {
        if (t >= t1) return;  // uniform
        KvTile& to = sm.tile[t & 1];
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int key = key0 + 8 * PW * i;
          put(k_chunk(to, key, 2 * chunk), k_chunk(to, key, 2 * chunk + 1), rk[i], k_ok ? pick(ks[i]) : NAN, pick(kb[i]));
        }
      };
      auto stage_v = [&](int t) {
        if (t >= t1) return;
        KvTile& to = sm.tile[t & 1];
        const bool masked = t >= t_masked || t < t_open;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int key = key0 + 8 * PW * i;
          float s = pick(vs[i]), z = pick(vb[i]);
          if (masked || !v_ok) {  // uniform
            const bool none = !v_ok || TKEYS * t + key >= sq.len;  // no such position
            const bool w = !none && wild(s, z);
            if (w) atomicOr(&sm.wild[t % 3][key >> 5], 1u << (key & 31));
            if (none || w) s = z = 0.0f;
          }
          put(v_chunk(to, key, 2 * chunk), v_chunk(to, key, 2 * chunk + 1), rv[i], s, z);
        }
      };

      lds_barrier();  // the block before is done with LDS
      if (t0 < t1) load_k(t0);

      // ---- the wave's rows
      const int f0 = b.blk * ROWS + 16 * NT * wv;
      TileRows<NT> st;
      int lim[NT];  // last key of the lane's row, -1: none
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int f = f0 + 16 * nt + lc;
        const int i = (int)fdiv_u((uint32_t)min(f, sq.R - 1), a.g);
        const int head = min(f, sq.R - 1) - i * a.G;
        lim[nt] = f < sq.R ? sq.base + i : -1;
        const uint16_t* qr = a.q + (int64_t)(q0 + i) * a.q_tok + (hk * a.G + head) * a.q_head + 8 * lq4;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          st.q[nt][kk] = u4_as_bf8(signed_q(*reinterpret_cast<const uint4*>(qr + 32 * kk), a.sl2));
      }
      st.clear();
      // keys that all, and that some, of the wave's rows see
      const int lim_lo = f0 < sq.R ? sq.base + (int)fdiv_u((uint32_t)f0, a.g) : -1;
      const int open_from =
          f0 < sq.R ? sq.base + (int)fdiv_u((uint32_t)min(f0 + 16 * NT - 1, sq.R - 1), a.g) - a.window + 1 : 0;

      f4_t c[NT][4];
      bf16x8_t p[NT][2];
      if (t0 < t1) {
        if (tid < 6) sm.wild[tid >> 1][tid & 1] = 0;
        stage_k(t0);
        int id_v = id_k;
        load_k(t0 + 1);
        load_v(id_v);
        lds_barrier();
        tile_scores<NT>(sm.tile[t0 & 1].k, st, lane, c);
        stage_k(t0 + 1);
        stage_v(t0);
        id_v = id_k;
        load_k(t0 + 2);
        load_v(id_v);
        for (int t = t0; t < t1; ++t) {
          lds_barrier();
          stage_k(t + 2);
          stage_v(t + 1);
          id_v = id_k;
          load_k(t + 3);
          load_v(id_v);
          if (TKEYS * t + TKEYS - 1 > lim_lo || TKEYS * t < open_from) {  // wave-uniform: masked for some row
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int key = TKEYS * t + 16 * mt + 4 * lq4 + r;
                  c[nt][mt][r] = key <= lim[nt] && key > lim[nt] - a.window ? c[nt][mt][r] : -INFINITY;
                }
          }
          Ahead ahead;
          tile_ahead(sm.tile[(t + 1) & 1].k, lane, ahead);
          tile_softmax<NT>(c, st, scale, p);
          // Q.K^T of tile t + 1 (behind the last one, of a tile nobody uses), P.V of tile t
          tile_matrix<NT>(sm.tile[(t + 1) & 1].k, sm.tile[t & 1].v, st, lane, c, p, ahead);
          if (t >= t_masked || t < t_open) {
            uint64_t w = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.wild[t % 3][0]) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.wild[t % 3][1]) << 32;
            for (; w; w &= w - 1) {  // rare
              const int key = __builtin_ctzll(w);
              bool ok;
              const int64_t row = pool_row(__builtin_amdgcn_readfirstlane(ids[t]), ok);
              add_wild<NT>(a.buf, row + key, key, TKEYS * t + key, st, lane, p, lim, a.window);
            }
          }
          // last read before the barrier ahead of this phase: what tile t + 2 will note
          if (tid < 2) sm.wild[(t + 2) % 3][tid] = 0;
        }
      }

      // ---- rows out: dims 16 w + 4 lq4 + r
      const bool part = c1 - c0 < b.tiles;
      const int64_t prow = ((int64_t)(2 * share + (c0 == 0)) * a.Hkv + hk) * ROWS;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int f = f0 + 16 * nt + lc;
        if (f >= sq.R) continue;
        if (part) {
          const int64_t pr = prow + 16 * (NT * wv + nt) + lc;
#pragma unroll
          for (int w = 0; w < 8; ++w)
            *reinterpret_cast<f4_t*>(a.part_acc + pr * D + 16 * w + 4 * lq4) = st.o[nt][w];
          if (lq4 == 0) a.part_ml[pr] = make_float2(st.m[nt], st.l[nt][0]);
          continue;
        }
        const int i = (int)fdiv_u((uint32_t)f, a.g), head = f - i * a.G;
        uint16_t* o = a.out + ((int64_t)(q0 + i) * a.Hkv * a.G + hk * a.G + head) * D + 4 * lq4;
        const float inv = sq.len < 0 ? NAN : st.l[nt][0] == 0.0f ? 0.0f : 1.0f / st.l[nt][0];
#pragma unroll
        for (int w = 0; w < 8; ++w)
          *reinterpret_cast<uint2*>(o + 16 * w) =
              make_uint2(pack_bf2(st.o[nt][w][0] * inv, st.o[nt][w][1] * inv),
                         pack_bf2(st.o[nt][w][2] * inv, st.o[nt][w][3] * inv));
      }
    }
    // the next block
    const int next = b.begin + b.tiles + BLOCK_COST;
    more = next < u1;
    if (more) {
      int ns = b.seq, place = b.place + 1;
      if (place * ROWS >= sq.R) {
        place = 0;
        ++ns;
      }
      const Seq nq = seq_of(a, ns);
      const int blk = block_at(place, (nq.R + ROWS - 1) / ROWS);
      const Span sp = block_span<ROWS>(a, nq, blk);
      b = Block{ns, blk, sp.lo, sp.n, next, place};
    }
  }
}

constexpr int MERGE_ROWS = 32;  // of a workgroup
// The parts of a block into output rows, by the workgroups of its first cut: share j's end. 32 lanes x 4
// dims per row.
template <int ROWS>
__global__ __launch_bounds__(256) void chunk_merge_kernel(const ChunkArgs a) {
  const int j = blockIdx.x / a.Hkv, hk = blockIdx.x - j * a.Hkv, lane = threadIdx.x & 63;
  const Deal deal = deal_out<ROWS>(a, lane);
  const int u = deal.share * (j + 1);
  if (u >= deal.total) return;
  const Block b = find_block<ROWS>(a, deal, u, lane);
  const int t = cut_tile(b, u);
  if (t == 0 || t == b.tiles || cut_tile(b, u - deal.share) != 0) return;  // no cut, or not its first
  const Seq sq = seq_of(a, b.seq);
  const int d = 4 * (threadIdx.x & 31);
  int n = 1;  // parts
  while (cut_tile(b, u + n * deal.share - deal.share) < b.tiles) ++n;
  constexpr int RT = MERGE_ROWS / 8;  // rows per thread: all their loads of a part together
  const int row0 = MERGE_ROWS * blockIdx.y + (threadIdx.x >> 5);
  if (b.blk * ROWS + MERGE_ROWS * (int)blockIdx.y >= sq.R) return;
  float M[RT], den[RT];
  f4_t acc[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    M[i] = -INFINITY;
    den[i] = 0.0f;
    acc[i] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 2
  for (int k = 0; k < n; ++k) {
    const int64_t part = ((int64_t)(2 * (j + k) + (k == 0)) * a.Hkv + hk) * ROWS;
    float2 ml[RT];
    f4_t o[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {  // rows past the sequence's are read, of the workspace, and not used
      ml[i] = a.part_ml[part + row0 + 8 * i];
      o[i] = *reinterpret_cast<const f4_t*>(a.part_acc + (part + row0 + 8 * i) * D + d);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) merge_into(M[i], den[i], acc[i], ml[i].x, ml[i].y, o[i]);
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int f = b.blk * ROWS + row0 + 8 * i;
    if (f >= sq.R) return;
    const float inv = den[i] == 0.0f ? 0.0f : 1.0f / den[i];
    const int p = (int)fdiv_u((uint32_t)f, a.g), head = f - p * a.G;
    *reinterpret_cast<uint2*>(a.out + ((int64_t)(a.row0[b.seq] + p) * a.Hkv * a.G + hk * a.G + head) * D + d) =
        make_uint2(pack_bf2(acc[i][0] * inv, acc[i][1] * inv), pack_bf2(acc[i][2] * inv, acc[i][3] * inv));
  }
}

// How a call's sequences are dealt out.
struct ChunkPlan {
  int nseq, lanes, shares;
  int seq[LQ_MAX_SEQS], row0[LQ_MAX_SEQS], rows[LQ_MAX_SEQS];
};
constexpr int ROWS = 64;
ChunkPlan chunk_plan(const int32_t* counts, int64_t nseq, int64_t Hkv, int64_t G, int cus) {
  ChunkPlan p{};
  int at = 0;
  for (int s = 0; s < nseq; ++s) {
    if (counts[s]) {
      p.seq[p.nseq] = s;
      p.row0[p.nseq] = at;
      p.rows[p.nseq++] = counts[s];
    }
    at += counts[s];
  }
  p.lanes = 6;
  while ((p.nseq << p.lanes) > 64) --p.lanes;
  p.shares = (int)std::max<int64_t>(1, 2 * cus / Hkv);
  return p;
}
int64_t chunk_bytes(const ChunkPlan& p, int64_t Hkv) {
  return 2 * p.shares * Hkv * ROWS * (int64_t)(D * sizeof(float) + sizeof(float2));
}

int check_chunk(int64_t Hq, int64_t Hkv, const int32_t* counts, int64_t nseq) {
  LQ_CHECK_ARG(Hkv >= 1 && Hkv <= 1024 && Hq >= Hkv && Hq % Hkv == 0 && Hq / Hkv <= 64,
               "Hq=%lld must be 1 to 64 times Hkv=%lld", (long long)Hq, (long long)Hkv);
  LQ_CHECK_ARG(nseq >= 1 && nseq <= LQ_MAX_SEQS && counts, "%lld sequences are not in [1, %d], or no counts",
               (long long)nseq, LQ_MAX_SEQS);
  int64_t rows = 0;
  for (int s = 0; s < nseq; ++s) {
    LQ_CHECK_ARG(counts[s] >= 0 && counts[s] <= (1 << 24) && counts[s] * (Hq / Hkv) < (1 << 30),
                 "row count %d of sequence %d", (int)counts[s], s);
    rows += counts[s];
  }
  LQ_CHECK_ARG(rows < (1 << 30), "too many rows");
  return LQ_OK;
}

}  // namespace
}  // namespace lq

extern "C" int64_t lq_paged_chunk_workspace_bytes(const int32_t* counts_host, int64_t nseq, int64_t Hq, int64_t Hkv) {
  using namespace lq;
  clear_error();
  if (check_chunk(Hq, Hkv, counts_host, nseq)) return -1;
  return chunk_bytes(chunk_plan(counts_host, nseq, Hkv, Hq / Hkv, device_cu_count()), Hkv);
}

extern "C" int lq_paged_chunk_attn(const uint16_t* q, int64_t q_tok, int64_t q_head, const uint8_t* kc,
                                   const uint16_t* ks, const uint16_t* kb, const uint8_t* vc, const uint16_t* vs,
                                   const uint16_t* vb, int64_t pages, int64_t Hq, int64_t Hkv, int64_t D,
                                   const int32_t* table, int64_t table_stride, int64_t table_width,
                                   const int32_t* lens, const int32_t* counts_host, int64_t nseq, int64_t window,
                                   float scale, uint16_t* out, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  using namespace lq;
  clear_error();
  ChunkArgs a{};
  a.buf = {const_cast<uint8_t*>(kc), const_cast<uint16_t*>(ks), const_cast<uint16_t*>(kb),
           const_cast<uint8_t*>(vc), const_cast<uint16_t*>(vs), const_cast<uint16_t*>(vb)};
  a.tab = {table, table_stride, (int)table_width, (int)pages};
  if (const int st = check_pool(a.buf, a.tab, table_stride, table_width, pages, Hkv, D)) return st;
  if (const int st = check_chunk(Hq, Hkv, counts_host, nseq)) return st;
  LQ_CHECK_ARG(window >= 0, "a window of %lld positions", (long long)window);
  LQ_CHECK_ARG(std::isfinite(scale), "the softmax scale is not finite");
  const int64_t G = Hq / Hkv;
  const ChunkPlan plan = chunk_plan(counts_host, nseq, Hkv, G, device_cu_count());
  if (plan.nseq == 0) return LQ_OK;
  LQ_CHECK_ARG(q && lens && out, "null pointer");
  LQ_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && ((q_tok | q_head) & 7) == 0,
               "rows must be 16-byte aligned (strides a multiple of 8)");
  int64_t most = 0;  // cost, if every block sees the whole table
  for (int s = 0; s < plan.nseq; ++s)
    most += (plan.rows[s] * G + lq::ROWS - 1) / lq::ROWS * (table_width + lq::BLOCK_COST);
  LQ_CHECK_ARG(most < (1ll << 31) - (1 << 20), "too many rows for table rows of %lld pages", (long long)table_width);
  const int64_t need = chunk_bytes(plan, Hkv);
  if (!workspace || workspace_bytes < need) {
    set_error("workspace of %lld bytes is smaller than the %lld needed", (long long)workspace_bytes, (long long)need);
    return LQ_EWORKSPACE;
  }
  LQ_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  a.q = q;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.lens = lens;
  a.out = out;
  a.part_acc = (float*)workspace;
  a.part_ml = (float2*)(a.part_acc + 2 * plan.shares * Hkv * lq::ROWS * 128);
  a.Hkv = (int)Hkv;
  a.G = (int)G;
  a.g = make_fastdiv((uint32_t)G);
  a.sl2 = scale * 1.4426950408889634f;
  a.window = window == 0 ? NO_WINDOW : (int)std::min<int64_t>(window, NO_WINDOW);
  a.shares = plan.shares;
  a.nseq = plan.nseq;
  a.lanes = plan.lanes;
  std::copy(plan.seq, plan.seq + LQ_MAX_SEQS, a.seq);
  std::copy(plan.row0, plan.row0 + LQ_MAX_SEQS, a.row0);
  std::copy(plan.rows, plan.rows + LQ_MAX_SEQS, a.rows);
  chunk_kernel<4, 1><<<dim3((unsigned)(plan.shares * Hkv)), dim3(256), 0, (hipStream_t)stream>>>(a);
  LQ_CHECK_LAUNCH("chunk_kernel");
  if (plan.shares > 1) {
    chunk_merge_kernel<lq::ROWS><<<dim3((unsigned)((plan.shares - 1) * Hkv), lq::ROWS / MERGE_ROWS), dim3(256), 0,
                                   (hipStream_t)stream>>>(a);
    LQ_CHECK_LAUNCH("chunk_merge_kernel");
  }
  return LQ_OK;
}
