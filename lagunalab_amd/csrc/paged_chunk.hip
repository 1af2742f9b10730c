// Attention of the last rows of several sequences -- a token, a verified block, a chunk of a prompt -- over a
// paged 8-bit cache, causal, over everything before a row or within a window. Sequence b has counts[b] query
// rows (host), packed one sequence behind the other, which are its last positions: row i is position
// p = lens[b] - counts[b] + i and sees max(0, p - window + 1) .. p. lens is read on the device, so that a
// recorded call follows growing sequences.
//
// Query rows of a KV head are numbered position-major (row f is position f / G of query head f % G), so that any
// grouping fills a matrix tile; a wave has 32 of them as the columns of v_mfma_f32_32x32x16_bf16 (attn_tile32.h). K and V
// are dequantized, scale * code + bias in fp32, to the bf16 rows that paged_gather reads. Softmax in fp32 with a running
// maximum; the weights are rounded to bf16, in the values and in the row sums alike: outputs are 0.0023 of their size off
// those in 64 bits, where the rounding of the output alone makes 0.0017.
//
// Sequences of many rows go as blocks of 256 rows (128 where no sequence has more): a workgroup walks the pages that its
// block sees, one tile of 64 keys each, dequantized once into LDS. Those of few rows (up to FEW_ROWS) go through waves
// that take half pages each (further down). Blocks are taken whole, or all blocks stand one behind the other, a block
// costing its tiles and BLOCK_COST for its start and end, and a workgroup takes an equal share of that, which may begin
// and end inside blocks: parts go to the workspace and a second launch merges them. Every workgroup adds the costs up
// itself, from the lengths. The rules and what they measured are at chunk_plan.
//
// Keys that a row does not see reach it in no way: masked scores are -infinity, pages that no row of a block
// sees are not read, and a V row with infinities or NaN in a tile that is masked for some row is taken out of
// the product and added for the rows that see it (0 times it would be NaN). A page outside the pool is NaN to
// the rows that see one of its positions, a length outside the table to all rows of the sequence.
#include <algorithm>

#include "attn_tile32.h"
#include "paged_tile.h"

namespace lq {
namespace {

using namespace attn;

constexpr int BLOCK_COST = 4;  // of a block's start and end, in tiles
constexpr int MIN_PART = 2;    // tiles of a block's part: nearer cuts move to the block's end
constexpr int NO_WINDOW = 1 << 25;
constexpr int FEW_WAVES = 4;
constexpr int SHARE_MIN = 4;  // half pages of a share of few rows: one per wave
constexpr int SEQ_COST = 8;   // of starting on a sequence, in half pages

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
  int shares;          // per KV head; 0: a workgroup takes a whole block
  int blocks;          // of the sequence with the most rows (few rows)
  int row_bits;        // log2 of a block's rows (few rows)
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
  Seq q;
};
// The block at a place among nb: the last, the first, the last but one, .., so that two neighbours cost about
// the same and cuts are few.
__device__ __forceinline__ int block_at(int place, int nb) {
  return place & 1 ? place >> 1 : nb - 1 - (place >> 1);
}

// What the call deals out: a lane's inclusive sum of costs (2^lanes of them per sequence) and its sequence, the whole
// and a share.
struct Deal {
  int upto;
  Seq q;
  int total, share;
};
// The sequence of a lane.
__device__ __forceinline__ Seq seq_at(const Deal& d, int lane) {
  return {__builtin_amdgcn_readlane(d.q.R, lane), __builtin_amdgcn_readlane(d.q.len, lane),
          __builtin_amdgcn_readlane(d.q.base, lane)};
}
template <int ROWS>
__device__ __forceinline__ Deal deal_out(const ChunkArgs& a, int lane) {
  const int s = lane >> a.lanes;
  int cost = 0;
  Seq q{0, 0, 0};
  if (s < a.nseq) {
    q = seq_of(a, s);
    for (int b = lane & ((1 << a.lanes) - 1); b * ROWS < q.R; b += 1 << a.lanes)
      cost += block_span<ROWS>(a, q, b).n + BLOCK_COST;
  }
  const int upto = wave_scan_i(cost);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  return {upto, q, total, max(BLOCK_COST + MIN_PART, (total + a.shares - 1) / a.shares)};
}
// The block that holds cost u (below the total).
template <int ROWS>
__device__ __forceinline__ Block find_block(const ChunkArgs& a, const Deal& d, int u, int lane) {
  const int last = (1 << a.lanes) - 1;  // a sequence's last lane has its end
  const int s = __builtin_popcountll(__builtin_amdgcn_ballot_w64((lane & last) == last && d.upto <= u));
  int before = s ? __builtin_amdgcn_readlane(d.upto, (s << a.lanes) - 1) : 0;
  const Seq q = seq_at(d, s << a.lanes);
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
              before + __builtin_amdgcn_readlane(upto - c, l), i + l, q};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
}
// The tile of a block at which a cut at cost u (anywhere) lies: not within MIN_PART of its ends.
__device__ __forceinline__ int cut_tile(const Block& b, int u) {
  const int t = u - b.begin - BLOCK_COST;
  return t >= b.tiles ? b.tiles : t < MIN_PART ? 0 : t > b.tiles - MIN_PART ? b.tiles : t;
}

// The block of rank x when all are in order of their tiles, most first: how many have at least n tiles is a sum over
// the sequences, a lane each, and the largest n that more than x have is found by halving. Behind a window all cost
// about the same and stand one sequence behind the other. Its cost is counted from its own begin.
template <int ROWS>
__device__ __forceinline__ Block ranked_block(const ChunkArgs& a, int x, int lane) {
  const Seq q = lane < a.nseq ? seq_of(a, lane) : Seq{0, 0, 0};
  const int nb = (q.R + ROWS - 1) / ROWS;
  Deal d{0, q, 0, 0};
  int s, blk;
  if (a.window < NO_WINDOW) {
    const int upto = wave_scan_i(nb);
    s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x));
    blk = __builtin_amdgcn_readlane(upto, s) - 1 - x;
  } else {
    auto from = [&](int n) {  // first block of the lane's sequence with at least n tiles (of nb: none)
      const int64_t y = (int64_t)a.G * ((int64_t)TKEYS * (n - 1) - q.base);  // the row that has to be reached
      return n <= 0 || y <= 0 ? 0 : y > q.R - 1 ? nb : (int)(y / ROWS);
    };
    int lo = 0, hi = a.tab.width + 1;  // all have lo, none has hi
    int above = 0;                     // blocks with at least hi tiles
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, n = __builtin_amdgcn_readfirstlane(wave_sum_i(nb - from(mid)));
      if (n > x) {
        lo = mid;
      } else {
        hi = mid;
        above = n;
      }
    }
    const int n = from(lo + 1) - from(lo), upto = wave_scan_i(n);
    s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x - above));
    blk = __builtin_amdgcn_readlane(from(lo), s) + x - above - __builtin_amdgcn_readlane(upto - n, s);
  }
  const Seq sq = seq_at(d, s);
  const Span sp = block_span<ROWS>(a, sq, blk);
  return {s, blk, sp.lo, sp.n, 0, 0, sq};
}

// Whether a V scale and bias may give something that is no finite bf16.
__device__ __forceinline__ bool wild(float s, float z) { return !(fabsf(s) * 255.0f + fabsf(z) < 3.3e38f); }

// The wild groups of one V row (key `key` of a tile whose P is p, `rel` behind the lane's row, row `row` of the
// pool), for the rows that see it: O^T took 0 in their place.
template <int E>
__device__ __forceinline__ void add_wild(const PagedBufs& buf, int64_t row, int key, int rel, Rows32& st, int lane,
                                         const bf16x8_t (&p)[E], int window) {
  const float pk = weight32(p, key, lane);
  const bool sees = (uint32_t)rel < (uint32_t)window;
  const uint32_t sw = reinterpret_cast<const uint32_t*>(buf.vs)[row], zw = reinterpret_cast<const uint32_t*>(buf.vb)[row];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float s = g ? bf16_hi(sw) : bf16_lo(sw), z = g ? bf16_hi(zw) : bf16_lo(zw);
    if (!wild(s, z)) continue;  // uniform
#pragma unroll
    for (int w = 2 * g; w < 2 * g + 2; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 v2 = dequant4(
            *reinterpret_cast<const uint32_t*>(buf.vc + row * D + 32 * w + 8 * j + 4 * (lane >> 5)), s, z);
        const float v[4] = {bf16_lo(v2.x), bf16_hi(v2.x), bf16_lo(v2.y), bf16_hi(v2.y)};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (sees) st.o[w][4 * j + r] = fmaf(pk, v[r], st.o[w][4 * j + r]);
      }
  }
}

// An entry of an array at a wave-uniform place, by the scalar cache: nothing of a call writes what it reads.
__device__ __forceinline__ int scalar(const int32_t* p, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p)[i];
}
// A wave-uniform pointer into global memory, kept apart from the lanes' offsets: loads take it as a scalar base.
template <typename T>
using global_ptr = const __attribute__((address_space(1))) T*;
template <typename T>
__device__ __forceinline__ global_ptr<T> uniform(const T* p) {
  global_ptr<T> g = (global_ptr<T>)p;
  asm volatile("" : "+s"(g));
  return g;
}

__device__ __forceinline__ uint32_t lane_offset(uint32_t o) {
  asm volatile("" : "+v"(o));
  return o;
}

// lds_barrier, with its wait known to the compiler: operands read ahead of it need none of their own behind it, where
// one would wait for later reads as well.
__device__ __forceinline__ void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int STAGES>
struct ChunkSmem {
  KvTile tile[STAGES];       // K of tile t in tile[t % STAGES], V likewise
  uint32_t wild[3][2];       // keys of tile t % 3, if masked, whose V is wild
};

// Blocks of many rows. Eight waves are two halves that run a phase apart: while one has the matrix cores (S of tile t + 1,
// O of tile t), the other does softmax and brings a tile in, its codes loaded two tiles ahead and K staged there, V a code
// at a time beside the MFMAs; one barrier per phase, and the waves in the matrix phase go first (s_setprio). Bound by the
// phases' own lengths (a wave's vector phase 1,850 cycles, of them 400 staging and 270 exponentials; its matrix phase 1,640
// for 32 MFMAs of 32) and, in long calls, by power. 2,048 rows of 32/8 heads behind 32,771 positions 1,060 to 1,090 us,
// 1,040 to 1,070 TFLOP/s. There, without priorities 1,115, with the vector phase first 1,180; V staged two codes behind
// every second MFMA 1,085; K staged in the matrix phase too 1,127 (the vector phase 1,640, the matrix phase 1,950); the
// row maximum between the MFMAs 1,072 instead of 1,063; where the row sums go: attn_tile32.h. Rows read back as bf16 and
// attended by the packed prompt kernel are faster in such calls and slower in shorter or smaller ones (us, here / read
// back): 2,048 rows behind 32,771 1,058 / 963, of 48/8 heads behind 7,000 402 / 371, 512 of 48/8 behind 7,681 117 / 122,
// of 32/8 behind 82,159 649 / 670, 256 of 48/8 behind 1,000 30 / 43, 64 of 32/8 behind 20,000 53 / 82. Four waves, two
// workgroups per CU, run a tile's phases one behind the other.
template <int PW>  // waves, of 32 rows each: 8 or 4
__global__ __launch_bounds__(64 * PW, 2) void chunk_kernel(const ChunkArgs a) {
  constexpr bool HALVES = PW == 8;
  constexpr int ROWS = 32 * PW, STAGES = HALVES ? 3 : 2;
  constexpr int C = 8 / PW;  // 16-byte chunks of K (of V) that a thread brings per tile
  __shared__ ChunkSmem<STAGES> sm;
  const int share = blockIdx.x / a.Hkv, hk = blockIdx.x - share * a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool grp_a = HALVES && wv < PW / 2;
  const int ln = lane & 31, h = lane >> 5;
  const float scale = abs_scale(a.sl2);
  int u0 = 0, u1;
  Block b;
  if (a.shares) {
    const Deal deal = deal_out<ROWS>(a, lane);
    u0 = deal.share * share;
    u1 = min(u0 + deal.share, deal.total);
    if (u0 >= u1) return;
    b = find_block<ROWS>(a, deal, u0, lane);
  } else {  // a whole block
    b = ranked_block<ROWS>(a, share, lane);
    u1 = b.tiles + BLOCK_COST;
  }

  // ---- a tile: thread tid brings 16 codes (chunk tid % 8) of key tid / 8 (and + 8 PW)
  const int key0 = tid >> 3, chunk = tid & 7;
  const uint32_t group = chunk < 4 ? SEL_LO : SEL_HI;  // of the thread's codes
  int c0, c1, t0, t1;  // the share's tiles of the block, from its own first and from the sequence's
  bool mine;
  const int32_t* ids;
  u4_t rk[C], rv[C], fk[C];
  uint32_t ks[C], kb[C], vs[C], vb[C], fs[C], fb[C];  // words of both groups
  // whether there are such pages, and their rows: of the K loaded last, of the one before it, the V loaded last, the
  // K loaded next; the first
  bool k_ok, before_ok, v_ok, next_ok, f_ok;
  int64_t row_k, row_before, row_next;
  int id_next;
  auto load_codes = [&](const uint8_t* codes, int64_t row, u4_t (&c)[C]) {
    const global_ptr<uint8_t> cp = uniform(codes + row * D);
    const uint32_t o = lane_offset(16u * tid);
#pragma unroll
    for (int i = 0; i < C; ++i) c[i] = *(global_ptr<u4_t>)(cp + (o + 1024 * PW * i));
  };
  auto load_words = [&](const uint16_t* words, int64_t row, uint32_t (&w)[C]) {
    const global_ptr<uint8_t> p = uniform(reinterpret_cast<const uint8_t*>(words + 2 * row));
    const uint32_t o = lane_offset(4u * key0);
#pragma unroll
    for (int i = 0; i < C; ++i) w[i] = *(global_ptr<uint32_t>)(p + (o + 32 * PW * i));
  };
  // K of the tiles in order, V of each one behind
  auto next_row = [&](int t) {  // of tile t, behind the last loaded
    next_ok = id_next >= 0 && id_next < a.tab.pages;
    row_next = ((int64_t)(next_ok ? id_next : 0) * a.Hkv + hk) * PAGE;
    id_next = scalar(ids, min(t + 1, t1 - 1));
  };
  auto load_k = [&]() {
    row_before = row_k;
    before_ok = k_ok;
    row_k = row_next;
    k_ok = next_ok;
    load_codes(a.buf.kc, row_k, rk);
    load_words(a.buf.ks, row_k, ks);
    load_words(a.buf.kb, row_k, kb);
  };
  auto load_v = [&]() {
    v_ok = before_ok;
    load_codes(a.buf.vc, row_before, rv);
    load_words(a.buf.vs, row_before, vs);
    load_words(a.buf.vb, row_before, vb);
  };

  // ---- a block: the wave's rows, and its first loads, out before the rows of the block before are written: the
  // first tile's K, the second's and the first's V
  int f, i, head;
  Rows32 st;
  auto open = [&]() {
    c0 = cut_tile(b, u0);
    c1 = cut_tile(b, u1);
    t0 = b.lo + c0;
    t1 = b.lo + c1;
    // a block without a tile (rows without keys) belongs to the share that its begin lies in
    mine = c0 < c1 || (b.tiles == 0 && b.begin >= u0 && b.begin < u1);
    if (!mine) return;
    ids = a.tab.ids + (int64_t)a.seq[b.seq] * a.tab.stride;
    if (t0 < t1) {
      k_ok = before_ok = true;
      row_k = row_before = 0;
      id_next = scalar(ids, t0);
      next_row(t0);
      load_k();
#pragma unroll
      for (int i = 0; i < C; ++i) {
        fk[i] = rk[i];
        fs[i] = ks[i];
        fb[i] = kb[i];
      }
      f_ok = k_ok;
      next_row(t0 + 1);
      load_k();
      load_v();
      next_row(t0 + 2);
    }
    f = b.blk * ROWS + 32 * wv + ln;
    i = (int)fdiv_u((uint32_t)min(f, b.q.R - 1), a.g);
    head = min(f, b.q.R - 1) - i * a.G;
    const uint16_t* qr = a.q + (int64_t)(a.row0[b.seq] + i) * a.q_tok + (hk * a.G + head) * a.q_head + 8 * h;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) st.q[kk] = u4_as_bf8(*reinterpret_cast<const uint4*>(qr + 16 * kk));
  };
  open();

  for (bool more = true; more;) {
    const Seq sq = b.q;
    uint16_t* out = nullptr;  // the lane's row, or its part
    float* part_acc = nullptr;
    float2* part_ml = nullptr;
    float inv = 0.0f;
    if (mine) {
      // tiles in [t_open, t_masked) are open to all rows of the block
      const int first = sq.base + (int)fdiv_u((uint32_t)(b.blk * ROWS), a.g);
      const int last = sq.base + (int)fdiv_u((uint32_t)min(b.blk * ROWS + ROWS - 1, sq.R - 1), a.g);
      const int t_masked = first < 0 ? 0 : (first + 1) / TKEYS;
      const int t_open = (max(0, last - a.window + 1) + TKEYS - 1) / TKEYS;
      auto put = [&](uint4* lo, uint4* hi, u4_t c, float s, float z) {
        const uint2 d0 = dequant4(c.x, s, z), d1 = dequant4(c.y, s, z);
        const uint2 d2 = dequant4(c.z, s, z), d3 = dequant4(c.w, s, z);
        *lo = make_uint4(d0.x, d0.y, d1.x, d1.y);
        *hi = make_uint4(d2.x, d2.y, d3.x, d3.y);
      };
      auto stage_k = [&](int t, const u4_t (&rk)[C], const uint32_t (&ks)[C], const uint32_t (&kb)[C], bool k_ok) {
        if (t >= t1) return;  // uniform
        KvTile& to = sm.tile[t % STAGES];
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int key = key0 + 8 * PW * i;
          put(k_chunk(to, key, 2 * chunk), k_chunk(to, key, 2 * chunk + 1), rk[i],
              bf16_pick(k_ok ? ks[i] : 0x7fc07fc0u, group), bf16_pick(kb[i], group));
        }
      };
      // V of tile t (of no tile behind the last: its place is free) in steps: its words settled, then a chunk's halves.
      auto settle_v = [&](int t) {
        if (!v_ok || t >= t_masked || t < t_open) {  // uniform
#pragma unroll
          for (int i = 0; i < C; ++i) {
            const int key = key0 + 8 * PW * i;
            const bool none = !v_ok || TKEYS * t + key >= sq.len;  // no such position
            const bool w = !none && wild(bf16_pick(vs[i], group), bf16_pick(vb[i], group));
            if (w && t < t1) atomicOr(&sm.wild[t % 3][key >> 5], 1u << (key & 31));
            if (none || w) vs[i] = vb[i] = 0;
          }
        }
      };
      // one code of each chunk at a time, 16 of them
      uint32_t vd[C][4];
      float before[C];
      auto stage_v = [&](int t, int n) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float sc = bf16_pick(vs[i], group), z = bf16_pick(vb[i], group);
          const float x = fmaf(sc, (float)((rv[i][n >> 2] >> (8 * (n & 3))) & 0xffu), z);
          if (n & 1)
            vd[i][(n >> 1) & 3] = pack_bf2(before[i], x);
          else
            before[i] = x;
          if ((n & 7) == 7)
            *v_chunk32(sm.tile[t % STAGES], key0 + 8 * PW * i, 2 * chunk + (n >> 3)) =
                make_uint4(vd[i][0], vd[i][1], vd[i][2], vd[i][3]);
        }
      };

      const int f0 = b.blk * ROWS + 32 * wv;
      const int lim = f < sq.R ? sq.base + i : -1;  // last key of the lane's row, below 0: none
      // keys up to here, and from there on, are seen by all of the wave's rows
      const int lim_lo = f0 < sq.R ? sq.base + (int)fdiv_u((uint32_t)f0, a.g) : -1;
      const int open_from =
          f0 < sq.R ? sq.base + (int)fdiv_u((uint32_t)min(f0 + 31, sq.R - 1), a.g) - a.window + 1 : 0;
      f16v_t c[2];
      bf16x8_t p[4];
      const uint32_t k_at = k_lane32(sm.tile[0], lane), v_at = v_lane32(sm.tile[0], lane);
      auto tile_at = [](int t) { return (uint32_t)(t % STAGES) * (uint32_t)sizeof(KvTile); };
      tile_barrier();  // the block before is done with LDS
      if (a.sl2 < 0.0f) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) st.q[kk] = u4_as_bf8(signed_q(__builtin_bit_cast(uint4, st.q[kk]), a.sl2));
      }
      st.clear();
      if (t0 < t1) {
        if (tid < 6) sm.wild[tid >> 1][tid & 1] = 0;
        stage_k(t0, fk, fs, fb, f_ok);
        auto begin = [&]() {  // K of the second tile, V of the first; the next ones loaded
          stage_k(t0 + 1, rk, ks, kb, k_ok);
          settle_v(t0);
#pragma unroll
          for (int n = 0; n < 16; ++n) stage_v(t0, n);
          load_k();
          load_v();
        };
        tile_barrier();
        if (HALVES && !grp_a) {  // half a tile behind
          begin();
          tile_barrier();
        }
        scores32(k_at + tile_at(t0), st, c);
        if (!HALVES || grp_a) begin();
        for (int t = t0; t < t1; ++t) {
          tile_barrier();
          // vector phase
          __builtin_amdgcn_s_setprio(0);
          next_row(t + 3);
          stage_k(t + 2, rk, ks, kb, k_ok);
          load_k();
          if (TKEYS * t + TKEYS - 1 > lim_lo || TKEYS * t < open_from) {  // wave-uniform: masked for some row
            mask32(c, lim - TKEYS * t - 4 * h, a.window);
          }
          Ahead32 ahead;
          const uint32_t kt = k_at + tile_at(t + 1);
          if constexpr (HALVES) {
            softmax32(c, st, scale, p, [&]() {
              ahead32(kt, ahead);
              __builtin_amdgcn_sched_barrier(0);
            });
            tile_barrier();
          } else {
            ahead32(kt, ahead);
            softmax32(c, st, scale, p);
          }
          // matrix phase: Q.K^T of tile t + 1 (behind the last one, of a tile nobody uses), P.V of tile t
          __builtin_amdgcn_s_setprio(1);
          // between them V of tile t + 1 is staged, and the tiles behind are loaded
          settle_v(t + 1);
          matrix32(kt, v_at + tile_at(t), st, c, p, ahead, [&](int n) {
            if (n < 16) stage_v(t + 1, n);
            if (n == 16) load_v();
          });
          if (t >= t_masked || t < t_open) {
            uint64_t w = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.wild[t % 3][0]) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.wild[t % 3][1]) << 32;
            for (; w; w &= w - 1) {  // rare
              const int key = __builtin_ctzll(w);
              const int64_t row = ((int64_t)scalar(ids, t) * a.Hkv + hk) * PAGE + key;  // a page of the pool
              add_wild(a.buf, row, key, lim - TKEYS * t - key, st, lane, p, a.window);
            }
          }
          // last read before the barrier ahead of this phase: what tile t + 2 will note
          if (tid < 2) sm.wild[(t + 2) % 3][tid] = 0;
        }
        if (HALVES && grp_a) tile_barrier();
      }

      // ---- rows out: dims 32 w + 8 j + 4 h ..
      st.l = sum_xor32(st.l);
      if (c1 - c0 < b.tiles) {
        const int64_t pr = ((int64_t)(2 * share + (c0 == 0)) * a.Hkv + hk) * ROWS + 32 * wv + ln;
        part_acc = a.part_acc + pr * D;
        part_ml = a.part_ml + pr;
      } else {
        out = a.out + ((int64_t)(a.row0[b.seq] + i) * a.Hkv * a.G + hk * a.G + head) * D;
        inv = sq.len < 0 ? NAN : st.l == 0.0f ? 0.0f : 1.0f / st.l;
      }
    }
    const bool write = mine && f < sq.R;
    // the next block
    const int next = b.begin + b.tiles + BLOCK_COST;
    more = next < u1;
    if (more) {
      int ns = b.seq, place = b.place + 1;
      if (place * ROWS >= sq.R) {
        place = 0;
        ++ns;
      }
      if (ns != b.seq) b.q = seq_of(a, ns);
      const int blk = block_at(place, (b.q.R + ROWS - 1) / ROWS);
      const Span sp = block_span<ROWS>(a, b.q, blk);
      b = Block{ns, blk, sp.lo, sp.n, next, place, b.q};
      open();
    }
    if (part_acc) {  // uniform, as out
      if (write) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f4_t*>(part_acc + 32 * w + 8 * j + 4 * h) =
                f4_t{st.o[w][4 * j], st.o[w][4 * j + 1], st.o[w][4 * j + 2], st.o[w][4 * j + 3]};
        if (h == 0) *part_ml = make_float2(st.m, st.l);
      }
    } else if (out) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          // dims 8 j .. of the lower lanes' rows and 8 (j + 1) .. of the upper ones' come together: 16 bytes each
          const auto lo = __builtin_amdgcn_permlane32_swap(pack_bf2(st.o[w][4 * j] * inv, st.o[w][4 * j + 1] * inv),
                                                           pack_bf2(st.o[w][4 * j + 4] * inv, st.o[w][4 * j + 5] * inv),
                                                           false, false);
          const auto hi = __builtin_amdgcn_permlane32_swap(pack_bf2(st.o[w][4 * j + 2] * inv, st.o[w][4 * j + 3] * inv),
                                                           pack_bf2(st.o[w][4 * j + 6] * inv, st.o[w][4 * j + 7] * inv),
                                                           false, false);
          if (write) *reinterpret_cast<uint4*>(out + 32 * w + 8 * (j + h)) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
        }
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
  const Seq sq = b.q;
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

// ---- sequences of few rows (single tokens, verified blocks): 32 query rows per workgroup, or 64, all of them in every
// wave, which takes half a page (32 keys) at a time through LDS of its own (no barriers), dequantized on its way into the
// matrix cores, the next one's loads out. Reading the pages bounds long calls of one block (5 rows behind 65,536
// positions, 8 KV heads: 39 us, 3.6 TB/s; 8 single tokens of 42,771 to 82,671 194, 5.6), dequantization and softmax those
// of more rows (about 2,800 cycles of vector work per half page), the way through a half page short ones. Whole pages per
// wave took 44.6 for the first, and 25.0 instead of 20.8 for 64 tokens of windows of 512.
constexpr int UNIT = 32;  // keys of a wave's step

template <int WV, int NB>  // waves, 32 rows each of a block
struct FewSmem {
  // a wave's keys: 16-byte chunk c of row r of K at c ^ kswz(r), of V at c ^ vfew(r); at the end 16 of its rows'
  // values, 16-byte chunk c of row r at c ^ r
  alignas(256) uint8_t codes[WV][2][UNIT * D];
  alignas(16) float w[WV][4][2][UNIT];  // K scales, K biases, V scales, V biases of the two groups
  uint4 q[NB][8][64];                   // the rows of q as B operands, a lane's place in each
  float2 ml[WV][32 * NB];
};
// Rows of V that a transposed read takes together, 4 h + 8 i + r: in different banks.
__device__ __forceinline__ int vfew(int r) { return (r & 3) | ((r >> 1) & 4); }

// First unit that the rows of a sequence see, and how many.
struct Units {
  int lo, n;
};
__device__ __forceinline__ Units few_units(const ChunkArgs& a, const Seq& q) {
  const int lo = max(0, q.base - a.window + 1) / UNIT;
  return {lo, q.len <= 0 ? 0 : (q.len + UNIT - 1) / UNIT - lo};
}
__device__ __forceinline__ Deal few_deal(const ChunkArgs& a, int lane) {
  const Seq q = lane < a.nseq ? seq_of(a, lane) : Seq{0, 0, 0};
  const int n = few_units(a, q).n;
  const int upto = wave_scan_i(n ? n + SEQ_COST : 0);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  return {upto, q, total, max(SHARE_MIN, (total + a.shares - 1) / a.shares)};
}

// Units [p0, p1) of sequence s for its rows f0 .. f0 + 32 NB - 1: partial rows to slot .., or with WHOLE output rows.
// AGAIN: other blocks read the pages too, and they stay in the L2 (streaming / staying, us: 48 rows of 16
// sessions of 100 to 4,100 positions 42.6 / 39.2; of one block 64 single tokens of up to 8,200 118 / 124). Sequences
// taken whole stream their pages whatever their blocks, which run side by side and are few pages apart: staying is
// within 5% either way there (48 rows of 16 windows of 512 14.9 / 15.4, of 16 sessions of 1,000 19.2 / 19.9, 96 of 8
// windows 14.0 / 14.1, of 32 32.2 / 30.6, of 64 57.2 / 55.5, 80 of 16 of 2 KV heads 13.6 / 13.2).
template <int NB, bool WHOLE, bool AGAIN, int WV, int MB>
__device__ __forceinline__ void few_part(const ChunkArgs& a, FewSmem<WV, MB>& sm, int s, const Seq& sq, int f0, int hk,
                                         int p0, int p1, int64_t slot) {
  int tid = threadIdx.x;  // re-read, so that no lane value made of it is kept across sequences
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, h = lane >> 5;

  const int32_t* ids = a.tab.ids + (int64_t)a.seq[s] * a.tab.stride;
  u4_t rk[4], rv[4];
  uint32_t kw, vw;  // of key ln: scale words (h == 0) or bias words of both groups
  bool next_ok = true;
  int64_t row_next = 0;
  auto read = [](const auto* from) {
    if constexpr (AGAIN)
      return *from;
    else
      return __builtin_nontemporal_load(from);
  };
  auto load = [&](int p) {
    const int id = scalar(ids, p / (PAGE / UNIT));
    next_ok = id >= 0 && id < a.tab.pages;
    row_next = ((int64_t)(next_ok ? id : 0) * a.Hkv + hk) * PAGE + p % (PAGE / UNIT) * UNIT;
    const u4_t* k = reinterpret_cast<const u4_t*>(a.buf.kc + row_next * D) + lane;
    const u4_t* v = reinterpret_cast<const u4_t*>(a.buf.vc + row_next * D) + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) rk[i] = read(k + 64 * i);
    kw = read(reinterpret_cast<const uint32_t*>(h ? a.buf.kb : a.buf.ks) + row_next + ln);
#pragma unroll
    for (int i = 0; i < 4; ++i) rv[i] = read(v + 64 * i);
    vw = read(reinterpret_cast<const uint32_t*>(h ? a.buf.vb : a.buf.vs) + row_next + ln);
  };
  int p = p0 + wv;
  if (p < p1) load(p);

  const float scale = abs_scale(a.sl2);
  int lim[NB];  // a row's position
#pragma unroll
  for (int t = 0; t < NB; ++t) {
    const int f = f0 + 32 * t + ln;
    lim[t] = f < sq.R ? sq.base + (int)fdiv_u((uint32_t)f, a.g) : -1;
  }
  __syncthreads();  // the sequence before is written
  // q in K's order of dims: step 2 j + x holds dims 16 (2 j + h) + 8 x .. + 7
#pragma unroll
  for (int t = 0; t < NB; ++t) {
    const int f = min(f0 + 32 * t + ln, sq.R - 1), i = (int)fdiv_u((uint32_t)f, a.g);
    const uint16_t* qr = a.q + (int64_t)(a.row0[s] + i) * a.q_tok + (hk * a.G + f - i * a.G) * a.q_head + 16 * h;
    for (int kk = wv; kk < 8; kk += WV)
      sm.q[t][kk][lane] = signed_q(*reinterpret_cast<const uint4*>(qr + 32 * (kk >> 1) + 8 * (kk & 1)), a.sl2);
  }
  Rows32 st[NB];
#pragma unroll
  for (int t = 0; t < NB; ++t) st[t].clear();
  const int lim_lo = sq.base + (int)fdiv_u((uint32_t)f0, a.g);
  const int open_from = sq.base + (int)fdiv_u((uint32_t)min(f0 + 32 * NB - 1, sq.R - 1), a.g) - a.window + 1;
  uint8_t* const kp = sm.codes[wv][0];
  uint8_t* const vp = sm.codes[wv][1];
  __syncthreads();  // q
  for (; p < p1; p += WV) {
    const int64_t row = row_next;
    const bool ok = next_ok;
    const bool masked = UNIT * p + UNIT - 1 > lim_lo || UNIT * p < open_from;
    wave_fence();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 3), c = lane & 7;
      reinterpret_cast<u4_t*>(kp)[8 * r + (c ^ kswz(r))] = rk[i];
      reinterpret_cast<u4_t*>(vp)[8 * r + (c ^ vfew(r))] = rv[i];
    }
    // no V of positions that are not there, nor of those that are not finite where some row does not see them
    const bool none = !ok || UNIT * p + ln >= sq.len;
    uint32_t keep = none ? 0u : 0xffffffffu;
    uint64_t wilds = 0;
    if (masked) {  // uniform
      const uint32_t other = __shfl_xor(vw, 32, 64), sw = h ? other : vw, zw = h ? vw : other;
      if (wild(bf16_lo(sw), bf16_lo(zw))) keep &= 0xffff0000u;
      if (wild(bf16_hi(sw), bf16_hi(zw))) keep &= 0x0000ffffu;
      wilds = __builtin_amdgcn_ballot_w64(!none && keep != 0xffffffffu) & 0xffffffffu;
    }
    if (!ok && h == 0) kw = 0x7fc07fc0u;
    sm.w[wv][h][0][ln] = bf16_lo(kw);
    sm.w[wv][h][1][ln] = bf16_hi(kw);
    sm.w[wv][2 + h][0][ln] = bf16_lo(vw & keep);
    sm.w[wv][2 + h][1][ln] = bf16_hi(vw & keep);
    if (p + WV < p1) load(p + WV);
    wave_fence();
    // scores
    f16v_t c[NB][1];
#pragma unroll
    for (int t = 0; t < NB; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) c[t][0][i] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float sc = sm.w[wv][0][j >> 1][ln], z = sm.w[wv][1][j >> 1][ln];
      const u4_t w = reinterpret_cast<const u4_t*>(kp)[8 * ln + ((2 * j + h) ^ kswz(ln))];
      const uint2 d0 = dequant4(w[0], sc, z), d1 = dequant4(w[1], sc, z);
      const uint2 d2 = dequant4(w[2], sc, z), d3 = dequant4(w[3], sc, z);
#pragma unroll
      for (int t = 0; t < NB; ++t) {
        c[t][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(words_as_bf8(d0.x, d0.y, d1.x, d1.y),
                                                          u4_as_bf8(sm.q[t][2 * j][lane]), c[t][0], 0, 0, 0);
        c[t][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(words_as_bf8(d2.x, d2.y, d3.x, d3.y),
                                                          u4_as_bf8(sm.q[t][2 * j + 1][lane]), c[t][0], 0, 0, 0);
      }
    }
    bf16x8_t pr[NB][2];
#pragma unroll
    for (int t = 0; t < NB; ++t) {
      if (masked) mask32(c[t], lim[t] - UNIT * p - 4 * h, a.window);  // uniform
      softmax32(c[t], st[t], scale, pr[t]);
      sums32(st[t], pr[t]);
    }
    // values: of keys 16 e + 8 (j / 4) + 4 h + j % 4, j < 8, this lane's dim of each window of 32
    const int r8 = (lane >> 1) & 7, src = 4 * h + 8 * (r8 >> 2) + (r8 & 3);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float sc[8], z[8];
        *reinterpret_cast<f4_t*>(sc) = *reinterpret_cast<const f4_t*>(&sm.w[wv][2][g][16 * e + 4 * h]);
        *reinterpret_cast<f4_t*>(sc + 4) = *reinterpret_cast<const f4_t*>(&sm.w[wv][2][g][16 * e + 8 + 4 * h]);
        *reinterpret_cast<f4_t*>(z) = *reinterpret_cast<const f4_t*>(&sm.w[wv][3][g][16 * e + 4 * h]);
        *reinterpret_cast<f4_t*>(z + 4) = *reinterpret_cast<const f4_t*>(&sm.w[wv][3][g][16 * e + 8 + 4 * h]);
#pragma unroll
        for (int w = 2 * g; w < 2 * g + 2; ++w) {
          const int chunk = 2 * w + ((lane >> 4) & 1);
          const v2i_t raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (lds_v2i_t*)(vp + (16 * e + src) * D + 16 * (chunk ^ vfew(src)) + 8 * (lane & 1)));
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[j] = fmaf(sc[j], (float)(((uint32_t)(j < 4 ? raw.x : raw.y) >> (8 * (j & 3))) & 0xffu), z[j]);
          const bf16x8_t vb = words_as_bf8(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]),
                                           pack_bf2(v[6], v[7]));
#pragma unroll
          for (int t = 0; t < NB; ++t)
            st[t].o[w] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb, pr[t][e], st[t].o[w], 0, 0, 0);
        }
      }
    for (; wilds; wilds &= wilds - 1) {  // rare
      const int key = __builtin_ctzll(wilds);
#pragma unroll
      for (int t = 0; t < NB; ++t)
        add_wild(a.buf, row + key, key, lim[t] - UNIT * p - key, st[t], lane, pr[t], a.window);
    }
  }

  // ---- the waves' rows meet in LDS, 16 at a time
  const int R = min(32 * NB, sq.R - f0);
  f4_t* acc = reinterpret_cast<f4_t*>(sm.codes[wv]);
#pragma unroll
  for (int t = 0; t < NB; ++t) {
    const float l = sum_xor32(st[t].l);
    if (h == 0) sm.ml[wv][32 * t + ln] = make_float2(st[t].m, l);
  }
#pragma unroll
  for (int part = 0; part < 2 * NB; ++part) {
    const Rows32& rt = st[part >> 1];
    if (16 * part >= R) break;  // uniform
    if (part) __syncthreads();  // the 16 before are read
    wave_fence();
    if (ln >> 4 == (part & 1)) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[32 * (ln & 15) + ((8 * w + 2 * j + h) ^ (ln & 15))] =
              f4_t{rt.o[w][4 * j], rt.o[w][4 * j + 1], rt.o[w][4 * j + 2], rt.o[w][4 * j + 3]};
    }
    __syncthreads();
    for (int x = tid; x < 32 * min(16, R - 16 * part); x += 64 * WV) {
      const int r = x >> 5, ch = x & 31, row = 16 * part + r;
      float M = -INFINITY, L = 0.0f;
      f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WV; ++w) M = max_ieee(M, sm.ml[w][row].x);
      const float Mr = M == -INFINITY ? 0.0f : M;
#pragma unroll
      for (int w = 0; w < WV; ++w) {
        const float2 ml = sm.ml[w][row];
        const float e = exp2_nonpos(ml.x - Mr);  // of no keys: 0, and a sum that is NaN stays
        o += reinterpret_cast<const f4_t*>(sm.codes[w])[32 * r + (ch ^ r)] * e;
        L += ml.y * e;
      }
      if constexpr (WHOLE) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const int q = (int)fdiv_u((uint32_t)(f0 + row), a.g), head = f0 + row - q * a.G;
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(a.row0[s] + q) * a.Hkv * a.G + hk * a.G + head) * D + 4 * ch) =
            make_uint2(pack_bf2(o[0] * inv, o[1] * inv), pack_bf2(o[2] * inv, o[3] * inv));
      } else {
        *reinterpret_cast<f4_t*>(a.part_acc + (slot + row) * D + 4 * ch) = o;
        if (ch == 0) a.part_ml[slot + row] = make_float2(M, L);
      }
    }
  }
}

// Partial rows of a KV head and row block: a block's for each share and sequence (along both each part adds one to
// their sum).
__device__ __forceinline__ int64_t few_slot(const ChunkArgs& a, int hk, int rb, int x) {
  return ((int64_t)(hk * a.blocks + rb) * (a.shares + a.nseq) + x) << a.row_bits;
}
template <int NB, bool WHOLE, bool AGAIN, int WV>
__device__ __forceinline__ void few_rows(const ChunkArgs& a, FewSmem<WV, NB>& sm, int s, const Seq& sq, int f0, int hk,
                                         int p0, int p1, int64_t slot) {
  if (sq.R - f0 > 32)  // uniform
    few_part<NB, WHOLE, AGAIN>(a, sm, s, sq, f0, hk, p0, p1, slot);
  else if (sq.R > f0)
    few_part<1, WHOLE, AGAIN>(a, sm, s, sq, f0, hk, p0, p1, slot);
}

// A share of the sequences' half pages, dealt out one sequence behind the other.
template <int NB, bool AGAIN>
__global__ __launch_bounds__(64 * FEW_WAVES, 2) void few_kernel(const ChunkArgs a) {
  __shared__ FewSmem<FEW_WAVES, NB> sm;
  const int hk = blockIdx.x % a.Hkv, y = blockIdx.x / a.Hkv, x = y / a.blocks, rb = y - x * a.blocks;
  const int lane = threadIdx.x & 63;
  const Deal deal = few_deal(a, lane);
  const int u0 = x * deal.share, u1 = min(u0 + deal.share, deal.total);
  if (u0 >= u1) return;
  int s = __builtin_popcountll(__builtin_amdgcn_ballot_w64(deal.upto <= u0));
  int begin = s ? __builtin_amdgcn_readlane(deal.upto, s - 1) : 0;
  for (int u = u0; u < u1; ++s) {
    const Seq sq = seq_at(deal, s);
    const Units pg = few_units(a, sq);
    if (pg.n == 0) continue;
    begin += SEQ_COST;
    const int p0 = max(u - begin, 0), p1 = min(u1 - begin, pg.n);
    if (p0 < p1)
      few_rows<NB, false, AGAIN>(a, sm, s, sq, 32 * NB * rb, hk, pg.lo + p0, pg.lo + p1, few_slot(a, hk, rb, x + s));
    begin += pg.n;
    u = begin;
  }
}

// A whole sequence per workgroup: nothing to merge.
template <int NB, int WV>
__global__ __launch_bounds__(64 * WV, 2) void few_whole_kernel(const ChunkArgs a) {
  __shared__ FewSmem<WV, NB> sm;
  const int hk = blockIdx.x % a.Hkv, y = blockIdx.x / a.Hkv, s = y / a.blocks, f0 = 32 * NB * (y - s * a.blocks);
  const Seq sq = seq_of(a, s);
  const int R = min(32 * NB, sq.R - f0);
  if (sq.len < 0) {
    for (int x = threadIdx.x; x < R * D; x += 64 * WV) {
      const int f = f0 + x / D, p = (int)fdiv_u((uint32_t)f, a.g);
      a.out[((int64_t)(a.row0[s] + p) * a.Hkv * a.G + hk * a.G + f - p * a.G) * D + x % D] = 0x7fc0;
    }
    return;
  }
  const Units pg = few_units(a, sq);
  few_rows<NB, true, false>(a, sm, s, sq, f0, hk, pg.lo, pg.lo + pg.n, 0);
}

// An output row by GR groups of 32 lanes (4 dims each), 8 / GR rows per workgroup: group g takes every GR-th
// partial, four at a time, and the groups meet in LDS.
template <int GR>
__global__ __launch_bounds__(256) void few_merge_kernel(const ChunkArgs a) {
  __shared__ float2 sh_ml[8];
  __shared__ f4_t sh_acc[8][32];
  const int lane = threadIdx.x & 63;
  // wave-uniform: a row has at least a wave. Rows of a sequence and KV head: as many as its blocks'
  const int row = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (8 / GR) + threadIdx.x / (32 * GR)));
  const int per = a.blocks << a.row_bits, y = row / per, f = row - y * per, s = min(y / a.Hkv, a.nseq - 1), hk = y % a.Hkv;
  const Deal deal = few_deal(a, lane);
  const Seq sq = seq_at(deal, s);
  const int pages = few_units(a, sq).n;
  const int before = (s ? __builtin_amdgcn_readlane(deal.upto, s - 1) : 0) + SEQ_COST;
  const int first = before / deal.share;
  const bool mine = f < sq.R;
  const int parts = mine && pages ? (before + pages - 1) / deal.share - first + 1 : 0;
  const int64_t slot = few_slot(a, hk, f >> a.row_bits, first + s) + (f & ((1 << a.row_bits) - 1));
  const int grp = (threadIdx.x >> 5) % GR, ch = threadIdx.x & 31;
  float M = -INFINITY, den = 0.0f;
  f4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = grp; i0 < parts; i0 += 4 * GR) {
    float2 ml[4];
    f4_t x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = slot + ((int64_t)min(i0 + GR * j, parts - 1) << a.row_bits);
      ml[j] = a.part_ml[at];
      x[j] = *reinterpret_cast<const f4_t*>(a.part_acc + at * D + 4 * ch);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + GR * j < parts) merge_into(M, den, acc, ml[j].x, ml[j].y, x[j]);
  }
  const int at = threadIdx.x >> 5;
  sh_acc[at][ch] = acc;
  if (ch == 0) sh_ml[at] = make_float2(M, den);
  __syncthreads();
  if (grp != 0 || !mine) return;
#pragma unroll
  for (int j = 1; j < GR; ++j) merge_into(M, den, acc, sh_ml[at + j].x, sh_ml[at + j].y, sh_acc[at + j][ch]);
  const float inv = sq.len < 0 ? NAN : den == 0.0f ? 0.0f : 1.0f / den;
  const int p = (int)fdiv_u((uint32_t)f, a.g);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)(a.row0[s] + p) * a.Hkv * a.G + hk * a.G + f - p * a.G) * D + 4 * ch) =
      make_uint2(pack_bf2(acc[0] * inv, acc[1] * inv), pack_bf2(acc[2] * inv, acc[3] * inv));
}

// How a call's sequences are dealt out. The lengths are the device's: the rules below take the table's width for them
// (the window's, where it is shorter), so a table wider than its sequences may get the way that suits long ones. us,
// table as wide as the sequences / 1,300 pages: a row behind 1,037 positions 15.0 / 9.5, of each of 64 sessions of 100 to
// 1,500 34.5 / 39.6, 8 of 16 of 97 to 4,099 40 / 42, 8 prompts of 300 rows 26 / 35, 512 rows behind 1,000 41.9 / 42.1,
// behind 7,681 121 / 121, 5 behind 65,536 39.0 / 38.3.
struct ChunkPart {  // the sequences of few rows, or of many
  int nseq, rows_of, shares, blocks;  // rows of a block, shares (0: whole blocks) and blocks per KV head
  int seq[LQ_MAX_SEQS], row0[LQ_MAX_SEQS], rows[LQ_MAX_SEQS];
  int64_t slots;  // partial rows, all heads; 0: no parts
};
struct ChunkPlan {
  ChunkPart few, many;
};
// Up to FEW_ROWS query rows of a sequence and KV head go as blocks of 32 (64) that read the pages each, those dealt out
// from the L2 but the first, more as blocks that share a dequantized page. us, shared / each, 8 KV heads: 36 rows behind
// 20,000 positions 54 / 27, 64 behind 65,536 87 / 60, 96 behind 65,536 86 / 74, behind 5,000 27 / 22, of 4 sessions of
// 9,000 51 / 53, of 16 of 4,099 65 / 81, 48 of 16 of 100 to 4,100 44 / 45; above the limit 126 behind 65,536 88 / 91,
// behind 20,000 57 / 40, behind 5,000 26 / 24, of 4 of 9,000 51 / 59, of 16 of 4,099 69 / 95: one session of up to 20,000
// would gain, several lose more.
constexpr int64_t FEW_ROWS = 96;
// Blocks of many rows are taken whole, a workgroup each and the longest first, where that leaves few compute units
// idle: IDLE_TILES per block, were all blocks as long as the table (or window) lets them be. Else the call is dealt out
// in shares, which end together but write, merge and start on parts. How the lengths differ is not known here, and one
// long block among short ones would be waited for: whole blocks have at most LONGEST tiles, or those that the rows see
// of each other alone keep the other workgroups busy for as long. us, shares / whole, 48/8 heads: 2,048 rows of a window
// of 512 66.8 / 57.4, of 4,096 240 / 263, 1,024 behind 1,000 68.4 / 67.5, behind 8,000 235 / 258, 7 prompts of up to
// 4,099 653 / 623, 24 chunks of up to 301 rows behind up to 6,007 365 / 348 (in shares all the same); 32/8 heads: 5
// prompts of up to 2,049 rows 123 / 103, 4 of 500 38 / 27, one of 5,000 254 / 244, 64 of 400 220 / 234.
constexpr int64_t IDLE_TILES = 8, LONGEST = 40;
// Of more than 32 rows, 64 go as one block where a workgroup (two per CU) has TWO_UNITS half pages or more, or a sequence
// and KV head of its own: its waves dequantize a page once for both halves, but have as much to join at the end. us, 32 /
// 64 rows: 48 of 16 sessions of 100 to 4,100 positions 39 / 43, of 2,050 each (17 half pages) 41 / 42, of 4,099 (32) 60
// / 57, of 4,608 (36) 65 / 60, of 6,000 77 / 67, of 8,000 97 / 81, of 100 to 8,000 60 / 55; 48 of 4 of 20,000 75 / 63, of
// one 27 / 34; 64 behind 65,536 61 / 57; 48 of 64 windows of 512 40 / 34, of 8 13.5 / 21. Half pages by the table's
// width: sequences that fill it gain from 32 on, those of half its width on average still lose there.
constexpr int64_t TWO_UNITS = 36;
// Calls of few pages per sequence take each whole: one launch, nothing to merge. Many sequences also where they are
// longer. us on the GPU, dealt out / whole: 1 session of 512 positions, 8 KV heads 9.3 / 10.2, of 1,038 9.5 / 15.0 (with
// the host, whose launches bound such a call, 16.3 / 14: the limit is set for calls made one by one, a recorded step
// would take shares from the first pages on); 8 of 1,500 16.4 / 20.3, 16 windows of 1,100 20.6 / 17.6, 32 of 1,500 32.1 /
// 24.3, 64 of 100 to 1,500 39.1 / 33.2.
constexpr int64_t WHOLE_PAGES = 20, WHOLE_PAGES_MANY = 32;
ChunkPlan chunk_plan(const int32_t* counts, int64_t nseq, int64_t Hkv, int64_t G, int64_t width, int64_t window, int cus) {
  ChunkPlan p{};
  int at = 0;
  int64_t most = 0, few = 0;  // query rows of a sequence
  for (int s = 0; s < nseq; ++s) {
    if (counts[s]) {
      const int64_t R = counts[s] * G;
      ChunkPart& c = R <= FEW_ROWS ? p.few : p.many;
      c.seq[c.nseq] = s;
      c.row0[c.nseq] = at;
      c.rows[c.nseq++] = counts[s];
      (R <= FEW_ROWS ? few : most) = std::max(R <= FEW_ROWS ? few : most, R);
    }
    at += counts[s];
  }
  // pages that a window lets n positions see
  auto seen = [&](int64_t n) { return window == 0 ? width : std::min(width, (window + n - 2 + PAGE - 1) / PAGE + 1); };
  p.many.rows_of = most > 128 ? 256 : 128;
  int64_t blocks = 0, own = 0;  // tiles that a KV head's rows see of each other
  for (int s = 0; s < p.many.nseq; ++s) {
    const int64_t n = (p.many.rows[s] * G + p.many.rows_of - 1) / p.many.rows_of;
    blocks += n;
    own += n * std::min<int64_t>(seen(1), p.many.rows[s] / (2 * PAGE));
  }
  p.many.blocks = (int)std::min<int64_t>(blocks, INT32_MAX);
  const int64_t slots = p.many.rows_of == 256 ? cus : 2 * cus;  // workgroups at a time
  const int64_t idle = (slots - blocks * Hkv % slots) % slots;
  const int64_t tiles = seen(p.many.rows_of / G + 1);
  if (idle * tiles > IDLE_TILES * blocks * Hkv || tiles > std::max(LONGEST, own * Hkv / slots))
    p.many.shares = (int)std::max<int64_t>(1, slots / Hkv);
  p.many.slots = p.many.nseq && p.many.shares > 1 ? 2 * p.many.shares * Hkv * p.many.rows_of : 0;
  int rows = 0;
  for (int s = 0; s < p.few.nseq; ++s) rows = std::max(rows, p.few.rows[s]);
  const int64_t units = p.few.nseq * Hkv * seen(rows) * (PAGE / UNIT);
  const bool two = few > 32 && (units >= TWO_UNITS * 2 * cus || p.few.nseq * Hkv >= 2 * cus);
  p.few.rows_of = two ? 64 : 32;
  p.few.blocks = (int)((few + p.few.rows_of - 1) / p.few.rows_of);
  const int64_t wgs = p.few.nseq * p.few.blocks * Hkv;
  if (seen(rows) > (2 * wgs >= cus ? WHOLE_PAGES_MANY : WHOLE_PAGES)) {
    p.few.shares = (int)std::max<int64_t>(1, 2 * cus / (Hkv * std::max(1, p.few.blocks)));
    p.few.slots = Hkv * p.few.blocks * (int64_t)(p.few.shares + p.few.nseq) * p.few.rows_of;
  }
  return p;
}
int64_t chunk_bytes(const ChunkPlan& p) {
  return std::max(p.few.slots, p.many.slots) * (int64_t)(D * sizeof(float) + sizeof(float2));
}

int check_chunk(int64_t Hq, int64_t Hkv, const int32_t* counts, int64_t nseq, int64_t width, int64_t window) {
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
  LQ_CHECK_ARG(width >= 1 && window >= 0 && window < ((int64_t)1 << 40),
               "a window of %lld positions, or table rows of %lld pages", (long long)window, (long long)width);
  return LQ_OK;
}

int launch_many(const ChunkArgs& a, const ChunkPart& c, hipStream_t st) {
  const dim3 grid((unsigned)((a.shares ? a.shares : c.blocks) * a.Hkv));
  if (c.rows_of == 256)
    chunk_kernel<8><<<grid, dim3(512), 0, st>>>(a);
  else
    chunk_kernel<4><<<grid, dim3(256), 0, st>>>(a);
  LQ_CHECK_LAUNCH("chunk_kernel");
  if (a.shares > 1) {
    auto* merge = c.rows_of == 256 ? chunk_merge_kernel<256> : chunk_merge_kernel<128>;
    merge<<<dim3((unsigned)((a.shares - 1) * a.Hkv), c.rows_of / MERGE_ROWS), dim3(256), 0, st>>>(a);
    LQ_CHECK_LAUNCH("chunk_merge_kernel");
  }
  return LQ_OK;
}

int launch_few(const ChunkArgs& a, const ChunkPart& c, hipStream_t st) {
  if (a.shares == 0) {
    const int64_t wgs = (int64_t)c.nseq * c.blocks * a.Hkv;
    const bool wide = c.rows_of == 32 && wgs <= device_cu_count();
    // blocks of 64 rows are only formed for more workgroups than CUs
    auto* whole = c.rows_of > 32 ? few_whole_kernel<2, 4> : wide ? few_whole_kernel<1, 8> : few_whole_kernel<1, 4>;
    whole<<<dim3((unsigned)wgs), dim3(wide ? 512 : 256), 0, st>>>(a);
    LQ_CHECK_LAUNCH("few_whole_kernel");
    return LQ_OK;
  }
  const bool again = c.blocks > 1;
  auto* few = c.rows_of > 32 ? again ? few_kernel<2, true> : few_kernel<2, false>
                             : again ? few_kernel<1, true> : few_kernel<1, false>;
  few<<<dim3((unsigned)(a.shares * c.blocks * a.Hkv)), dim3(64 * FEW_WAVES), 0, st>>>(a);
  LQ_CHECK_LAUNCH("few_kernel");
  const int64_t n = (int64_t)c.nseq * a.Hkv * c.rows_of * c.blocks;
  if (a.shares / std::min(c.nseq, 4) > 16)
    few_merge_kernel<8><<<dim3((unsigned)n), dim3(256), 0, st>>>(a);
  else
    few_merge_kernel<2><<<dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st>>>(a);
  LQ_CHECK_LAUNCH("few_merge_kernel");
  return LQ_OK;
}

}  // namespace
}  // namespace lq

extern "C" int64_t lq_paged_chunk_workspace_bytes(const int32_t* counts_host, int64_t nseq, int64_t Hq, int64_t Hkv,
                                                  int64_t table_width, int64_t window) {
  using namespace lq;
  clear_error();
  if (check_chunk(Hq, Hkv, counts_host, nseq, table_width, window)) return -1;
  return chunk_bytes(chunk_plan(counts_host, nseq, Hkv, Hq / Hkv, table_width, window, device_cu_count()));
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
  if (const int st = check_chunk(Hq, Hkv, counts_host, nseq, table_width, window)) return st;
  LQ_CHECK_ARG(std::isfinite(scale), "the softmax scale is not finite");
  const int64_t G = Hq / Hkv;
  const ChunkPlan plan = chunk_plan(counts_host, nseq, Hkv, G, table_width, window, device_cu_count());
  if (plan.few.nseq + plan.many.nseq == 0) return LQ_OK;
  LQ_CHECK_ARG(q && lens && out, "null pointer");
  LQ_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && ((q_tok | q_head) & 7) == 0,
               "rows must be 16-byte aligned (strides a multiple of 8)");
  LQ_CHECK_ARG((int64_t)plan.many.blocks * Hkv <= 1 << 22, "too many rows");  // workgroups of a launch
  int64_t most = 0;  // cost, if every block sees the whole table: twice as much has to fit 32 bits
  for (int s = 0; s < plan.many.nseq; ++s)
    most += (plan.many.rows[s] * G + plan.many.rows_of - 1) / plan.many.rows_of * (table_width + lq::BLOCK_COST);
  most = std::max<int64_t>(most, plan.few.nseq * (2 * table_width + lq::SEQ_COST));
  LQ_CHECK_ARG(most < 1ll << 30, "too many rows for table rows of %lld pages", (long long)table_width);
  const int64_t need = chunk_bytes(plan);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    set_error("workspace of %lld bytes is smaller than the %lld needed", (long long)workspace_bytes, (long long)need);
    return LQ_EWORKSPACE;
  }
  LQ_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  a.q = q;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.lens = lens;
  a.out = out;
  a.Hkv = (int)Hkv;
  a.G = (int)G;
  a.g = make_fastdiv((uint32_t)G);
  a.sl2 = scale * 1.4426950408889634f;
  a.window = window == 0 ? NO_WINDOW : (int)std::min<int64_t>(window, NO_WINDOW);
  const hipStream_t st = (hipStream_t)stream;
  for (const ChunkPart* c : {&plan.many, &plan.few}) {
    if (c->nseq == 0) continue;
    a.part_acc = (float*)workspace;
    a.part_ml = (float2*)(a.part_acc + c->slots * 128);
    a.shares = c->shares;
    a.blocks = c->blocks;
    a.row_bits = c->rows_of > 32 ? 6 : 5;
    a.nseq = c->nseq;
    a.lanes = 6;
    while ((c->nseq << a.lanes) > 64) --a.lanes;
    std::copy(c->seq, c->seq + LQ_MAX_SEQS, a.seq);
    std::copy(c->row0, c->row0 + LQ_MAX_SEQS, a.row0);
    std::copy(c->rows, c->rows + LQ_MAX_SEQS, a.rows);
    const int status = c == &plan.many ? launch_many(a, *c, st) : launch_few(a, *c, st);
    if (status) return status;
  }
  return LQ_OK;
}
