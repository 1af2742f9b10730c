// Causal attention of packed prompts: the rows of up to 64 sequences of different lengths, one behind the
// other, bf16 q [rows, Hq, 128] over k and v [keys, Hkv, 128] with any token and head strides, no padding
// and no score matrix. Sequence s has q_lens[s] rows and k_lens[s] keys, aligned at their ends: row i sees
// keys 0 .. k_lens[s] - q_lens[s] + i, so a prompt has as many of both and a chunk of one more keys. Rows
// without a key are 0.
//
// Work: a workgroup of 8 waves (or 4, see below) takes 256 query rows (128) of a KV head, numbered
// position-major (row f is position f / G of query head f % G), so that any grouping fills the matrix
// cores and a block's rows see nearly the same keys; a wave has 32 of them. It walks the 64-key tiles up
// to its last row's bound, each copied into LDS once for all waves (three buffers of K and of V, copies
// two tiles ahead) and run through attn_tile.h. A SIMD holds one wave of each half of the workgroup, and
// the halves run one phase apart, so that one's matrix phase (P.V of a tile, Q.K^T of the next) lies
// beside the other's vector phase (softmax, copies), with a barrier after each:
//
//   slot    group A                   group B
//   2t      Q.K^T(t), P.V(t-1)        softmax(t-1), copies K(t+2) V(t+1)
//   2t+1    softmax(t), copies        Q.K^T(t), P.V(t-1)
//
// The small workgroups have 4 waves, 128 rows and two buffers each, a barrier per tile, and share a CU in
// twos: what the halves above do for each other, the two do by chance. Slower by 3% where blocks are long,
// faster where they are short (prompt_plan has the rule and what it measured).
//
// The work is dealt out in whole blocks, longest first, or in equal shares of tiles. For these the blocks of
// all sequences stand one behind the other (of a sequence the last, the first, the last but one, .., so that
// two neighbours cost about the same everywhere and cuts are few), a block costing its tiles and BLOCK_COST
// for its start and end, and a workgroup takes one share, which may begin and end inside blocks. Parts of
// blocks go to the workspace and a second launch merges them. A workgroup finds its block or share by scanning
// the blocks, a lane each; nothing of the plan but the sequences' costs comes from the host. Where all small
// workgroups are resident at once, those beyond one per CU stand in ascending order, so that a CU holds a
// long and a short one (2,048 rows, 32/8 heads: 53.3 -> 51.4 us). The KV head is the fastest index, so that
// neighbouring workgroups (XCDs) hold different heads and each XCD's L2 the K and V of few.
//
// Keys that a row does not see reach it in no way: masked scores are -infinity, and an infinity or NaN in
// V of a tile that is masked for some row of the block goes only to the rows that see its key (0 times it
// would be NaN): such tiles are rare and take the two-pass form.
#include <algorithm>

#include "attn_tile.h"

namespace lq {
namespace {

using namespace attn;

constexpr int NT = 2;          // 16-row tiles per wave
constexpr int PROWS = 256;     // rows of a block; SROWS where the workgroups are small
constexpr int SROWS = 128;
constexpr int BLOCK_COST = 4;  // of a block's start and end, in tiles
constexpr int MIN_PART = 2;    // tiles of a block's part: nearer cuts move to the block's end

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;           // [rows, Hq, 128]
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  float* part_acc;         // [2 x shares x Hkv][256][128] rows of parts: slot 0 of a share those of the block
  float2* part_ml;         // that began in an earlier one, slot 1 of the block that goes on in a later one
  int Hkv, G, nseq;
  FastDiv g;
  float sl2;
  int64_t share;           // cost of a share; 0: a workgroup takes one whole block
  int longest;             // tiles of the longest block
  int paired;              // whole blocks from this rank on in ascending order, -1: none
  int q_begin[LQ_MAX_SEQS + 1], k_begin[LQ_MAX_SEQS + 1];
  int64_t cost[LQ_MAX_SEQS + 1];  // of the blocks before each sequence
};

// 64-key tiles that block blk (of ROWS rows) of a sequence of R rows needs; base: row i sees keys <= base + i.
template <int ROWS = PROWS>
__host__ __device__ __forceinline__ int block_tiles(int blk, int R, FastDiv g, int base) {
  const int last = base + (int)fdiv_u((uint32_t)min(blk * ROWS + ROWS - 1, R - 1), g);
  return last < 0 ? 0 : last / TKEYS + 1;
}

// A block, its place among its sequence's blocks and where its cost begins.
struct Block {
  int seq, blk, tiles;
  int64_t begin;
  int place;
};
// The block at a place among nb: the last, the first, the last but one, ..
__device__ __forceinline__ int block_at(int place, int nb) {
  return place & 1 ? place >> 1 : nb - 1 - (place >> 1);
}
__device__ __forceinline__ int seq_rows(const PromptArgs& a, int s) {
  return (a.q_begin[s + 1] - a.q_begin[s]) * a.G;
}
__device__ __forceinline__ int seq_base(const PromptArgs& a, int s) {
  return a.k_begin[s + 1] - a.k_begin[s] - (a.q_begin[s + 1] - a.q_begin[s]);
}
// The block that holds cost u (below the total): the sequence by a lane each, then its blocks 64 at a time.
__device__ __forceinline__ Block find_block(const PromptArgs& a, int64_t u, int lane) {
  const int64_t end = lane < a.nseq ? a.cost[lane + 1] : INT64_MAX;
  const int s = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= u));
  const int R = seq_rows(a, s), base = seq_base(a, s), nb = (R + PROWS - 1) / PROWS;
  int64_t before = a.cost[s];
  for (int i = 0;; i += 64) {
    const int tiles = i + lane < nb ? block_tiles(block_at(i + lane, nb), R, a.g, base) : 0;
    const int c = i + lane < nb ? tiles + BLOCK_COST : 0;
    const int upto = wave_scan_i(c);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > u);
    if (past || i + 64 >= nb) {
      const int l = past ? __builtin_ctzll(past) : 0;
      return {s, block_at(i + l, nb), __builtin_amdgcn_readlane(tiles, l),
              before + __builtin_amdgcn_readlane(upto - c, l), i + l};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
}
// The block of rank x when all are in order of their tiles, most first: how many have at least n tiles is a
// sum over the sequences, a lane each, and the largest n that more than x have is found by halving. Its cost
// is counted from its own begin.
template <int ROWS>
__device__ __forceinline__ Block ranked_block(const PromptArgs& a, int x, int lane) {
  const int sl = min(lane, a.nseq - 1);
  const int R = lane < a.nseq ? seq_rows(a, sl) : 0, base = seq_base(a, sl), nb = (R + ROWS - 1) / ROWS;
  auto from = [&](int n) {  // first block of the lane's sequence with at least n tiles (of nb: none)
    const int64_t y = a.G * ((int64_t)TKEYS * (n - 1) - base);  // the row that has to be reached
    return n <= 0 || y <= 0 ? 0 : y > R - 1 ? nb : (int)(y / ROWS);
  };
  int lo = 0, hi = a.longest + 1;  // all have lo, none has hi
  int above = 0;                   // blocks with at least hi tiles
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, n = __builtin_amdgcn_readfirstlane(wave_sum_i(nb - from(mid)));
    if (n > x) {
      lo = mid;
    } else {
      hi = mid;
      above = n;
    }
  }
  const int n = from(lo + 1) - from(lo);
  const int upto = wave_scan_i(n);
  const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x - above));
  return {l, __builtin_amdgcn_readlane(from(lo), l) + x - above - __builtin_amdgcn_readlane(upto - n, l), lo, 0, 0};
}
// The tile of a block at which a cut at cost u (anywhere) lies: not within MIN_PART of its ends.
__device__ __forceinline__ int cut_tile(const Block& b, int64_t u) {
  const int64_t t = u - b.begin - BLOCK_COST;
  return t >= b.tiles ? b.tiles : t < MIN_PART ? 0 : t > b.tiles - MIN_PART ? b.tiles : (int)t;
}

template <int STAGES>  // tiles of K and of V in LDS
struct PromptSmem {
  alignas(256) uint16_t k[STAGES][TKEYS * D];
  alignas(256) uint16_t v[STAGES][TKEYS * D];
  uint32_t nonfinite[3][2];  // keys of tile t % 3, if masked, whose V holds an infinity or NaN
};

template <int PW>  // waves: 8, or 4 for small workgroups, two per CU
__global__ __launch_bounds__(64 * PW, 2) void prompt_attn_kernel(const PromptArgs a) {
  constexpr bool HALVES = PW == 8;
  constexpr int ROWS = 16 * NT * PW, STAGES = HALVES ? 3 : 2;
  constexpr int CP = 16 / PW;  // copies of a wave per tile, K and V each
  static_assert(ROWS == (HALVES ? PROWS : SROWS), "block sizes");
  __shared__ PromptSmem<STAGES> sm;
  const int share = blockIdx.x / a.Hkv, hk = blockIdx.x - share * a.Hkv;
  const int blocks = gridDim.x / a.Hkv;
  const int rank = (uint32_t)share < (uint32_t)a.paired ? share : blocks - 1 - (share - a.paired);
  Block b = HALVES && a.share ? find_block(a, a.share * share, threadIdx.x & 63)
                              : ranked_block<ROWS>(a, rank, threadIdx.x & 63);
  const int64_t u0 = a.share * share;  // 0 for a whole block
  const int64_t u1 = a.share ? min(u0 + a.share, a.cost[a.nseq]) : b.tiles + BLOCK_COST;
  for (bool more = true; more;) {
    // re-read per block, so that no lane value made of it is kept across blocks
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool grp_a = HALVES && wv < PW / 2;
    const int lc = lane & 15, lq4 = lane >> 4;
    const int s = b.seq, blk = b.blk;
    const int q0 = a.q_begin[s], lq = a.q_begin[s + 1] - q0;
    const int k0 = a.k_begin[s], lk = a.k_begin[s + 1] - k0;
    const int R = lq * a.G, base = lk - lq;
    const int tiles = b.tiles;
    const int t0 = HALVES ? cut_tile(b, u0) : 0, t1 = HALVES ? cut_tile(b, u1) : tiles;
    // a block without a tile (rows without keys) belongs to the share that its begin lies in
    const bool mine = t0 < t1 || (tiles == 0 && b.begin >= u0 && b.begin < u1);
    if (mine) {
      const float scale = abs_scale(a.sl2);
      // tiles from here on are masked for some row of the block (or end behind the last key)
      const int low = base + (int)fdiv_u((uint32_t)(blk * ROWS), a.g);
      const int t_masked = low < 0 ? 0 : (low + 1) / TKEYS;

      // ---- copies: wave wv brings 4 CP keys from 4 CP wv on of every tile, K and V 1 KB (4 keys) at a
      // time; a lane's 16 bytes land at lane x 16, so the swizzle is in the chunk it reads. Keys past the
      // last one read it again.
      const int krow = 4 * CP * wv + (lane >> 4);  // and + 4, ..
      const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.k + (int64_t)k0 * a.k_tok + hk * a.k_head);
      const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.v + (int64_t)k0 * a.v_tok + hk * a.v_head);
      const uint32_t k_at = lds_u32(sm.k) + 1024u * CP * wv, v_at = lds_u32(sm.v) + 1024u * CP * wv;
      // A tile's base is scalar, a lane's offset in it fixed but in the tile that ends behind the last key.
      auto copy = [&](const uint8_t* from, int64_t tok, int t, uint32_t to, const uint32_t (&at)[CP],
                      bool is_v) {
        const int tt = min(t, t1 - 1);
        const uint8_t* sb = from + 2 * TKEYS * tok * tt;
        const uint32_t m = __builtin_amdgcn_readfirstlane(to + (uint32_t)(t % STAGES) * (TKEYS * D * 2));
        uint32_t o[CP];
#pragma unroll
        for (int i = 0; i < CP; ++i) o[i] = at[i];
        if (TKEYS * tt + TKEYS > lk) {  // uniform
#pragma unroll
          for (int i = 0; i < CP; ++i) {
            const int r = krow + 4 * i;
            o[i] = 2 * (uint32_t)tok * (uint32_t)min(r, lk - 1 - TKEYS * tt) +
                   16 * (lc ^ (is_v ? 2 * (r & 7) : r & 15));
          }
        }
#pragma unroll
        for (int i = 0; i < CP; ++i)
          asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                       :: "v"(o[i]), "s"(sb), "s"(m + 1024u * i) : "memory");
      };
      uint32_t ko[CP], vo[CP];
#pragma unroll
      for (int i = 0; i < CP; ++i) {
        const int r = krow + 4 * i;
        ko[i] = 2 * (uint32_t)a.k_tok * r + 16 * (lc ^ (r & 15));
        vo[i] = 2 * (uint32_t)a.v_tok * r + 16 * (lc ^ (2 * (r & 7)));
      }
      auto copy_k = [&](int t) { copy(kbase, a.k_tok, t, k_at, ko, false); };
      auto copy_v = [&](int t) { copy(vbase, a.v_tok, t, v_at, vo, true); };
      // The wave's own V rows of tile t, in LDS: infinities and NaN become 0 and their keys are noted.
      auto scan_v = [&](int t) {
#pragma unroll
        for (int i = 0; i < CP; ++i) {
          uint4* at = reinterpret_cast<uint4*>(&sm.v[t % STAGES][(4 * CP * wv + 4 * i) * D + 8 * lane]);
          const uint4 u = *at;
          uint32_t m = bf16x2_absmax_bits(bf16x2_absmax_bits(0, u.x), u.y);
          m = bf16x2_absmax_bits(bf16x2_absmax_bits(m, u.z), u.w);
          const int key = krow + 4 * i;
          if ((m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u) {
            *at = make_uint4(finite_bf2(u.x), finite_bf2(u.y), finite_bf2(u.z), finite_bf2(u.w));
            atomicOr(&sm.nonfinite[t % 3][key >> 5], 1u << (key & 31));
          }
        }
      };

      lds_barrier();  // the other half is done with the block before
      if (t0 < t1) {  // out before the rows of q are asked for
        copy_k(t0);
        copy_k(t0 + 1);
        copy_v(t0);
      }

      // ---- the wave's rows
      const int f0 = blk * ROWS + 16 * NT * wv;
      TileRows<NT> st;
      int lim[NT];  // last key of the lane's row, -1: none
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int f = f0 + 16 * nt + lc;
        const int i = (int)fdiv_u((uint32_t)min(f, R - 1), a.g);
        const int head = min(f, R - 1) - i * a.G;
        lim[nt] = f < R ? base + i : -1;
        const uint16_t* qr = a.q + (int64_t)(q0 + i) * a.q_tok + (hk * a.G + head) * a.q_head + 8 * lq4;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          st.q[nt][kk] = u4_as_bf8(signed_q(*reinterpret_cast<const uint4*>(qr + 32 * kk), a.sl2));
      }
      st.clear();
      const int lim_lo = f0 < R ? base + (int)fdiv_u((uint32_t)f0, a.g) : -1;

      f4_t c[NT][4];
      bf16x8_t p[NT][2];
      // V(t) of the wave's copies has landed (with 8 waves 4 newer ones are out)
      auto landed = [&](int t) {
        if constexpr (HALVES)
          asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // and K(t + 1)
        if (t >= t_masked) scan_v(t);  // workgroup-uniform
      };
      if (t0 < t1) {
        if (tid < 6) sm.nonfinite[tid >> 1][tid & 1] = 0;
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * CP) : "memory");  // K(t0)
        lds_barrier();
        if (HALVES && !grp_a) {  // half a tile behind
          copy_k(t0 + 2);
          copy_v(t0 + 1);
          asm volatile("s_waitcnt vmcnt(6)" ::: "memory");  // K(t0 + 1)
          lds_barrier();
        }
        tile_scores<NT>(sm.k[t0 % STAGES], st, lane, c);
        for (int t = t0; t < t1; ++t) {
          if (grp_a)
            asm volatile("s_waitcnt vmcnt(2)" ::: "memory");  // K(t + 1)
          else
            landed(t);
          lds_barrier();
          // vector phase
          __builtin_amdgcn_s_setprio(HALVES);
          copy_k(t + (grp_a || !HALVES ? 2 : 3));
          copy_v(t + (grp_a || !HALVES ? 1 : 2));
          if (TKEYS * t + TKEYS - 1 > lim_lo) {  // wave-uniform: masked for some row
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  c[nt][mt][r] = TKEYS * t + 16 * mt + 4 * lq4 + r <= lim[nt] ? c[nt][mt][r] : -INFINITY;
          }
          Ahead ahead;
          if constexpr (HALVES) {
            tile_softmax<NT>(c, st, scale, p);
            tile_ahead(sm.k[(t + 1) % STAGES], lane, ahead);
            if (grp_a)
              landed(t);
            else
              asm volatile("s_waitcnt vmcnt(6)" ::: "memory");  // K(t + 2)
            lds_barrier();
          } else {
            tile_ahead(sm.k[(t + 1) % STAGES], lane, ahead);
            tile_softmax<NT>(c, st, scale, p);
          }
          // matrix phase: Q.K^T of tile t + 1 (behind the last one, of a copy nobody reads), P.V of tile t
          __builtin_amdgcn_s_setprio(!HALVES);
          tile_matrix<NT>(sm.k[(t + 1) % STAGES], sm.v[t % STAGES], st, lane, c, p, ahead);
          if (t >= t_masked) {
            uint64_t nf = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.nonfinite[t % 3][0]) |
                          (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.nonfinite[t % 3][1]) << 32;
            for (; nf; nf &= nf - 1) {  // rare
              const int key = __builtin_ctzll(nf), at = TKEYS * t + key;
              if (at < lk) tile_nonfinite<NT>(vbase + 2 * a.v_tok * at, key, at, st, lane, p, lim);
            }
          }
          // last read before the barrier ahead of this phase: what tile t + 2 will note
          if (tid < 2) sm.nonfinite[(t + 2) % 3][tid] = 0;
        }
        if (HALVES && grp_a) lds_barrier();
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the last tile
      }

      // ---- rows out: dims 16 w + 4 lq4 + r
      const bool part = HALVES && t1 - t0 < tiles;
      const int64_t prow = ((int64_t)(2 * share + (t0 == 0)) * a.Hkv + hk) * ROWS;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int f = f0 + 16 * nt + lc;
        if (f >= R) continue;
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
        const float inv = st.l[nt][0] == 0.0f ? 0.0f : 1.0f / st.l[nt][0];
#pragma unroll
        for (int w = 0; w < 8; ++w)
          *reinterpret_cast<uint2*>(o + 16 * w) =
              make_uint2(pack_bf2(st.o[nt][w][0] * inv, st.o[nt][w][1] * inv),
                         pack_bf2(st.o[nt][w][2] * inv, st.o[nt][w][3] * inv));
      }
    }
    // the next block
    const int64_t next = b.begin + b.tiles + BLOCK_COST;
    more = HALVES && next < u1;
    if (more) {
      int ns = b.seq, place = b.place + 1;
      if (place * PROWS >= R) {
        place = 0;
        do ++ns;
        while (a.cost[ns + 1] == a.cost[ns]);  // sequences without rows cost nothing
      }
      const int nr = seq_rows(a, ns), nblk = block_at(place, (nr + PROWS - 1) / PROWS);
      b = Block{ns, nblk, block_tiles(nblk, nr, a.g, seq_base(a, ns)), next, place};
    }
  }
}

constexpr int MERGE_ROWS = 32;  // of a workgroup
// The parts of a block into output rows, by the workgroups of its first cut: share j's end. 32 lanes x 4
// dims per row.
__global__ __launch_bounds__(256) void prompt_merge_kernel(const PromptArgs a) {
  const int j = blockIdx.x / a.Hkv, hk = blockIdx.x - j * a.Hkv;
  const int64_t u = a.share * (j + 1);
  const Block b = find_block(a, u, threadIdx.x & 63);
  const int t = cut_tile(b, u);
  if (t == 0 || t == b.tiles || cut_tile(b, u - a.share) != 0) return;  // no cut, or not its first
  const int R = seq_rows(a, b.seq);
  const int d = 4 * (threadIdx.x & 31);
  int n = 1;  // parts
  while (cut_tile(b, u + n * a.share - a.share) < b.tiles) ++n;
  constexpr int RT = MERGE_ROWS / 8;  // rows per thread: all their loads of a part together
  const int row0 = MERGE_ROWS * blockIdx.y + (threadIdx.x >> 5);
  if (b.blk * PROWS + MERGE_ROWS * (int)blockIdx.y >= R) return;
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
    const int64_t part = ((int64_t)(2 * (j + k) + (k == 0)) * a.Hkv + hk) * PROWS;
    float2 ml[RT];
    f4_t o[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {  // rows past the sequence's are read, of the workspace, and not used
      ml[i] = a.part_ml[part + row0 + 8 * i];
      o[i] = *reinterpret_cast<const f4_t*>(a.part_acc + (part + row0 + 8 * i) * D + d);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const float mn = max_ieee(M[i], ml[i].x);
      const float mr = mn == -INFINITY ? 0.0f : mn;
      const float e0 = exp2_nonpos(M[i] - mr), e1 = exp2_nonpos(ml[i].x - mr);
      acc[i] = acc[i] * e0 + o[i] * e1;
      den[i] = den[i] * e0 + ml[i].y * e1;
      M[i] = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int f = b.blk * PROWS + row0 + 8 * i;
    if (f >= R) return;
    const float inv = den[i] == 0.0f ? 0.0f : 1.0f / den[i];
    const int p = (int)fdiv_u((uint32_t)f, a.g), head = f - p * a.G;
    *reinterpret_cast<uint2*>(a.out + ((int64_t)(a.q_begin[b.seq] + p) * a.Hkv * a.G + hk * a.G + head) * D + d) =
        make_uint2(pack_bf2(acc[i][0] * inv, acc[i][1] * inv), pack_bf2(acc[i][2] * inv, acc[i][3] * inv));
  }
}

// How the work is dealt out, with the cost of the blocks of every sequence. Three ways (us at 32/8 heads but
// where said; on gfx950, 256 CUs):
//
//  - whole blocks of 256 rows, longest first, where there are WHOLE_ROUNDS and more for each CU and they are
//    long: the last round evens itself out, nothing is merged, and the workgroups of a head walk its keys
//    together, which the L2 likes (16,384 rows: 1,840, in shares 2,040, small 1,905).
//  - small workgroups, whole blocks of 128 rows, two per CU: nothing is merged either, a block's start and end
//    lie beside the other workgroup's tiles, and the rows that a short sequence leaves unused in its last block
//    are fewer (128 rows: 12.9, in shares 17.0; 2,048: 51.4 and 59.0; 5,000: 200 and 214; 64 prompts of 400
//    rows: 198, as whole blocks of 256 rows 241).
//  - shares of equal cost, one per CU, where the blocks are few and long, so that whole ones would leave CUs
//    idle (512 rows on 7,681: 82, small 169).
//
// Small workgroups are taken where their time comes out lower, in units of 0.03 us: 40 per tile of the longest
// block (alone on its CU), 31 per tile of all and 31 per tile that a CU with fewer blocks has to wait (counted
// as the shortest; 40 where the last block is alone), against 60 per tile of a share and 240 for parts and
// merge. Over 170 shapes of 1 to 64 sequences and 8 to 64 heads the choice was the faster by up to 45%, and
// the slower by more than 2% in one (8 prompts of 1,000 rows: 95.4, in shares 92.6).
constexpr int64_t WHOLE_ROUNDS = 6;
constexpr int64_t WHOLE_TILES = 48;  // per block of 128 rows
struct PromptPlan {
  int64_t cost[LQ_MAX_SEQS + 1], share, shares;  // share 0: whole blocks, `shares` of them
  int longest, paired;
  bool small;  // whole blocks of SROWS rows
};
PromptPlan prompt_plan(const int32_t* q_lens, const int32_t* k_lens, int64_t nseq, int64_t Hkv, int64_t G,
                       int cus) {
  PromptPlan p{};
  const FastDiv g = make_fastdiv((uint32_t)G);
  int64_t blocks = 0, sblocks = 0, stiles = 0, shortest = INT64_MAX;
  for (int s = 0; s < LQ_MAX_SEQS; ++s) {
    int64_t c = 0;
    const int R = s < nseq ? (int)(q_lens[s] * G) : 0;
    for (int b = 0; (int64_t)b * PROWS < R; ++b) {
      const int t = block_tiles(b, R, g, k_lens[s] - q_lens[s]);
      p.longest = std::max(p.longest, t);
      c += t + BLOCK_COST;
      ++blocks;
      const int ts = block_tiles<SROWS>(2 * b, R, g, k_lens[s] - q_lens[s]);
      const bool two = b * PROWS + SROWS < R;
      sblocks += 1 + two;
      stiles += ts + (two ? t : 0);
      shortest = std::min<int64_t>(shortest, ts);
    }
    p.cost[s + 1] = p.cost[s] + c;
  }
  p.paired = -1;
  if (blocks * Hkv >= WHOLE_ROUNDS * cus && stiles >= WHOLE_TILES * sblocks) {
    p.shares = blocks;
    return p;
  }
  const int64_t total = p.cost[nseq], per_head = std::max<int64_t>(1, cus / Hkv);
  p.share = std::max<int64_t>(BLOCK_COST + MIN_PART, (total + per_head - 1) / per_head);
  p.shares = (total + p.share - 1) / p.share;
  const int64_t n = sblocks * Hkv, most = (n + cus - 1) / cus;  // small blocks, and of a CU
  const int64_t idle = 31 * (most * cus - n) * shortest / cus + most % 2 * 9 * shortest;
  if (std::max<int64_t>(40 * p.longest, 31 * stiles * Hkv / cus + idle) <= 60 * p.share + 240) {
    p.small = true;
    p.share = 0;
    p.shares = sblocks;
    if (n <= 2 * cus) p.paired = (int)per_head;
  }
  return p;
}

int64_t prompt_bytes(const PromptPlan& p, int64_t Hkv) {
  return p.share && p.shares > 1 ? 2 * p.shares * Hkv * PROWS * (int64_t)(D * sizeof(float) + sizeof(float2)) : 0;
}

int check_prompt(int64_t Hq, int64_t Hkv, int64_t D, const int32_t* q_lens, const int32_t* k_lens,
                 int64_t nseq) {
  LQ_CHECK_ARG(D == 128, "head_dim must be 128 (got %lld)", (long long)D);
  LQ_CHECK_ARG(Hkv >= 1 && Hkv <= 1024 && Hq >= Hkv && Hq % Hkv == 0 && Hq / Hkv <= 64,
               "Hq=%lld must be 1 to 64 times Hkv=%lld", (long long)Hq, (long long)Hkv);
  LQ_CHECK_ARG(nseq >= 1 && nseq <= LQ_MAX_SEQS, "%lld sequences are not in [1, %d]", (long long)nseq,
               LQ_MAX_SEQS);
  LQ_CHECK_ARG(q_lens && k_lens, "null pointer");
  int64_t tq = 0, tk = 0;
  for (int s = 0; s < nseq; ++s) {
    LQ_CHECK_ARG(q_lens[s] >= 0 && k_lens[s] >= 0 && q_lens[s] <= (1 << 24) && k_lens[s] <= (1 << 24),
                 "sequence %d has %d rows and %d keys (at most 2^24)", s, (int)q_lens[s], (int)k_lens[s]);
    LQ_CHECK_ARG((int64_t)q_lens[s] * (Hq / Hkv) < (1 << 30), "%d rows of one sequence are too many",
                 (int)q_lens[s]);
    tq += q_lens[s];
    tk += k_lens[s];
  }
  LQ_CHECK_ARG(tq < (1 << 30) && tk < (1 << 30), "too many rows");
  return LQ_OK;
}

}  // namespace
}  // namespace lq

extern "C" int64_t lq_prompt_workspace_bytes(const int32_t* q_lens_host, const int32_t* k_lens_host,
                                             int64_t nseq, int64_t Hq, int64_t Hkv) {
  using namespace lq;
  clear_error();
  if (check_prompt(Hq, Hkv, 128, q_lens_host, k_lens_host, nseq)) return -1;
  return prompt_bytes(prompt_plan(q_lens_host, k_lens_host, nseq, Hkv, Hq / Hkv, device_cu_count()), Hkv);
}

extern "C" int lq_prompt_attn(const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t q_tok,
                              int64_t q_head, int64_t k_tok, int64_t k_head, int64_t v_tok,
                              int64_t v_head, const int32_t* q_lens_host, const int32_t* k_lens_host,
                              int64_t nseq, int64_t Hq, int64_t Hkv, int64_t D, float scale,
                              uint16_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lq;
  clear_error();
  if (const int st = check_prompt(Hq, Hkv, D, q_lens_host, k_lens_host, nseq)) return st;
  int64_t tq = 0, tk = 0;
  for (int s = 0; s < nseq; ++s) {
    tq += q_lens_host[s];
    tk += k_lens_host[s];
  }
  if (tq == 0) return LQ_OK;
  LQ_CHECK_ARG(q && out && (tk == 0 || (k && v)), "null pointer");
  LQ_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 &&
                   ((q_tok | q_head | k_tok | k_head | v_tok | v_head) & 7) == 0,
               "rows must be 16-byte aligned (strides a multiple of 8)");
  LQ_CHECK_ARG(k_tok >= 0 && v_tok >= 0 && k_tok < (1 << 24) && v_tok < (1 << 24),
               "rows of k or v 2^24 values apart or more");
  LQ_CHECK_ARG(std::isfinite(scale), "the softmax scale is not finite");
  const PromptPlan plan = prompt_plan(q_lens_host, k_lens_host, nseq, Hkv, Hq / Hkv, device_cu_count());
  const int64_t need = prompt_bytes(plan, Hkv);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    set_error("workspace of %lld bytes is smaller than the %lld needed", (long long)workspace_bytes,
              (long long)need);
    return LQ_EWORKSPACE;
  }
  LQ_CHECK_ARG(plan.shares * Hkv < (1 << 23), "too many workgroups");
  LQ_CHECK_ARG(need == 0 || ((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  PromptArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.k_tok = k_tok;
  a.k_head = k_head;
  a.v_tok = v_tok;
  a.v_head = v_head;
  a.part_acc = (float*)workspace;
  a.part_ml = need ? (float2*)(a.part_acc + 2 * plan.shares * Hkv * PROWS * lq::D) : nullptr;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.nseq = (int)nseq;
  a.g = make_fastdiv((uint32_t)a.G);
  a.sl2 = scale * 1.4426950408889634f;
  a.share = plan.share;
  a.longest = plan.longest;
  a.paired = plan.paired;
  a.q_begin[0] = a.k_begin[0] = 0;
  for (int s = 0; s < LQ_MAX_SEQS; ++s) {
    a.q_begin[s + 1] = a.q_begin[s] + (s < nseq ? q_lens_host[s] : 0);
    a.k_begin[s + 1] = a.k_begin[s] + (s < nseq ? k_lens_host[s] : 0);
    a.cost[s] = plan.cost[s];
  }
  a.cost[LQ_MAX_SEQS] = plan.cost[LQ_MAX_SEQS];
  const dim3 grid((unsigned)(plan.shares * Hkv));
  if (plan.small)
    prompt_attn_kernel<4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
  else
    prompt_attn_kernel<8><<<grid, dim3(512), 0, (hipStream_t)stream>>>(a);
  LQ_CHECK_LAUNCH("prompt_attn_kernel");
  if (need > 0) {
    prompt_merge_kernel<<<dim3((unsigned)((plan.shares - 1) * Hkv), PROWS / MERGE_ROWS), dim3(256), 0,
                          (hipStream_t)stream>>>(a);
    LQ_CHECK_LAUNCH("prompt_merge_kernel");
  }
  return LQ_OK;
}
