// Causal attention of packed prompts: the rows of up to 64 sequences of different lengths, one behind the
// other, bf16 q [rows, Hq, 128] over k and v [keys, Hkv, 128] with any token and head strides, no padding
// and no score matrix. Sequence s has q_lens[s] rows and k_lens[s] keys, aligned at their ends: row i sees
// keys 0 .. k_lens[s] - q_lens[s] + i, so a prompt has as many of both and a chunk of one more keys. Rows
// without a key are 0.
//
// Work: a workgroup of 8 waves takes 256 query rows of a KV head, numbered position-major (row f is
// position f / G of query head f % G), so that any grouping fills the matrix cores and a block's rows see
// nearly the same keys; a wave has 32 of them. It walks the 64-key tiles up to its last row's bound, each
// copied into LDS once for all waves (three buffers of K and of V, copies two tiles ahead) and run through
// attn_tile.h. A SIMD holds one wave of each half of the workgroup, and the halves run one phase apart, so
// that one's matrix phase (P.V of a tile, Q.K^T of the next) lies beside the other's vector phase (softmax,
// copies), with a barrier after each:
//
//   slot    group A                   group B
//   2t      Q.K^T(t), P.V(t-1)        softmax(t-1), copies K(t+2) V(t+1)
//   2t+1    softmax(t), copies        Q.K^T(t), P.V(t-1)
//
// Where whole blocks would leave CUs idle
// (short or few prompts behind long pasts) a block's tiles are cut into parts whose partial rows a second
// launch merges.
//
// The blocks of a launch come as a list in the kernel's arguments, made on the host from the lengths,
// longest first; the KV head is the fastest index, so that neighbouring workgroups (XCDs) hold different
// heads and each XCD's L2 the K and V of few.
//
// Keys that a row does not see reach it in no way: masked scores are -infinity, and an infinity or NaN in
// V of a tile that is masked for some row of the block goes only to the rows that see its key (0 times it
// would be NaN): such tiles are rare and take the two-pass form.
#include <algorithm>
#include <vector>

#include "attn_tile.h"

namespace lq {
namespace {

using namespace attn;

constexpr int PW = 8;          // waves per workgroup
constexpr int NT = 2;          // 16-row tiles per wave
constexpr int PROWS = 16 * NT * PW;
constexpr int LIST = 768;      // blocks of one launch: kernel arguments are limited to 4 KB
constexpr int MAX_PARTS = 63;

// A block of a sequence (or part j of n of its tiles): seq | block << 6 | j << 20 | n << 26.
struct Entry {
  uint32_t x;
  __host__ __device__ int seq() const { return x & 63; }
  __host__ __device__ int block() const { return (x >> 6) & 16383; }
  __host__ __device__ int part() const { return (x >> 20) & 63; }
  __host__ __device__ int parts() const { return x >> 26; }
};

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;           // [rows, Hq, 128]
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  float* part_acc;         // [entries of the call x Hkv][256][128], of entries that are parts
  float2* part_ml;
  int Hkv, G;
  FastDiv g;
  float sl2;
  int q_begin[LQ_MAX_SEQS + 1], k_begin[LQ_MAX_SEQS + 1];
  Entry list[LIST];
};

// 64-key tiles that block blk of a sequence of R rows needs; base: row i sees keys <= base + i.
__host__ __device__ __forceinline__ int block_tiles(int blk, int R, FastDiv g, int base) {
  const int last = base + (int)fdiv_u((uint32_t)min(blk * PROWS + PROWS - 1, R - 1), g);
  return last < 0 ? 0 : last / TKEYS + 1;
}

constexpr int STAGES = 3;  // tiles of K and of V in LDS
struct PromptSmem {
  alignas(256) uint16_t k[STAGES][TKEYS * D];
  alignas(256) uint16_t v[STAGES][TKEYS * D];
  uint32_t nonfinite[STAGES][2];  // keys of a masked tile whose V holds an infinity or NaN
};

__global__ __launch_bounds__(64 * PW, 2) void prompt_attn_kernel(const PromptArgs a, int first) {
  __shared__ PromptSmem sm;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool grp_a = wv < PW / 2;
  const int lc = lane & 15, lq4 = lane >> 4;
  const int x = blockIdx.x / a.Hkv, hk = blockIdx.x - x * a.Hkv;
  const Entry en = a.list[x];
  if (en.parts() == 0) return;  // fills up a launch
  const int s = en.seq(), blk = en.block();
  const int q0 = a.q_begin[s], lq = a.q_begin[s + 1] - q0;
  const int k0 = a.k_begin[s], lk = a.k_begin[s + 1] - k0;
  const int R = lq * a.G, base = lk - lq;
  const int tiles = block_tiles(blk, R, a.g, base);
  const int t0 = (int)((int64_t)tiles * en.part() / en.parts());
  const int t1 = (int)((int64_t)tiles * (en.part() + 1) / en.parts());
  const float scale = abs_scale(a.sl2);
  // tiles from here on are masked for some row of the block (or end behind the last key)
  const int low = base + (int)fdiv_u((uint32_t)(blk * PROWS), a.g);
  const int t_masked = low < 0 ? 0 : (low + 1) / TKEYS;

  // ---- copies: wave wv brings keys 8 wv .. 8 wv + 7 of every tile, K and V 1 KB (4 keys) at a time; a
  // lane's 16 bytes land at lane x 16, so the swizzle is in the chunk it reads. Keys past the last one
  // read it again.
  const int krow = 8 * wv + (lane >> 4);  // and + 4
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.k + (int64_t)k0 * a.k_tok + hk * a.k_head);
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.v + (int64_t)k0 * a.v_tok + hk * a.v_head);
  const uint32_t k_at = lds_u32(sm.k) + 2048u * wv, v_at = lds_u32(sm.v) + 2048u * wv;
  // A tile's base is scalar, a lane's offset in it fixed but in the tile that ends behind the last key.
  auto copy = [&](const uint8_t* from, int64_t tok, int t, uint32_t to, const uint32_t (&at)[2], bool is_v) {
    const int tt = min(t, t1 - 1);
    const uint8_t* sb = from + 2 * TKEYS * tok * tt;
    const uint32_t m = __builtin_amdgcn_readfirstlane(to + (uint32_t)(t % STAGES) * (TKEYS * D * 2));
    uint32_t o[2] = {at[0], at[1]};
    if (TKEYS * tt + TKEYS > lk) {  // uniform
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = krow + 4 * i;
        o[i] = 2 * (uint32_t)tok * (uint32_t)min(r, lk - 1 - TKEYS * tt) + 16 * (lc ^ (is_v ? 2 * (r & 7) : r & 15));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                   :: "v"(o[i]), "s"(sb), "s"(m + 1024u * i) : "memory");
  };
  uint32_t ko[2], vo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = krow + 4 * i;
    ko[i] = 2 * (uint32_t)a.k_tok * r + 16 * (lc ^ (r & 15));
    vo[i] = 2 * (uint32_t)a.v_tok * r + 16 * (lc ^ (2 * (r & 7)));
  }
  auto copy_k = [&](int t) { copy(kbase, a.k_tok, t, k_at, ko, false); };
  auto copy_v = [&](int t) { copy(vbase, a.v_tok, t, v_at, vo, true); };
  // The wave's own V rows of tile t, in LDS: infinities and NaN become 0 and their keys are noted.
  auto scan_v = [&](int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint4* at = reinterpret_cast<uint4*>(&sm.v[t % STAGES][(8 * wv + 4 * i) * D + 8 * lane]);
      const uint4 u = *at;
      uint32_t m = bf16x2_absmax_bits(bf16x2_absmax_bits(0, u.x), u.y);
      m = bf16x2_absmax_bits(bf16x2_absmax_bits(m, u.z), u.w);
      const int key = krow + 4 * i;
      if ((m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u) {
        *at = make_uint4(finite_bf2(u.x), finite_bf2(u.y), finite_bf2(u.z), finite_bf2(u.w));
        atomicOr(&sm.nonfinite[t % STAGES][key >> 5], 1u << (key & 31));
      }
    }
  };

  // ---- the wave's rows
  const int f0 = blk * PROWS + 16 * NT * wv;
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
  // V(t) of the wave's copies has landed (4 newer ones are out)
  auto landed = [&](int t) {
    asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    if (t >= t_masked) scan_v(t);  // workgroup-uniform
  };
  if (t0 < t1) {
    if (tid < 2 * STAGES) sm.nonfinite[tid >> 1][tid & 1] = 0;
    copy_k(t0);
    copy_k(t0 + 1);
    copy_v(t0);
    asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    lds_barrier();
    if (!grp_a) {  // half a tile behind
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
      __builtin_amdgcn_s_setprio(1);
      copy_k(t + (grp_a ? 2 : 3));
      copy_v(t + (grp_a ? 1 : 2));
      if (TKEYS * t + TKEYS - 1 > lim_lo) {  // wave-uniform: masked for some row
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              c[nt][mt][r] = TKEYS * t + 16 * mt + 4 * lq4 + r <= lim[nt] ? c[nt][mt][r] : -INFINITY;
      }
      tile_softmax<NT>(c, st, scale, p);
      Ahead ahead;
      tile_ahead(sm.k[(t + 1) % STAGES], lane, ahead);
      if (grp_a)
        landed(t);
      else
        asm volatile("s_waitcnt vmcnt(6)" ::: "memory");  // K(t + 2)
      lds_barrier();
      // matrix phase: Q.K^T of tile t + 1 (behind the last one, of a copy nobody reads), P.V of tile t
      __builtin_amdgcn_s_setprio(0);
      tile_matrix<NT>(sm.k[(t + 1) % STAGES], sm.v[t % STAGES], st, lane, c, p, ahead);
      if (t >= t_masked) {
        uint64_t nf = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.nonfinite[t % STAGES][0]) |
                      (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sm.nonfinite[t % STAGES][1]) << 32;
        for (; nf; nf &= nf - 1) {  // rare
          const int key = __builtin_ctzll(nf), at = TKEYS * t + key;
          if (at < lk) tile_nonfinite<NT>(vbase + 2 * a.v_tok * at, key, at, st, lane, p, lim);
        }
      }
      // read by the other half for the last time a slot ago: group A clears what tile t + 2 will note
      if (tid < 2) sm.nonfinite[(t + 2) % STAGES][tid] = 0;
    }
    if (grp_a) lds_barrier();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the last tile
  }

  // ---- rows out: dims 16 w + 4 lq4 + r
  const int64_t prow = ((int64_t)(first + x) * a.Hkv + hk) * PROWS;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int f = f0 + 16 * nt + lc;
    if (f >= R) continue;
    if (en.parts() > 1) {
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

// The parts of a block (consecutive entries) into output rows: 32 lanes x 4 dims per row, 8 rows per
// workgroup.
__global__ __launch_bounds__(256) void prompt_merge_kernel(const PromptArgs a, int first) {
  const int x = blockIdx.x / a.Hkv, hk = blockIdx.x - x * a.Hkv;
  const Entry en = a.list[x];
  if (en.parts() < 2 || en.part() != 0) return;
  const int s = en.seq();
  const int q0 = a.q_begin[s], R = (a.q_begin[s + 1] - q0) * a.G;
  const int wrow = 8 * blockIdx.y + (threadIdx.x >> 5), d = 4 * (threadIdx.x & 31);
  const int f = en.block() * PROWS + wrow;
  if (f >= R) return;
  float M = -INFINITY, den = 0.0f;
  f4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < en.parts(); ++j) {
    const int64_t pr = ((int64_t)(first + x + j) * a.Hkv + hk) * PROWS + wrow;
    const float2 ml = a.part_ml[pr];
    const f4_t o = *reinterpret_cast<const f4_t*>(a.part_acc + pr * D + d);
    const float mn = max_ieee(M, ml.x);
    const float mr = mn == -INFINITY ? 0.0f : mn;
    const float e0 = M == -INFINITY ? 0.0f : exp2_nonpos(M - mr);
    const float e1 = ml.x == -INFINITY ? 0.0f : exp2_nonpos(ml.x - mr);
    acc = acc * e0 + o * e1;
    den = den * e0 + ml.y * e1;
    M = mn;
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  const int i = (int)fdiv_u((uint32_t)f, a.g), head = f - i * a.G;
  *reinterpret_cast<uint2*>(a.out + ((int64_t)(q0 + i) * a.Hkv * a.G + hk * a.G + head) * D + d) =
      make_uint2(pack_bf2(acc[0] * inv, acc[1] * inv), pack_bf2(acc[2] * inv, acc[3] * inv));
}

struct PromptPlan {
  std::vector<Entry> list;
  bool split = false;
};

// The blocks of the call, longest first, cut into parts where whole blocks would not fill the CUs.
// Returns an LQ_ status.
int prompt_plan(const int32_t* q_lens, const int32_t* k_lens, int64_t nseq, int64_t Hkv, int64_t G,
                int cus, PromptPlan* plan) {
  struct Block {
    int tiles, seq, blk;
  };
  const FastDiv g = make_fastdiv((uint32_t)G);
  std::vector<Block> blocks;
  int64_t total = 0;
  int longest = 0;
  for (int s = 0; s < nseq; ++s) {
    const int64_t R = (int64_t)q_lens[s] * G;
    LQ_CHECK_ARG((R + PROWS - 1) / PROWS <= 16384, "%d query rows of one sequence are too many",
                 (int)q_lens[s]);
    for (int b = 0; b * PROWS < R; ++b) {
      const int t = block_tiles(b, (int)R, g, k_lens[s] - q_lens[s]);
      blocks.push_back({t, s, b});
      total += t;
      longest = std::max(longest, t);
    }
  }
  // a CU's equal share of the tiles, as the size of a part
  const int64_t share = std::max<int64_t>(4, (total * Hkv + cus - 1) / cus);
  plan->split = longest > share + share / 4;
  auto parts = [&](int t) {
    return plan->split ? (int)std::min<int64_t>(MAX_PARTS, std::max<int64_t>(1, (t + share - 1) / share))
                       : 1;
  };
  std::stable_sort(blocks.begin(), blocks.end(), [&](const Block& x, const Block& y) {
    return x.tiles * parts(y.tiles) > y.tiles * parts(x.tiles);
  });
  for (const Block& b : blocks) {
    const int n = parts(b.tiles);
    // a block's parts stay in one launch
    if ((int)(plan->list.size() % LIST) + n > LIST)
      while (plan->list.size() % LIST) plan->list.push_back({0u});
    for (int j = 0; j < n; ++j)
      plan->list.push_back({(uint32_t)b.seq | (uint32_t)b.blk << 6 | (uint32_t)j << 20 | (uint32_t)n << 26});
  }
  return LQ_OK;
}

int64_t prompt_bytes(const PromptPlan& p, int64_t Hkv) {
  return p.split ? (int64_t)p.list.size() * Hkv * PROWS * (int64_t)(D * sizeof(float) + sizeof(float2)) : 0;
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
  try {
    PromptPlan plan;
    if (prompt_plan(q_lens_host, k_lens_host, nseq, Hkv, Hq / Hkv, device_cu_count(), &plan)) return -1;
    return prompt_bytes(plan, Hkv);
  } catch (...) {
    set_error("no host memory for the plan");
    return -1;
  }
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
  PromptArgs a;
  std::vector<Entry> list;
  try {
    PromptPlan plan;
    if (const int st = prompt_plan(q_lens_host, k_lens_host, nseq, Hkv, Hq / Hkv, device_cu_count(), &plan))
      return st;
    const int64_t need = prompt_bytes(plan, Hkv);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
      set_error("workspace of %lld bytes is smaller than the %lld needed", (long long)workspace_bytes,
                (long long)need);
      return LQ_EWORKSPACE;
    }
    LQ_CHECK_ARG(need == 0 || ((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
    a.part_acc = (float*)workspace;
    a.part_ml = need ? (float2*)(a.part_acc + (int64_t)plan.list.size() * Hkv * PROWS * 128) : nullptr;
    list.swap(plan.list);
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
    a.Hkv = (int)Hkv;
    a.G = (int)(Hq / Hkv);
    a.g = make_fastdiv((uint32_t)a.G);
    a.sl2 = scale * 1.4426950408889634f;
    a.q_begin[0] = a.k_begin[0] = 0;
    for (int s = 0; s < LQ_MAX_SEQS; ++s) {
      a.q_begin[s + 1] = a.q_begin[s] + (s < nseq ? q_lens_host[s] : 0);
      a.k_begin[s + 1] = a.k_begin[s] + (s < nseq ? k_lens_host[s] : 0);
    }
    const bool split = plan.split;
    for (size_t at = 0; at < list.size(); at += LIST) {
      const int n = (int)std::min<size_t>(LIST, list.size() - at);
      for (int i = 0; i < LIST; ++i) a.list[i] = i < n ? list[at + i] : Entry{0u};
      prompt_attn_kernel<<<dim3((unsigned)(n * Hkv)), dim3(64 * PW), 0, (hipStream_t)stream>>>(a, (int)at);
      LQ_CHECK_LAUNCH("prompt_attn_kernel");
      if (split) {
        prompt_merge_kernel<<<dim3((unsigned)(n * Hkv), PROWS / 8), dim3(256), 0, (hipStream_t)stream>>>(
            a, (int)at);
        LQ_CHECK_LAUNCH("prompt_merge_kernel");
      }
    }
  } catch (...) {
    set_error("no host memory for the plan");
    return LQ_EHIP;
  }
  return LQ_OK;
}
