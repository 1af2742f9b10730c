// Paged 8-bit cache: the pool's buffers and the checks shared by the entry points that take them.
//
// A page holds 64 positions of every KV head of one layer: codes uint8 [pages, Hkv, 64, 128], scales
// and biases bf16 [pages, Hkv, 64, 2], for K and for V -- each page the contiguous cache layout of 64
// rows. Row b of a table (int32 [B, width], device) lists the pages of sequence b in order: position p
// lies in slot p % 64 of page table[b, p / 64].
#pragma once

#include "common.h"

namespace lq {

constexpr int PAGE = 64;

struct PagedBufs {
  uint8_t* kc;
  uint16_t* ks;
  uint16_t* kb;
  uint8_t* vc;
  uint16_t* vs;
  uint16_t* vb;
};

struct PageTable {
  const int32_t* ids;
  int64_t stride;  // entries from a sequence's row to the next
  int width;       // pages of a row
  int pages;       // pages of the pool: other ids are not followed
};

inline int check_pool(const PagedBufs& p, const PageTable& t, int64_t stride, int64_t width,
                      int64_t pages, int64_t Hkv, int64_t D) {
  LQ_CHECK_ARG(D == 128, "head_dim must be 128 (got %lld)", (long long)D);
  LQ_CHECK_ARG(Hkv >= 1 && Hkv <= 1024, "%lld KV heads are not in [1, 1024]", (long long)Hkv);
  LQ_CHECK_ARG(pages >= 1 && pages <= INT32_MAX / PAGE, "%lld pages are not in [1, 2^25)",
               (long long)pages);
  LQ_CHECK_ARG(width >= 1 && width <= (1 << 24) / PAGE && stride >= 0,
               "a table row of %lld pages is not in [1, 2^18]", (long long)width);
  LQ_CHECK_ARG(p.kc && p.ks && p.kb && p.vc && p.vs && p.vb && t.ids, "null pointer");
  LQ_CHECK_ARG((((uintptr_t)p.kc | (uintptr_t)p.vc) & 15) == 0 &&
                   (((uintptr_t)p.ks | (uintptr_t)p.kb | (uintptr_t)p.vs | (uintptr_t)p.vb) & 15) == 0,
               "pool buffers must be 16-byte aligned");
  return LQ_OK;
}

}  // namespace lq
