// A KV cache in pages: where its rows lie, and the checks that every entry point over it makes.
#pragma once

#include "tg_common.h"

namespace tg {
namespace {

// One layer's pages: row r of KV head h in page p lies p ps + h hs + r rs elements behind the base.  Key j of sequence b is row
// j % page of page table[b][j / page]; an entry outside 0 .. n_pages - 1 names none.
struct PagePool {
  bf16_t *k, *v;
  int64_t k_ps, k_hs, k_rs, v_ps, v_hs, v_rs;
  int n_pages, lg;               // a page has 1 << lg rows
};

// A logit that its scale took below fp32's range (a mask's lowest float, at scales above ln 2) is the lowest float, so that it
// weighs nothing beside others, but is not hidden.  (A not-a-number stays one.)
__device__ __forceinline__ float in_range(float z) { return z < -3.402823466e38f ? -3.402823466e38f : z; }

inline int check_pool(const char *what, const void *k, const void *v, const int64_t (&ks)[3], const int64_t (&vs)[3],
                      int32_t num_pages, int32_t page_rows, int32_t num_heads_k, int32_t head_dim, PagePool *p) {
  TG_CHECK(head_dim == kHeadDim, "%s: head_dim must be 128", what);
  TG_CHECK(num_heads_k > 0 && num_heads_k <= 256, "%s: KV heads must be in 1..256", what);
  TG_CHECK(num_pages > 0, "%s: the cache has no pages", what);
  TG_CHECK(page_rows >= 16 && page_rows <= 65536 && (page_rows & (page_rows - 1)) == 0,
           "%s: page rows must be a power of two from 16 to 65536 (got %d)", what, page_rows);
  TG_CHECK((int64_t)num_pages * page_rows < (1ll << 31), "%s: a cache must have less than 2^31 rows", what);
  TG_CHECK(k && v, "%s: null cache pointer", what);
  TG_CHECK(aligned16(k) && aligned16(v), "%s: cache pointers must be 16-byte aligned", what);
  for (int i = 0; i < 3; ++i)
    TG_CHECK(ks[i] >= 0 && vs[i] >= 0 && ks[i] % 8 == 0 && vs[i] % 8 == 0,
             "%s: cache strides must be multiples of 8 elements", what);
  TG_CHECK(page_rows * ks[2] < (1 << 29) && page_rows * vs[2] < (1 << 29), "%s: a page must span less than 1 GiB", what);
  *p = PagePool{static_cast<bf16_t *>(const_cast<void *>(k)), static_cast<bf16_t *>(const_cast<void *>(v)),
                ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], num_pages, __builtin_ctz((unsigned)page_rows)};
  return 0;
}
inline int check_table(const char *what, const int32_t *table, int64_t table_stride, int32_t table_cols, int32_t num_seqs) {
  TG_CHECK(table != nullptr, "%s: null page table", what);
  TG_CHECK(table_cols > 0 && (num_seqs <= 1 || table_stride >= 0), "%s: the page table has no columns", what);
  return 0;
}

}  // namespace
}  // namespace tg
