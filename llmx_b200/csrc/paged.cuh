// The paged 16-bit key/value cache as the kernels address it
// (include/llmx_attn.h), shared by the store and eviction (paged_cache.cu) and
// the attention over it (attn_paged.cu, attn_paged_tc.cu).
#pragma once

#include "common.cuh"

namespace llmx_b200 {

// A validated cache.
struct PagedArgs {
  void *k, *v;
  long long ks[3], vs[3];  // elements: page, kv head, token
  const int *table;        // nullable
  long long table_stride;
  float *w;  // nullable
  long long ws[2];
  int n_pages, max_pages, page_size, Hkv, D;
  unsigned int *err;
};

// Checks *c for sequences b < batch; fills *k (without the error word).
llmx_status validate_paged(const llmx_paged_cache *c, int batch, PagedArgs *k);

// The page of page slot `slot` of sequence b in a table (NULL: the sequence's
// `columns` pages one after the other), or -1 (and the error word set) where it
// lies outside the cache or its table.
__device__ __forceinline__ int paged_page(const PagedArgs &a, const int *table, long long stride, int columns, int b,
                                          long long slot) {
  if (slot >= 0 && slot < columns) {
    const long long id = table != nullptr ? (long long)table[b * stride + slot] : (long long)b * columns + slot;
    if (id >= 0 && id < a.n_pages) return (int)id;
  }
  raise_error(a.err, kDevErrBadPage);
  return -1;
}
__device__ __forceinline__ int paged_page(const PagedArgs &a, int b, long long slot) {
  return paged_page(a, a.table, a.table_stride, a.max_pages, b, slot);
}

}  // namespace llmx_b200
