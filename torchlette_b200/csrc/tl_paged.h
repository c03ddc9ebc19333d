// Where the tokens of a paged cache are, for the kernels (tl_paged_append.cu, tl_paged_attention.cu) and for a test on the host: everything
// that an index read on the device has to pass before it becomes an address.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define TL_HD __host__ __device__ __forceinline__
#else
#define TL_HD inline
#endif

// Indexes that a kernel skipped, as bits of word 1 of the context's status words
enum { kBadPosition = 1, kBadSequence = 2, kBadPage = 4 };

// A token at position pos >= 0 of sequence seq: 0, or why it is skipped.  table_rows < 0: no rotation tables.
TL_HD int tl_bad_token(int32_t pos, int64_t seq, int32_t n_seqs, int32_t max_pages, int32_t page_size, int64_t table_rows) {
  if (seq < 0 || seq >= n_seqs) return kBadSequence;
  if (pos / page_size >= max_pages || (table_rows >= 0 && pos >= table_rows)) return kBadPosition;
  return 0;
}
TL_HD bool tl_bad_page(int32_t page, int64_t n_pages) { return page < 0 || page >= n_pages; }
// Element offset of head 0's vector at slot `slot` of a page; heads are page_size * head_dim apart
TL_HD int64_t tl_page_at(int32_t page, int32_t slot, int32_t n_kv_heads, int32_t page_size, int32_t head_dim) {
  return (int64_t(page) * n_kv_heads * page_size + slot) * head_dim;
}
