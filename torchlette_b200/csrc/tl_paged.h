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

// ---- how attention's work is split -------------------------------------------------------------------------------------------
// A unit is `keys` neighbouring keys of one token and one group of query heads.  The units of a call, token after token, are
// dealt out to `ctas` CTAs in equal contiguous shares, so a CTA's share may begin and end inside a token's keys: those parts meet in scratch.
TL_HD int32_t tl_units(int32_t first_key, int32_t end_key, int32_t keys) { return end_key > first_key ? (end_key - first_key + keys - 1) / keys : 0; }
TL_HD int64_t tl_share_begin(int64_t units, int32_t ctas, int32_t cta) { return units * cta / ctas; }
// The CTA whose share holds a unit: the largest c with units * c / ctas <= unit
TL_HD int32_t tl_share_owner(int64_t units, int32_t ctas, int64_t unit) { return int32_t(((unit + 1) * ctas - 1) / units); }
// CTAs that a call of so many units uses: with fewer units each, a CTA's fixed costs outweigh what it reads
TL_HD int32_t tl_share_ctas(int64_t units, int32_t most, int32_t least_units) {
  const int64_t c = (units + least_units - 1) / least_units;
  return c < 1 ? 1 : c < most ? int32_t(c) : most;
}
// n / d for 0 <= n < 2^31 as (n * mul) >> shift: mul = ceil(2^shift / d), shift = 31 + ceil(log2 d), so that the
// error mul * d - 2^shift < d <= 2^(shift - 31) stays below one step of n / d for every such n; mul fits 32 bits
struct TlDivide {
  uint32_t mul, shift;
};
inline TlDivide tl_divide_by(int32_t d) {
  uint32_t log = 0;
  while ((int64_t(1) << log) < d) ++log;
  const uint64_t one = uint64_t(1) << (31 + log);
  return {uint32_t((one + uint64_t(d) - 1) / uint64_t(d)), 31 + log};
}
TL_HD int32_t tl_divide(int32_t n, TlDivide by) { return int32_t((uint64_t(uint32_t(n)) * by.mul) >> by.shift); }
