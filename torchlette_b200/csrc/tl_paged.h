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
  if (pos >= int64_t(max_pages) * page_size || (table_rows >= 0 && pos >= table_rows)) return kBadPosition;
  return 0;
}
TL_HD bool tl_bad_page(int32_t page, int64_t n_pages) { return page < 0 || page >= n_pages; }
// Element offset of head 0's vector at slot `slot` of a page; heads are page_size * head_dim apart
TL_HD int64_t tl_page_at(int32_t page, int32_t slot, int32_t n_kv_heads, int32_t page_size, int32_t head_dim) {
  return (int64_t(page) * n_kv_heads * page_size + slot) * head_dim;
}

// ---- how attention's work is split -------------------------------------------------------------------------------------------
// A part is the keys of one token for one group of query heads, tile after tile.  What it costs is counted in tiles, kLead of them for what a
// part costs by itself (its queries, the meeting of the warps, its output); so a part of n tiles takes up kLead + n units, the lead first.
// The units of a call, part after part, are dealt out to `ctas` CTAs in equal contiguous shares.  A share may begin and end inside a
// part's tiles: what its CTAs make of it meets in scratch.
// (Without a lead, 64 ragged sequences up to 8000: 160 us against 137, the CTAs with many short ones ending last; 3, 6 and 9 are alike since cuts meet at the
// end of a share, but f32 shares of few tiles: 14.4 us with 3, 11.6 with 6 and 9.)
constexpr int kLead = 6;
TL_HD int32_t tl_tiles(int32_t first_key, int32_t end_key, int32_t keys) {
  return end_key > first_key ? (end_key - 1) / keys + 1 - first_key / keys : 0;
}
struct TlShares {
  int64_t units, each;  // each: of a share; the first `more` have one more
  int32_t ctas, more;
};
TL_HD int64_t tl_quotient(int64_t a, int64_t b) { return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b; }
// CTAs that a call uses: a share of fewer than least_units does not pay for a CTA's fixed costs, unless it is a part by itself
// (short sequences side by side rather than one after another); every share has a tile
TL_HD TlShares tl_shares(int64_t units, int32_t most, int32_t least_units, int64_t parts) {
  int64_t c = units / least_units;  // a constant where it is called
  if (c < parts) c = parts;
  if (c > most) c = most;
  if (c * (kLead + 1) > units) c = units / (kLead + 1);
  if (c < 1) c = 1;
  const int64_t each = tl_quotient(units, c);
  return {units, each, int32_t(c), int32_t(units - each * c)};
}
TL_HD int64_t tl_share_begin(const TlShares& s, int32_t cta) { return s.each * cta + (cta < s.more ? cta : s.more); }
// The CTA whose share holds a unit
TL_HD int32_t tl_share_owner(const TlShares& s, int64_t unit) {
  const int64_t big = (s.each + 1) * s.more;
  return int32_t(unit < big ? tl_quotient(unit, s.each + 1) : s.more + tl_quotient(unit - big, s.each));
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
