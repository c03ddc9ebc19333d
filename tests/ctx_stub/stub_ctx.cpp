// A context of the library made without a GPU, for calls that refuse their arguments before anything is launched.
#include "tl_common.cuh"

TlBlockPool::TlBlockPool() = default;
TlBlockPool::~TlBlockPool() = default;

extern "C" void* stub_ctx() {
  tl_ctx* ctx = new tl_ctx();
  ctx->sm_count = 148;
  return ctx;
}
extern "C" int stub_bad_token(int pos, long long seq, int n_seqs, int max_pages, int page_size, long long rows) {
  return tl_bad_token(pos, seq, n_seqs, max_pages, page_size, rows);
}
extern "C" int stub_bad_page(int page, long long n_pages) { return tl_bad_page(page, n_pages); }
extern "C" long long stub_page_at(int page, int slot, int heads, int page_size, int dim) { return tl_page_at(page, slot, heads, page_size, dim); }
extern "C" int stub_lead() { return kLead; }
extern "C" int stub_tiles(int first, int end, int keys) { return tl_tiles(first, end, keys); }
extern "C" int stub_share_ctas(long long units, int most, int least, long long parts) { return tl_shares(units, most, least, parts).ctas; }
extern "C" long long stub_share_begin(long long units, int most, int least, long long parts, int cta) { return tl_share_begin(tl_shares(units, most, least, parts), cta); }
extern "C" int stub_share_owner(long long units, int most, int least, long long parts, long long unit) { return tl_share_owner(tl_shares(units, most, least, parts), unit); }
// The first n at which the quotient by d is wrong, of `count` neighbours of every multiple that is tried; -1: none
extern "C" long long stub_divide_wrong(int d, int tries) {
  const TlDivide by = tl_divide_by(d);
  const long long most = 2147483647;
  for (int i = 0; i <= tries; ++i) {
    const long long m = most / d * i / tries * d;
    for (long long n = m - 2; n <= m + 2; ++n)
      if (n >= 0 && n <= most && tl_divide(int(n), by) != n / d) return n;
  }
  for (long long n = most - 2 * (long long)(d); n <= most; n += d > 1000 ? d / 500 : 1)
    if (n >= 0 && tl_divide(int(n), by) != n / d) return n;
  return -1;
}
