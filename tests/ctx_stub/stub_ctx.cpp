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
