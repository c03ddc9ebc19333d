// Attention of one new token per row over a paged cache (include/tlcuda.h, tl_paged_attention).
//
//   x_j = cap(q . k_j * scale) + slope (j - p),   out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m)
//
// one pass over the keys with the running maximum, sum and output of the softmax in f32.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "tl_vec.cuh"

namespace {

struct PagedArgs {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int32_t *page_table, *positions, *token_seq;
  const float* slopes;
  int64_t qt, qh, n_pages;
  int32_t tokens, n_heads, n_kv_heads, rep, head_dim, page_size, n_seqs, max_pages, window, dtype;
  float scale, softcap;
  int* status;
};

// A CTA per token and query head; a warp per key, a lane per 32nd dimension.
__global__ void __launch_bounds__(128) paged_attention_kernel(PagedArgs p) {
  __shared__ float sm[4], sl[4], so[4][256];
  tl_pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, kvh = h / p.rep, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t out_at = (int64_t(t) * p.n_heads + h) * p.head_dim, q_at = int64_t(t) * p.qt + h * p.qh;
  int pos = p.positions[t];
  int64_t seq = p.token_seq ? p.token_seq[t] : t;
  if (pos >= 0) {
    const int bad = tl_bad_token(pos, seq, p.n_seqs, p.max_pages, p.page_size, -1);
    if (bad) { atomicOr(p.status, bad); pos = -1; }
  }
  const int lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    o[i] = 0.f;
    q[i] = lane + 32 * i < p.head_dim ? ld_f32(p.q, p.dtype, q_at + lane + 32 * i) : 0.f;
  }
  for (int j = lo + warp; j <= pos; j += 4) {
    const int index = j / p.page_size, page = p.page_table[seq * p.max_pages + index];
    if (tl_bad_page(page, p.n_pages)) { atomicOr(p.status, kBadPage); continue; }
    const int64_t at = tl_page_at(page, j - index * p.page_size, p.n_kv_heads, p.page_size, p.head_dim) + int64_t(kvh) * p.page_size * p.head_dim;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.head_dim) x = fmaf(q[i], ld_f32(p.k_pages, p.dtype, at + lane + 32 * i), x);
    x = warp_sum(x) * p.scale;
    if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
    if (p.slopes) x = fmaf(p.slopes[h], float(j - pos), x);
    const float nm = fmaxf(m, x);
    if (nm == -INFINITY) continue;
    const float f = expf(m - nm), e = expf(x - nm);
    m = nm;
    l = fmaf(l, f, e);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.head_dim) o[i] = fmaf(o[i], f, e * ld_f32(p.v_pages, p.dtype, at + lane + 32 * i));
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  for (int d = threadIdx.x; d < p.head_dim; d += 128) {
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = sl[w] == 0.f ? 0.f : sm[w] == mx ? 1.f : expf(sm[w] - mx);
      if (f != 0.f) { num = fmaf(f, so[w][d], num); den = fmaf(f, sl[w], den); }
    }
    tl_store_out(p.out, p.dtype, out_at + d, den == 0.f ? 0.f : num / den);
  }
}

}  // namespace

extern "C" {

int32_t tl_paged_attention(tl_ctx* ctx, const tl_paged_cache* cache, const int32_t* positions, const int32_t* token_seq, int64_t tokens, const void* q,
                           int64_t q_token_stride, int64_t q_head_stride, int64_t n_heads, void* out, float scale, float softcap, int32_t window,
                           const float* slopes) {
  TL_CHECK_CTX(ctx);
  int32_t rc = tl_check_paged(ctx, "tl_paged_attention", cache, positions, token_seq, tokens);
  if (rc != TL_OK) return rc;
  if (n_heads < 1 || n_heads % cache->n_kv_heads != 0 || n_heads > 65535)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: %lld heads over %d kv heads", (long long)n_heads, cache->n_kv_heads);
  if (cache->head_dim % 8 != 0 || cache->head_dim > 256)
    return tl_set_error(ctx, TL_ERR_UNSUPPORTED, "tl_paged_attention: head_dim must be a multiple of 8 and at most 256, got %d", cache->head_dim);
  if (!std::isfinite(scale) || !std::isfinite(softcap) || softcap < 0.f || window < 0)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: scale and softcap must be finite, softcap and window not negative");
  if (tokens == 0) return TL_OK;
  if (!q || !out) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: null pointer");
  const int64_t esz = int64_t(tl_dtype_size(cache->dtype));
  if (q_token_stride < 0 || q_head_stride < 0 || (q_token_stride * esz) % 16 != 0 || (q_head_stride * esz) % 16 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache->k_pages) |
        reinterpret_cast<uintptr_t>(cache->v_pages)) & 15) != 0)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: pages, q, out and q's strides must be multiples of 16 bytes");
  DeviceGuard guard(ctx->device);
  PagedArgs p{};
  p.q = q; p.k_pages = cache->k_pages; p.v_pages = cache->v_pages; p.out = out;
  p.page_table = cache->page_table; p.positions = positions; p.token_seq = token_seq; p.slopes = slopes;
  p.qt = q_token_stride; p.qh = q_head_stride; p.n_pages = cache->n_pages;
  p.tokens = int32_t(tokens); p.n_heads = int32_t(n_heads); p.n_kv_heads = cache->n_kv_heads; p.rep = int32_t(n_heads / cache->n_kv_heads);
  p.head_dim = cache->head_dim; p.page_size = cache->page_size; p.n_seqs = cache->n_seqs; p.max_pages = cache->max_pages;
  p.window = window; p.dtype = cache->dtype; p.scale = scale; p.softcap = softcap; p.status = ctx->dev_status + 1;
  TL_CUDA(ctx, tl_launch_waiting(paged_attention_kernel, dim3(unsigned(tokens), unsigned(n_heads)), dim3(128), ctx->stream, p));
  ctx->counters[TL_COUNTER_KERNEL_LAUNCHES]++;
  tl_wrote(ctx, out, tokens * n_heads * cache->head_dim * esz, true);
  return TL_OK;
}

}  // extern "C"
