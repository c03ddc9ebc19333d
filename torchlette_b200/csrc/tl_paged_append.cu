// Appending to a paged cache: the per-head norm of q and k, the rotation at each token's own position and the append of k and v, in one
// launch where the separate ops take five (tl_rmsnorm and tl_rope for q and for k, a copy each for k and v with one position for all
// sequences).
//
//   x^ = x * rsqrt(mean(x^2) + eps) * w;   y[d] = x^[d] c[d] - x^[d + D/2] s[d],  y[d + D/2] = x^[d + D/2] c[d] + x^[d] s[d]
//
// f32 arithmetic, one rounding at the store; v is copied bit for bit.
//
// Bound: HBM for prompts (every element is read and written once), launch and the chain position -> page -> store for a step's few tokens.  A head
// is a group of lanes; a thread keeps its dimensions' rotation in registers and takes several heads of its token, whose loads are on their way together.
// Measured: 8001 tokens x 48 heads x 128 bf16: 40.8 us (198 MB, 4.85 TB/s), f32 65.2 (6.1 TB/s); a step's 64 tokens 4.6 us through the Python API, its host time.
#include <algorithm>
#include <type_traits>

#include "tl_vec.cuh"

namespace {

struct AppendArgs {
  const void *q, *k, *v;
  void* q_out;
  int64_t qt, qh, ot, oh, kt, kh, vt, vh;  // strides in elements: tokens, heads
  void *k_pages, *v_pages;
  const int32_t *page_table, *positions, *token_seq;
  const void *q_weight, *k_weight;
  const float *cos_t, *sin_t;
  int64_t tokens, table_rows, n_pages;
  int32_t n_heads, n_kv_heads, head_dim, page_size, n_seqs, max_pages, dtype, w_dtype;
  float eps;
  TlDivide page_div;
  int* status;
};

// Whether token t is there: nothing but its position and sequence is read of one that is not
__device__ __forceinline__ bool is_there(const AppendArgs& p, int64_t t, int& pos, int64_t& seq) {
  pos = p.positions[t];
  if (pos < 0) return false;
  seq = p.token_seq ? int64_t(p.token_seq[t]) : t;
  const int bad = tl_bad_token(pos, seq, p.n_seqs, p.max_pages, p.page_size, p.cos_t ? p.table_rows : -1);
  if (bad) atomicOr(p.status, bad);
  return !bad;
}
// Where it goes: the element offset in k_pages and v_pages of head 0, or -1 if its page is not there.  index: of the page in its sequence
__device__ __forceinline__ int64_t place(const AppendArgs& p, int pos, int index, int page) {
  if (!tl_bad_page(page, p.n_pages)) return tl_page_at(page, pos - index * p.page_size, p.n_kv_heads, p.page_size, p.head_dim);
  atomicOr(p.status, kBadPage);
  return -1;
}

// Any strides and even head_dim: a warp per token and head (q's, then k's, then v's), a lane per pair of dimensions.
__global__ void __launch_bounds__(128) append_kernel(AppendArgs p) {
  tl_pdl_wait();
  const int lane = threadIdx.x & 31, half = p.head_dim >> 1;
  const int rows = (p.q ? p.n_heads : 0) + 2 * p.n_kv_heads;
  const int64_t all = p.tokens * rows, step = int64_t(gridDim.x) * 4;
  for (int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5); w < all; w += step) {
    const int64_t t = w / rows;
    int r = int(w - t * rows), pos;
    int64_t seq;
    if (!is_there(p, t, pos, seq)) continue;
    const int index = tl_divide(pos, p.page_div);
    const int64_t at = place(p, pos, index, p.page_table[seq * p.max_pages + index]);
    const void *x, *weight;
    void* y;
    int64_t xi, yi;
    if (p.q && r < p.n_heads) {
      x = p.q; y = p.q_out; weight = p.q_weight;
      xi = t * p.qt + r * p.qh; yi = t * p.ot + r * p.oh;
    } else {
      if (p.q) r -= p.n_heads;
      if (at < 0) continue;
      const bool is_k = r < p.n_kv_heads;
      if (!is_k) r -= p.n_kv_heads;
      x = is_k ? p.k : p.v; y = is_k ? p.k_pages : p.v_pages; weight = p.k_weight;
      xi = is_k ? t * p.kt + r * p.kh : t * p.vt + r * p.vh;
      yi = at + int64_t(r) * p.page_size * p.head_dim;
      if (!is_k) {
        for (int d = lane; d < p.head_dim; d += 32) tl_store_out(y, p.dtype, yi + d, ld_f32(x, p.dtype, xi + d));
        continue;
      }
    }
    float inv = 1.f;
    if (weight) {
      float ss = 0.f;
      for (int d = lane; d < p.head_dim; d += 32) {
        const float e = ld_f32(x, p.dtype, xi + d);
        ss = fmaf(e, e, ss);
      }
      inv = rsqrtf(warp_sum(ss) / float(p.head_dim) + p.eps);
      __syncwarp();
    }
    for (int d = lane; d < half; d += 32) {
      float a = ld_f32(x, p.dtype, xi + d), b = ld_f32(x, p.dtype, xi + d + half);
      if (weight) {
        a = a * inv * ld_f32(weight, p.w_dtype, d);
        b = b * inv * ld_f32(weight, p.w_dtype, d + half);
      }
      float c = 1.f, s = 0.f;
      if (p.cos_t) { c = p.cos_t[int64_t(pos) * half + d]; s = p.sin_t[int64_t(pos) * half + d]; }
      tl_store_out(y, p.dtype, yi + d, a * c - b * s);
      tl_store_out(y, p.dtype, yi + d + half, b * c + a * s);
    }
  }
}

// Four elements as they are stored
template <typename T> struct Four {
  using Bits = std::conditional_t<sizeof(T) == 4, uint4, uint2>;
  Bits u;
  __device__ __forceinline__ void load(const T* p) { u = __ldcs(reinterpret_cast<const Bits*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Bits*>(p) = u; }
  __device__ __forceinline__ void values(float (&v)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = DT<T>::to_f32(reinterpret_cast<const T*>(&u)[e]);
  }
  __device__ __forceinline__ void take(const float (&v)[4]) {
    if constexpr (std::is_same_v<T, __half>) {
      const __half2 h[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
      u = *reinterpret_cast<const Bits*>(h);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
      u = *reinterpret_cast<const Bits*>(h);
    } else {
      u = *reinterpret_cast<const Bits*>(v);
    }
  }
};
__device__ __forceinline__ void load4_any(const void* p, int dtype, int i, float (&v)[4]) {
  if (dtype == TL_F32) {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else if (dtype == TL_F16) {
    Four<__half> f;
    f.u = *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(p) + i);
    f.values(v);
  } else {
    Four<__nv_bfloat16> f;
    f.u = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
    f.values(v);
  }
}
// A group of LANES lanes (a power of two that holds head_dim / 8) a head, HEADS heads a thread, a CTA for a token's next THREADS / LANES * HEADS heads.  A
// lane has four dimensions of the first half and the same four of the second, which the rotation mixes: no lane needs another's.  The rows are held as
// stored until their turn, so that several CTAs an SM have loads on their way.  (Eight neighbouring dimensions a lane and shuffles: 52 us for
// 8001 tokens x 48 heads x 128 bf16, 197 MB, by the instructions that it issued.)
template <typename T, int LANES, int HEADS, int THREADS>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 1024 / THREADS : 768 / THREADS) append_vec_kernel(const __grid_constant__ AppendArgs p) {
  tl_pdl_wait();
  const int64_t t = blockIdx.x;
  int pos;
  int64_t seq;
  if (!is_there(p, t, pos, seq)) return;  // the same in all threads
  const int index = tl_divide(pos, p.page_div), page = p.page_table[seq * p.max_pages + index];  // on its way with the rows
  const int half = p.head_dim >> 1, d = 4 * int(threadIdx.x % LANES);
  const int n_q = p.q ? p.n_heads : 0, n_qk = n_q + p.n_kv_heads, rows = n_qk + p.n_kv_heads;
  constexpr int kStep = THREADS / LANES;
  const int first = int(blockIdx.y) * (kStep * HEADS) + int(threadIdx.x) / LANES;
  const bool lane_in = d < half;

  // (heads are at most 2^31 elements apart here, so that a head costs no 64-bit product)
  const T *q = reinterpret_cast<const T*>(p.q) + t * p.qt + d, *k = reinterpret_cast<const T*>(p.k) + t * p.kt + d, *v = reinterpret_cast<const T*>(p.v) + t * p.vt + d;
  const int qh = int(p.qh), kh = int(p.kh), vh = int(p.vh), oh = int(p.oh), gh = p.page_size * p.head_dim;
  Four<T> x[HEADS][2];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int r = first + i * kStep;
    if (lane_in && r < rows) {
      const T* from = r < n_q ? q + r * qh : r < n_qk ? k + (r - n_q) * kh : v + (r - n_qk) * vh;
      x[i][0].load(from);
      x[i][1].load(from + half);
    }
  }
  const int64_t at = place(p, pos, index, page);
  float c[4], s[4];
  if (lane_in && p.cos_t) {
    load4_any(p.cos_t + int64_t(pos) * half, TL_F32, d, c);
    load4_any(p.sin_t + int64_t(pos) * half, TL_F32, d, s);
  }
  T *q_out = reinterpret_cast<T*>(p.q_out) + t * p.ot + d, *k_out = reinterpret_cast<T*>(p.k_pages) + at + d, *v_out = reinterpret_cast<T*>(p.v_pages) + at + d;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int r = first + i * kStep;
    const bool here = lane_in && r < rows, is_q = r < n_q, is_v = r >= n_qk;
    const void* weight = is_q ? p.q_weight : p.k_weight;
    float a[4], b[4], inv = 1.f;
    if (here && !is_v) {
      x[i][0].values(a);
      x[i][1].values(b);
    }
    if (p.q_weight || p.k_weight) {
      float ss = 0.f;
      if (here && !is_v)
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, LANES);
      inv = rsqrtf(ss / float(p.head_dim) + p.eps);
    }
    if (!here) continue;
    if (!is_v) {
      if (weight) {
        float w[4];
        load4_any(weight, p.w_dtype, d, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = a[e] * inv * w[e];
        load4_any(weight, p.w_dtype, d + half, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = b[e] * inv * w[e];
      }
      if (p.cos_t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = a[e] * c[e] - b[e] * s[e];
          b[e] = b[e] * c[e] + a[e] * s[e];
          a[e] = y;
        }
      x[i][0].take(a);
      x[i][1].take(b);
    }
    if (!is_q && at < 0) continue;
    T* to = is_q ? q_out + r * oh : is_v ? v_out + (r - n_qk) * gh : k_out + (r - n_q) * gh;
    x[i][0].store(to);
    x[i][1].store(to + half);
  }
}

// A thread takes one head while the tokens are too few to fill the chip (their loads all at once), else as many of a token's as six, in smaller
// CTAs: what a thread works out once (its token's place, pages and rotation) costs about as many instructions as two heads (8001 tokens x 48
// heads x 128 bf16: 47 us with three heads a thread, when six took 44.6).
template <typename T, int LANES, int HEADS, int THREADS> cudaError_t launch_heads(tl_ctx* ctx, const AppendArgs& p, int rows) {
  constexpr int kRows = THREADS / LANES * HEADS;
  return tl_launch_waiting(append_vec_kernel<T, LANES, HEADS, THREADS>, dim3(unsigned(p.tokens), unsigned((rows + kRows - 1) / kRows)), dim3(THREADS), ctx->stream, p);
}
template <typename T, int LANES> cudaError_t launch_vec(tl_ctx* ctx, const AppendArgs& p, int rows) {
  if (int64_t(p.tokens) * rows < int64_t(ctx->sm_count) * 8 * (256 / LANES)) return launch_heads<T, LANES, 1, 256>(ctx, p, rows);
  const int each = (rows + 128 / LANES - 1) / (128 / LANES);  // heads for a thread of a CTA that takes the token whole
  if (each <= 2) return launch_heads<T, LANES, 2, 128>(ctx, p, rows);
  if (each <= 4) return launch_heads<T, LANES, 4, 128>(ctx, p, rows);
  return launch_heads<T, LANES, 6, 128>(ctx, p, rows);
}
template <typename T> cudaError_t launch_lanes(tl_ctx* ctx, const AppendArgs& p, int rows) {
  if (p.head_dim <= 64) return launch_vec<T, 8>(ctx, p, rows);  // a lane: 4 + 4 dimensions
  if (p.head_dim <= 128) return launch_vec<T, 16>(ctx, p, rows);
  return launch_vec<T, 32>(ctx, p, rows);
}

}  // namespace

int32_t tl_check_paged(tl_ctx* ctx, const char* who, const tl_paged_cache* c, const int32_t* positions, const int32_t* token_seq, int64_t tokens) {
  if (!c) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "%s: null cache", who);
  if (c->n_pages < 0 || c->page_size < 1 || c->n_kv_heads < 1 || c->head_dim < 1 || c->n_seqs < 0 || c->max_pages < 0 || tokens < 0)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "%s: bad shape (pages %lld of %d, kv heads %d, head dim %d, sequences %d of %d pages, tokens %lld)", who,
                        (long long)c->n_pages, c->page_size, c->n_kv_heads, c->head_dim, c->n_seqs, c->max_pages, (long long)tokens);
  if (!tl_dtype_valid(c->dtype)) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "%s: unknown dtype", who);
  if (tokens == 0) return TL_OK;
  if (!positions || !c->k_pages || !c->v_pages || !c->page_table) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!token_seq && tokens > c->n_seqs)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "%s: %lld tokens for %d sequences need token_seq", who, (long long)tokens, c->n_seqs);
  // positions are int32 (a tile behind the last one too), and an offset inside a page
  if (int64_t(c->max_pages) * c->page_size > INT32_MAX - 64 || int64_t(c->n_kv_heads) * c->page_size * c->head_dim > INT32_MAX || tokens > INT32_MAX)
    return tl_set_error(ctx, TL_ERR_UNSUPPORTED, "%s: positions (2^31 - 64), a page's elements and tokens are limited to 2^31", who);
  return TL_OK;
}

extern "C" {

int32_t tl_paged_append(tl_ctx* ctx, const tl_paged_cache* cache, const int32_t* positions, const int32_t* token_seq, int64_t tokens, const void* q,
                        int64_t q_token_stride, int64_t q_head_stride, int64_t n_heads, void* q_out, int64_t out_token_stride, int64_t out_head_stride,
                        const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                        const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps, const float* cos_table, const float* sin_table,
                        int64_t table_rows) {
  TL_CHECK_CTX(ctx);
  int32_t rc = tl_check_paged(ctx, "tl_paged_append", cache, positions, token_seq, tokens);
  if (rc != TL_OK) return rc;
  if (cache->head_dim % 2 != 0 || cache->head_dim > 1024)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: head_dim must be even and at most 1024, got %d", cache->head_dim);
  if ((q_weight || k_weight) && !tl_dtype_valid(weight_dtype)) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: unknown weight dtype");
  if (!cos_table != !sin_table || (cos_table && table_rows < 0))
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: the rotation needs both tables and their rows");
  if (q && (n_heads < 1 || n_heads > 65535)) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: bad n_heads %lld", (long long)n_heads);
  if (tokens == 0) return TL_OK;
  if (!k || !v || !q != !q_out) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: null k or v, or only one of q and q_out");
  if (q == q_out && q && (q_token_stride != out_token_stride || q_head_stride != out_head_stride))
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: in place q_out has q's strides");
  if ((q && (q_token_stride < 0 || q_head_stride < 0 || out_token_stride < 0 || out_head_stride < 0)) || k_token_stride < 0 || k_head_stride < 0 ||
      v_token_stride < 0 || v_head_stride < 0)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_append: negative stride");
  DeviceGuard guard(ctx->device);
  AppendArgs p{};
  p.q = q; p.k = k; p.v = v; p.q_out = q_out;
  p.qt = q_token_stride; p.qh = q_head_stride; p.ot = out_token_stride; p.oh = out_head_stride;
  p.kt = k_token_stride; p.kh = k_head_stride; p.vt = v_token_stride; p.vh = v_head_stride;
  p.k_pages = cache->k_pages; p.v_pages = cache->v_pages; p.page_table = cache->page_table; p.positions = positions; p.token_seq = token_seq;
  p.q_weight = q_weight; p.k_weight = k_weight; p.cos_t = cos_table; p.sin_t = sin_table;
  p.tokens = tokens; p.table_rows = table_rows; p.n_pages = cache->n_pages;
  p.n_heads = int32_t(n_heads); p.n_kv_heads = cache->n_kv_heads; p.head_dim = cache->head_dim; p.page_size = cache->page_size;
  p.n_seqs = cache->n_seqs; p.max_pages = cache->max_pages; p.dtype = cache->dtype; p.w_dtype = weight_dtype;
  p.page_div = tl_divide_by(cache->page_size);
  p.eps = eps; p.status = ctx->dev_status + 1;
  const int64_t rows = (q ? n_heads : 0) + 2 * int64_t(cache->n_kv_heads), esz = int64_t(tl_dtype_size(cache->dtype));
  const int64_t widest = std::max({q_head_stride * (q != nullptr), out_head_stride * (q != nullptr), k_head_stride, v_head_stride, int64_t(cache->page_size) * cache->head_dim});
  // Both halves of a head are whole vectors of four, and every row, weight and table starts on 16 bytes
  uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(cache->k_pages) |
                   reinterpret_cast<uintptr_t>(cache->v_pages) | reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight) |
                   reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table) |
                   uintptr_t((k_token_stride | k_head_stride | v_token_stride | v_head_stride) * esz);
  if (q) bits |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | uintptr_t((q_token_stride | q_head_stride | out_token_stride | out_head_stride) * esz);
  if (cache->head_dim % 8 == 0 && cache->head_dim <= 256 && (bits & 15) == 0 && rows <= 65535 && rows * widest <= INT32_MAX) {
    TL_CUDA(ctx, cache->dtype == TL_F32 ? launch_lanes<float>(ctx, p, int(rows))
                                        : cache->dtype == TL_F16 ? launch_lanes<__half>(ctx, p, int(rows)) : launch_lanes<__nv_bfloat16>(ctx, p, int(rows)));
  } else {
    const int64_t grid = std::min<int64_t>((tokens * rows + 3) / 4, int64_t(ctx->sm_count) * 16);
    TL_CUDA(ctx, tl_launch_waiting(append_kernel, dim3(unsigned(grid)), dim3(128), ctx->stream, p));
  }
  ctx->counters[TL_COUNTER_KERNEL_LAUNCHES]++;
  const int64_t page_bytes = cache->n_pages * cache->n_kv_heads * cache->page_size * cache->head_dim * int64_t(tl_dtype_size(cache->dtype));
  tl_wrote(ctx, cache->k_pages, page_bytes, true);
  tl_wrote(ctx, cache->v_pages, page_bytes);
  if (q_out)
    tl_wrote(ctx, q_out, ((tokens - 1) * out_token_stride + (n_heads - 1) * out_head_stride + cache->head_dim) * int64_t(tl_dtype_size(cache->dtype)));
  return TL_OK;
}

}  // extern "C"
