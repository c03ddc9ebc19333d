// A token of each row of logits from given random numbers: temperature, top-k, top-p and min-p (include/tlcuda.h, tl_sample).
//
//   w_i = exp((x_i - max) / T), the kept tokens as declared there, token = first i with sum_{j <= i, kept} w_j > u * sum_kept w_j
//
// The order of tokens by size is that of (key, lowest index first), where key is the logit's bits as an unsigned integer of the same
// order; a set of kept tokens is a smallest key and, among the tokens that have it, a last index.  Masses are whole multiples of 2^-shift
// (44 bits behind the point for vocabularies up to 2^18), computed in 64 bits: their sums are exact, so that neither the order of atomics nor the split
// over CTAs changes a token, and a border is where it is in 64-bit arithmetic.
//
// A cluster of CTAs owns a row, each a contiguous slice; what the CTAs tell each other goes through distributed shared memory.  No scratch, no
// second launch.
#include <algorithm>
#include <climits>
#include <cmath>

#include <cooperative_groups.h>

#include "tl_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 16, kBins = 2048;
constexpr uint32_t kNone = 0x007fffffu;  // key of -infinity: never kept

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  const float *temperature, *top_p, *min_p, *uniforms;
  const int32_t* top_k;
  int32_t* out;
  int32_t vocab, per_cta, shift, vec;  // per_cta: elements of a slice, a multiple of 8; vec: rows start on 16 bytes
};

struct Shared {
  unsigned long long warp_max[kMaxCluster * kWarps];  // (key, ~index) of every warp of the cluster
  unsigned long long told[2][kMaxCluster];            // one value a CTA, two turns
  unsigned long long mass[kBins];
  unsigned long long part[kWarps];
  uint32_t count[kBins];
  uint32_t low, high, bin, bin_count, token;
  unsigned long long above;
};

__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// NaN is -infinity, -0 is 0
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }

// A row's view of one CTA: its slice, the tokens kept so far, and the cluster around it.
template <typename T> struct Row {
  const T* x;
  int begin, end, rank, ctas, turn;
  bool vec;
  float max;
  double inv_t, one;
  uint32_t threshold, min_key;  // kept: key > threshold, or equal and index <= last; and key >= min_key once min-p counts
  int last;
  Shared* s;

  // f(index, value) for the elements of the slice that are this thread's, eight neighbours at a time
  template <typename F> __device__ __forceinline__ void each_of(int i, F&& f) const {
    if (i >= end) return;
    float v[8];
    if (vec && i + 8 <= end) {
      constexpr int kLoads = sizeof(T) == 4 ? 2 : 1;
      uint4 u[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) u[j] = __ldg(reinterpret_cast<const uint4*>(x + i) + j);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = clean(DT<T>::to_f32(reinterpret_cast<const T*>(u)[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i + e < end ? clean(DT<T>::to_f32(x[i + e])) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f(i + e, v[e]);
  }
  template <typename F> __device__ __forceinline__ void each(F&& f) const {
    for (int i = begin + int(threadIdx.x) * 8; i < end; i += kThreads * 8) each_of(i, f);
  }
  __device__ __forceinline__ bool kept(int i, uint32_t key) const { return key > threshold || (key == threshold && i <= last); }
  __device__ __forceinline__ unsigned long long mass_of(float v) const {
    if (v == max) return static_cast<unsigned long long>(one);
    const double d = double(v) - double(max);
    return d == -INFINITY ? 0ull : static_cast<unsigned long long>(__double2ll_rn(exp(d * inv_t) * one));
  }
  __device__ __forceinline__ unsigned long long block_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s->part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += s->part[w];
    return v;
  }
  // Running sum over the CTA's threads, v included, and the whole
  __device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long& whole) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) s->part[warp] = v;
    __syncthreads();
    whole = 0;
    unsigned long long before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s->part[w];
      whole += s->part[w];
    }
    return v + before;
  }
  // Every CTA's value in s->told[turn]: two turns, so that a CTA may tell the next while another still reads this one
  __device__ __forceinline__ const unsigned long long* tell(unsigned long long v) {
    turn ^= 1;
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x < ctas) cluster.map_shared_rank(s->told[turn], threadIdx.x)[rank] = v;
    cluster.sync();
    return s->told[turn];
  }
  __device__ __forceinline__ unsigned long long cluster_sum(unsigned long long v, unsigned long long& before) {
    const unsigned long long* all = tell(block_sum(v));
    unsigned long long whole = 0;
    before = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank) before += all[c];
      whole += all[c];
    }
    return whole;
  }
  // The first index of the row at which the running sum of f reaches `need` (>= 1, at most the whole), which starts with `before` in this
  // CTA; all ones where that is not in this CTA's slice.
  template <typename F> __device__ __forceinline__ uint32_t search(F&& f, unsigned long long before, unsigned long long need) {
    if (threadIdx.x == 0) s->token = 0xffffffffu;
    if (before >= need) { __syncthreads(); return 0xffffffffu; }
    for (int b = begin; b < end; b += kThreads * 8) {  // uniform
      const int i = b + int(threadIdx.x) * 8;
      unsigned long long mine = 0, whole;
      each_of(i, [&](int j, float v) { mine += f(j, v); });
      const unsigned long long to = block_scan(mine, whole) + before;
      if (to >= need && to - mine < need) {
        unsigned long long run = to - mine;
        bool done = false;
        each_of(i, [&](int j, float v) {
          run += f(j, v);
          if (!done && run >= need) { s->token = uint32_t(j); done = true; }
        });
      }
      if (before + whole >= need) break;
      before += whole;
    }
    __syncthreads();
    return s->token;
  }

  // Narrows the kept tokens to the shortest prefix by size whose count (MASS: mass) reaches `need`.
  template <bool MASS> __device__ void narrow(unsigned long long need, float lowest) {
    cg::cluster_group cluster = cg::this_cluster();
    uint32_t low = threshold > kNone ? threshold : kNone + 1, high = key_of(max);
    unsigned long long above = 0, ties = 0;
    const float scale = float(kBins) / (max - lowest);
    bool linear = isfinite(scale) && scale > 0.f && max - lowest > 0.f && isfinite(max) && isfinite(lowest);
    bool first = true;
    while (first || low < high) {
      first = false;
      const uint32_t span = high - low;
      const int shift = max_(0, 32 - __clz(span) - 11);
      auto bin_of = [&](float v, uint32_t key) -> int {
        // both fall with the value, so a bin's tokens are next to each other by size
        return linear ? min(kBins - 1, int(fminf((max - v) * scale, float(kBins)))) : int((high - key) >> shift);
      };
      for (int b = threadIdx.x; b < kBins; b += kThreads) { s->mass[b] = 0; s->count[b] = 0; }
      __syncthreads();
      each([&](int i, float v) {
        const uint32_t key = key_of(v);
        if (key >= low && key <= high && kept(i, key)) {
          const int b = bin_of(v, key);
          atomicAdd(&s->count[b], 1u);
          if (MASS) {
            const unsigned long long w = mass_of(v);
            if (w) atomicAdd(&s->mass[b], w);
          }
        }
      });
      cluster.sync();
      constexpr int kPer = kBins / kThreads;
      unsigned long long metric[kPer], counts[kPer], mine = 0, whole;
#pragma unroll
      for (int j = 0; j < kPer; ++j) metric[j] = counts[j] = 0;
      for (int c = 0; c < ctas; ++c) {
        const uint32_t* rc = cluster.map_shared_rank(s->count, c);
        const unsigned long long* rm = cluster.map_shared_rank(s->mass, c);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          counts[j] += rc[threadIdx.x * kPer + j];
          if (MASS) metric[j] += rm[threadIdx.x * kPer + j];
        }
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (!MASS) metric[j] = counts[j];
        mine += metric[j];
      }
      const unsigned long long to = block_scan(mine, whole) + above;
      if (to >= need && to - mine < need) {
        unsigned long long run = to - mine;
        bool done = false;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (!done && run + metric[j] >= need) {
            s->bin = threadIdx.x * kPer + j;
            s->bin_count = uint32_t(counts[j]);
            s->above = run;
            done = true;
          }
          run += metric[j];
        }
      }
      if (threadIdx.x == 0) { s->low = 0xffffffffu; s->high = 0; }
      __syncthreads();
      if (above + whole < need) return;  // all of them do not reach it: all stay (uniform over the cluster)
      const int bin = int(s->bin);
      ties = s->bin_count;
      above = s->above;
      if (linear) {  // the keys of that bin
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](int i, float v) {
          const uint32_t key = key_of(v);
          if (key >= low && key <= high && kept(i, key) && bin_of(v, key) == bin) { lo = min(lo, key); hi = max_(hi, key); }
        });
        atomicMin(&s->low, lo);
        atomicMax(&s->high, hi);
        __syncthreads();
        const unsigned long long* all = tell((static_cast<unsigned long long>(s->low) << 32) | s->high);
        low = 0xffffffffu;
        high = 0;
        for (int c = 0; c < ctas; ++c) { low = min(low, uint32_t(all[c] >> 32)); high = max_(high, uint32_t(all[c])); }
        linear = false;
      } else {
        const uint32_t top = high - (uint32_t(bin) << shift), width = 1u << shift;
        low = top - low >= width ? top - width + 1 : low;
        high = top;
        cluster.sync();  // the bins are cleared next: all have read them
      }
    }
    // `ties` tokens have the key `low`; so many of them are needed
    const unsigned long long w = MASS ? mass_of(of_key(low)) : 1ull;
    const unsigned long long n = w ? (need - above + w - 1) / w : 1ull;
    int cut = INT_MAX;
    if (n < ties) {
      const int old_last = low == threshold ? last : INT_MAX;
      auto tie = [&](int i, float v) -> unsigned long long { return key_of(v) == low && i <= old_last ? 1ull : 0ull; };
      unsigned long long mine = 0, before;
      each([&](int i, float v) { mine += tie(i, v); });
      cluster_sum(mine, before);
      const uint32_t at = search(tie, before, n);
      const unsigned long long* all = tell(at);
      uint32_t where = 0xffffffffu;
      for (int c = 0; c < ctas; ++c) where = min(where, uint32_t(all[c]));
      cut = int(where);
    } else if (low == threshold) {
      cut = last;
    }
    threshold = low;
    last = cut;
  }
  static __device__ __forceinline__ int max_(int a, int b) { return a > b ? a : b; }
  static __device__ __forceinline__ uint32_t max_(uint32_t a, uint32_t b) { return a > b ? a : b; }
};

// How much mass the running sum has to reach: the first sum above u * whole is the first that is >= this
__device__ __forceinline__ unsigned long long to_reach(double u, unsigned long long whole) {
  const double t = floor(u * double(whole));
  const unsigned long long n = t > 0 ? static_cast<unsigned long long>(t) + 1 : 1ull;
  return n < whole ? n : whole;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs p) {
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank()), row = int(blockIdx.x) / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Row<T> r;
  r.x = reinterpret_cast<const T*>(p.logits) + int64_t(row) * p.row_stride;
  r.begin = int(min(int64_t(p.vocab), int64_t(rank) * p.per_cta));
  r.end = int(min(int64_t(p.vocab), int64_t(r.begin) + p.per_cta));
  r.rank = rank; r.ctas = ctas; r.turn = 0; r.vec = p.vec != 0; r.s = &s;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !p.uniforms || !(t > 0.f);

  // the largest logit
  unsigned long long best = 0;
  float least = INFINITY;
  r.each([&](int i, float v) {
    const unsigned long long e = (static_cast<unsigned long long>(key_of(v)) << 32) | uint32_t(~i);
    if (i < r.end) {
      best = best > e ? best : e;
      if (v > -INFINITY) least = fminf(least, v);
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long e = __shfl_xor_sync(0xffffffffu, best, o);
    best = best > e ? best : e;
  }
  if (lane < ctas) cluster.map_shared_rank(s.warp_max, lane)[rank * kWarps + warp] = best;
  cluster.sync();
  unsigned long long top = 0;
  for (int w = lane; w < ctas * kWarps; w += 32) top = top > s.warp_max[w] ? top : s.warp_max[w];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long e = __shfl_xor_sync(0xffffffffu, top, o);
    top = top > e ? top : e;
  }
  if (uint32_t(top >> 32) <= kNone || greedy) {  // the same in all CTAs of the row
    if (rank == 0 && threadIdx.x == 0) p.out[row] = uint32_t(top >> 32) <= kNone ? -1 : int(~uint32_t(top));
    return;
  }
  r.max = of_key(uint32_t(top >> 32));
  r.inv_t = 1.0 / double(t);
  r.one = ldexp(1.0, p.shift);
  r.threshold = kNone;
  r.last = -1;
  r.min_key = 0;
  if (p.min_p && p.min_p[row] > 0.f) {
    const double least_kept = p.min_p[row] < 1.f ? double(r.max) + double(t) * log(double(p.min_p[row])) : double(r.max);
    float f = float(least_kept);
    if (double(f) < least_kept) f = nextafterf(f, INFINITY);
    r.min_key = key_of(clean(f));
  }
  float u = p.uniforms[row];
  u = u > 0.f ? fminf(u, 1.f) : 0.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;

  if (k > 0 && k < p.vocab) {
    float lowest = 0.f;
    {
      // the smallest finite logit of the row
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
      if (threadIdx.x == 0) s.low = 0xffffffffu;
      __syncthreads();
      if (lane == 0) atomicMin(&s.low, key_of(least));
      __syncthreads();
      const unsigned long long* all = r.tell(s.low);
      uint32_t lo = 0xffffffffu;
      for (int c = 0; c < ctas; ++c) lo = min(lo, uint32_t(all[c]));
      lowest = of_key(lo);
    }
    r.template narrow<false>(static_cast<unsigned long long>(k), lowest);
  }
  if (top_p < 1.f) {
    unsigned long long mine = 0, before;
    r.each([&](int i, float v) { if (r.kept(i, key_of(v))) mine += r.mass_of(v); });
    const unsigned long long whole = r.cluster_sum(mine, before);
    const double want = ceil(double(fmaxf(top_p, 0.f)) * double(whole));
    r.template narrow<true>(want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull, r.max - 31.f * t);
  }
  auto weight = [&](int i, float v) -> unsigned long long {
    const uint32_t key = key_of(v);
    return key >= r.min_key && r.kept(i, key) ? r.mass_of(v) : 0ull;
  };
  unsigned long long mine = 0, before;
  r.each([&](int i, float v) { mine += weight(i, v); });
  const unsigned long long whole = r.cluster_sum(mine, before);
  const uint32_t token = r.search(weight, before, to_reach(double(u), whole));
  if (threadIdx.x == 0 && token != 0xffffffffu) p.out[row] = int(token);
}

}  // namespace

extern "C" {

int32_t tl_sample(tl_ctx* ctx, const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride, const float* temperature,
                  const int32_t* top_k, const float* top_p, const float* min_p, const float* uniforms, int32_t* out_tokens) {
  TL_CHECK_CTX(ctx);
  if (!tl_dtype_valid(dtype)) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_sample: unknown dtype");
  if (rows < 0 || vocab < 1 || (rows > 1 && row_stride < vocab))
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_sample: bad shape (rows %lld, vocab %lld, row stride %lld)", (long long)rows, (long long)vocab,
                        (long long)row_stride);
  if (vocab > (int64_t(1) << 24) || rows > (int64_t(1) << 24))
    return tl_set_error(ctx, TL_ERR_UNSUPPORTED, "tl_sample: at most 2^24 rows and logits a row");
  if (rows == 0) return TL_OK;
  if (!logits || !out_tokens) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_sample: null pointer");
  DeviceGuard guard(ctx->device);
  SampleArgs p{};
  p.logits = logits; p.row_stride = row_stride;
  p.temperature = temperature; p.top_p = top_p; p.min_p = min_p; p.uniforms = uniforms; p.top_k = top_k; p.out = out_tokens;
  p.vocab = int32_t(vocab);
  p.shift = 44;
  while (p.shift > 38 && (vocab >> (62 - p.shift)) != 0) --p.shift;  // the whole mass stays below 2^63
  int ctas = 1;
  while (ctas < 8 && vocab > int64_t(ctas) * kThreads * 8) ctas *= 2;
  p.per_cta = int32_t(((vocab + ctas - 1) / ctas + 7) / 8 * 8);
  const size_t esz = tl_dtype_size(dtype);
  p.vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (rows == 1 || (row_stride * int64_t(esz)) % 16 == 0);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TL_CUDA(ctx, dtype == TL_F32 ? cudaLaunchKernelEx(&cfg, sample_kernel<float>, p)
                               : dtype == TL_F16 ? cudaLaunchKernelEx(&cfg, sample_kernel<__half>, p) : cudaLaunchKernelEx(&cfg, sample_kernel<__nv_bfloat16>, p));
  ctx->counters[TL_COUNTER_KERNEL_LAUNCHES]++;
  tl_wrote(ctx, out_tokens, rows * int64_t(sizeof(int32_t)));
  return TL_OK;
}

}  // extern "C"
