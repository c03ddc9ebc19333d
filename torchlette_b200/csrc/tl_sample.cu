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
// second launch.  Bound: HBM for the first pass over a row, L2 and the cluster's meetings after it.
//
//   one pass    the row's maximum, and the maxima of 256 groups of its elements.
//   top-k       up to kMaxQuick: the k-th largest of the group maxima is no more than the k-th largest logit, and little is between them (k = 50: about 55
//               candidates).  A second pass sends what is not below it to the first CTA, which ranks the candidates by counting and draws.
//   the rest    a set of kept tokens is narrowed by 2048 bins of counts or masses, linear in the logit, and the bin that holds the border
//               is resolved by ranking its tokens; where ties or a spread over all magnitudes leave too many in it, by bins of the keys down to one key.
//               Then a pass over the masses, and the CTA that holds the answer walks its slice.
//
// exp in 64 bits by a table of 2^(j/128) and a polynomial on what is left (Tang's table-driven method, 1989): ten operations where the library's exp takes
// about three times as many.
//
// Measured: 64 rows x 151 936 f32, top-k 50 and top-p .95: 25.2 us (39 MB: 6 us of HBM, the rest is the cluster's meetings and the first CTA's ranking);
// 16 such rows in f16, top-p .9 and min-p .02: 44 us, 8 of them the pass into bins (exponentials and shared atomics), 4 each the pass
// that sends a bin's tokens and the one over the kept masses, the rest meetings and reads of other CTAs' bins.
#include <algorithm>
#include <climits>
#include <cmath>

#include <cooperative_groups.h>

#include "tl_common.cuh"
#include "tl_tma.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 16, kBins = 2048, kGroups = 256, kMaxQuick = 192, kCandidates = 1024;
constexpr uint32_t kNone = 0x007fffffu;  // key of -infinity: never kept

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  const float *temperature, *top_p, *min_p, *uniforms;
  const int32_t* top_k;
  int32_t* out;
  int32_t vocab, per_cta, shift, vec;  // per_cta: elements of a slice, a multiple of 8; vec: rows start on 16 bytes
};

using u64 = unsigned long long;
struct Shared {
  u64 group_max[kGroups];      // (key, ~index) of every group of the cluster
  u64 told[2][2 * kMaxCluster];  // one or two values a CTA, two turns
  u64 part[kWarps];
  double table[128];           // 2^(j / 128)
  uint32_t count[kBins], mass_low[kBins], mass_high[kBins];  // of this CTA's slice
  u64 cand[kCandidates];       // in the first CTA: (key, ~index)
  u64 sorted[kCandidates], weight[kCandidates];
  uint32_t n_cand, low, high, bin, bin_count, token, border_key, border_index;
  u64 above;
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
  int begin, end, rank_in, ctas, turn;
  bool vec;
  float max;
  double scale, offset, lowest;  // 128 log2 of a weight is logit * scale + offset; below lowest nothing is left
  int shift;
  uint32_t threshold, min_key;  // kept: key > threshold, or equal and index <= last; and key >= min_key once min-p counts
  int last;
  Shared* s;

  static constexpr int kLoads = sizeof(T) == 4 ? 2 : 1;
  struct Eight {
    uint4 u[kLoads];
  };
  __device__ __forceinline__ bool whole(int i) const { return vec && i + 8 <= end; }
  __device__ __forceinline__ void fetch(int i, Eight& e) const {
    if (whole(i))
#pragma unroll
      for (int j = 0; j < kLoads; ++j) e.u[j] = __ldg(reinterpret_cast<const uint4*>(x + i) + j);
  }
  // CLEAN: NaN is -infinity and -0 is 0; else as stored
  template <bool CLEAN, typename F> __device__ __forceinline__ void take(int i, const Eight& u, F&& f) const {
    if (i >= end) return;
    float v[8];
    if (whole(i)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = DT<T>::to_f32(reinterpret_cast<const T*>(u.u)[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i + e < end ? DT<T>::to_f32(x[i + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f(i + e, CLEAN ? clean(v[e]) : v[e]);
  }
  // f(index, value) for the elements of the slice that are this thread's, eight neighbours at a time
  template <bool CLEAN = true, typename F> __device__ __forceinline__ void each_of(int i, F&& f) const {
    Eight e;
    fetch(i, e);
    take<CLEAN>(i, e, f);
  }
  template <bool CLEAN = true, typename F> __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 2
    for (int i = begin + int(threadIdx.x) * 8; i < end; i += kThreads * 8) each_of<CLEAN>(i, f);
  }
  __device__ __forceinline__ bool kept(int i, uint32_t key) const { return key > threshold || (key == threshold && i <= last); }
  __device__ __forceinline__ u64 mass_of(float v) const {
    if (v == max) return u64(1) << shift;
    const double t = fma(double(v), scale, offset);  // 128 log2 of the weight
    if (!(t >= lowest)) return 0;                    // rounds to none; -infinity, and what is infinitely far from the largest
    const double m = t + 6755399441055744.0;         // 1.5 * 2^52: its low word is t rounded
    const int n = __double2loint(m);
    const double r = t - (m - 6755399441055744.0);   // |r| <= 1/2: 2^(r / 128) by its series, the fifth term is below 2^-49
    constexpr double a1 = 0.0054152123481245725, a2 = a1 * a1 / 2, a3 = a1 * a1 * a1 / 6, a4 = a1 * a1 * a1 * a1 / 24;  // a1 = ln 2 / 128
    const double q = r * fma(r, fma(r, fma(r, a4, a3), a2), a1), w = s->table[n & 127];
    const double x = fma(w, q, w);                   // [1, 2) or just past it, times 2^(n >> 7)
    const double y = __hiloint2double(__double2hiint(x) + (((n >> 7) + shift) << 20), __double2loint(x));
    return static_cast<u64>(__double_as_longlong(y + 4503599627370496.0) - __double_as_longlong(4503599627370496.0));  // 2^52: rounded to a whole number
  }
  __device__ __forceinline__ u64 block_sum(u64 v) {
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
  __device__ __forceinline__ u64 block_scan(u64 v, u64& whole) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) s->part[warp] = v;
    __syncthreads();
    whole = 0;
    u64 before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s->part[w];
      whole += s->part[w];
    }
    return v + before;
  }
  // Every CTA's value in s->told[turn]: two turns, so that a CTA may tell the next while another still reads this one
  __device__ __forceinline__ const u64* tell(u64 v, u64 second = 0) {
    turn ^= 1;
    cg::cluster_group cluster = cg::this_cluster();
    if (int(threadIdx.x) < ctas) {
      u64* to = cluster.map_shared_rank(s->told[turn], threadIdx.x);
      to[rank_in] = v;
      to[kMaxCluster + rank_in] = second;
    }
    cluster.sync();
    return s->told[turn];
  }
  __device__ __forceinline__ u64 cluster_sum(u64 v, u64& before) { return totals(block_sum(v), before); }
  // The first index of the row at which the running sum of f reaches `need` (>= 1, at most the whole), which starts with `before` in this
  // CTA; all ones where that is not in this CTA's slice.
  template <typename F> __device__ __forceinline__ uint32_t search(F&& f, u64 before, u64 need) {
    if (threadIdx.x == 0) s->token = 0xffffffffu;
    if (before >= need) { __syncthreads(); return 0xffffffffu; }
    for (int b = begin; b < end; b += kThreads * 8) {  // uniform
      const int i = b + int(threadIdx.x) * 8;
      u64 mine = 0, whole;
      each_of(i, [&](int j, float v) { mine += f(j, v); });
      const u64 to = block_scan(mine, whole) + before;
      if (to >= need && to - mine < need) {
        u64 run = to - mine;
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

  // In the first CTA: the candidates of s->cand by size in s->sorted (up to `most` of them), `n` in all
  __device__ __forceinline__ void rank(int n, int most) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u64 mine = s->cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += s->cand[j] > mine;
      if (before < most) s->sorted[before] = mine;
    }
    __syncthreads();
  }
  // An element to the first CTA's candidates
  __device__ __forceinline__ void send(int i, uint32_t key) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t at = atomicAdd(cluster.map_shared_rank(&s->n_cand, 0), 1u);
    if (at < kCandidates) cluster.map_shared_rank(s->cand, 0)[at] = (u64(key) << 32) | uint32_t(~i);
  }

  // Narrows the kept tokens to the shortest prefix by size whose count reaches `need`, or (MASS) whose mass reaches the fraction p of all of theirs.
  template <bool MASS> __device__ void narrow(u64 need, double p, float least) {
    cg::cluster_group cluster = cg::this_cluster();
    uint32_t low = threshold > kNone ? threshold : kNone + 1, high = key_of(max);
    u64 above = 0, ties = 0;
    const float per_bin = float(kBins) / (max - least);
    bool linear = isfinite(per_bin) && per_bin > 0.f && max - least > 0.f && isfinite(max) && isfinite(least);
    bool first = true;
    const int slice = kBins / ctas;  // bins that this CTA adds up over the cluster
    while (first || low < high) {
      const uint32_t span = high - low;
      const int shift_of = max_(0, 32 - __clz(span) - 11);
      auto bin_of = [&](float v, uint32_t key) -> int {
        // both fall with the value, so a bin's tokens are next to each other by size
        return linear ? min(kBins - 1, int(fminf((max - v) * per_bin, float(kBins)))) : int((high - key) >> shift_of);
      };
      for (int b = threadIdx.x; b < kBins; b += kThreads) {
        s->count[b] = 0;
        if (MASS) s->mass_low[b] = s->mass_high[b] = 0;
      }
      __syncthreads();
      each([&](int i, float v) {
        const uint32_t key = key_of(v);
        if (key >= low && key <= high && kept(i, key)) {
          const int b = bin_of(v, key);
          atomicAdd(&s->count[b], 1u);
          if (MASS) {
            const u64 w = mass_of(v);
            if (w) {  // 64 bits by two atomics: whoever makes the low word overflow carries
              const uint32_t lo = uint32_t(w), old = atomicAdd(&s->mass_low[b], lo), hi = uint32_t(w >> 32) + (old + lo < old ? 1u : 0u);
              if (hi) atomicAdd(&s->mass_high[b], hi);
            }
          }
        }
      });
      if (threadIdx.x == 0) { s->n_cand = 0; s->low = 0xffffffffu; s->high = 0; s->bin = 0xffffffffu; }
      cluster.sync();
      // This CTA's bins, neighbouring ones by a thread
      const int per = (slice + kThreads - 1) / kThreads, b0 = rank_of_slice(slice) + int(threadIdx.x) * per;
      const bool has = int(threadIdx.x) * per < slice;
      u64 metric[4], mine = 0;
      uint32_t counts[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) { metric[j] = 0; counts[j] = 0; }
      if (has) {
        if (per == 1) {  // eight CTAs' at once: a remote load takes as long as a meeting
          for (int c0 = 0; c0 < ctas; c0 += 8) {
            uint32_t n[8], lo[8], hi[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const bool there = c0 + c < ctas;
              const int from = there ? c0 + c : 0;
              n[c] = there ? cluster.map_shared_rank(s->count, from)[b0] : 0u;
              lo[c] = MASS && there ? cluster.map_shared_rank(s->mass_low, from)[b0] : 0u;
              hi[c] = MASS && there ? cluster.map_shared_rank(s->mass_high, from)[b0] : 0u;
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              counts[0] += n[c];
              metric[0] += (u64(hi[c]) << 32) + lo[c];
            }
          }
        } else {
          for (int c = 0; c < ctas; ++c) {
            const uint32_t* rc = cluster.map_shared_rank(s->count, c);
            const uint32_t* rl = cluster.map_shared_rank(s->mass_low, c);
            const uint32_t* rh = cluster.map_shared_rank(s->mass_high, c);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < per) {
                counts[j] += rc[b0 + j];
                if (MASS) metric[j] += (u64(rh[b0 + j]) << 32) + rl[b0 + j];
              }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!MASS) metric[j] = counts[j];
        mine += metric[j];
      }
      u64 here, before;
      const u64 to = block_scan(mine, here);
      const u64 whole = totals(here, before);
      if (MASS && first) {
        const double want = ceil(p * double(whole));
        need = want >= 1.0 ? static_cast<u64>(want) : 1ull;
        if (need > whole) need = whole;
      }
      if (above + whole < need) return;  // all of them do not reach it: all stay (uniform over the cluster)
      u64 run = above + before + to - mine;
      if (run < need && run + mine >= need) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (run < need && run + metric[j] >= need) {
            s->bin = b0 + j;
            s->bin_count = counts[j];
            s->above = run;
          }
          run += metric[j];
        }
      }
      __syncthreads();
      // from the CTA that found it to all
      const u64* where = tell((u64(s->bin) << 32) | s->bin_count, s->above);
      int owner = 0;
      for (int c = 0; c < ctas; ++c)
        if (uint32_t(where[c] >> 32) != 0xffffffffu) owner = c;
      const int bin = int(where[owner] >> 32);
      ties = uint32_t(where[owner]);
      above = where[kMaxCluster + owner];
      first = false;
      if (ties <= kCandidates && (linear || shift_of > 0)) {
        // few: ranked by the first CTA
        each([&](int i, float v) {
          const uint32_t key = key_of(v);
          if (key >= low && key <= high && kept(i, key) && bin_of(v, key) == bin) send(i, key);
        });
        cluster.sync();
        if (rank_in == 0) {
          const int n = int(ties);
          this->rank(n, n);
          u64 sum = 0;
          const int per_thread = kCandidates / kThreads;
          u64 w[per_thread];
#pragma unroll
          for (int j = 0; j < per_thread; ++j) {
            const int i = int(threadIdx.x) * per_thread + j;
            w[j] = i < n ? (MASS ? mass_of(of_key(uint32_t(s->sorted[i] >> 32))) : 1ull) : 0ull;
            sum += w[j];
          }
          u64 all;
          u64 at = above + block_scan(sum, all) - sum;
#pragma unroll
          for (int j = 0; j < per_thread; ++j) {
            if (at < need && at + w[j] >= need) {
              const u64 e = s->sorted[threadIdx.x * per_thread + j];
              s->border_key = uint32_t(e >> 32);
              s->border_index = ~uint32_t(e);
            }
            at += w[j];
          }
          __syncthreads();
        }
        const u64 border = tell((u64(s->border_key) << 32) | s->border_index)[0];
        threshold = uint32_t(border >> 32);
        last = int(uint32_t(border));
        return;
      }
      if (linear) {  // the keys of that bin
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](int i, float v) {
          const uint32_t key = key_of(v);
          if (key >= low && key <= high && kept(i, key) && bin_of(v, key) == bin) { lo = min(lo, key); hi = max_(hi, key); }
        });
        atomicMin(&s->low, lo);
        atomicMax(&s->high, hi);
        __syncthreads();
        const u64* all = tell((u64(s->low) << 32) | s->high);
        low = 0xffffffffu;
        high = 0;
        for (int c = 0; c < ctas; ++c) { low = min(low, uint32_t(all[c] >> 32)); high = max_(high, uint32_t(all[c])); }
        linear = false;
      } else {
        const uint32_t top = high - (uint32_t(bin) << shift_of), width = 1u << shift_of;
        low = top - low >= width ? top - width + 1 : low;
        high = top;
      }
    }
    // `ties` tokens have the key `low`; so many of them are needed
    const u64 w = MASS ? mass_of(of_key(low)) : 1ull;
    const u64 n = w ? (need - above + w - 1) / w : 1ull;
    int cut = INT_MAX;
    if (n < ties) {
      const int old_last = low == threshold ? last : INT_MAX;
      auto tie = [&](int i, float v) -> u64 { return key_of(v) == low && i <= old_last ? 1ull : 0ull; };
      u64 mine = 0, before;
      each([&](int i, float v) { mine += tie(i, v); });
      cluster_sum(mine, before);
      const uint32_t at = search(tie, before, n);
      const u64* all = tell(at);
      uint32_t where = 0xffffffffu;
      for (int c = 0; c < ctas; ++c) where = min(where, uint32_t(all[c]));
      cut = int(where);
    } else if (low == threshold) {
      cut = last;
    }
    threshold = low;
    last = cut;
  }
  __device__ __forceinline__ int rank_of_slice(int slice) const { return rank_in * slice; }
  // The sum over the cluster of a value that is the same in all threads of a CTA, and what the CTAs before this one have of it
  __device__ __forceinline__ u64 totals(u64 v, u64& before) {
    const u64* all = tell(v);
    u64 whole = 0;
    before = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank_in) before += all[c];
      whole += all[c];
    }
    return whole;
  }
  static __device__ __forceinline__ int max_(int a, int b) { return a > b ? a : b; }
  static __device__ __forceinline__ uint32_t max_(uint32_t a, uint32_t b) { return a > b ? a : b; }
};

// How much mass the running sum has to reach: the first sum above u * whole is the first that is >= this
__device__ __forceinline__ u64 to_reach(double u, u64 whole) {
  const double t = floor(u * double(whole));
  const u64 n = t > 0 ? static_cast<u64>(t) + 1 : 1ull;
  return n < whole ? n : whole;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs p) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  Shared& s = *reinterpret_cast<Shared*>(dynamic);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank()), row = int(blockIdx.x) / ctas;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 128) s.table[threadIdx.x] = exp2(double(threadIdx.x) * (1.0 / 128));
  if (threadIdx.x == 0) s.n_cand = 0;
  // All CTAs of the cluster run before one of them writes to another's shared memory: said here, waited for behind the first pass
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  tl_pdl_wait();
  Row<T> r;
  r.x = reinterpret_cast<const T*>(p.logits) + int64_t(row) * p.row_stride;
  r.begin = int(min(int64_t(p.vocab), int64_t(rank) * p.per_cta));
  r.end = int(min(int64_t(p.vocab), int64_t(r.begin) + p.per_cta));
  r.rank_in = rank; r.ctas = ctas; r.turn = 0; r.vec = p.vec != 0; r.s = &s;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !p.uniforms || !(t > 0.f);
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
  float u = p.uniforms ? p.uniforms[row] : 0.f;
  u = u > 0.f ? fminf(u, 1.f) : 0.f;

  // the largest logit, the lowest index of equal ones, of 256 groups of them (NaN is never larger)
  float most = -INFINITY;
  int at = -1;
  r.template each<false>([&](int i, float v) {
    if (v > most) { most = v; at = i; }
  });
  u64 best = at < 0 ? 0 : (u64(key_of(clean(most))) << 32) | uint32_t(~at);
  const int width = 2 * ctas;  // lanes of a group: 256 / ctas groups in a CTA
  for (int o = width >> 1; o > 0; o >>= 1) {
    const u64 e = __shfl_xor_sync(0xffffffffu, best, o);
    best = best > e ? best : e;
  }
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  {
    const int groups = kGroups / ctas, group = int(threadIdx.x) / width;
    for (int c = lane & (width - 1); c < ctas; c += width) cluster.map_shared_rank(s.group_max, c)[rank * groups + group] = best;
  }
  cluster.sync();
  u64 top = 0;
  for (int w = lane; w < kGroups; w += 32) top = top > s.group_max[w] ? top : s.group_max[w];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 e = __shfl_xor_sync(0xffffffffu, top, o);
    top = top > e ? top : e;
  }
  if (uint32_t(top >> 32) <= kNone || greedy) {  // the same in all CTAs of the row
    if (rank == 0 && threadIdx.x == 0) p.out[row] = uint32_t(top >> 32) <= kNone ? -1 : int(~uint32_t(top));
    return;
  }
  r.max = of_key(uint32_t(top >> 32));
  r.shift = p.shift;
  r.scale = 128 * 1.4426950408889634 / double(t);
  r.offset = -double(r.max) * r.scale;
  r.lowest = -128.0 * (p.shift + 1);
  r.threshold = kNone;
  r.last = -1;
  r.min_key = 0;
  if (min_p > 0.f) {
    const double least_kept = min_p < 1.f ? double(r.max) + double(t) * log(double(min_p)) : double(r.max);
    float f = float(least_kept);
    if (double(f) < least_kept) f = nextafterf(f, INFINITY);
    r.min_key = key_of(clean(f));
  }

  if (k > 0 && k <= kMaxQuick && k < p.vocab) {
    // The k-th largest of the groups' maxima, its first 20 bits: at least k logits are not below it.  Bit by bit, by every warp for itself.
    uint32_t mine[kGroups / 32], from = 0;
#pragma unroll
    for (int j = 0; j < kGroups / 32; ++j) mine[j] = uint32_t(s.group_max[j * 32 + lane] >> 32);
    for (int bit = 31; bit >= 12; --bit) {
      const uint32_t tried = from | (1u << bit);
      int above = 0;
#pragma unroll
      for (int j = 0; j < kGroups / 32; ++j) above += __popc(__ballot_sync(0xffffffffu, mine[j] >= tried));
      if (above >= k) from = tried;
    }
    from = Row<T>::max_(from, kNone + 1);
    const float least = of_key(from);
    r.template each<false>([&](int i, float v) {
      if (v >= least) r.send(i, key_of(clean(v)));
    });
    cluster.sync();
    const int n = int(*cluster.map_shared_rank(&s.n_cand, 0));
    if (n <= kCandidates) {
      if (rank == 0) {
        const int kept = min(k, n), i = threadIdx.x;
        r.rank(n, kept);
        const u64 e = i < kept ? s.sorted[i] : 0;
        u64 w = i < kept ? r.mass_of(of_key(uint32_t(e >> 32))) : 0, whole;
        if (top_p < 1.f) {
          const u64 to = r.block_scan(w, whole);
          const double want = ceil(double(fmaxf(top_p, 0.f)) * double(whole));
          if (to - w >= (want >= 1.0 ? static_cast<u64>(want) : 1ull)) w = 0;
        }
        if (uint32_t(e >> 32) < r.min_key) w = 0;
        s.weight[i] = w;
        whole = r.block_sum(w);
        const u64 need = to_reach(double(u), whole);
        if (w) {  // the running mass in the order of the vocabulary
          u64 before = 0;
          for (int j = 0; j < kept; ++j) before += uint32_t(s.sorted[j]) > uint32_t(e) ? s.weight[j] : 0;  // ~index
          if (before < need && before + w >= need) p.out[row] = int(~uint32_t(e));
        }
      }
      cluster.sync();  // the count has been read by all
      return;
    }
    cluster.sync();
  }
  if (k > 0 && k < p.vocab) {
    // the smallest finite logit of the row
    float least = INFINITY;
    r.each([&](int, float v) { if (v > -INFINITY) least = fminf(least, v); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
    __syncthreads();
    if (threadIdx.x == 0) s.low = 0xffffffffu;
    __syncthreads();
    if (lane == 0) atomicMin(&s.low, key_of(least));
    __syncthreads();
    const u64* all = r.tell(s.low);
    uint32_t lo = 0xffffffffu;
    for (int c = 0; c < ctas; ++c) lo = min(lo, uint32_t(all[c]));
    r.template narrow<false>(u64(k), 0.0, of_key(lo));
  }
  if (top_p < 1.f) r.template narrow<true>(0, double(fmaxf(top_p, 0.f)), r.max - 16.f * t);  // what is further behind shares the last bin
  auto weight = [&](int i, float v) -> u64 {
    const uint32_t key = key_of(v);
    return key >= r.min_key && r.kept(i, key) ? r.mass_of(v) : 0ull;
  };
  const int turns = (p.per_cta + kThreads * 8 - 1) / (kThreads * 8);
  if (turns * kWarps <= kCandidates) {
    // The mass of every turn of every warp is kept, so that the CTA with the answer looks at one warp's 256 logits again
    int turn = 0;
    u64 mine = 0, before;
    for (int i = r.begin + int(threadIdx.x) * 8; turn < turns; ++turn, i += kThreads * 8) {
      u64 w = 0;
      r.each_of(i, [&](int j, float v) { w += weight(j, v); });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      if (lane == 0) { s.weight[turn * kWarps + (threadIdx.x >> 5)] = w; mine += w; }
    }
    const u64 whole = r.cluster_sum(mine, before), need = to_reach(double(u), whole);
    const int first = int(threadIdx.x) * 2;
    const u64 a = first < turns * kWarps ? s.weight[first] : 0, b = first + 1 < turns * kWarps ? s.weight[first + 1] : 0;
    u64 here;
    const u64 to = r.block_scan(a + b, here) + before - a - b;
    if (threadIdx.x == 0) s.n_cand = 0xffffffffu;
    __syncthreads();
    if (to < need && to + a >= need) { s.n_cand = first; s.above = to; }
    if (to + a < need && to + a + b >= need) { s.n_cand = first + 1; s.above = to + a; }
    __syncthreads();
    if (threadIdx.x < 32 && s.n_cand != 0xffffffffu) {
      const int i = r.begin + (int(s.n_cand) / kWarps * kThreads + int(s.n_cand) % kWarps * 32 + lane) * 8;
      u64 w = 0;
      r.each_of(i, [&](int j, float v) { w += weight(j, v); });
      u64 run = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
      }
      run += s.above - w;
      if (run < need && run + w >= need)
        r.each_of(i, [&](int j, float v) {
          const u64 x = weight(j, v);
          if (run < need && run + x >= need) p.out[row] = j;
          run += x;
        });
    }
    return;
  }
  u64 mine = 0, before;
  r.each([&](int i, float v) { mine += weight(i, v); });
  const u64 whole = r.cluster_sum(mine, before);
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
  // CTAs of a row: as many as leave two places an SM for all rows' (a row's lie in one GPC, so that some rows may start late all the same), each with a vector a thread;
  // top-p over 151 936 logits with 16 against 8: 16 rows 45 and 53 us, one row 35 and 44
  int ctas = 1;
  while (ctas < kMaxCluster && vocab > int64_t(ctas) * kThreads * 8 && rows * ctas * 2 <= 2 * int64_t(ctx->sm_count)) ctas *= 2;
  p.per_cta = int32_t(((vocab + ctas - 1) / ctas + 7) / 8 * 8);
  const size_t esz = tl_dtype_size(dtype);
  p.vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (rows == 1 || (row_stride * int64_t(esz)) % 16 == 0);
  const auto kernel = dtype == TL_F32 ? sample_kernel<float> : dtype == TL_F16 ? sample_kernel<__half> : sample_kernel<__nv_bfloat16>;
  TL_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Shared))));
  if (ctas > 8) TL_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[1] = tl_pdl_attribute();
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TL_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, p));
  ctx->counters[TL_COUNTER_KERNEL_LAUNCHES]++;
  tl_wrote(ctx, out_tokens, rows * int64_t(sizeof(int32_t)), true);
  return TL_OK;
}

}  // extern "C"
