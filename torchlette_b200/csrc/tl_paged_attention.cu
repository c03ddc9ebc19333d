// Attention of one new token per row over a paged cache (include/tlcuda.h, tl_paged_attention).
//
//   x_j = cap(q . k_j * scale) + slope (j - p),   out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m)
//
// in one pass over the keys, with the running maximum m, sum and output of the softmax in f32 registers.  Bound: HBM, the cache is read once.
//
// Work.  The keys of all tokens are cut into tiles (16 of one token and one KV head's query heads, f32 8), and the tiles dealt out to
// a fixed number of resident CTAs in equal contiguous shares (tl_paged.h): sequences of any lengths load all SMs alike, and nothing on the host
// depends on a length, so that a captured call serves sequences that grow.  A producer warp looks up the pages, a batch of tiles ahead, and fills a ring of tiles
// in shared memory across the borders of tokens and heads; the consumer warps take the tiles in turn, each with a softmax of its own, and
// meet at the end of a token's keys.  Where a share ends inside a token's keys the CTA leaves maximum, sum and output in scratch, and whoever of that
// token's CTAs comes last joins them in the order of the keys (in groups of 13 first, where they are many), so that no result depends on timing.
//
// The ring.  Where a tile's rows are neighbours in a page (page_size a multiple of the tile), TMA boxes of 128-byte columns, 128-byte swizzle: an
// instruction for each 2 KB.  Other page sizes: cp.async into the same layout, 16 bytes a lane.
// (A ring of each warp's own, filled by its own cp.async, was 63 us on 8 sequences x 8 KV heads x 4000 keys x 128 f16: 700 instructions a tile, most of
// them addresses, and a wait for the page table in every one.)
//
// f16 / bf16.  The rows of a tile are the A operand of S^T = K q^T (ldmatrix) and, transposed on the way, of O^T = V^T p; the probabilities go
// from accumulators to the B operand in the register file (movmatrix), split into 16-bit terms that keep nearly all bits (tl_attention.cuh).
// f32: CUDA cores, a lane per D / 32 dimensions; the partial dot products of eight keys are summed over the lanes by exchanging halves.
//
// Measured: 8 sequences x 4000 keys, 32 query / 8 KV heads x 128 f16: 31.4 us (131 MB, 4.2 TB/s; about 4 us until the first tile, 20 of copies at 6, 7 of
// meeting and joining); 64 ragged sequences up to 8000, bf16: 119 us (5.9 TB/s); one of 100 003 keys, 2 KV heads: 29.8 us.
//
// Rows of a tile that the token does not see never count: their scores are replaced, not multiplied, and their values zeroed before the
// product, whatever the pages hold there.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "tl_attention.cuh"
#include "tl_mma_frag.cuh"
#include "tl_tma.cuh"

namespace {

// Two CTAs an SM of three consumer warps and a producer (128 threads: all registers but a few): 64 ragged sequences up to 8000 took 139 us with one CTA of
// seven consumers, whose one producer does not keep up (2 CTAs: 120), 147 with five consumers a CTA; the others within 5 %.
constexpr int kCtas = 2, kConsumerWarps = 3;
constexpr int kGroup = 13;       // parts joined at once: two levels for the 296 CTAs of one long sequence
constexpr int kMaxStages = 48;
constexpr int kLeastUnits = 12;  // least share of a CTA, see tl_shares

struct PagedArgs {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int32_t *page_table, *positions, *token_seq;
  const float* slopes;
  int64_t qt, qh, n_pages;
  int32_t tokens, n_heads, n_kv_heads, rep, head_dim, page_size, n_seqs, max_pages, window, row_tiles, stages;
  TlDivide page_div, stage_div;
  float scale, softcap, cap_inv, cap_exp;
  int *status, *wait_status;
  float* slots;        // [2 * CTAs] parts of tokens
  unsigned* arrivals;  // [3 * CTAs], zero between launches: CTAs of a group that have left their part, groups of a token
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {  // 16 bytes, or zeros with bytes == 0
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives once this thread's copies so far have landed
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// What is seen of a stage's tile (low half) and the lap of the ring that it belongs to (high half), written before the tile is asked for.  A parity wait passes
// in the phase before the one that it means too, and a consumer may come to a stage before the lap in front of its own has landed there, since
// the tiles in between are other warps'.  So it waits for its lap's word first: the producer writes it once the lap before has been consumed.
__device__ __forceinline__ void publish(uint32_t* at, int lap, uint32_t seen) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(at)), "r"((uint32_t(lap) << 16) | seen) : "memory");
}
// By a whole warp; false: gave up
__device__ __forceinline__ bool tile_ready(uint32_t* at, uint64_t* full, int lap, volatile int* abort_flag, uint32_t& seen) {
  uint32_t word = 0;
  bool here = false;
  for (int it = 0; it < kWaitTimeoutIters && !here; ++it) {
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(word) : "r"(smem_u32(at)) : "memory");
    here = word >> 16 == (uint32_t(lap) & 0xffffu);
    if ((it & 63) == 63 && *abort_flag) break;
  }
  if (!__all_sync(0xffffffffu, here)) return false;
  seen = word & 0xffffu;
  return mbar_wait_all(full, lap & 1, abort_flag);
}
template <class Tile> constexpr int kConsumers = 32 * Tile::WARPS;
template <class Tile> __device__ __forceinline__ void consumers_meet() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers<Tile>) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The keys that token t sees, [lo, hi) of sequence seq; none of them if it is not there.
struct Token {
  int32_t lo, hi, seq;
};
__device__ __forceinline__ Token token_of(const PagedArgs& p, int t, bool report) {
  Token k{0, 0, 0};
  const int pos = p.positions[t];
  if (pos < 0) return k;
  k.seq = p.token_seq ? p.token_seq[t] : t;
  const int bad = tl_bad_token(pos, k.seq, p.n_seqs, p.max_pages, p.page_size, -1);
  if (bad) {
    if (report) atomicOr(p.status, bad);
    return k;
  }
  k.lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  k.hi = pos + 1;
  return k;
}

// A place in the call's tiles: tile `u` of the `n` of token t and its group `seg` = (KV head, tile of its query heads).  Tiles lie at multiples of
// KEYS in the sequence.
struct Cursor {
  int t, seg, u, n, kvh, tile;
  Token k;
  template <int KEYS> __device__ __forceinline__ void open(const PagedArgs& p) {
    k = token_of(p, t, false);
    n = tl_tiles(k.lo, k.hi, KEYS);
  }
  __device__ __forceinline__ void head(const PagedArgs& p) {
    if (p.row_tiles == 1) { kvh = seg; tile = 0; }
    else { kvh = seg / p.row_tiles; tile = seg - kvh * p.row_tiles; }
  }
  // from u == n to the next group's first tile
  template <int KEYS> __device__ __forceinline__ void next(const PagedArgs& p) {
    u = 0;
    if (++seg == p.n_kv_heads * p.row_tiles) {
      seg = 0;
      do {
        if (++t >= p.tokens) { n = 0; return; }
        open<KEYS>(p);
      } while (n == 0);
    }
    head(p);
  }
  template <int KEYS> __device__ __forceinline__ int first_key(int i) const { return (k.lo / KEYS + i) * KEYS; }
};

// c tanh(x / c), within a few 2^-23 of itself whatever c is.  From |x / c| = 1/4 on it is c (1 - 2 / (1 + exp(2 x / c))), scale = 2 log2(e) / c, whose error is a
// few 2^-23 of c, as the value is; below, where that form cancels and a large cap would take the scores with it, x times the first five terms of tanh(y) / y
// (the sixth is below 2^-26 there).  (16 sequences x <= 6000 keys x 256: 32.5 us, without the near form 32.0; tanhf's two branches were
// a third of the kernel's instructions.)
__device__ __forceinline__ float cap(float x, float c, float inv, float scale) {
  float t;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(x * scale));
  const float far = fmaf(-2.f * __fdividef(1.f, 1.f + t), c, c), y = x * inv, y2 = y * y;
  const float near = x * fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835, -17.f / 315), 2.f / 15), -1.f / 3), 1.f);
  return fabsf(y) < .25f ? near : far;
}

// Infinite values and the terms of a probability: one that is zero or negative makes NaN of an infinity.  A NaN of this kind, which no conversion makes, is stored where
// an output is NaN and the sum of its row's probabilities is not, and look_again() finds it there.
constexpr uint16_t kUnsettled = 0xfff1;
template <typename AT> __device__ __forceinline__ bool unsettled(const AT& x) { return reinterpret_cast<const uint16_t&>(x) == kUnsettled; }
// The part's outputs that are not settled, by all threads of the CTA: what the row sees in that dimension decides.  One infinity is infinity, both, a NaN, and an infinity
// whose score is -infinity are NaN.  found: [rows][DPAD] words.
template <typename AT, int DPAD, int THREADS>
__device__ __noinline__ void look_again(const PagedArgs& p, const Token& k, int t, int kvh, int h0, int rows, uint32_t* found) {
  constexpr int kAhead = 4;
  enum { kUp = 1, kDown = 2, kNan = 4 };
  const int lane = threadIdx.x & 31, d0 = 8 * lane, all = rows * p.head_dim;
  AT* out = reinterpret_cast<AT*>(p.out) + (int64_t(t) * p.n_heads + h0) * p.head_dim;
  bool any = false;
  for (int i = threadIdx.x; i < all; i += THREADS) any |= unsettled(out[i]);
  for (int i = threadIdx.x; i < rows * DPAD; i += THREADS) found[i] = 0;
  if (!__syncthreads_or(any)) return;
  for (int j0 = k.lo + kAhead * (int(threadIdx.x) >> 5); j0 < k.hi; j0 += kAhead * (THREADS / 32)) {
    int64_t at[kAhead];
    uint4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = min(j0 + i, k.hi - 1), index = tl_divide(j, p.page_div), page = p.page_table[int64_t(k.seq) * p.max_pages + index];
      at[i] = tl_bad_page(page, p.n_pages) || j0 + i >= k.hi ? -1 : tl_page_at(page, j - index * p.page_size, p.n_kv_heads, p.page_size, p.head_dim) + int64_t(kvh) * p.page_size * p.head_dim + d0;
      v[i] = make_uint4(0, 0, 0, 0);
      if (at[i] >= 0 && d0 < p.head_dim) v[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const AT*>(p.v_pages) + at[i]);
    }
#pragma unroll 1
    for (int i = 0; i < kAhead; ++i) {
      const AT* e = reinterpret_cast<const AT*>(&v[i]);
      uint32_t kind = 0;  // three bits for each of the eight
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const float x = DT<AT>::to_f32(e[d]);
        kind |= uint32_t(isfinite(x) ? 0 : x != x ? kNan : x > 0.f ? kUp : kDown) << (3 * d);
      }
      if (!__any_sync(0xffffffffu, kind != 0)) continue;
#pragma unroll 1
      for (int r = 0; r < rows; ++r) {
        float x = 0.f;
        if (d0 < p.head_dim) {
          const AT *q = reinterpret_cast<const AT*>(p.q) + int64_t(t) * p.qt + int64_t(h0 + r) * p.qh + d0, *kp = reinterpret_cast<const AT*>(p.k_pages) + at[i];
#pragma unroll
          for (int d = 0; d < 8; ++d) x = fmaf(DT<AT>::to_f32(q[d]), DT<AT>::to_f32(kp[d]), x);
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        x *= p.scale;
        if (p.softcap > 0.f) x = cap(x, p.softcap, p.cap_inv, p.cap_exp);
        if (p.slopes) x = fmaf(p.slopes[h0 + r], float(int(j0 + i + 1) - k.hi), x);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const uint32_t is = (kind >> (3 * d)) & 7;
          if (is) atomicOr(&found[r * DPAD + d0 + d], x == -INFINITY ? uint32_t(kNan) : is);
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < all; i += THREADS) {
    const int r = i / p.head_dim;
    const uint32_t is = found[r * DPAD + i - r * p.head_dim];
    if (unsettled(out[i])) out[i] = DT<AT>::from_f32(is == kUp ? INFINITY : is == kDown ? -INFINITY : NAN);
  }
  __syncthreads();
}

// Probabilities are held times 2^10 in f16: the low term of their split stays clear of f16's subnormals.
template <typename AT> constexpr float kProbBias = 0.f;
template <> constexpr float kProbBias<__half> = 10.f;

// What a warp holds of the softmax of its keys, and how it takes a tile of them in: 16-bit types on the tensor cores.  A maximum of -infinity says that no key has
// been seen, and only that: from the first one on it is no less than -FLT_MAX, so that scores that are NaN (which no maximum keeps) or all -infinity end as NaN in
// the sum or as a sum of zero, whose outputs are NaN, and not as the zeros of a row that sees nothing.
// NT = 1: up to 8 query heads of a KV head, NT = 2: up to 16.
template <typename AT_, int DPAD_, int NT>
struct MmaTile {
  using AT = AT_;
  static constexpr int DPAD = DPAD_, ROWS = 8 * NT, KEYS = 16, TERMS = ProbSplit<AT>::kTerms, CTAS = kCtas, WARPS = kConsumerWarps;
  static constexpr bool kLookAgain = true;  // infinite values need it: terms of probabilities
  uint32_t q[NT][DPAD / 16][2];
  float o[NT][DPAD / 16][4], m[NT][2], l[NT][2], slope[NT][2];

  // The queries of a part, which may still be on their way while the one before it ends
  __device__ __forceinline__ void load(const PagedArgs& p, int t, int kvh, int tile) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = tile * ROWS + nt * 8 + g;
      const AT* qp = reinterpret_cast<const AT*>(p.q) + int64_t(t) * p.qt + int64_t(kvh * p.rep + row) * p.qh + 2 * c;
#pragma unroll
      for (int i = 0; i < DPAD / 16; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          q[nt][i][j] = row < p.rep && 16 * i + 8 * j < p.head_dim ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * i + 8 * j)) : 0u;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = tile * ROWS + nt * 8 + 2 * c + e;
        slope[nt][e] = p.slopes && r < p.rep ? p.slopes[kvh * p.rep + r] * kLog2e : 0.f;
      }
    }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < DPAD / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
    }
  }
  // ks, vs: the tile's keys and values; bit j of `seen`: key j counts; key0 - pos: how far the first one lies behind
  template <bool OPTIONS> __device__ __forceinline__ void take(const PagedArgs& p, uint32_t ks, uint32_t vs, uint32_t seen, int behind) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    float s[NT][4];
    {
      const int r = (lane & 7) + ((lane >> 3) & 1) * 8, half = lane >> 4;
      const uint32_t at = ks + 128 * r, x = ((r & 7) ^ half) << 4;  // 16-byte chunk 2 i + half of row r, swizzled
      float s0[NT][4], s1[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s0[nt][e] = s1[nt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < DPAD / 16; ++i) {
        uint32_t a[4];
        ldmatrix4(at + (i >> 2) * (KEYS * 128) + (x ^ ((2 * (i & 3)) << 4)), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) MmaOps<AT>::mma_free(i & 1 ? s1[nt] : s0[nt], a[0], a[1], a[2], a[3], q[nt][i][0], q[nt][i][1]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = s0[nt][e] + s1[nt][e];
    }
    uint32_t pf[NT][TERMS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // element e: key g + 8 * (e >> 1), query row 2c + (e & 1); in powers of two from here on
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = g + 8 * (e >> 1);
        float x;
        if (OPTIONS) {
          x = s[nt][e] * p.scale;
          if (p.softcap > 0.f) x = cap(x, p.softcap, p.cap_inv, p.cap_exp);
          x = fmaf(slope[nt][e & 1], float(behind + key), x * kLog2e);
        } else {
          x = s[nt][e] * (p.scale * kLog2e);
        }
        s[nt][e] = seen == 0xffffu || (seen >> key) & 1 ? x : -INFINITY;
      }
      float nm[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = fmaxf(s[nt][e], s[nt][e + 2]);
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        nm[e] = fmaxf(fmaxf(m[nt][e], v), -FLT_MAX);
      }
      if (__any_sync(0xffffffffu, nm[0] != m[nt][0] || nm[1] != m[nt][1])) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f[e] = nm[e] == m[nt][e] ? 1.f : exp2f(m[nt][e] - nm[e]);  // the first keys: exp2(-inf) = 0 on zeros
          l[nt][e] *= f[e];
          m[nt][e] = nm[e];
        }
#pragma unroll
        for (int i = 0; i < DPAD / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][i][e] *= f[e & 1];
      }
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[e] = exp2f(s[nt][e] - m[nt][e & 1] + kProbBias<AT>);
        l[nt][e & 1] += pr[e];
      }
      uint32_t a[TERMS], b[TERMS];
      ProbSplit<AT>::split(make_float2(pr[0], pr[1]), a);
      ProbSplit<AT>::split(make_float2(pr[2], pr[3]), b);
#pragma unroll
      for (int i = 0; i < TERMS; ++i) {
        pf[nt][i][0] = transpose8x8(a[i]);
        pf[nt][i][1] = transpose8x8(b[i]);
      }
    }
    const int r = (lane & 7) + (lane >> 4) * 8, half = (lane >> 3) & 1;
    const uint32_t at = vs + 128 * r, x = ((r & 7) ^ half) << 4;
#pragma unroll
    for (int i = 0; i < DPAD / 16; ++i) {
      uint32_t a[4];
      ldmatrix4_trans(at + (i >> 2) * (KEYS * 128) + (x ^ ((2 * (i & 3)) << 4)), a);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < TERMS; ++j) MmaOps<AT>::mma_free(o[nt][i], a[0], a[1], a[2], a[3], pf[nt][j][0], pf[nt][j][1]);
    }
  }
  // The warp's maxima, sums and outputs to wm[row], wl[row], wo[row * pitch + d], rows below `rows` only
  __device__ __forceinline__ void end(float* wm, float* wl, float* wo, int pitch, int rows) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = l[nt][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const int r = nt * 8 + 2 * c + e;
        if (r < rows) {
          if (g == 0) { wm[r] = m[nt][e]; wl[r] = v; }
#pragma unroll
          for (int i = 0; i < DPAD / 16; ++i) {
            wo[r * pitch + 16 * i + g] = o[nt][i][e];
            wo[r * pitch + 16 * i + g + 8] = o[nt][i][e + 2];
          }
        }
      }
  }
  // The rows' outputs straight from the registers, where the warp's keys are all there are; true if one of this lane's is not settled
  __device__ __forceinline__ bool finish(AT* out, int dim, int rows) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    bool odd = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = l[nt][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const float inv = m[nt][e] == -INFINITY ? 0.f : 1.f / v;
        const int r = nt * 8 + 2 * c + e;
        if (r < rows) {
          float none = 0.f;  // NaN if one of them is not finite
#pragma unroll
          for (int i = 0; i < DPAD / 8; ++i) {
            const float x = o[nt][i >> 1][e + 2 * (i & 1)] * inv;
            if (8 * i < dim) out[r * dim + 8 * i + g] = DT<AT>::from_f32(x);
            none = fmaf(x, 0.f, none);
          }
          if (none != none && v > 0.f) {
#pragma unroll 1
            for (int d = g; d < dim; d += 8) {
              const float x = DT<AT>::to_f32(out[r * dim + d]);
              if (x != x) { reinterpret_cast<uint16_t*>(out)[r * dim + d] = kUnsettled; odd = true; }
            }
          }
        }
      }
    return odd;
  }
};

// Sums N values over the warp, each lane ending with the one of number lane_value<N>(lane): at every step a lane keeps half of its values and hands
// over the rest, N - 1 + (5 - log2 N) shuffles in all instead of 5 N.
template <int N, int BIT = 16> __device__ __forceinline__ float sum_exchange(const float (&v)[N]) {
  if constexpr (N > 1) {
    const bool up = (threadIdx.x & BIT) != 0;
    float half[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) half[i] = (up ? v[i + N / 2] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + N / 2], BIT);
    return sum_exchange<N / 2, BIT / 2>(half);
  } else {
    float x = v[0];
#pragma unroll
    for (int b = BIT; b > 0; b >>= 1) x += __shfl_xor_sync(0xffffffffu, x, b);
    return x;
  }
}
// f32: a lane owns E neighbouring dimensions of all keys and rows; eight keys a tile.
template <int DPAD_, int ROWS_>
struct F32Tile {
  using AT = float;
  static constexpr int DPAD = DPAD_, ROWS = ROWS_, KEYS = 8, E = DPAD / 32, CTAS = kCtas, WARPS = kConsumerWarps;
  static constexpr bool kLookAgain = false;
  static constexpr int kSets = ROWS * KEYS > 32 ? ROWS * KEYS / 32 : 1, kN = ROWS * KEYS / kSets;  // kN values are summed at once
  static constexpr int kRowsOfSet = ROWS / kSets, kLog = kN == 32 ? 5 : kN == 16 ? 4 : 3;
  float q[ROWS][E], o[ROWS][E];
  float m[kSets], l[kSets], slope[kSets];  // of the row whose score this lane ends up with: its maximum, and the sum over this lane's keys

  __device__ __forceinline__ void load(const PagedArgs& p, int t, int kvh, int tile) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int row = tile * ROWS + r;
      const float* qp = reinterpret_cast<const float*>(p.q) + int64_t(t) * p.qt + int64_t(kvh * p.rep + row) * p.qh + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) q[r][e] = row < p.rep && lane * E + e < p.head_dim ? __ldg(qp + e) : 0.f;
    }
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const int row = tile * ROWS + s * kRowsOfSet + (lane >> (5 - kLog)) / KEYS;
      slope[s] = p.slopes && row < p.rep ? p.slopes[kvh * p.rep + row] * kLog2e : 0.f;
    }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] = 0.f;
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      m[s] = -INFINITY;
      l[s] = 0.f;
    }
  }
  // this lane's dimensions of row r
  static __device__ __forceinline__ void row_of(uint32_t tile_at, int r, float (&v)[E]) {
    const int lane = threadIdx.x & 31;
    if (E == 2) {
      const int c = lane >> 1;
      const uint32_t at = tile_at + (c >> 3) * (KEYS * 128) + r * 128 + (((c & 7) ^ r) << 4) + 8 * (lane & 1);
      asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[E - 1]) : "r"(at));
    } else {
#pragma unroll
      for (int e = 0; e + 3 < E; e += 4) {
        const int c = (lane * E + e) >> 2;
        const uint32_t at = tile_at + (c >> 3) * (KEYS * 128) + r * 128 + (((c & 7) ^ r) << 4);
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[e]), "=f"(v[e + 1]), "=f"(v[e + 2]), "=f"(v[e + 3]) : "r"(at));
      }
    }
  }
  template <bool OPTIONS> __device__ __forceinline__ void take(const PagedArgs& p, uint32_t ks, uint32_t vs, uint32_t seen, int behind) {
    const int lane = threadIdx.x & 31;
    float dot[kSets][kN];  // value row * KEYS + key of a set
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      float k[E];
      row_of(ks, j, k);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x = fmaf(q[r][e], k[e], x);
        dot[r / kRowsOfSet][(r % kRowsOfSet) * KEYS + j] = x;
      }
    }
    float pr[kSets];
    const int key = (lane >> (5 - kLog)) % KEYS;
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float x = sum_exchange<kN>(dot[s]);
      if (OPTIONS) {
        x *= p.scale;
        if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
        x = fmaf(slope[s], float(behind + key), x * kLog2e);
      } else {
        x *= p.scale * kLog2e;
      }
      x = (seen >> key) & 1 ? x : -INFINITY;
      float top = x;  // over the keys of a row: lanes that differ in the key's bits
#pragma unroll
      for (int b = 1 << (5 - kLog); b < KEYS << (5 - kLog); b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
      const float nm = fmaxf(fmaxf(m[s], top), -FLT_MAX);
      if (__any_sync(0xffffffffu, nm != m[s])) {
        const float f = nm == m[s] ? 1.f : exp2f(m[s] - nm);
        m[s] = nm;
        l[s] *= f;
#pragma unroll
        for (int i = 0; i < kRowsOfSet; ++i) {
          const float g = __shfl_sync(0xffffffffu, f, (i * KEYS) << (5 - kLog));
#pragma unroll
          for (int e = 0; e < E; ++e) o[s * kRowsOfSet + i][e] *= g;
        }
      }
      pr[s] = exp2f(x - nm);
      l[s] += pr[s];
    }
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      float v[E];
      row_of(vs, j, v);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float w = __shfl_sync(0xffffffffu, pr[r / kRowsOfSet], ((r % kRowsOfSet) * KEYS + j) << (5 - kLog));
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = fmaf(w, v[e], o[r][e]);
      }
    }
  }
  __device__ __forceinline__ void end(float* wm, float* wl, float* wo, int pitch, int rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float v = l[s];
#pragma unroll
      for (int b = 1 << (5 - kLog); b < KEYS << (5 - kLog); b <<= 1) v += __shfl_xor_sync(0xffffffffu, v, b);
      const int r = s * kRowsOfSet + (lane >> (5 - kLog)) / KEYS;
      if ((lane & ((KEYS << (5 - kLog)) - 1)) == 0 && r < rows) { wm[r] = m[s]; wl[r] = v; }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < rows)
#pragma unroll
        for (int e = 0; e < E; ++e) wo[r * pitch + lane * E + e] = o[r][e];
  }
  __device__ __forceinline__ bool finish(float* out, int dim, int rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float v = l[s];
#pragma unroll
      for (int b = 1 << (5 - kLog); b < KEYS << (5 - kLog); b <<= 1) v += __shfl_xor_sync(0xffffffffu, v, b);
      const float inv = m[s] == -INFINITY ? 0.f : 1.f / v;
#pragma unroll
      for (int i = 0; i < kRowsOfSet; ++i) {
        const float f = __shfl_sync(0xffffffffu, inv, (i * KEYS) << (5 - kLog));
        const int r = s * kRowsOfSet + i;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (r < rows && lane * E + e < dim) out[r * dim + lane * E + e] = o[r][e] * f;
      }
    }
    return false;
  }
};

// A stage of the ring: a tile's keys, then its values, each in boxes of KEYS rows of 128 bytes (16-byte chunk c of row r at c ^ (r & 7)).
template <class Tile> constexpr int kBoxBytes = Tile::KEYS * 128;
template <class Tile> constexpr int kBoxes = Tile::DPAD * int(sizeof(typename Tile::AT)) / 128;
template <class Tile> constexpr int kStageBytes = 2 * kBoxes<Tile> * kBoxBytes<Tile>;
// Behind the ring: [warps][rows][DPAD + 4] outputs, [warps][rows] maxima and [warps][rows] sums of the consumer warps (the pitch keeps the lanes of a quad in
// banks of their own), which join() uses too.
template <class Tile> constexpr int kPitch = Tile::DPAD + 4;
template <class Tile> constexpr int area_bytes(int rows) { return Tile::WARPS * rows * (2 + kPitch<Tile>) * int(sizeof(float)); }
// A part in scratch: [ROWS][DPAD] outputs, then [ROWS] maxima and [ROWS] sums; whole 16-byte vectors
template <class Tile> __host__ __device__ constexpr int slot_floats() { return Tile::ROWS * Tile::DPAD + (2 * Tile::ROWS + 3) / 4 * 4; }
template <class Tile> constexpr int kSlotMax = Tile::ROWS * Tile::DPAD;
template <class Tile> constexpr int kSlotSum = kSlotMax<Tile> + Tile::ROWS;

// The slot in which CTA first + i of a token's CTAs leaves its part: the first of them starts the token, the others have it begun elsewhere.
__device__ __forceinline__ int slot_of(int first, int i) { return 2 * (first + i) + (i == 0 ? 1 : 0); }
// Parts i = from, from + step, ... of a token, `count` of them (at most 32), by all threads of the CTA: write(e, output, maximum, sum) gets four
// neighbouring values of [rows][DPAD] from e on, not yet divided by the sum.  The loads of kGroup of them are on their way together.  area: rows * 34 floats.
template <class Tile, typename W> __device__ __forceinline__ void join(const float* slots, int first, int from, int step, int count, int rows, float* area, W&& write) {
  constexpr int kThreads = 32 + kConsumers<Tile>, kItems = (Tile::ROWS * Tile::DPAD / 4 + kThreads - 1) / kThreads, kTogether = kItems > 2 ? 2 : kItems;
  float *maxima = area, *sums = maxima + rows, *factor = sums + rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto part = [&](int i) { return slots + int64_t(slot_of(first, from + i * step)) * slot_floats<Tile>(); };
  float4 v[kTogether][kGroup];
  auto fetch = [&](int e0, int i0) {
#pragma unroll
    for (int k = 0; k < kTogether; ++k)
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int e = e0 + 4 * (k * kThreads + int(threadIdx.x));
        if (i0 + i < count && e < rows * Tile::DPAD) v[k][i] = __ldcg(reinterpret_cast<const float4*>(part(i0 + i) + e));
      }
  };
  fetch(0, 0);
  for (int r = warp; r < rows; r += kThreads / 32) {
    float mx = -INFINITY, sum = 0.f;
    if (lane < count) { mx = __ldcg(part(lane) + kSlotMax<Tile> + r); sum = __ldcg(part(lane) + kSlotSum<Tile> + r); }
    float top = mx;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = mx == -INFINITY ? 0.f : exp2f(mx - top);
    sum *= f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < count) factor[r * 32 + lane] = f;
    if (lane == 0) { maxima[r] = top; sums[r] = sum; }
  }
  __syncthreads();
#pragma unroll 1
  for (int e0 = 0; e0 < rows * Tile::DPAD; e0 += 4 * kTogether * kThreads) {
    float4 a[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += kGroup) {
      if (e0 + i0 > 0) fetch(e0, i0);
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const int r = min((e0 + 4 * (k * kThreads + int(threadIdx.x))) / Tile::DPAD, rows - 1);
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          if (i0 + i < count) {
            const float f = factor[r * 32 + i0 + i];
            a[k].x = fmaf(f, v[k][i].x, a[k].x); a[k].y = fmaf(f, v[k][i].y, a[k].y);
            a[k].z = fmaf(f, v[k][i].z, a[k].z); a[k].w = fmaf(f, v[k][i].w, a[k].w);
          }
      }
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int e = e0 + 4 * (k * kThreads + int(threadIdx.x)), r = min(e / Tile::DPAD, rows - 1);
      write(e, a[k], maxima[r], sums[r]);  // by whole warps; e may lie past the end
    }
  }
}
// What the CTAs of a part have left in their slots before this is seen by the one that comes last
__device__ __forceinline__ bool arrive(unsigned* at, int of) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(at) : "memory");
  if (old != unsigned(of) - 1) return false;
  *at = 0;  // for the next launch
  return true;
}

template <class Tile, bool OPTIONS, bool TMA>
__global__ void __launch_bounds__(32 + kConsumers<Tile>, Tile::CTAS)
    paged_attention_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using AT = typename Tile::AT;
  constexpr int DPAD = Tile::DPAD, KEYS = Tile::KEYS, WARPS = Tile::WARPS, kThreads = 32 + kConsumers<Tile>;
  constexpr int kHalf = kStageBytes<Tile> / 2, kPerChunk = 16 / int(sizeof(AT));
  constexpr uint32_t kAll = (1u << KEYS) - 1;
  extern __shared__ __align__(1024) uint8_t sm[];
  struct Part {
    int t, kvh, tile, n;
    Token k;
    long long tile0;
    int left;  // in a slot: other CTAs have tiles of it too
  };
  __shared__ Part first, cut[2];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ uint32_t seen_of[kMaxStages];
  __shared__ long long found_begin, scan[kThreads / 32];
  __shared__ int found_token, is_last[2], groups_done, any_unsettled, abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = int(blockIdx.x);
  if (int(threadIdx.x) < p.stages) {
    mbar_init(&full[threadIdx.x], TMA ? 1 : 33);  // cp.async: every lane's copies, and the word of what is seen
    mbar_init(&empty[threadIdx.x], 1);
    seen_of[threadIdx.x] = 0xffff0000u;  // no lap's
    mbar_fence_init();
  }
  if (threadIdx.x == 0) {
    any_unsettled = abort_flag = is_last[0] = is_last[1] = cut[0].left = cut[1].left = 0;
    if (TMA) { tma_prefetch_desc(&k_map); tma_prefetch_desc(&v_map); }
  }
  if (p.head_dim < DPAD) {  // no copy writes the padding: it is zero from here on
    for (int i = threadIdx.x; i < p.stages * (kStageBytes<Tile> / 16); i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  tl_pdl_wait();

  // What all tokens cost, and where this CTA's share begins: by every warp for itself where tokens are few, else by the threads together
  const int segs = p.n_kv_heads * p.row_tiles;
  const bool wide = p.tokens > 256;
  const int id = wide ? int(threadIdx.x) : lane, chunk = (p.tokens + (wide ? kThreads : 32) - 1) / (wide ? kThreads : 32);
  const int t_first = min(p.tokens, id * chunk), t_end = min(p.tokens, t_first + chunk);
  auto cost_of = [&](const Token& k) {
    const int n = tl_tiles(k.lo, k.hi, KEYS);
    return n ? n + kLead : 0;
  };
  long long mine = 0;
  bool nothing = false;  // one of these tokens sees nothing
  Token k{0, 0, 0};
  for (int t = t_first; t < t_end; ++t) {
    k = token_of(p, t, false);
    mine += cost_of(k);
    nothing |= k.hi == 0;
  }
  long long to = mine, whole;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, to, o);
    if (lane >= o) to += v;
  }
  whole = __shfl_sync(0xffffffffu, to, 31);
  if (wide) {
    if (lane == 31) scan[warp] = to;
    __syncthreads();
    whole = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) to += scan[w];
      whole += scan[w];
    }
  }
  if (wide ? __syncthreads_or(nothing) : __any_sync(0xffffffffu, nothing))
    for (int t = cta; t < p.tokens; t += int(gridDim.x))
      if (token_of(p, t, threadIdx.x == 0).hi == 0)
        for (int e = threadIdx.x; e < p.n_heads * p.head_dim; e += kThreads)
          reinterpret_cast<AT*>(p.out)[int64_t(t) * p.n_heads * p.head_dim + e] = DT<AT>::from_f32(0.f);
  if (whole == 0) return;
  const TlShares shares = tl_shares(whole * segs, int(gridDim.x), kLeastUnits, (long long)(p.tokens) * segs);
  if (cta >= shares.ctas) return;
  const long long begin = tl_share_begin(shares, cta), end = tl_share_begin(shares, cta + 1);
  Cursor c;
  long long into = 0;  // how far the share's begin lies in the units of its token
  const bool found = (to - mine) * segs <= begin && begin < to * segs;  // one thread's
  c.t = t_first;
  if (found) {
    into = begin - (to - mine) * segs;
    if (chunk > 1)
      for (;; ++c.t) {
        k = token_of(p, c.t, false);
        const long long n = (long long)(cost_of(k)) * segs;
        if (into < n) break;
        into -= n;
      }
  }
  if (wide) {
    if (found) { found_token = c.t; found_begin = into; }
    __syncthreads();
    c.t = found_token;
    into = found_begin;
    c.template open<KEYS>(p);
  } else {
    const int from = __ffs(__ballot_sync(0xffffffffu, found)) - 1;
    c.t = __shfl_sync(0xffffffffu, c.t, from);
    into = __shfl_sync(0xffffffffu, into, from);
    c.k.lo = __shfl_sync(0xffffffffu, k.lo, from);
    c.k.hi = __shfl_sync(0xffffffffu, k.hi, from);
    c.k.seq = __shfl_sync(0xffffffffu, k.seq, from);
    c.n = tl_tiles(c.k.lo, c.k.hi, KEYS);
  }
  c.seg = int(tl_quotient(into, c.n + kLead));
  c.head(p);
  long long tile0 = begin - (into - (long long)(c.seg) * (c.n + kLead)) + kLead;  // the unit of the part's first tile
  // The part's tiles in the share are [c.u, stop)
  int stop;
  auto clip = [&]() {
    c.u = int(max(0ll, begin - tile0));
    stop = int(min((long long)(c.n), end - tile0));
  };
  auto advance = [&]() {  // to the next part; false: the share ends here
    tile0 += c.n + kLead;
    if (tile0 >= end) return false;
    c.template next<KEYS>(p);
    clip();
    return true;
  };
  clip();
  if (Tile::kLookAgain && threadIdx.x == 0) first = Part{c.t, c.kvh, c.tile, c.n, c.k, tile0, 0};

  if (warp == WARPS) {
    // ---- the producer.  A lane looks up a tile's page (cp.async: a row's) a batch before it is copied, so that the table is read on the way.
    constexpr int kBatch = TMA ? 32 : 1;
    struct Batch {
      int n, key0, kvh, key, page;  // n tiles from key0 on; this lane's key and its page
      Token k;
    };
    bool more = true;
    auto look_up = [&]() {
      Batch b;
      b.n = 0;
      while (more && c.u >= stop) more = advance();
      if (!more) return b;
      b.n = min(kBatch, stop - c.u);
      b.k = c.k;
      b.kvh = c.kvh;
      b.key0 = c.template first_key<KEYS>(c.u);
      b.key = b.key0 + (TMA ? lane * KEYS : lane);
      b.page = -1;
      if (TMA ? lane < b.n : lane < KEYS && b.key >= b.k.lo && b.key < b.k.hi) b.page = __ldg(p.page_table + int64_t(b.k.seq) * p.max_pages + tl_divide(b.key, p.page_div));
      c.u += b.n;
      return b;
    };
    Batch now = look_up();
    int stage = 0, lap = 0, issued = 0;
    const int boxes = 2 * ((p.head_dim * int(sizeof(AT)) + 127) / 128), at_once = min(min(4, 32 / boxes), p.stages), my_tile = lane / boxes, my_box = lane % boxes;
    bool ok = true;
    while (now.n > 0 && ok) {
      const Batch then = look_up();
      const bool wanted = TMA ? lane < now.n : lane < KEYS && now.key >= now.k.lo && now.key < now.k.hi, there = wanted && !tl_bad_page(now.page, p.n_pages);
      if (wanted && !there) atomicOr(p.status, kBadPage);
      const int in_page = now.key - tl_divide(now.key, p.page_div) * p.page_size;
      const int64_t row = (int64_t(now.page) * p.n_kv_heads + now.kvh) * p.page_size + in_page;
      if (TMA) {
        // Some tiles at once, a lane for each box: a copy costs a warp about 50 ns to issue, whichever lanes do
        for (int j = 0; j < now.n; j += at_once) {
          const int n = min(at_once, now.n - j), key0 = now.key0 + (j + my_tile) * KEYS;
          const int y = __shfl_sync(0xffffffffu, int(row), j + my_tile);
          const bool mine = my_tile < n, copied = __shfl_sync(0xffffffffu, int(there), j + my_tile) != 0;
          int to_stage = stage + my_tile, to_lap = lap;
          if (to_stage >= p.stages) { to_stage -= p.stages; ++to_lap; }
          // (the first lap: the phase before the first)
          if (!__all_sync(0xffffffffu, !mine || mbar_wait(&empty[to_stage], (to_lap & 1) ^ 1, &abort_flag))) { ok = false; break; }
          if (mine && my_box == 0) {
            uint32_t seen = kAll;
            if (key0 < now.k.lo) seen &= kAll << (now.k.lo - key0);
            if (key0 + KEYS > now.k.hi) seen &= kAll >> (key0 + KEYS - now.k.hi);
            publish(&seen_of[to_stage], to_lap, copied ? seen : 0);
            if (copied) mbar_expect_tx(&full[to_stage], uint32_t(boxes * kBoxBytes<Tile>));
            else mbar_arrive(&full[to_stage]);
          }
          __syncwarp();
          if (mine && copied) {
            const int half = boxes >> 1, b = my_box < half ? my_box : my_box - half;
            tma_load_2d(sm + to_stage * kStageBytes<Tile> + (my_box < half ? 0 : kHalf) + b * kBoxBytes<Tile>, my_box < half ? &k_map : &v_map,
                        b * (128 / int(sizeof(AT))), y, &full[to_stage]);
          }
          issued += n;
          stage += n;
          if (stage >= p.stages) { stage -= p.stages; ++lap; }
        }
      } else {
        if (!mbar_wait_all(&empty[stage], (lap & 1) ^ 1, &abort_flag)) { ok = false; break; }
        const uint32_t seen = __ballot_sync(0xffffffffu, there);
        const uint32_t ks = smem_u32(sm + stage * kStageBytes<Tile>), vs = ks + kHalf;
        const int chunks = p.head_dim / kPerChunk;
        for (int r = 0; r < KEYS; ++r) {
          const int64_t from = __shfl_sync(0xffffffffu, row, r) * p.head_dim;
          const int bytes = (seen >> r) & 1 ? 16 : 0;
          for (int ch = lane; ch < chunks; ch += 32) {
            const uint32_t to_at = (ch >> 3) * kBoxBytes<Tile> + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
            const int64_t e = bytes ? from + ch * kPerChunk : 0;
            copy16(ks + to_at, reinterpret_cast<const AT*>(p.k_pages) + e, bytes);
            copy16(vs + to_at, reinterpret_cast<const AT*>(p.v_pages) + e, bytes);
          }
        }
        copy_arrive(&full[stage]);
        if (lane == 0) {
          publish(&seen_of[stage], lap, seen);
          mbar_arrive(&full[stage]);
        }
        if (++stage == p.stages) { stage = 0; ++lap; }
      }
      now = then;
    }
    if (!ok) {
      if (lane == 0) { atomicExch(&abort_flag, 1); atomicExch(p.wait_status, TL_DEV_TIMEOUT_EMPTY); }
      if (TMA && lane == 0) tma_drain(full, p.stages, issued);
      if (!TMA) asm volatile("cp.async.wait_all;" ::: "memory");
    }
  }

  // ---- the consumers take the share's tiles in turn; a part of few tiles is one warp's, which then needs nobody else
  constexpr int kSmall = 4;
  float* area = reinterpret_cast<float*>(sm + p.stages * kStageBytes<Tile>);
  // Four neighbouring values of a row by each thread
  auto store = [&](const Part& w, int h0, int e, float4 o, float top, float sum) {
    const int r = e / DPAD, d = e - r * DPAD;
    const float inv = top == -INFINITY ? 0.f : 1.f / sum;  // 0: no key's page is there, nothing is seen
    const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    if (d < p.head_dim) {
      AT* to_at = reinterpret_cast<AT*>(p.out) + (int64_t(w.t) * p.n_heads + h0 + r) * p.head_dim + d;
      if (sizeof(AT) == 4) {
        *reinterpret_cast<float4*>(to_at) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        AT h[4];
        float none = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[j] = DT<AT>::from_f32(v[j]);
          none = fmaf(v[j], 0.f, none);
        }
        if (none != none && sum > 0.f) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (v[j] != v[j]) {
              reinterpret_cast<uint16_t&>(h[j]) = kUnsettled;
              any_unsettled = 1;
            }
        }
        *reinterpret_cast<uint2*>(to_at) = *reinterpret_cast<const uint2*>(h);
      }
    }
  };
  if (warp < WARPS) {
    int before = 0, small = 0;  // the share's tiles before this part; parts that were one warp's
    bool ok = true, met = true;
    auto settle = [&](bool more) {
      while (more && c.u >= stop) more = advance();
      return more;
    };
    Tile tile;
    bool more = settle(true);
    if (more) tile.load(p, c.t, c.kvh, c.tile);
    while (more) {
      const int u = c.u, count = stop - u;
      const bool starts = u == 0, ends = stop == c.n, alone = starts && ends && c.n <= kSmall, mine = !alone || small++ % WARPS == warp;
      const Part part{c.t, c.kvh, c.tile, c.n, c.k, tile0, !(starts && ends)};
      const int rows = min(Tile::ROWS, p.rep - part.tile * Tile::ROWS), h0 = part.kvh * p.rep + part.tile * Tile::ROWS;
      if (mine) {
        tile.reset();
        for (int j = alone ? 0 : (warp + WARPS - before % WARPS) % WARPS; j < count; j += alone ? 1 : WARPS) {
          const int lap = tl_divide(before + j, p.stage_div), stage = before + j - lap * p.stages;
          uint32_t seen = 0;
          if (ok && !tile_ready(&seen_of[stage], &full[stage], lap, &abort_flag, seen)) {
            ok = false;
            if (lane == 0) { atomicExch(&abort_flag, 1); atomicExch(p.wait_status, TL_DEV_TIMEOUT_FULL); }
          }
          if (ok) {
            const uint32_t ks = smem_u32(sm + stage * kStageBytes<Tile>);
            if (seen) {
              if (TMA && seen != kAll) {  // values that do not count, whatever they are
                for (int i = lane; i < KEYS * kBoxes<Tile> * 8; i += 32) {
                  const int r = (i >> 3) % KEYS;
                  if (!((seen >> r) & 1)) reinterpret_cast<uint4*>(sm + stage * kStageBytes<Tile> + kHalf)[i] = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
              }
              tile.template take<OPTIONS>(p, ks, ks + kHalf, seen, c.template first_key<KEYS>(u + j) + 1 - part.k.hi);
              if (TMA && seen != kAll) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
          }
        }
      }
      before += count;
      more = settle(advance());
      if (more) tile.load(p, c.t, c.kvh, c.tile);

      // The end of the part, or of this CTA's share of it
      if (alone) {
        if (mine) {
          const bool odd = tile.finish(reinterpret_cast<AT*>(p.out) + (int64_t(part.t) * p.n_heads + h0) * p.head_dim, p.head_dim, rows);
          if (odd) any_unsettled = 1;
        }
        continue;
      }
      float *wo = area, *wm = wo + WARPS * rows * kPitch<Tile>, *wl = wm + WARPS * rows;
      if (!met) consumers_meet<Tile>();  // the area is free again
      met = false;
      tile.end(wm + warp * rows, wl + warp * rows, wo + warp * rows * kPitch<Tile>, kPitch<Tile>, rows);
      consumers_meet<Tile>();
      float* slot = p.slots + int64_t(2 * cta + (starts ? 1 : 0)) * slot_floats<Tile>();
      for (int e0 = warp * 128; e0 < rows * DPAD; e0 += WARPS * 128) {
        const int e = e0 + 4 * lane, r = min(e, rows * DPAD - 1) / DPAD, d = e - r * DPAD;
        const bool here = e < rows * DPAD;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
        if (here) {
#pragma unroll
          for (int i = 0; i < WARPS; ++i) top = fmaxf(top, wm[i * rows + r]);
#pragma unroll
          for (int i = 0; i < WARPS; ++i) {
            const float mx = wm[i * rows + r], g = mx == -INFINITY ? 0.f : exp2f(mx - top);
            const float4 w = *reinterpret_cast<const float4*>(wo + (i * rows + r) * kPitch<Tile> + d);
            sum = fmaf(wl[i * rows + r], g, sum);
            o.x = fmaf(w.x, g, o.x); o.y = fmaf(w.y, g, o.y); o.z = fmaf(w.z, g, o.z); o.w = fmaf(w.w, g, o.w);
          }
        }
        if (!here) continue;
        if (!part.left) {
          store(part, h0, e, o, top, sum);
        } else {
          if (d == 0) { __stcg(slot + kSlotMax<Tile> + r, top); __stcg(slot + kSlotSum<Tile> + r, sum); }
          __stcg(reinterpret_cast<float4*>(slot + e), o);
        }
      }
      if (part.left && threadIdx.x == 0) cut[starts ? 1 : 0] = part;
    }
  }

  // What others have tiles of too: at most the part that the share's begin cuts and the one that its end cuts.  Only now: a fence and an atomic take microseconds
  // while the copies are at full rate, and the next part's tiles would wait behind them (8 x 8 x 4000 keys: CTAs with a cut inside their share
  // ended 5 to 9 us after the others).  A part's CTAs are head .. head + ctas - 1; whoever comes last of a group of kGroup joins what the group
  // has left, in the place of the first of them, and whoever ends the last group joins the groups'.
  __syncthreads();
  struct Crowd {
    int head, group, groups, members;
  };
  auto crowd_of = [&](const Part& w) {
    Crowd g;
    g.head = tl_share_owner(shares, w.tile0);
    const int ctas = tl_share_owner(shares, w.tile0 + w.n - 1) - g.head + 1;
    g.group = (cta - g.head) / kGroup;
    g.groups = (ctas + kGroup - 1) / kGroup;
    g.members = min(kGroup, ctas - g.group * kGroup);
    return g;
  };
  if (threadIdx.x < 2 && cut[threadIdx.x].left) {
    const Crowd g = crowd_of(cut[threadIdx.x]);
    is_last[threadIdx.x] = arrive(p.arrivals + slot_of(g.head, g.group * kGroup), g.members);
  }
  __syncthreads();
  if ((is_last[0] | is_last[1] | any_unsettled) == 0) return;
  unsigned joined = 0;
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (!is_last[i]) continue;
    const Part w = cut[i];
    const Crowd g = crowd_of(w);
    const int rows = min(Tile::ROWS, p.rep - w.tile * Tile::ROWS), h0 = w.kvh * p.rep + w.tile * Tile::ROWS;
    bool whole_part = g.groups == 1;
#pragma unroll 1
    for (int level = 0; level < 2; ++level) {
      float* to_slot = p.slots + int64_t(slot_of(g.head, g.group * kGroup)) * slot_floats<Tile>();
      __syncthreads();  // the area is free
      join<Tile>(p.slots, g.head, level == 0 ? g.group * kGroup : 0, level == 0 ? 1 : kGroup, level == 0 ? g.members : g.groups, rows, area,
                 [&](int e, float4 o, float top, float sum) {
                   const bool here = e < rows * DPAD;
                   if (!here) return;
                   if (whole_part) {
                     store(w, h0, e, o, top, sum);
                   } else {
                     __stcg(reinterpret_cast<float4*>(to_slot + e), o);
                     if (e % DPAD == 0) { __stcg(to_slot + kSlotMax<Tile> + e / DPAD, top); __stcg(to_slot + kSlotSum<Tile> + e / DPAD, sum); }
                   }
                 });
      if (whole_part) break;
      __syncthreads();
      if (threadIdx.x == 0) groups_done = arrive(p.arrivals + 2 * gridDim.x + g.head, g.groups);
      __syncthreads();
      if (!groups_done) break;
      whole_part = true;
    }
    joined |= unsigned(whole_part) << i;
  }

  // Outputs that are not settled, now that the ring is empty: while one warp walked a sequence the others' waits would run out
  if constexpr (Tile::kLookAgain) {
    __syncthreads();
    if (!any_unsettled) return;
    auto again = [&](int t, int kvh, int tile, const Token& k) {
      look_again<AT, DPAD, kThreads>(p, k, t, kvh, kvh * p.rep + tile * Tile::ROWS, min(Tile::ROWS, p.rep - tile * Tile::ROWS), reinterpret_cast<uint32_t*>(area));
    };
#pragma unroll 1
    for (int i = 0; i < 2; ++i)
      if ((joined >> i) & 1) again(cut[i].t, cut[i].kvh, cut[i].tile, cut[i].k);
    c.t = first.t; c.kvh = first.kvh; c.tile = first.tile; c.n = first.n; c.k = first.k;
    c.seg = c.kvh * p.row_tiles + c.tile;
    tile0 = first.tile0;
    clip();
    do {
      if (c.u == 0 && stop == c.n) again(c.t, c.kvh, c.tile, c.k);
    } while (advance());
  }
}

template <class Tile, bool OPTIONS, bool TMA>
cudaError_t launch(tl_ctx* ctx, PagedArgs& p, const CUtensorMap& k_map, const CUtensorMap& v_map, int64_t most_units) {
  // Shared memory in equal parts for the resident CTAs (1 KB of each is the system's, the barriers take less than another)
  const int rows = std::min(Tile::ROWS, p.rep), room = (228 / Tile::CTAS - 1) * 1024 - 2048 - area_bytes<Tile>(rows);
  p.stages = std::min(kMaxStages, room / kStageBytes<Tile>);
  p.stage_div = tl_divide_by(p.stages);
  const int smem = p.stages * kStageBytes<Tile> + area_bytes<Tile>(rows);
  auto kernel = paged_attention_kernel<Tile, OPTIONS, TMA>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(std::min<int64_t>(int64_t(ctx->sm_count) * Tile::CTAS, std::max<int64_t>(1, most_units))));
  cfg.blockDim = dim3(32 + kConsumers<Tile>);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1] = {tl_pdl_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, k_map, v_map);
}
template <class Tile> cudaError_t launch_tile(tl_ctx* ctx, PagedArgs& p, int64_t longest) {
  using AT = typename Tile::AT;
  p.row_tiles = (p.rep + Tile::ROWS - 1) / Tile::ROWS;
  const int64_t most = int64_t(p.tokens) * p.n_kv_heads * p.row_tiles * (longest / Tile::KEYS + 2);
  // TMA boxes are whole 128-byte columns of a tile's rows, which are neighbours where a page holds whole tiles; their coordinates are int32
  const int64_t all_rows = p.n_pages * p.n_kv_heads * p.page_size;
  CUtensorMap k_map{}, v_map{};
  constexpr int kColumns = 128 / int(sizeof(AT));
  const bool tma = p.page_size % Tile::KEYS == 0 && p.head_dim >= kColumns && all_rows > 0 && all_rows <= INT32_MAX &&
                   tl_encode_tmap_2d(&k_map, int(sizeof(AT)), p.k_pages, uint64_t(p.head_dim), uint64_t(all_rows), uint64_t(p.head_dim) * sizeof(AT), kColumns,
                                     Tile::KEYS, 3) &&
                   tl_encode_tmap_2d(&v_map, int(sizeof(AT)), p.v_pages, uint64_t(p.head_dim), uint64_t(all_rows), uint64_t(p.head_dim) * sizeof(AT), kColumns,
                                     Tile::KEYS, 3);
  const bool options = p.softcap > 0.f || p.slopes;
  if (tma) return options ? launch<Tile, true, true>(ctx, p, k_map, v_map, most) : launch<Tile, false, true>(ctx, p, k_map, v_map, most);
  return options ? launch<Tile, true, false>(ctx, p, k_map, v_map, most) : launch<Tile, false, false>(ctx, p, k_map, v_map, most);
}
// Up to 8 query heads of a KV head on one tile, up to 16 on a tile of two, more on several; 256 dimensions leave registers for 8 (f32: 4).
template <typename AT> cudaError_t launch_mma(tl_ctx* ctx, PagedArgs& p, int64_t longest) {
  if (p.head_dim <= 64) return p.rep <= 8 ? launch_tile<MmaTile<AT, 64, 1>>(ctx, p, longest) : launch_tile<MmaTile<AT, 64, 2>>(ctx, p, longest);
  if (p.head_dim <= 128) return p.rep <= 8 ? launch_tile<MmaTile<AT, 128, 1>>(ctx, p, longest) : launch_tile<MmaTile<AT, 128, 2>>(ctx, p, longest);
  return launch_tile<MmaTile<AT, 256, 1>>(ctx, p, longest);
}
cudaError_t launch_f32(tl_ctx* ctx, PagedArgs& p, int64_t longest) {
  if (p.head_dim <= 64)
    return p.rep == 1 ? launch_tile<F32Tile<64, 1>>(ctx, p, longest) : p.rep <= 4 ? launch_tile<F32Tile<64, 4>>(ctx, p, longest) : launch_tile<F32Tile<64, 8>>(ctx, p, longest);
  if (p.head_dim <= 128)
    return p.rep == 1 ? launch_tile<F32Tile<128, 1>>(ctx, p, longest) : p.rep <= 4 ? launch_tile<F32Tile<128, 4>>(ctx, p, longest) : launch_tile<F32Tile<128, 8>>(ctx, p, longest);
  return p.rep == 1 ? launch_tile<F32Tile<256, 1>>(ctx, p, longest) : launch_tile<F32Tile<256, 4>>(ctx, p, longest);
}

// Parts of tokens for two CTAs an SM of the largest slot, and the arrivals: one size for all calls, so that no captured call's scratch is replaced.
constexpr int kSlotFloats = 16 * 130;
static_assert(kGroup * 32 >= 160 * kCtas, "two levels are enough for so many SMs");
static_assert(kMaxStages <= 32 + 32 * kConsumerWarps, "a barrier a thread");
static_assert(slot_floats<MmaTile<__half, 64, 2>>() <= kSlotFloats && slot_floats<F32Tile<256, 4>>() <= kSlotFloats && slot_floats<F32Tile<128, 8>>() <= kSlotFloats, "slots");
static_assert(slot_floats<MmaTile<__half, 256, 1>>() <= kSlotFloats && slot_floats<MmaTile<__half, 128, 2>>() <= kSlotFloats, "slots");
int32_t secure_scratch(tl_ctx* ctx) {
  if (ctx->paged_scratch) return TL_OK;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (!ctx->capturing) TL_CUDA(ctx, cudaStreamIsCapturing(ctx->stream, &capture));
  if (ctx->capturing || capture != cudaStreamCaptureStatusNone)
    return tl_set_error(ctx, TL_ERR_UNSUPPORTED, "tl_paged_attention: its scratch is not there yet during graph capture; run the call once before capturing");
  const size_t ctas = size_t(ctx->sm_count) * 2, bytes = ctas * (2 * kSlotFloats * sizeof(float) + 3 * sizeof(unsigned));
  const cudaError_t e = tl_zeroed(ctx->pool, &ctx->paged_scratch, bytes, ctx->stream);
  if (e == cudaErrorMemoryAllocation) {
    cudaGetLastError();
    return tl_set_error(ctx, TL_ERR_OOM, "tl_paged_attention: scratch of %zu bytes failed: %s", bytes, cudaGetErrorString(e));
  }
  TL_CUDA(ctx, e);
  ctx->paged_scratch_bytes = bytes;
  return TL_OK;
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
  if (!std::isfinite(scale) || !std::isfinite(softcap) || (softcap != 0.f && softcap < 1e-30f) || window < 0)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: scale and softcap must be finite, softcap 0 or at least 1e-30, window not negative");
  if (tokens == 0) return TL_OK;
  if (!q || !out) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: null pointer");
  const int64_t esz = int64_t(tl_dtype_size(cache->dtype));
  if (q_token_stride < 0 || q_head_stride < 0 || (q_token_stride * esz) % 16 != 0 || (q_head_stride * esz) % 16 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache->k_pages) |
        reinterpret_cast<uintptr_t>(cache->v_pages)) & 15) != 0)
    return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: pages, q, out and q's strides must be multiples of 16 bytes");
  // A token's queries are read by more than one CTA, and again behind its first outputs where values are infinite
  if (q == out) return tl_set_error(ctx, TL_ERR_INVALID_ARG, "tl_paged_attention: out overlaps q");
  DeviceGuard guard(ctx->device);
  rc = secure_scratch(ctx);
  if (rc != TL_OK) return rc;
  PagedArgs p{};
  p.q = q; p.k_pages = cache->k_pages; p.v_pages = cache->v_pages; p.out = out;
  p.page_table = cache->page_table; p.positions = positions; p.token_seq = token_seq; p.slopes = slopes;
  p.qt = q_token_stride; p.qh = q_head_stride; p.n_pages = cache->n_pages;
  p.tokens = int32_t(tokens); p.n_heads = int32_t(n_heads); p.n_kv_heads = cache->n_kv_heads; p.rep = int32_t(n_heads / cache->n_kv_heads);
  p.head_dim = cache->head_dim; p.page_size = cache->page_size; p.n_seqs = cache->n_seqs; p.max_pages = cache->max_pages;
  p.window = window; p.scale = scale; p.softcap = softcap; p.cap_inv = softcap > 0.f ? 1.f / softcap : 0.f; p.cap_exp = softcap > 0.f ? 2.f * kLog2e / softcap : 0.f;
  p.page_div = tl_divide_by(cache->page_size);
  p.status = ctx->dev_status + 1;
  p.wait_status = ctx->dev_status;
  p.slots = reinterpret_cast<float*>(ctx->paged_scratch);
  p.arrivals = reinterpret_cast<unsigned*>(p.slots + size_t(ctx->sm_count) * 2 * 2 * kSlotFloats);
  int64_t longest = int64_t(cache->max_pages) * cache->page_size;
  if (window > 0) longest = std::min<int64_t>(longest, window);
  TL_CUDA(ctx, cache->dtype == TL_F32 ? launch_f32(ctx, p, longest)
                                      : cache->dtype == TL_F16 ? launch_mma<__half>(ctx, p, longest) : launch_mma<__nv_bfloat16>(ctx, p, longest));
  ctx->counters[TL_COUNTER_KERNEL_LAUNCHES]++;
  tl_wrote(ctx, out, tokens * n_heads * cache->head_dim * esz, true);
  return TL_OK;
}

}  // extern "C"
