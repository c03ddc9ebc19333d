// Attention of one new token per row over a paged cache (include/tlcuda.h, tl_paged_attention).
//
//   x_j = cap(q . k_j * scale) + slope (j - p),   out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m)
//
// in one pass over the keys, with the running maximum m, sum and output of the softmax in f32 registers.  Bound: HBM, the cache is read once.
//
// Work.  The keys of all tokens are cut into units (64 keys of one token and one KV head's query heads), and the units dealt out to
// a fixed number of resident CTAs in equal contiguous shares (tl_paged.h): sequences of any lengths load all SMs alike, and nothing on the host
// depends on a length, so that a captured call serves sequences that grow.  A warp takes 16 keys of every unit, for which it keeps a ring of its
// own in shared memory, filled by cp.async a few units ahead across the borders of tokens and heads: no barrier inside a token's keys.
// Where a share ends inside a token's keys the CTA leaves maximum, sum and output in scratch, and whoever of that token's CTAs comes last
// joins them in the order of the keys (in groups of 16 first, where they are many), so that no result depends on timing.
//
// f16 / bf16.  The rows of a tile are the A operand of S^T = K q^T (ldmatrix) and, transposed on the way, of O^T = V^T p; the probabilities go
// from accumulators to the B operand in the register file (movmatrix), split into 16-bit terms that keep nearly all bits (tl_attention.cuh).
// f32: CUDA cores, a lane per D / 32 dimensions; the partial dot products of eight keys are summed over the lanes by exchanging halves.
//
// Keys that no token sees are not read: rows of a tile past a token's end are zero-filled by the copy, whatever the pages hold there.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "tl_attention.cuh"
#include "tl_mma_frag.cuh"

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kGroup = 16;

struct PagedArgs {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int32_t *page_table, *positions, *token_seq;
  const float* slopes;
  int64_t qt, qh, n_pages;
  int32_t tokens, n_heads, n_kv_heads, rep, head_dim, page_size, n_seqs, max_pages, window, row_tiles, least_units;
  TlDivide page_div;
  float scale, softcap;
  int* status;
  float* slots;        // [2 * CTAs] parts of tokens
  unsigned* arrivals;  // [3 * CTAs], zero between launches: CTAs of a group that have left their part, groups of a token
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {  // 16 bytes, or zeros with bytes == 0
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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
  int32_t lo, hi;
  int64_t seq;
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

// A place in the call's units: unit `u` of the `n` of token t and its group `seg` = (KV head, tile of its query heads)
struct Cursor {
  int t, seg, u, n, kvh, tile;
  Token k;
  template <int KEYS> __device__ __forceinline__ void open(const PagedArgs& p) {
    k = token_of(p, t, false);
    n = tl_units(k.lo, k.hi, KEYS);
  }
  __device__ __forceinline__ void head(const PagedArgs& p) {
    if (p.row_tiles == 1) { kvh = seg; tile = 0; }
    else { kvh = seg / p.row_tiles; tile = seg - kvh * p.row_tiles; }
  }
  template <int KEYS> __device__ __forceinline__ void next(const PagedArgs& p) {
    if (++u < n) return;
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
};

// One row again, by one warp and over exactly the keys that it sees: its result is not finite, and whether that is what the cache holds or an infinite value times
// a probability's low term (zero, or negative) only whole probabilities tell.  Two passes; dimensions d0 .. d0 + 31 are stored.
template <typename AT>
__device__ __noinline__ void row_again(const PagedArgs& p, const Token& k, int pos, int t, int h, int kvh, int d0) {
  const int lane = threadIdx.x & 31;
  const AT* q = reinterpret_cast<const AT*>(p.q) + int64_t(t) * p.qt + int64_t(h) * p.qh;
  float mx = -FLT_MAX, sum = 0.f, o = 0.f;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
    for (int j = k.lo; j < k.hi; ++j) {
      const int index = tl_divide(j, p.page_div), page = p.page_table[k.seq * p.max_pages + index];
      if (tl_bad_page(page, p.n_pages)) continue;
      const int64_t at = tl_page_at(page, j - index * p.page_size, p.n_kv_heads, p.page_size, p.head_dim) + int64_t(kvh) * p.page_size * p.head_dim;
      const AT* kp = reinterpret_cast<const AT*>(p.k_pages) + at;
      float x = 0.f;
      for (int d = lane; d < p.head_dim; d += 32) x = fmaf(DT<AT>::to_f32(q[d]), DT<AT>::to_f32(kp[d]), x);
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
      x *= p.scale;
      if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
      if (p.slopes) x = fmaf(p.slopes[h], float(j - pos), x);
      if (pass == 0) {
        mx = fmaxf(mx, x);
      } else {
        const float e = expf(x - mx);
        sum += e;
        if (d0 + lane < p.head_dim) o = fmaf(e, DT<AT>::to_f32(reinterpret_cast<const AT*>(p.v_pages)[at + d0 + lane]), o);
      }
    }
  }
  if (d0 + lane < p.head_dim) reinterpret_cast<AT*>(p.out)[(int64_t(t) * p.n_heads + h) * p.head_dim + d0 + lane] = DT<AT>::from_f32(o / sum);
}

// Probabilities are held times 2^10 in f16: the low term of their split stays clear of f16's subnormals.
template <typename AT> constexpr float kProbBias = 0.f;
template <> constexpr float kProbBias<__half> = 10.f;

// What a warp holds of the softmax of its keys, and how it takes a tile of them in: 16-bit types on the tensor cores.
// NT = 1: up to 8 query heads of a KV head, NT = 2: up to 16.
template <typename AT_, int DPAD_, int NT, int STAGES_>
struct MmaTile {
  using AT = AT_;
  static constexpr int DPAD = DPAD_, ROWS = 8 * NT, KEYS = 16, STAGES = STAGES_, CHUNKS = DPAD / 8, TERMS = ProbSplit<AT>::kTerms;
  static constexpr bool kRedo = true;  // infinite values need it
  uint32_t q[NT][DPAD / 16][2];
  float o[NT][DPAD / 16][4], m[NT][2], l[NT][2], slope[NT][2];

  // chunk c of row r, 16 bytes each, so that the eight rows that ldmatrix reads at once lie in different banks
  static __device__ __forceinline__ int chunk_at(int r, int c) { return r * CHUNKS + (c ^ (r & 7)); }

  __device__ __forceinline__ void begin(const PagedArgs& p, int t, int kvh, int tile) {
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
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
        const int r = tile * ROWS + nt * 8 + 2 * c + e;
        slope[nt][e] = p.slopes && r < p.rep ? p.slopes[kvh * p.rep + r] * kLog2e : 0.f;
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
      float s0[NT][4], s1[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s0[nt][e] = s1[nt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < DPAD / 16; ++i) {
        uint32_t a[4];
        ldmatrix4(ks + 16 * chunk_at(r, 2 * i + half), a);
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
          if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
          x = fmaf(slope[nt][e & 1], float(behind + key), x * kLog2e);
        } else {
          x = s[nt][e] * (p.scale * kLog2e);
        }
        s[nt][e] = (seen >> key) & 1 ? x : -INFINITY;
      }
      float nm[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = fmaxf(s[nt][e], s[nt][e + 2]);
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        nm[e] = fmaxf(m[nt][e], v);
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
        const float mm = m[nt][e & 1];
        pr[e] = mm == -INFINITY ? 0.f : exp2f(s[nt][e] - mm + kProbBias<AT>);
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
#pragma unroll
    for (int i = 0; i < DPAD / 16; ++i) {
      uint32_t a[4];
      ldmatrix4_trans(vs + 16 * chunk_at(r, 2 * i + half), a);
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
};

// Sums N values over the warp, each lane ending with the one of number lane_value<N>(lane): at every step a lane keeps half of its values and hands
// over the rest, N - 1 + (5 - log2 N) shuffles in all instead of 5 N.
template <int N> __device__ __forceinline__ float sum_exchange(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int bit = 16;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, bit >>= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float give = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
    }
  }
#pragma unroll
  for (; bit > 0; bit >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
  return v[0];
}
// f32: a lane owns E neighbouring dimensions of all keys and rows; eight keys a tile.
template <int DPAD_, int ROWS_, int STAGES_>
struct F32Tile {
  using AT = float;
  static constexpr int DPAD = DPAD_, ROWS = ROWS_, KEYS = 8, STAGES = STAGES_, CHUNKS = DPAD / 4, E = DPAD / 32;
  static constexpr bool kRedo = false;
  static constexpr int kSets = ROWS * KEYS > 32 ? ROWS * KEYS / 32 : 1, kN = ROWS * KEYS / kSets;  // kN values are summed at once
  static constexpr int kRowsOfSet = ROWS / kSets, kLog = kN == 32 ? 5 : kN == 16 ? 4 : 3;
  float q[ROWS][E], o[ROWS][E], m[ROWS], l[ROWS];  // m: the same in all lanes; l: a lane's own
  float slope[kSets];
  static __device__ __forceinline__ int chunk_at(int r, int c) { return r * CHUNKS + c; }

  __device__ __forceinline__ void begin(const PagedArgs& p, int t, int kvh, int tile) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int row = tile * ROWS + r;
      const float* qp = reinterpret_cast<const float*>(p.q) + int64_t(t) * p.qt + int64_t(kvh * p.rep + row) * p.qh + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        q[r][e] = row < p.rep && lane * E + e < p.head_dim ? __ldg(qp + e) : 0.f;
        o[r][e] = 0.f;
      }
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const int row = tile * ROWS + s * kRowsOfSet + (lane >> (5 - kLog)) / KEYS;
      slope[s] = p.slopes && row < p.rep ? p.slopes[kvh * p.rep + row] * kLog2e : 0.f;
    }
  }
  static __device__ __forceinline__ void load(uint32_t at, float (&v)[E]) {
    if (E == 2) {
      asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[E - 1]) : "r"(at));
    } else {
#pragma unroll
      for (int e = 0; e + 3 < E; e += 4)
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[e]), "=f"(v[e + 1]), "=f"(v[e + 2]), "=f"(v[e + 3]) : "r"(at + 4 * e));
    }
  }
  template <bool OPTIONS> __device__ __forceinline__ void take(const PagedArgs& p, uint32_t ks, uint32_t vs, uint32_t seen, int behind) {
    const int lane = threadIdx.x & 31;
    float dot[kSets][kN];  // value row * KEYS + key of a set
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      float k[E];
      load(ks + 4 * (j * DPAD + lane * E), k);
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
#pragma unroll
      for (int i = 0; i < kRowsOfSet; ++i) {
        const int r = s * kRowsOfSet + i;
        const float nm = fmaxf(m[r], __shfl_sync(0xffffffffu, top, (i * KEYS) << (5 - kLog)));
        if (nm != m[r]) {  // the same in all lanes
          const float f = exp2f(m[r] - nm);
          m[r] = nm;
          l[r] *= f;
#pragma unroll
          for (int e = 0; e < E; ++e) o[r][e] *= f;
        }
      }
      float mm = m[s * kRowsOfSet];
#pragma unroll
      for (int i = 1; i < kRowsOfSet; ++i) mm = (lane >> (5 - kLog)) / KEYS == i ? m[s * kRowsOfSet + i] : mm;
      pr[s] = mm == -INFINITY ? 0.f : exp2f(x - mm);
    }
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      float v[E];
      load(vs + 4 * (j * DPAD + lane * E), v);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float w = __shfl_sync(0xffffffffu, pr[r / kRowsOfSet], ((r % kRowsOfSet) * KEYS + j) << (5 - kLog));
        l[r] += w;  // all lanes hold the whole sum
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = fmaf(w, v[e], o[r][e]);
      }
    }
  }
  __device__ __forceinline__ void end(float* wm, float* wl, float* wo, int pitch, int rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < rows) {
        if (lane == 0) { wm[r] = m[r]; wl[r] = l[r]; }
#pragma unroll
        for (int e = 0; e < E; ++e) wo[r * pitch + lane * E + e] = o[r][e];
      }
  }
};

// Dynamic shared memory: the warps' rings, then [4][rows] maxima, [4][rows] sums and [4][rows][DPAD + 4] outputs (the pitch keeps the lanes of a
// quad in banks of their own), which join() uses too.
template <class Tile> constexpr int kRingBytes = kWarps * Tile::STAGES * 2 * Tile::KEYS * Tile::DPAD * int(sizeof(typename Tile::AT));
template <class Tile> constexpr int kPitch = Tile::DPAD + 4;
template <class Tile> constexpr int area_bytes(int rows) { return kWarps * rows * (2 + kPitch<Tile>) * int(sizeof(float)); }
// A part in scratch: [ROWS][DPAD] outputs, then [ROWS] maxima and [ROWS] sums; whole 16-byte vectors
template <class Tile> __host__ __device__ constexpr int slot_floats() { return Tile::ROWS * Tile::DPAD + (2 * Tile::ROWS + 3) / 4 * 4; }
template <class Tile> constexpr int kSlotMax = Tile::ROWS * Tile::DPAD;
template <class Tile> constexpr int kSlotSum = kSlotMax<Tile> + Tile::ROWS;

// The slot in which CTA first + i of a token's CTAs leaves its part: the first of them starts the token, the others have it begun elsewhere.
__device__ __forceinline__ int slot_of(int first, int i) { return 2 * (first + i) + (i == 0 ? 1 : 0); }
// Parts i = from, from + step, ... of a token, `count` of them (at most 32), become one in area: [rows][DPAD] outputs, [rows] maxima, [rows] sums, and
// then the [rows][count] factors used.
template <class Tile> __device__ void join(const float* slots, int first, int from, int step, int count, int rows, float* area) {
  float *maxima = area + rows * Tile::DPAD, *sums = maxima + rows, *factor = sums + rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < rows; r += kWarps) {
    float mx = -INFINITY, sum = 0.f;
    const float* at = slots + int64_t(slot_of(first, from + min(lane, count - 1) * step)) * slot_floats<Tile>() + r;
    if (lane < count) { mx = __ldcg(at + kSlotMax<Tile>); sum = __ldcg(at + kSlotSum<Tile>); }
    float top = mx;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = mx == -INFINITY ? 0.f : exp2f(mx - top);
    sum *= f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < count) factor[r * count + lane] = f;
    if (lane == 0) { maxima[r] = top; sums[r] = sum; }
  }
  __syncthreads();
  for (int e = threadIdx.x * 4; e < rows * Tile::DPAD; e += kThreads * 4) {
    const int r = e / Tile::DPAD;
    const float* at = slots + e;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(at + int64_t(slot_of(first, from + i * step)) * slot_floats<Tile>()));
      const float f = factor[r * count + i];
      a.x = fmaf(f, v.x, a.x); a.y = fmaf(f, v.y, a.y); a.z = fmaf(f, v.z, a.z); a.w = fmaf(f, v.w, a.w);
    }
    *reinterpret_cast<float4*>(area + e) = a;
  }
  __syncthreads();
}

template <class Tile, bool OPTIONS>
__global__ void __launch_bounds__(kThreads) paged_attention_kernel(const __grid_constant__ PagedArgs p) {
  using AT = typename Tile::AT;
  constexpr int DPAD = Tile::DPAD, KEYS = Tile::KEYS, STAGES = Tile::STAGES, UNIT = KEYS * kWarps, CHUNKS = Tile::CHUNKS;
  constexpr int kTileBytes = KEYS * DPAD * int(sizeof(AT)), kCopies = KEYS * CHUNKS / 32, kPerChunk = 16 / int(sizeof(AT));
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ long long found_begin, scan[kWarps];
  __shared__ int found_token, is_last;
  __shared__ uint32_t seen_of[kWarps][STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = int(blockIdx.x);
  float* area = reinterpret_cast<float*>(sm + kRingBytes<Tile>);
  const uint32_t ring = smem_at(sm) + warp * STAGES * 2 * kTileBytes;
  if (p.head_dim < DPAD) {  // the copies leave the padding alone: it is zero from here on
    for (int i = threadIdx.x; i < kRingBytes<Tile> / 16; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  tl_pdl_wait();

  // Tokens that see nothing, and how many units the others have
  const int segs = p.n_kv_heads * p.row_tiles, chunk = (p.tokens + kThreads - 1) / kThreads;
  const int t_first = min(p.tokens, int(threadIdx.x) * chunk), t_end = min(p.tokens, t_first + chunk);
  long long mine = 0;
  for (int t = t_first; t < t_end; ++t) {
    const Token k = token_of(p, t, t % int(gridDim.x) == cta);
    mine += tl_units(k.lo, k.hi, UNIT);
  }
  for (int t = cta; t < p.tokens; t += int(gridDim.x)) {
    const Token k = token_of(p, t, false);
    if (k.hi == 0)
      for (int e = threadIdx.x; e < p.n_heads * p.head_dim; e += kThreads)
        reinterpret_cast<AT*>(p.out)[int64_t(t) * p.n_heads * p.head_dim + e] = DT<AT>::from_f32(0.f);
  }
  long long to = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, to, o);
    if (lane >= o) to += v;
  }
  if (lane == 31) scan[warp] = to;
  __syncthreads();
  long long whole = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) to += scan[w];
    whole += scan[w];
  }
  const long long units = whole * segs;
  const int ctas = tl_share_ctas(units, int(gridDim.x), p.least_units);
  if (units == 0 || cta >= ctas) return;
  const long long begin = tl_share_begin(units, ctas, cta), end = tl_share_begin(units, ctas, cta + 1);
  if ((to - mine) * segs <= begin && begin < to * segs) {  // one thread's
    long long at = (to - mine) * segs;
    for (int t = t_first; t < t_end; ++t) {
      const Token k = token_of(p, t, false);
      const long long n = (long long)(tl_units(k.lo, k.hi, UNIT)) * segs;
      if (begin < at + n) {
        found_token = t;
        found_begin = begin - at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();

  Cursor c;
  c.t = found_token;
  c.template open<UNIT>(p);
  c.seg = int(found_begin / c.n);
  c.u = int(found_begin - (long long)(c.seg) * c.n);
  c.head(p);
  Cursor f = c;  // what is fetched next

  // A lane below KEYS finds its key's row a unit before it is copied: the table is read on the way
  bool row_seen;
  int64_t row_at;
  auto look_up = [&](bool more) {
    const int key = f.k.lo + f.u * UNIT + warp * KEYS + lane;
    row_seen = more && lane < KEYS && key < f.k.hi;
    row_at = 0;
    if (row_seen) {
      const int index = tl_divide(key, p.page_div), page = __ldg(p.page_table + f.k.seq * p.max_pages + index);
      if (tl_bad_page(page, p.n_pages)) {
        atomicOr(p.status, kBadPage);
        row_seen = false;
      } else {
        row_at = tl_page_at(page, key - index * p.page_size, p.n_kv_heads, p.page_size, p.head_dim) + int64_t(f.kvh) * p.page_size * p.head_dim;
      }
    }
  };
  auto fetch = [&](int stage) {
    const uint32_t seen = __ballot_sync(0xffffffffu, row_seen);
    if (lane == 0) seen_of[warp][stage] = seen;
    const uint32_t ks = ring + stage * 2 * kTileBytes, vs = ks + kTileBytes;
    if (seen) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int e = i * 32 + lane, r = e / CHUNKS, ch = e % CHUNKS;
        const int64_t at = __shfl_sync(0xffffffffu, row_at, r) + ch * kPerChunk;
        const int bytes = (seen >> r) & 1 ? 16 : 0;
        if (ch * kPerChunk < p.head_dim) {
          copy16(ks + 16 * Tile::chunk_at(r, ch), reinterpret_cast<const AT*>(p.k_pages) + at, bytes);
          copy16(vs + 16 * Tile::chunk_at(r, ch), reinterpret_cast<const AT*>(p.v_pages) + at, bytes);
        }
      }
    }
    copy_commit();
  };
  long long ahead = begin;  // units fetched
  look_up(true);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (ahead < end) {
      fetch(s);
      if (++ahead < end) { f.template next<UNIT>(p); look_up(true); }
    } else {
      copy_commit();
    }
  }

  Tile tile;
  tile.begin(p, c.t, c.kvh, c.tile);
  int stage = 0;
  for (long long w = begin; w < end; ++w) {
    copy_wait<STAGES - 2>();
    __syncwarp();  // this unit's rows have landed for all lanes, and all have read the last one's
    const uint32_t seen = seen_of[warp][stage];
    {
      const int to_fill = stage == 0 ? STAGES - 1 : stage - 1;
      if (ahead < end) {
        fetch(to_fill);
        if (++ahead < end) { f.template next<UNIT>(p); look_up(true); }
      } else {
        copy_commit();
      }
    }
    const uint32_t ks = ring + stage * 2 * kTileBytes;
    if (seen) tile.template take<OPTIONS>(p, ks, ks + kTileBytes, seen, c.k.lo + c.u * UNIT + warp * KEYS + 1 - c.k.hi);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (c.u + 1 < c.n && w + 1 < end) { ++c.u; continue; }

    // The last unit of this token and group, or of this CTA's share
    const int rows = min(Tile::ROWS, p.rep - c.tile * Tile::ROWS), h0 = c.kvh * p.rep + c.tile * Tile::ROWS;
    float *wm = area, *wl = wm + kWarps * rows, *wo = wl + kWarps * rows;
    const long long seg_begin = w - c.u, seg_end = seg_begin + c.n;
    const bool starts = seg_begin >= begin, ends = seg_end <= end;
    tile.end(wm + warp * rows, wl + warp * rows, wo + warp * rows * kPitch<Tile>, kPitch<Tile>, rows);
    __syncthreads();
    auto store = [&](int r, int d, float v) {  // a warp's 32 values are one row's
      if (Tile::kRedo && __any_sync(0xffffffffu, d < p.head_dim && !isfinite(v))) {
        row_again<AT>(p, c.k, c.k.hi - 1, c.t, h0 + r, c.kvh, d & ~31);
      } else if (d < p.head_dim) {
        reinterpret_cast<AT*>(p.out)[(int64_t(c.t) * p.n_heads + h0 + r) * p.head_dim + d] = DT<AT>::from_f32(v);
      }
    };
    float* slot = p.slots + int64_t(2 * cta + (starts ? 1 : 0)) * slot_floats<Tile>();
    for (int e = threadIdx.x; e < rows * DPAD; e += kThreads) {
      const int r = e / DPAD, d = e - r * DPAD;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = fmaxf(top, wm[i * rows + r]);
      float sum = 0.f, o = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float mx = wm[i * rows + r], g = mx == -INFINITY ? 0.f : exp2f(mx - top);
        sum = fmaf(wl[i * rows + r], g, sum);
        o = fmaf(wo[(i * rows + r) * kPitch<Tile> + d], g, o);
      }
      if (starts && ends) {
        store(r, d, sum == 0.f ? 0.f : o / sum);  // no key's page is there: nothing is seen
      } else {
        if (d == 0) { __stcg(slot + kSlotMax<Tile> + r, top); __stcg(slot + kSlotSum<Tile> + r, sum); }
        __stcg(slot + e, o);
      }
    }
    if (!(starts && ends)) {
      // The token's CTAs are first .. first + count - 1.  Whoever comes last of a group of kGroup joins the group's parts, in the place of the first of
      // them, and whoever ends the last group joins the groups'.
      const int first = tl_share_owner(units, ctas, seg_begin), count = tl_share_owner(units, ctas, seg_end - 1) - first + 1;
      const int group = (cta - first) / kGroup, groups = (count + kGroup - 1) / kGroup, members = min(kGroup, count - group * kGroup);
      auto last_of = [&](unsigned* arrived, int of) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          is_last = atomicAdd(arrived, 1u) == unsigned(of) - 1;
          if (is_last) *arrived = 0;  // for the next launch
        }
        __syncthreads();
        __threadfence();
        return is_last != 0;
      };
      bool done = last_of(p.arrivals + slot_of(first, group * kGroup), members);
      if (done) {
        join<Tile>(p.slots, first, group * kGroup, 1, members, rows, area);
        if (groups > 1) {
          float* to_slot = p.slots + int64_t(slot_of(first, group * kGroup)) * slot_floats<Tile>();
          for (int e = threadIdx.x; e < rows * DPAD; e += kThreads) __stcg(to_slot + e, area[e]);
          if (int(threadIdx.x) < rows) {
            __stcg(to_slot + kSlotMax<Tile> + threadIdx.x, area[rows * DPAD + threadIdx.x]);
            __stcg(to_slot + kSlotSum<Tile> + threadIdx.x, area[rows * DPAD + rows + threadIdx.x]);
          }
          done = last_of(p.arrivals + 2 * gridDim.x + first, groups);
          if (done) join<Tile>(p.slots, first, 0, kGroup, groups, rows, area);
        }
      }
      if (done)
        for (int e = threadIdx.x; e < rows * DPAD; e += kThreads) {
          const int r = e / DPAD;
          const float sum = area[rows * DPAD + rows + r];
          store(r, e - r * DPAD, sum == 0.f ? 0.f : area[e] / sum);
        }
    }
    __syncthreads();
    if (w + 1 < end) {
      c.template next<UNIT>(p);
      tile.begin(p, c.t, c.kvh, c.tile);
    }
  }
}

// CTAs that are resident together: by shared memory, two where the ring allows
template <class Tile> int resident(int rows) { return std::min(2, 233472 / (kRingBytes<Tile> + area_bytes<Tile>(rows) + 1024 + 512)); }

template <class Tile, bool OPTIONS> cudaError_t launch(tl_ctx* ctx, const PagedArgs& p, int64_t most_units) {
  const int rows = std::min(Tile::ROWS, p.rep), smem = kRingBytes<Tile> + area_bytes<Tile>(rows);
  auto kernel = paged_attention_kernel<Tile, OPTIONS>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(std::min<int64_t>(int64_t(ctx->sm_count) * resident<Tile>(rows), std::max<int64_t>(1, most_units))));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}
template <class Tile> cudaError_t launch_tile(tl_ctx* ctx, PagedArgs& p, int64_t longest) {
  p.row_tiles = (p.rep + Tile::ROWS - 1) / Tile::ROWS;
  constexpr int kUnit = Tile::KEYS * kWarps;
  const int64_t most = int64_t(p.tokens) * p.n_kv_heads * p.row_tiles * ((longest + kUnit - 1) / kUnit);
  return p.softcap > 0.f || p.slopes ? launch<Tile, true>(ctx, p, most) : launch<Tile, false>(ctx, p, most);
}
// Up to 8 query heads of a KV head on one tile, up to 16 on a tile of two, more on several; 256 dimensions leave registers for 8 (f32: 4).
template <typename AT> cudaError_t launch_mma(tl_ctx* ctx, PagedArgs& p, int64_t longest) {
  if (p.head_dim <= 64) return p.rep <= 8 ? launch_tile<MmaTile<AT, 64, 1, 4>>(ctx, p, longest) : launch_tile<MmaTile<AT, 64, 2, 4>>(ctx, p, longest);
  if (p.head_dim <= 128) return p.rep <= 8 ? launch_tile<MmaTile<AT, 128, 1, 3>>(ctx, p, longest) : launch_tile<MmaTile<AT, 128, 2, 3>>(ctx, p, longest);
  return launch_tile<MmaTile<AT, 256, 1, 3>>(ctx, p, longest);
}
cudaError_t launch_f32(tl_ctx* ctx, PagedArgs& p, int64_t longest) {
  if (p.head_dim <= 64)
    return p.rep == 1 ? launch_tile<F32Tile<64, 1, 4>>(ctx, p, longest) : p.rep <= 4 ? launch_tile<F32Tile<64, 4, 4>>(ctx, p, longest) : launch_tile<F32Tile<64, 8, 4>>(ctx, p, longest);
  if (p.head_dim <= 128)
    return p.rep == 1 ? launch_tile<F32Tile<128, 1, 3>>(ctx, p, longest) : p.rep <= 4 ? launch_tile<F32Tile<128, 4, 3>>(ctx, p, longest) : launch_tile<F32Tile<128, 8, 3>>(ctx, p, longest);
  return p.rep == 1 ? launch_tile<F32Tile<256, 1, 3>>(ctx, p, longest) : launch_tile<F32Tile<256, 4, 3>>(ctx, p, longest);
}

// Parts of tokens for two CTAs an SM of the largest slot, and the arrivals: one size for all calls, so that no captured call's scratch is replaced.
constexpr int kSlotFloats = 16 * 130, kLeastUnits = 4;
static_assert(slot_floats<MmaTile<__half, 64, 2, 4>>() <= kSlotFloats && slot_floats<F32Tile<256, 4, 3>>() <= kSlotFloats && slot_floats<F32Tile<128, 8, 3>>() <= kSlotFloats, "slots");
static_assert(slot_floats<MmaTile<__half, 256, 1, 3>>() <= kSlotFloats && slot_floats<MmaTile<__half, 128, 2, 3>>() <= kSlotFloats, "slots");
int32_t secure_scratch(tl_ctx* ctx) {
  if (ctx->paged_scratch) return TL_OK;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (!ctx->capturing) TL_CUDA(ctx, cudaStreamIsCapturing(ctx->stream, &capture));
  if (ctx->capturing || capture != cudaStreamCaptureStatusNone)
    return tl_set_error(ctx, TL_ERR_UNSUPPORTED, "tl_paged_attention: its scratch is not there yet during graph capture; run the call once before capturing");
  const size_t ctas = size_t(ctx->sm_count) * 2, bytes = ctas * (2 * kSlotFloats * sizeof(float) + 3 * sizeof(unsigned));
  void* at = nullptr;
  const cudaError_t e = ctx->pool.device_malloc(&at, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return tl_set_error(ctx, TL_ERR_OOM, "tl_paged_attention: scratch of %zu bytes failed: %s", bytes, cudaGetErrorString(e));
  }
  ctx->paged_scratch = at;
  TL_CUDA(ctx, cudaMemsetAsync(at, 0, bytes, ctx->stream));
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
  rc = secure_scratch(ctx);
  if (rc != TL_OK) return rc;
  PagedArgs p{};
  p.q = q; p.k_pages = cache->k_pages; p.v_pages = cache->v_pages; p.out = out;
  p.page_table = cache->page_table; p.positions = positions; p.token_seq = token_seq; p.slopes = slopes;
  p.qt = q_token_stride; p.qh = q_head_stride; p.n_pages = cache->n_pages;
  p.tokens = int32_t(tokens); p.n_heads = int32_t(n_heads); p.n_kv_heads = cache->n_kv_heads; p.rep = int32_t(n_heads / cache->n_kv_heads);
  p.head_dim = cache->head_dim; p.page_size = cache->page_size; p.n_seqs = cache->n_seqs; p.max_pages = cache->max_pages;
  p.window = window; p.scale = scale; p.softcap = softcap; p.least_units = kLeastUnits;
  p.page_div = tl_divide_by(cache->page_size);
  p.status = ctx->dev_status + 1;
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
