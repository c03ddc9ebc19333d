/*
 * The paged cache's calls and sampling through the addon: what a buffer handle does not hold is refused before the library is called, the rest arrives.
 * On the fake N-API of stub_napi.c; built by tests/test_napi_paged_cpu.py.
 */
#define main stub_main
#include "stub_napi.c"
#undef main

static struct { int append, attention, sample; tl_paged_cache cache; int64_t tokens, heads; const void *q, *out, *k, *logits; float scale; int32_t window; } seen;
int32_t tl_paged_append(tl_ctx* c, const tl_paged_cache* cache, const int32_t* positions, const int32_t* seq, int64_t tokens, const void* q, int64_t qt, int64_t qh, int64_t heads,
                        void* out, int64_t ot, int64_t oh, const void* k, int64_t kt, int64_t kh, const void* v, int64_t vt, int64_t vh, const void* qw, const void* kw, int32_t wd,
                        float eps, const float* cos, const float* sin, int64_t rows) {
  (void)c; (void)positions; (void)seq; (void)qt; (void)qh; (void)ot; (void)oh; (void)kt; (void)kh; (void)v; (void)vt; (void)vh; (void)qw; (void)kw; (void)wd; (void)eps; (void)cos;
  (void)sin; (void)rows;
  seen.append++; seen.cache = *cache; seen.tokens = tokens; seen.heads = heads; seen.q = q; seen.out = out; seen.k = k;
  return 0;
}
int32_t tl_paged_attention(tl_ctx* c, const tl_paged_cache* cache, const int32_t* positions, const int32_t* seq, int64_t tokens, const void* q, int64_t qt, int64_t qh, int64_t heads,
                           void* out, float scale, float softcap, int32_t window, const float* slopes) {
  (void)c; (void)positions; (void)seq; (void)qt; (void)qh; (void)softcap; (void)slopes;
  seen.attention++; seen.cache = *cache; seen.tokens = tokens; seen.heads = heads; seen.q = q; seen.out = out; seen.scale = scale; seen.window = window;
  return 0;
}
int32_t tl_sample(tl_ctx* c, const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t stride, const float* t, const int32_t* k, const float* p, const float* m,
                  const float* u, int32_t* out) {
  (void)c; (void)dtype; (void)rows; (void)vocab; (void)stride; (void)t; (void)k; (void)p; (void)m; (void)u;
  seen.sample++; seen.logits = logits; seen.out = out;
  return 0;
}

static V* ctx;
static V* buffer(double bytes) { V* a[2] = {ctx, number(bytes)}; return call("alloc", 2, a); }
static void* address(V* b) { V* a[1] = {b}; return (void*)(uintptr_t)call("ptrOf", 1, a)->big; }
static V* cache_of(V* k, V* v, V* table, int dtype) {  /* 5 pages of 2 heads x 16 x 64, 3 sequences of 4 pages */
  static const char* const names[] = {"kPages", "vPages", "pageTable", "nPages", "pageSize", "kvHeads", "headDim", "dtype", "nSeqs", "maxPages"};
  V* values[] = {k, v, table, number(5), number(16), number(2), number(64), number(dtype), number(3), number(4)};
  V* o = nv(T_OBJ);
  o->n = 10;
  for (int i = 0; i < 10; ++i) { o->keys[i] = names[i]; o->elems[i] = values[i]; }
  return o;
}
static int refused(const char* name, size_t argc, V** argv, const char* what) {
  const int calls = seen.append + seen.attention + seen.sample;
  call(name, argc, argv);
  return g_env.has_thrown && strstr(g_env.thrown, what) && seen.append + seen.attention + seen.sample == calls;
}

int main(void) {
  napi_register_module_v1(&g_env, nv(T_OBJ));
  V* a1[1] = {number(0)};
  ctx = call("ctxCreate", 1, a1);
  const double pages = 5 * 2 * 16 * 64;
  V *none = nv(T_NULL), *table = buffer(3 * 4 * 4), *pos = buffer(3 * 4);
  V *k16 = buffer(pages * 2), *v16 = buffer(pages * 2), *k32 = buffer(pages * 4), *v32 = buffer(pages * 4);
  V *half = cache_of(k16, v16, table, TL_F16), *single = cache_of(k32, v32, table, TL_F32);
  V *q16 = buffer(3 * 4 * 64 * 2), *q32 = buffer(3 * 4 * 64 * 4), *slopes = buffer(4 * 4);

  /* attention: three tokens, four heads */
  V* at[14] = {ctx, half, pos, none, number(3), q16, number(256), number(64), number(4), buffer(3 * 256 * 2), number(.25), number(0), number(7), slopes};
  call("pagedAttention", 14, at);
  EXPECT(!g_env.has_thrown && seen.attention == 1 && seen.q == address(q16) && seen.out == address(at[9]) && seen.tokens == 3 && seen.heads == 4 && seen.scale == .25f &&
         seen.window == 7 && seen.cache.k_pages == address(k16) && seen.cache.n_pages == 5 && seen.cache.max_pages == 4, "attention's arguments arrive");
  at[1] = single;
  EXPECT(refused("pagedAttention", 14, at, "of q"), "f16 queries beside an f32 cache are refused");
  at[5] = q32;
  EXPECT(refused("pagedAttention", 14, at, "of out"), "an f16 output beside an f32 cache is refused");
  at[9] = buffer(3 * 256 * 4);
  call("pagedAttention", 14, at);
  EXPECT(!g_env.has_thrown && seen.attention == 2, "f32 everywhere is fine");
  at[8] = number(6); at[6] = number(192); at[7] = number(32);
  EXPECT(refused("pagedAttention", 14, at, "of out"), "more heads than the output has are refused");
  at[8] = number(4); at[6] = number(256); at[7] = number(64);
  at[2] = buffer(2 * 4);
  EXPECT(refused("pagedAttention", 14, at, "of positions"), "too few positions are refused");
  at[2] = pos; at[3] = buffer(8);
  EXPECT(refused("pagedAttention", 14, at, "of tokenSeq"), "too few sequences are refused");
  at[3] = none; at[13] = buffer(8);
  EXPECT(refused("pagedAttention", 14, at, "of slopes"), "too few slopes are refused");
  at[13] = none; at[1] = cache_of(k16, v32, table, TL_F32);
  EXPECT(refused("pagedAttention", 14, at, "of kPages"), "pages of another type are refused");
  at[1] = cache_of(k32, v32, buffer(40), TL_F32);
  EXPECT(refused("pagedAttention", 14, at, "of pageTable"), "a short page table is refused");
  at[1] = single; at[5] = nv(T_BIG); at[5]->big = 0x1000;  /* an address: nothing is known of it */
  call("pagedAttention", 14, at);
  EXPECT(!g_env.has_thrown && seen.attention == 3 && seen.q == (void*)0x1000, "addresses pass");

  /* append: the rows of one product, eight heads of 64 */
  V *rows = buffer(3 * 512 * 2), *tables = buffer(50 * 32 * 4), *w = buffer(64 * 4);
  V* vk[2] = {rows, number(256 * 2)};
  V* vv[2] = {rows, number(384 * 2)};
  V *kk = call("view", 2, vk), *vvv = call("view", 2, vv);
  V* ap[25] = {ctx, half, pos, none, number(3), rows, number(512), number(64), number(4), buffer(3 * 256 * 2), number(256), number(64), kk, number(512), number(64), vvv,
               number(512), number(64), w, w, number(TL_F32), number(1e-6), tables, tables, number(50)};
  call("pagedAppend", 25, ap);
  EXPECT(!g_env.has_thrown && seen.append == 1 && seen.k == (char*)address(rows) + 512, "a product's columns arrive");
  struct { int at; V* bad; const char* what; } wrong[] = {
    {5, buffer(3 * 512 * 2 - 1024), "of q"}, {9, buffer(3 * 256 * 2 - 2), "of qOut"}, {12, buffer(128 * 2), "of k"}, {15, buffer(128 * 2), "of v"}, {18, buffer(63 * 4), "of qWeight"},
    {19, buffer(63 * 4), "of kWeight"}, {22, buffer(49 * 32 * 4), "of cos"}, {23, buffer(49 * 32 * 4), "of sin"}, {1, single, "of q"}, {2, buffer(4), "of positions"}};
  for (size_t i = 0; i < sizeof(wrong) / sizeof(wrong[0]); ++i) {
    V* good = ap[wrong[i].at];
    ap[wrong[i].at] = wrong[i].bad;
    EXPECT(refused("pagedAppend", 25, ap, wrong[i].what), wrong[i].what);
    ap[wrong[i].at] = good;
  }
  ap[4] = number(0);
  ap[5] = buffer(1);
  call("pagedAppend", 25, ap);
  EXPECT(!g_env.has_thrown && seen.append == 2, "no tokens need no rows");

  /* sampling: two rows of 100 */
  V *row = buffer(8), *logits = buffer(200 * 4);
  V* sa[12] = {ctx, logits, number(TL_F32), number(2), number(100), number(100), row, row, row, row, row, row};
  call("sample", 12, sa);
  EXPECT(!g_env.has_thrown && seen.sample == 1 && seen.logits == address(logits) && seen.out == address(row), "sampling's arguments arrive");
  static const char* const what[] = {"of temperature", "of topK", "of topP", "of minP", "of uniforms", "of out"};
  for (int i = 0; i < 6; ++i) {
    sa[6 + i] = buffer(4);
    EXPECT(refused("sample", 12, sa, what[i]), what[i]);
    sa[6 + i] = row;
  }
  sa[1] = buffer(200 * 2);
  EXPECT(refused("sample", 12, sa, "of logits"), "f16 logits called f32 are refused");
  sa[2] = number(TL_F16);
  call("sample", 12, sa);
  EXPECT(!g_env.has_thrown && seen.sample == 2, "f16 logits are fine");
  printf("ALL OK\n");
  return 0;
}
