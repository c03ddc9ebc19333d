// tl_zeroed (tl_pool.cuh) on a fake device whose calls can be made to fail, and a pool that only allocates.  Built by tests/test_zeroed_cpu.py.
#include "tl_pool.cuh"

#include <cstdio>
#include <cstdlib>
#include <cstring>

static int mallocs = 0, frees = 0, zeroed = 0;
static cudaError_t fail_malloc = cudaSuccess, fail_memset = cudaSuccess;
static char block[64];

TlBlockPool::TlBlockPool() = default;
TlBlockPool::~TlBlockPool() = default;
cudaError_t TlBlockPool::device_malloc(void** out, size_t) {
  if (fail_malloc != cudaSuccess) return fail_malloc;
  ++mallocs;
  *out = block;
  return cudaSuccess;
}
extern "C" {
cudaError_t cudaFree(void* p) {
  frees += p == block;
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* p, int value, size_t bytes, cudaStream_t) {
  if (fail_memset != cudaSuccess) return fail_memset;
  memset(p, value, bytes);
  ++zeroed;
  return cudaSuccess;
}
}

#define CHECK(x) \
  do { if (!(x)) { fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x); exit(1); } } while (0)

int main() {
  TlBlockPool pool;
  void* at = nullptr;
  memset(block, 1, sizeof(block));
  fail_malloc = cudaErrorMemoryAllocation;
  CHECK(tl_zeroed(pool, &at, sizeof(block), nullptr) == cudaErrorMemoryAllocation && !at && !frees);
  fail_malloc = cudaSuccess;
  fail_memset = cudaErrorInvalidValue;  // the next call finds nothing that nobody zeroed
  CHECK(tl_zeroed(pool, &at, sizeof(block), nullptr) == cudaErrorInvalidValue && !at && mallocs == 1 && frees == 1);
  fail_memset = cudaSuccess;
  CHECK(tl_zeroed(pool, &at, sizeof(block), nullptr) == cudaSuccess && at == block && mallocs == 2 && frees == 1 && zeroed == 1);
  for (char c : block) CHECK(c == 0);
  return 0;
}
