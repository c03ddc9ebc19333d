// Element access of the decode ops (tl_decode_ops.cu, tl_paged_append.cu): any storage type as f32, one element or eight
// at a time, and the sum over a warp.
#pragma once

#include "tl_common.cuh"

#ifdef __CUDACC__
__device__ __forceinline__ float ld_f32(const void* p, int dtype, int64_t i) {
  if (dtype == TL_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == TL_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Rows of whole 8-element vectors: the row is read once and held in registers, a vector (or CH of them) a thread, so a
// row costs one round trip to memory and one reduction.
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = DT<T>::to_f32(e[i]);
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = DT<T>::from_f32(v[i]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void load8_any(const void* p, int dtype, int64_t i, float (&v)[8]) {
  if (dtype == TL_F32) load8(reinterpret_cast<const float*>(p) + i, v);
  else if (dtype == TL_F16) load8(reinterpret_cast<const __half*>(p) + i, v);
  else load8(reinterpret_cast<const __nv_bfloat16*>(p) + i, v);
}
#endif  // __CUDACC__
