// Eight consecutive elements of fp32 / bf16 / fp16 at a time, in and out of fp32 registers. The vector accesses need the element's own alignment only (this
// target's global loads and stores take any address): rows and tensors that begin anywhere move as fast as aligned ones but for the lines they straddle.
#pragma once
#include "common.cuh"

typedef uint32_t vec8_u4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Raw8 { uint32_t w[2 * sizeof(T)]; };      // as they lie in memory

template <typename T> __device__ __forceinline__ float elem_ld(const T* p);
template <> __device__ __forceinline__ float elem_ld<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float elem_ld<bf16_t>(const bf16_t* p) { return bf2f(*p); }
template <> __device__ __forceinline__ float elem_ld<_Float16>(const _Float16* p) { return (float)*p; }
__device__ __forceinline__ void elem_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void elem_st(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void elem_st(_Float16* p, float v) { *p = (_Float16)v; }

template <typename T>
__device__ __forceinline__ Raw8<T> raw8_ld(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (unsigned j = 0; j < sizeof(T) / 2; ++j) {
    const vec8_u4 a = reinterpret_cast<const vec8_u4*>(p)[j];
    r.w[4 * j] = a.x; r.w[4 * j + 1] = a.y; r.w[4 * j + 2] = a.z; r.w[4 * j + 3] = a.w;
  }
  return r;
}
template <typename T, bool NT = false>
__device__ __forceinline__ void raw8_st(T* p, const Raw8<T>& r) {      // NT: past the caches
#pragma unroll
  for (unsigned j = 0; j < sizeof(T) / 2; ++j) {
    const vec8_u4 a = {r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]};
    if (NT) __builtin_nontemporal_store(a, reinterpret_cast<vec8_u4*>(p) + j);
    else reinterpret_cast<vec8_u4*>(p)[j] = a;
  }
}
__device__ __forceinline__ void raw8_unpack(const Raw8<float>& r, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(r.w[e]);
}
__device__ __forceinline__ void raw8_unpack(const Raw8<bf16_t>& r, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(e & 1 ? r.w[e >> 1] & 0xffff0000u : r.w[e >> 1] << 16);
}
__device__ __forceinline__ void raw8_unpack(const Raw8<_Float16>& r, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[e >> 1] >> (16 * (e & 1))));
}
__device__ __forceinline__ void raw8_pack(const float (&v)[8], Raw8<float>& r) {
#pragma unroll
  for (int e = 0; e < 8; ++e) r.w[e] = __float_as_uint(v[e]);
}
__device__ __forceinline__ void raw8_pack(const float (&v)[8], Raw8<bf16_t>& r) {
#pragma unroll
  for (int j = 0; j < 4; ++j) r.w[j] = f2bf2(v[2 * j], v[2 * j + 1]);
}
__device__ __forceinline__ void raw8_pack(const float (&v)[8], Raw8<_Float16>& r) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 a = {(_Float16)v[2 * j], (_Float16)v[2 * j + 1]};
    r.w[j] = __builtin_bit_cast(uint32_t, a);
  }
}
template <typename T> __device__ __forceinline__ void vec8_ld(const T* p, float (&o)[8]) { raw8_unpack(raw8_ld(p), o); }
template <typename T, bool NT = false>
__device__ __forceinline__ void vec8_st(T* p, const float (&v)[8]) {
  Raw8<T> r;
  raw8_pack(v, r);
  raw8_st<T, NT>(p, r);
}
