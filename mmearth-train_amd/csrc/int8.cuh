// Linear layer in 8-bit integers: y[m][n] = sx[m] sw[n] sum_k xq[m][k] wq[n][k] + bias[n].
//
//   sx[m] = max_k |x[m][k]| / 127,  xq[m][k] = round(127 x[m][k] / max_k |x[m][k]|)  (half to even), the same for the rows (output channels) of W.
//
// The integer sums are exact, so neither the order of k nor a split of it changes a result. A row that holds NaN or infinity has the scale NaN and
// codes 0: its outputs are NaN, the other rows are untouched. Rows of codes are padded with zeros to a multiple of I8_KPAD bytes.
#pragma once
#include "common.cuh"

#define I8_KPAD 128
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

template <typename T> struct I8Io;
template <> struct I8Io<float> {
  static __device__ __forceinline__ float ld(const float* p) { return *p; }
  static __device__ __forceinline__ void ld8v(const float* p, float (&o)[8]) { ld8(p, o); }
  static __device__ __forceinline__ void st(float* p, float v) { *p = v; }
};
template <> struct I8Io<bf16_t> {
  static __device__ __forceinline__ float ld(const bf16_t* p) { return bf2f(*p); }
  static __device__ __forceinline__ void ld8v(const bf16_t* p, float (&o)[8]) { ld8(p, o); }
  static __device__ __forceinline__ void st(bf16_t* p, float v) { *p = f2bf(v); }
};
template <> struct I8Io<_Float16> {
  typedef __attribute__((ext_vector_type(8))) _Float16 h8;
  static __device__ __forceinline__ float ld(const _Float16* p) { return (float)*p; }
  static __device__ __forceinline__ void ld8v(const _Float16* p, float (&o)[8]) {
    const h8 a = *reinterpret_cast<const h8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
  }
  static __device__ __forceinline__ void st(_Float16* p, float v) { *p = (_Float16)v; }
};
// eight elements of a row from element i on; those at or past K read as 0
template <typename T>
__device__ __forceinline__ void i8_ld8(const T* row, int i, int K, bool vec, float (&o)[8]) {
  if (vec && i + 8 <= K) { I8Io<T>::ld8v(row + i, o); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = i + e < K ? I8Io<T>::ld(row + i + e) : 0.f;
}
// eight codes. t = 127 x / a in fp32 is off by less than 5e-5, so its code is right except next to a half, where 127 x / a is formed in fp64: the product
// is exact there, and a quotient of numbers of at most 31 and 24 bits that is not a half differs from one by far more than a rounding.
__device__ __forceinline__ uint2 i8_codes(const float (&x)[8], float a, float inv) {
  uint2 q = make_uint2(0, 0);
  const bool tiny = a < 1e-30f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float t = x[e] * inv, r = rintf(t);
    if (tiny || fabsf(fabsf(t - r) - 0.5f) < 1e-3f) r = (float)rint(127.0 * (double)x[e] / (double)a);
    const unsigned b = (unsigned)(int)r & 255u;
    if (e < 4) q.x |= b << (8 * e); else q.y |= b << (8 * (e - 4));
  }
  return q;
}
template <int TPR>
__device__ __forceinline__ unsigned i8_row_max(unsigned mx, unsigned* red) {      // over the TPR threads of a row; 64: one wave, 256: the workgroup
#pragma unroll
  for (int d = 32; d; d >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, d));
  if (TPR == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  return mx;
}
// Rows to codes, the row held in registers between the maximum and the codes (NV vectors of eight per thread; NV = 0: any length, the row is read twice).
// Bound by memory: sizeof(T) + 1 bytes per element.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void i8_quant_kernel(const T* __restrict__ x, long long ldx, int M, int K, int8_t* __restrict__ q, int ldq,
                                                       float* __restrict__ scale) {
  __shared__ unsigned red[4];
  const int t = threadIdx.x % TPR;
  const bool vec = ((((uintptr_t)x) | ((uintptr_t)ldx * sizeof(T))) & 15) == 0;
  constexpr int NR = NV ? NV : 1;
  for (int m = blockIdx.x * (256 / TPR) + threadIdx.x / TPR; m < M; m += gridDim.x * (256 / TPR)) {
    const T* row = x + (size_t)m * ldx;
    float v[NR][8];
    unsigned mx = 0;
    if (NV) {
#pragma unroll
      for (int j = 0; j < NR; ++j) i8_ld8(row, (j * TPR + t) * 8, K, vec, v[j]);
#pragma unroll
      for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(v[j][e]) & 0x7fffffffu);
    } else {
      for (int i = t * 8; i < K; i += TPR * 8) {
        i8_ld8(row, i, K, vec, v[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(v[0][e]) & 0x7fffffffu);
      }
    }
    mx = i8_row_max<TPR>(mx, red);
    const bool bad = mx >= 0x7f800000u;
    const float a = __uint_as_float(mx), inv = 127.f / a;
    int8_t* out = q + (size_t)m * ldq;
    if (t == 0) scale[m] = bad ? NAN : (float)((double)a / 127.0);
    if (NV) {
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        const int i = (j * TPR + t) * 8;
        uint2 c = make_uint2(0, 0);
        if (!bad && mx) c = i8_codes(v[j], a, inv);
        if (i < ldq) *reinterpret_cast<uint2*>(out + i) = c;
      }
    } else {
      for (int i = t * 8; i < ldq; i += TPR * 8) {
        uint2 c = make_uint2(0, 0);
        i8_ld8(row, i, K, vec, v[0]);
        if (!bad && mx) c = i8_codes(v[0], a, inv);
        *reinterpret_cast<uint2*>(out + i) = c;
      }
    }
    if (TPR == 256) __syncthreads();      // red is written again
  }
}

// Any shape: 64 x 64 tile, wave w computes 64 rows x 16 columns straight from global memory. v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k of
// row / column l % 16 from (l / 16) * 16 on; the result lane l holds rows (l / 16) * 4 + i of column l % 16.
template <typename T>
__global__ __launch_bounds__(256) void i8_gemm_kernel(const int8_t* __restrict__ A, int lda, const float* __restrict__ sa, const int8_t* __restrict__ B, int ldb,
                                                      const float* __restrict__ sb, const float* __restrict__ bias, T* __restrict__ y, long long ldy, int M, int N,
                                                      int Kp) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int m0 = blockIdx.x * 64, n = blockIdx.y * 64 + w * 16 + (lane & 15);
  const int8_t* b = B + (size_t)min(n, N - 1) * ldb + (lane >> 4) * 16;
  const int8_t* a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = A + (size_t)min(m0 + i * 16 + (lane & 15), M - 1) * lda + (lane >> 4) * 16;
  i32x4_t acc[4] = {};
  for (int k = 0; k < Kp; k += 64) {
    const i32x4_t bv = *reinterpret_cast<const i32x4_t*>(b + k);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4_t*>(a[i] + k), bv, acc[i], 0, 0, 0);
  }
  if (n >= N) return;
  const float s = sb[n], c = bias ? bias[n] : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int m = m0 + i * 16 + (lane >> 4) * 4 + e;
      if (m < M) I8Io<T>::st(y + (size_t)m * ldy + n, (float)acc[i][e] * sa[m] * s + c);
    }
}
