// extern "C" surface of libmpmae_hip.so, 8-bit integer linear layer (int8.cuh). gfx950 only.
#include "capi_common.h"
#include "int8.cuh"
#include <algorithm>
using std::min;

template <typename T>
static void quant_rows(const T* x, long long ldx, int M, int K, int8_t* q, int ldq, float* scale, hipStream_t st) {
#define I8_Q(TPR, NV) LAUNCH((i8_quant_kernel<T, TPR, NV>), dim3(min(cdiv(M, 256 / TPR), 1 << 20)), dim3(256), 0, st, x, ldx, M, K, q, ldq, scale)
  // a wave per row while four vectors per lane hold it, then a workgroup per row, then a workgroup that reads the row twice
  if (ldq <= 512) I8_Q(64, 1);
  else if (ldq <= 1024) I8_Q(64, 2);
  else if (ldq <= 2048) I8_Q(64, 4);
  else if (ldq <= 4096) I8_Q(256, 2);
  else if (ldq <= 8192) I8_Q(256, 4);
  else if (ldq <= 16384) I8_Q(256, 8);
  else I8_Q(256, 0);
#undef I8_Q
}
template <typename T>
static void gemm_i8(const MpmaeI8Args& a, const int8_t* q, const float* sx, hipStream_t st) {
  LAUNCH(i8_gemm_kernel<T>, dim3(cdiv(a.M, 64), cdiv(a.N, 64)), dim3(256), 0, st, q, a.ldq, sx, a.w, a.ldw, a.sw, a.bias, (T*)a.y, a.ldy, a.M, a.N, a.ldq);
}
static bool bad_rows(int dt, const void* x, long long ldx, int M, int K, const void* q, int ldq, const float* scale) {
  return dt < 0 || dt > 2 || !x || !q || !scale || M < 1 || K < 1 || K > 131071 || ldx < 0 || ldq < K || ldq % I8_KPAD || ((uintptr_t)q & 15);
}

extern "C" {

int mpmae_quant_i8(int dt, const void* x, long long ldx, int M, int K, int8_t* q, int ldq, float* scale, mpmae_stream_t s) {
  if (bad_rows(dt, x, ldx, M, K, q, ldq, scale)) return (int)hipErrorInvalidValue;
  if (dt == 0) quant_rows((const float*)x, ldx, M, K, q, ldq, scale, S_(s));
  else if (dt == 1) quant_rows((const bf16_t*)x, ldx, M, K, q, ldq, scale, S_(s));
  else quant_rows((const _Float16*)x, ldx, M, K, q, ldq, scale, S_(s));
  RET();
}

int mpmae_linear_i8(int dt, const MpmaeI8Args* args, mpmae_stream_t s) {
  if (!args) return (int)hipErrorInvalidValue;
  const MpmaeI8Args a = *args;
  if (bad_rows(dt, a.x, a.ldx, a.M, a.K, a.q, a.ldq, a.sx) || !a.w || !a.sw || !a.y || a.N < 1 || a.ldy < a.N || a.ldw != a.ldq || ((uintptr_t)a.w & 15) ||
      cdiv(a.N, 64) > 65535)
    return (int)hipErrorInvalidValue;
  const int err = mpmae_quant_i8(dt, a.x, a.ldx, a.M, a.K, a.q, a.ldq, a.sx, s);
  if (err) return err;
  if (dt == 0) gemm_i8<float>(a, a.q, a.sx, S_(s));
  else if (dt == 1) gemm_i8<bf16_t>(a, a.q, a.sx, S_(s));
  else gemm_i8<_Float16>(a, a.q, a.sx, S_(s));
  RET();
}

}  // extern "C"
