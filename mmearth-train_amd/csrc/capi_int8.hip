// extern "C" surface of libmpmae_hip.so, 8-bit integer linear layer (int8.cuh). gfx950 only.
#include "capi_common.h"
#include "int8.cuh"
#include <algorithm>
using std::min;

template <typename T, bool RAGGED>
static void quant_rows_of(const T* x, long long ldx, int M, int K, int8_t* q, int ldq, float* scale, hipStream_t st) {
#define I8_Q(TPR, NV) LAUNCH((i8_quant_kernel<T, TPR, NV, RAGGED>), dim3(min(cdiv(M, 256 / TPR), 1 << 20)), dim3(256), 0, st, x, ldx, M, K, q, ldq, scale)
  // 16 or 32 lanes per short row (49050 x 18: a wave per row takes four times the waves), a wave per row while four vectors per lane hold it, then a workgroup per
  // row, then a workgroup that reads the row twice
  if (K < 8) I8_Q(16, -1);
  else if (ldq <= 128) I8_Q(16, 1);
  else if (ldq <= 256) I8_Q(32, 1);
  else if (ldq <= 512) I8_Q(64, 1);
  else if (ldq <= 1024) I8_Q(64, 2);
  else if (ldq <= 2048) I8_Q(64, 4);
  else if (ldq <= 4096) I8_Q(256, 2);
  else if (ldq <= 8192) I8_Q(256, 4);
  else if (ldq <= 16384) I8_Q(256, 8);
  else I8_Q(256, 0);
#undef I8_Q
}
template <typename T>
static void quant_rows(const T* x, long long ldx, int M, int K, int8_t* q, int ldq, float* scale, hipStream_t st) {
  if (K & 7) quant_rows_of<T, true>(x, ldx, M, K, q, ldq, scale, st);
  else quant_rows_of<T, false>(x, ldx, M, K, q, ldq, scale, st);
}
template <typename T, bool FUSED>
static void skinny(const MpmaeI8Args& a, hipStream_t st) {
  const size_t lds = 8 * 1024 + (FUSED ? (size_t)a.M * (a.ldq + 16) : 0);
  LAUNCH((i8_skinny_kernel<T, FUSED>), dim3(cdiv(a.N, 16)), dim3(512), lds, st, (const T*)a.x, a.ldx, (const int8_t*)a.q, (const float*)a.sx, a.w, a.sw,
         a.bias, (T*)a.y, a.ldy, a.M, a.N, a.K, a.ldq);
}
template <typename T, int BM, int BN, int WM, int WN, int BK, int ST>
static void tiles(const MpmaeI8Args& a, int count, const I8Tiles& tl, hipStream_t st) {
  LAUNCH((i8_tile_kernel<T, BM, BN, WM, WN, BK, ST, false>), dim3(count * tl.subm * tl.subn), dim3(WM * WN * 64), i8_tile_lds(BM, BN, BK, ST), st, (const int8_t*)a.q,
         (const float*)a.sx, a.w, a.sw, a.bias, (T*)a.y, a.ldy, a.M, a.N, a.ldq, tl, (int*)nullptr);
}
template <typename T, int BM, int BN, int WM, int WN, int BK, int ST>
static void tiles(const MpmaeI8Args& a, hipStream_t st) {
  const int mt = cdiv(a.M, BM), nt = cdiv(a.N, BN);
  tiles<T, BM, BN, WM, WN, BK, ST>(a, mt * nt, I8Tiles{mt, nt, 0, 1, 1}, st);
}
// Parts of k for a product with so few tiles that W would come in through a few compute units: about 512 workgroups, at least 1024 of k each.
// 64 x 11264 -> 1000: 20.8 us whole, 10.8 us in eight parts with the join; 300 x 4096 -> 320: 9.8 / 8.8 us in four; 100 x 2816 -> 320: 7.1 / 7.0 us, so
// shorter rows stay whole, and so do products of over 128 tiles (20 x 11264 -> 11264, 176 tiles: 32.8 / 33.1 us).
static bool i8_few(int M, int N) { return M <= 16 && cdiv(N, 16) <= 512; }
static int i8_splits(int M, int N, int Kp) {
  const long long t = (long long)cdiv(M, 32) * cdiv(N, 64);
  if (i8_few(M, N) || t > 128 || Kp < 4096) return 1;
  return (int)min<long long>(min<long long>(512 / t, Kp / 1024), 8);
}
template <typename T>
static void linear_i8(const MpmaeI8Args& a, hipStream_t st) {
  // Up to 8 rows of a moderate length: one launch that quantises and multiplies (1 x 1024 -> 4096: 4.1 us; 7.2 us in two launches). A workgroup holds the rows in
  // its registers; longer ones go through a launch of their own.
  if (a.M <= 8 && i8_vectors(a.M, a.ldq) <= I8_KEPT && a.K >= 8) return skinny<T, true>(a, st);
  quant_rows((const T*)a.x, a.ldx, a.M, a.K, a.q, a.ldq, a.sx, st);
  auto count = [&](int bm, int bn) { return (long long)cdiv(a.M, bm) * cdiv(a.N, bn); };
  const int splits = i8_splits(a.M, a.N, a.ldq);
  // 16 x 2816 -> 1000: 4.3 us with k split between the waves, 7.1 us in 32 x 64 tiles; -> 11264: 11.4 and 7.9 us
  if (i8_few(a.M, a.N)) return skinny<T, false>(a, st);
  if (splits > 1) {
    const int mt = cdiv(a.M, 32), nt = cdiv(a.N, 64);
    LAUNCH((i8_tile_kernel<T, 32, 64, 2, 2, 128, 4, true>), dim3(mt * nt, splits), dim3(256), i8_tile_lds(32, 64, 128, 4), st, (const int8_t*)a.q, (const float*)a.sx, a.w, a.sw,
           a.bias, (T*)a.y, a.ldy, a.M, a.N, a.ldq, (I8Tiles{mt, nt, 0, 1, 1}), a.part);
    LAUNCH(i8_join_kernel<T>, dim3(grid1d((long long)a.M * a.N, 256, 4096)), dim3(256), 0, st, (const int*)a.part, splits, (const float*)a.sx, a.sw, a.bias, (T*)a.y,
           a.ldy, a.M, a.N);
    return;
  }
  // Tile by the number of tiles that 256 compute units get (us of the product alone; M x K -> N; the last column with its remainder in pieces):
  //                          32 x 64   64 x 64  128 x 64  128 x 128  256 x 128  256 x 256
  //   49 x 2816 -> 11264         9.8      10.1      15.6       17.5       30.4       17.5
  //   784 x 2816 -> 2816        20.5      17.6      17.9       19.7       34.5       19.5
  //   12544 x 512 -> 2048       52.5      35.2      29.0       28.8       29.7       31.1
  //   1568 x 1024 -> 4096       23.1      17.9      17.2       14.7       18.3       14.1
  //   6272 x 2048 -> 2048       64.2      44.9      39.5       36.3       36.0       35.7
  //   25088 x 640 -> 2560      132.8      86.3      66.5       61.7       57.8       68.4
  //   25088 x 160 -> 640        25.5      19.2      15.7       15.5       15.3       20.9
  //   4096 x 4096 -> 4096      146.3     100.0      76.6       68.7       70.6       58.6
  //   12544 x 2048 -> 4096     247.2     164.7     124.6      114.1      122.8      102.7
  // 256 x 256 reads LDS least per product, but a workgroup has a compute unit to itself: it needs a long k to cover its first loads and its stores.
  if (count(32, 64) <= 512) return tiles<T, 32, 64, 2, 2, 128, 4>(a, st);
  if (count(64, 64) <= 1024) return tiles<T, 64, 64, 2, 2, 128, 3>(a, st);
  if (a.K >= 2048 && count(256, 256) >= 256) {
    // whole rounds of one tile per compute unit, and what is left over in pieces that fill one round (12544 x 11264 -> 2816: 539 tiles: 470 us in three rounds,
    // 360 us in two and 27 tiles in eighths)
    const int mt = cdiv(a.M, 256), nt = cdiv(a.N, 256), all = mt * nt, full = all % 256 > 224 ? all : all / 256 * 256;
    tiles<T, 256, 256, 2, 4, 128, 2>(a, full, I8Tiles{mt, nt, 0, 1, 1}, st);
    if (all - full > 32) tiles<T, 128, 128, 2, 2, 128, 2>(a, all - full, I8Tiles{mt, nt, full, 2, 2}, st);
    else if (all > full) tiles<T, 128, 64, 2, 2, 128, 4>(a, all - full, I8Tiles{mt, nt, full, 2, 4}, st);
    return;
  }
  if (count(256, 128) >= 1536) return tiles<T, 256, 128, 2, 2, 64, 2>(a, st);
  if (a.K >= 1024) return tiles<T, 128, 128, 2, 2, 128, 2>(a, st);
  tiles<T, 128, 64, 2, 2, 128, 2>(a, st);
}
// (ldq: K rounded up and nothing else, since the split of k, and with it the workspace, goes by K alone and rows of fewer than eight elements pad one I8_KPAD)
static int row_bytes(int K) { return (K + I8_KPAD - 1) / I8_KPAD * I8_KPAD; }
static bool bad_rows(int dt, const void* x, long long ldx, int M, int K, const void* q, int ldq, const float* scale) {
  return dt < 0 || dt > 2 || !x || !q || !scale || M < 1 || K < 1 || K > 131071 || ldx < 0 || ldq != row_bytes(K) || ((uintptr_t)q & 15);
}

extern "C" {

int mpmae_quant_i8(int dt, const void* x, long long ldx, int M, int K, int8_t* q, int ldq, float* scale, mpmae_stream_t s) {
  if (bad_rows(dt, x, ldx, M, K, q, ldq, scale)) return (int)hipErrorInvalidValue;
  if (dt == 0) quant_rows((const float*)x, ldx, M, K, q, ldq, scale, S_(s));
  else if (dt == 1) quant_rows((const bf16_t*)x, ldx, M, K, q, ldq, scale, S_(s));
  else quant_rows((const _Float16*)x, ldx, M, K, q, ldq, scale, S_(s));
  RET();
}

long long mpmae_linear_i8_part_bytes(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1 || K > 131071) return 0;
  const int s = i8_splits(M, N, row_bytes(K));
  return s > 1 ? (long long)s * M * N * 4 : 0;
}

int mpmae_linear_i8(int dt, const MpmaeI8Args* args, mpmae_stream_t s) {
  if (!args) return (int)hipErrorInvalidValue;
  const MpmaeI8Args a = *args;
  if (bad_rows(dt, a.x, a.ldx, a.M, a.K, a.q, a.ldq, a.sx) || !a.w || !a.sw || !a.y || a.N < 1 || a.ldy < a.N || a.ldw != a.ldq || ((uintptr_t)a.w & 15) ||
      (i8_splits(a.M, a.N, a.ldq) > 1 && !a.part) || ((uintptr_t)a.part & 15))
    return (int)hipErrorInvalidValue;
  if (dt == 0) linear_i8<float>(a, S_(s));
  else if (dt == 1) linear_i8<bf16_t>(a, S_(s));
  else linear_i8<_Float16>(a, S_(s));
  RET();
}

}  // extern "C"
