// Linear layer in 8-bit integers: y[m][n] = sx[m] sw[n] sum_k xq[m][k] wq[n][k] + bias[n].
//
//   sx[m] = max_k |x[m][k]| / 127,  xq[m][k] = round(127 x[m][k] / max_k |x[m][k]|)  (half to even), the same for the rows (output channels) of W.
//
// The integer sums are exact, so neither the order of k nor a split of it changes a result. A row that holds NaN or infinity has the scale NaN and
// codes 0: its outputs are NaN, the other rows are untouched. Rows of codes are padded with zeros to a multiple of I8_KPAD bytes.
//
// Measured (bf16, bias; quantisation + product in us, traced, after a hundred calls): 1 x 1024 -> 4096 4.1 in one launch; 8 x 2816 -> 1000 6.2 in one launch;
// 49 x 2816 -> 11264 3.6 + 9.4; 50176 x 512 -> 2048 16 + 82 (94 a call untraced; 27 % of the time in the matrix cores, output 205 MB); 12544 x 11264 -> 2816 75 + 303
// in whole rounds + 41 for the rest (2.3 PTOP/s). The library's int8 product reaches 2.4 PTOP/s at 16384^3 and takes 401 us for the last one, 120 us for
// the one before it, 21 us for 49 rows.
#pragma once
#include "vec8.cuh"
#include <type_traits>

#define I8_KPAD 128
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

// Eight elements of a row of at least eight from element i on: one load from a clamped address (a load behind a branch is waited for where the branch joins,
// and a row's loads would go one after the other). What lies past K becomes 0. Where K is no multiple of eight (RAGGED) the vector that straddles the end is
// replaced by `last`, which every lane loads, element by element, once per row.
template <typename T> __device__ __forceinline__ Raw8<T> i8_ld8(const T* row, int i, int K) { return raw8_ld(row + min(i, K - 8)); }
template <typename T, bool RAGGED>
__device__ __forceinline__ void i8_last8(const T* row, int K, float (&last)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) last[e] = RAGGED && (K & ~7) + e < K ? elem_ld(row + min((K & ~7) + e, K - 1)) : 0.f;
}
template <typename T, bool RAGGED>
__device__ __forceinline__ void i8_end8(int i, int K, const Raw8<T>& raw, const float (&last)[8], float (&o)[8]) {
  raw8_unpack(raw, o);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (RAGGED) o[e] = i + 8 <= K ? o[e] : i == (K & ~7) ? last[e] : 0.f;
    else o[e] = i < K ? o[e] : 0.f;
  }
}
// Eight codes. Adding 1.5 * 2^23 rounds x * (127 / a) to the nearest whole number (half to even) and leaves it, as a byte of two's complement, in the low
// bits of the sum. The rounded factor makes the product wrong by at most 127 * 2^-24 = 7.6e-6, so a code is certain unless the product lies within 2e-5 of a
// half; those (|x| = a / 2 is a common one in 16-bit types) are decided on the remainder 127 x - r a, which is exact: in fp32 for types of at most 11
// significant bits, in fp64 for fp32. up: 1, or 2^100 for a row whose reciprocal would overflow, 2^-100 where 127 a would; a and inv are those of the row times
// up (exact for every element that has a code but 0).
struct I8Row { float a, inv, up; };
__device__ __forceinline__ I8Row i8_row(unsigned mx) {
  I8Row r;
  r.a = __uint_as_float(mx);
  r.up = r.a < 1e-30f ? 0x1p100f : r.a > 1e30f ? 0x1p-100f : 1.f;
  r.a *= r.up;
  r.inv = 127.f / r.a;
  return r;
}
__device__ __forceinline__ float i8_scale(unsigned mx) { return mx >= 0x7f800000u ? NAN : __uint_as_float(mx) / 127.f; }
// An output. The sum meets the weight's scale first: with a row near the type's largest number (its lowest value as a mask) sum * sx alone would pass fp32's range.
__device__ __forceinline__ float i8_out(int sum, float sx, float sw, float bias) { return (float)sum * sw * sx + bias; }
template <typename T>
__device__ __forceinline__ uint2 i8_codes(const float (&x)[8], const I8Row& row) {
  constexpr float MAGIC = 12582912.f;
  unsigned u[8];
  float worst = 0.f, v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = x[e] * row.up;
    const float s = __builtin_fmaf(v[e], row.inv, MAGIC);
    worst = fmaxf(worst, fabsf(__builtin_fmaf(v[e], row.inv, -(s - MAGIC))));
    u[e] = __float_as_uint(s);
  }
  if (worst >= 0.49998f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      using F = typename std::conditional<sizeof(T) == 2, float, double>::type;
      const F r = (F)(__uint_as_float(u[e]) - MAGIC), rest = (F)127 * (F)v[e] - r * (F)row.a, twice = rest < 0 ? -2 * rest : 2 * rest;
      if (twice > (F)row.a || (twice == (F)row.a && (u[e] & 1))) u[e] += rest < 0 ? ~0u : 1u;
    }
  }
  uint2 q;
  q.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400), 0x05040100);
  q.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[7], u[6], 0x0c0c0400), __builtin_amdgcn_perm(u[5], u[4], 0x0c0c0400), 0x05040100);
  return q;
}
template <int TPR>
__device__ __forceinline__ unsigned i8_row_max(unsigned mx, unsigned* red) {      // over the TPR threads of a row: part of a wave, a wave, or (256) the workgroup
#pragma unroll
  for (int d = TPR < 64 ? TPR / 2 : 32; d; d >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, d));
  if (TPR == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  return mx;
}
// Rows to codes, the row held in registers between the maximum and the codes (NV vectors of eight per thread; NV = 0: any length of at least
// eight, the row is read twice; NV = -1: fewer than eight).
// Bound by memory: sizeof(T) + 1 bytes per element.
template <typename T, int TPR, int NV, bool RAGGED>
__device__ __forceinline__ void i8_quant_row(const T* row, int K, int8_t* out, int ldq, float* scale, int t, unsigned* red) {
  constexpr int NR = NV > 0 ? NV : 1;
  float v[NR][8], last[8];
  unsigned mx = 0;
  auto take = [&](const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(x[e]) & 0x7fffffffu);
  };
  if (NV > 0) {
    Raw8<T> raw[NR];
#pragma unroll
    for (int j = 0; j < NR; ++j) raw[j] = i8_ld8(row, (j * TPR + t) * 8, K);
    i8_last8<T, RAGGED>(row, K, last);
#pragma unroll
    for (int j = 0; j < NR; ++j) { i8_end8<T, RAGGED>((j * TPR + t) * 8, K, raw[j], last, v[j]); take(v[j]); }
  } else if (NV < 0) {                              // rows of fewer than eight elements
#pragma unroll
    for (int e = 0; e < 8; ++e) v[0][e] = t == 0 && e < K ? elem_ld(row + min(e, K - 1)) : 0.f;
    take(v[0]);
  } else {
    i8_last8<T, RAGGED>(row, K, last);
    for (int i = t * 8; i < K; i += TPR * 8) { i8_end8<T, RAGGED>(i, K, i8_ld8(row, i, K), last, v[0]); take(v[0]); }
  }
  mx = i8_row_max<TPR>(mx, red);
  const bool live = mx < 0x7f800000u && mx;
  const I8Row rw = i8_row(mx);
  if (t == 0) *scale = i8_scale(mx);
  if (NV != 0) {
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const int i = (j * TPR + t) * 8;
      uint2 c = make_uint2(0, 0);
      if (live) c = i8_codes<T>(v[j], rw);
      if (i < ldq) *reinterpret_cast<uint2*>(out + i) = c;
    }
  } else {
    for (int i = t * 8; i < ldq; i += TPR * 8) {
      uint2 c = make_uint2(0, 0);
      i8_end8<T, RAGGED>(i, K, i8_ld8(row, i, K), last, v[0]);
      if (live) c = i8_codes<T>(v[0], rw);
      *reinterpret_cast<uint2*>(out + i) = c;
    }
  }
}
template <typename T, int TPR, int NV, bool RAGGED>
__global__ __launch_bounds__(256) void i8_quant_kernel(const T* __restrict__ x, long long ldx, int M, int K, int8_t* __restrict__ q, int ldq,
                                                       float* __restrict__ scale) {
  __shared__ unsigned red[4];
  const int t = threadIdx.x % TPR;
  // (unsigned: the step past the last row, at most 2^24 rows on, may pass 31 bits)
  for (unsigned m = blockIdx.x * (256 / TPR) + threadIdx.x / TPR; m < (unsigned)M; m += gridDim.x * (256 / TPR)) {
    i8_quant_row<T, TPR, NV, RAGGED>(x + (size_t)m * ldx, K, q + (size_t)m * ldq, ldq, scale + m, t, red);
    if (TPR == 256) __syncthreads();      // red is written again
  }
}

// ---------------------------------------------------------------------------------
// Up to 16 rows: bound by reading W once. A workgroup of eight waves takes 16 columns and splits k between the waves, so that even a
// layer of 1000 columns has every load of W in flight at once; the eight integer partial sums meet in LDS. A wave's step is 128 bytes of k
// (two matrix operands of 64), so that every row of W is read in whole 128-byte lines. D[n][m] = W x^T: a lane ends with four consecutive columns of one row.
// FUSED: every workgroup quantises the rows itself, into LDS (x is small and in L2; the launch and the wait of a kernel of its own cost more).
// ---------------------------------------------------------------------------------
// M <= 8 rows to codes in LDS (row pitch Kp + 16: the matrix operands of 16 rows meet no bank twice), by eight waves: rows side by side, the waves that are
// left over share a row.
__host__ __device__ __forceinline__ int i8_waves_per_row(int M) { return M > 4 ? 1 : M > 2 ? 2 : M > 1 ? 4 : 8; }
// vectors of eight a lane holds of its row
__host__ __device__ __forceinline__ int i8_vectors(int M, int Kp) { return (Kp + 512 * i8_waves_per_row(M) - 1) / (512 * i8_waves_per_row(M)); }
constexpr int I8_KEPT = 6;
// A row's vectors, at most NV a lane, stay in registers between the maximum and the codes.
template <typename T, int NV, bool RAGGED>
__device__ __forceinline__ void i8_quant_kept(const T* __restrict__ x, long long ldx, int M, int K, int8_t* Al, int Kp, float* ssx, unsigned (*smax)[8]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wpr = i8_waves_per_row(M), r = w / wpr, part = w % wpr, step = wpr * 512, i0 = (part * 64 + lane) * 8;
  const T* row = x + (size_t)min(r, M - 1) * ldx;
  Raw8<T> raw[NV];
  float v[NV][8], last[8];
#pragma unroll
  for (int u = 0; u < NV; ++u) raw[u] = i8_ld8(row, i0 + u * step, K);
  i8_last8<T, RAGGED>(row, K, last);
  unsigned mx = 0;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    i8_end8<T, RAGGED>(i0 + u * step, K, raw[u], last, v[u]);
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(v[u][e]) & 0x7fffffffu);
  }
  mx = i8_row_max<64>(mx, nullptr);
  if (lane == 0) smax[r][part] = mx;
  __syncthreads();
  if (r < M) {
    mx = 0;
    for (int i = 0; i < wpr; ++i) mx = max(mx, smax[r][i]);
    const bool live = mx < 0x7f800000u && mx;
    const I8Row rw = i8_row(mx);
    if (part == 0 && lane == 0) ssx[r] = i8_scale(mx);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = i0 + u * step;
      uint2 c = i8_codes<T>(v[u], rw);
      c.x = live ? c.x : 0; c.y = live ? c.y : 0;
      if (i < Kp) *reinterpret_cast<uint2*>(Al + r * (Kp + 16) + i) = c;
    }
  }
  __syncthreads();
}
template <typename T, bool FUSED>
__global__ __launch_bounds__(512) void i8_skinny_kernel(const T* __restrict__ x, long long ldx, const int8_t* __restrict__ A, const float* __restrict__ sa,
                                                        const int8_t* __restrict__ B, const float* __restrict__ sb, const float* __restrict__ bias,
                                                        T* __restrict__ y, long long ldy, int M, int N, int K, int Kp) {
  extern __shared__ __attribute__((aligned(16))) unsigned char i8_smem[];
  int* red = reinterpret_cast<int*>(i8_smem);                                             // [8][16 m][16 n]
  int8_t* Al = reinterpret_cast<int8_t*>(i8_smem) + 8 * 1024;                             // [M][Kp + 16] (FUSED)
  __shared__ unsigned smax[8][8];
  __shared__ float ssx[8];
  // (matrix instructions ignore the lane mask: what decides whether a wave runs them is a scalar)
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int steps = Kp >> 7;
  const int8_t* b = B + (size_t)min(n0 + lr, N - 1) * Kp + lg * 16;
  constexpr int U = 4;                                      // steps whose loads are in flight together
  i32x4_t bv[U][2];
  auto load_w = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * 8 < steps) {
#pragma unroll
        for (int h = 0; h < 2; ++h) bv[u][h] = *reinterpret_cast<const i32x4_t*>(b + ((s0 + u * 8) << 7) + h * 64);
      }
  };
  load_w(w);                                                // the first weights are on their way while x is quantised
  if (FUSED) {
    const bool two = i8_vectors(M, Kp) <= 2;
    if ((K & 7) && two) i8_quant_kept<T, 2, true>(x, ldx, M, K, Al, Kp, ssx, smax);
    else if (K & 7) i8_quant_kept<T, I8_KEPT, true>(x, ldx, M, K, Al, Kp, ssx, smax);
    else if (two) i8_quant_kept<T, 2, false>(x, ldx, M, K, Al, Kp, ssx, smax);
    else i8_quant_kept<T, I8_KEPT, false>(x, ldx, M, K, Al, Kp, ssx, smax);
  }
  const int r = min(lr, M - 1);
  const int8_t* a = (FUSED ? Al + (size_t)r * (Kp + 16) : A + (size_t)r * Kp) + lg * 16;
  i32x4_t acc = {};
  for (int s0 = w; s0 < steps; s0 += 8 * U) {
    if (s0 != w) load_w(s0);
    i32x4_t av[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * 8 < steps) {
#pragma unroll
        for (int h = 0; h < 2; ++h) av[u][h] = *reinterpret_cast<const i32x4_t*>(a + ((s0 + u * 8) << 7) + h * 64);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * 8 < steps) {
#pragma unroll
        for (int h = 0; h < 2; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(bv[u][h], av[u][h], acc, 0, 0, 0);
      }
    }
  }
  *reinterpret_cast<i32x4_t*>(red + (w * 16 + lr) * 16 + lg * 4) = acc;      // lane: row lr, columns lg * 4 .. + 3
  __syncthreads();
  if (threadIdx.x < 256) {
    const int o = threadIdx.x, m = o >> 4, n = n0 + (o & 15);
    int sum = 0;
#pragma unroll
    for (int v = 0; v < 8; ++v) sum += red[v * 256 + o];
    if (m < M && n < N) elem_st(y + (size_t)m * ldy + n, i8_out(sum, FUSED ? ssx[m] : sa[m], sb[n], bias ? bias[n] : 0.f));
  }
}

// ---------------------------------------------------------------------------------
// Many rows. BM x BN tile, WM x WN waves, slabs of BK bytes of k that go global -> LDS directly (global_load_lds_dwordx4) into a ring of ST slots; one
// barrier per slab publishes slab kt and frees the slot that slab kt + ST - 1 lands in. A row of a slab is BK / 16 chunks of 16 bytes, unpadded; the chunk
// index is XORed with a function of the row, on the source address of the load and on the fragment read, so that 16 lanes that read one chunk of 16 rows
// meet no bank twice. D[n][m] = W x^T over pairs of column tiles with interleaved rows: a lane ends with eight consecutive columns of a row.
// ---------------------------------------------------------------------------------
typedef const __attribute__((address_space(1))) void* i8_gptr_t;
typedef __attribute__((address_space(3))) void* i8_lptr_t;

// ds_read_b128 is served in groups of sixteen lanes, {0-3, 12-15, 20-27} and so on: with these no group of either operand meets a bank twice (BK = 64 with the
// row's bits 2 and 3 instead: 36 % of the LDS cycles were conflicts)
template <int BK> __device__ __forceinline__ int i8_swz_a(int row) { return BK == 128 ? row & 7 : ((row >> 3) & 1) << 1; }
template <int BK> __device__ __forceinline__ int i8_swz_b(int row) { return BK == 128 ? ((row & 3) | (((row >> 3) & 1) << 2)) : ((row >> 3) & 1) << 1; }

constexpr int i8_tile_lds(int bm, int bn, int bk, int st) { return (bm + bn) * bk * st + (bm + 2 * bn) * 4; }
constexpr int i8_waves_per_simd(int lds, int waves) { return 160 * 1024 / lds * waves / 4 > 0 ? 160 * 1024 / lds * waves / 4 : 1; }
struct I8Tiles {
  int mt, nt;              // tiles of the whole product, of BM * subm rows and BN * subn columns
  int first, subm, subn;   // this launch: those from tile `first` on, each in subm * subn pieces
};

template <typename T, int BM, int BN, int WM, int WN, int BK, int ST, bool SPLIT>
__global__ __launch_bounds__(WM * WN * 64, i8_waves_per_simd(i8_tile_lds(BM, BN, BK, ST), WM * WN)) void i8_tile_kernel(
    const int8_t* __restrict__ A, const float* __restrict__ sa, const int8_t* __restrict__ B, const float* __restrict__ sb, const float* __restrict__ bias,
    T* __restrict__ y, long long ldy, int M, int N, int Kp, I8Tiles tl, int* __restrict__ part) {
  constexpr int NTH = WM * WN * 64, RCH = BK / 16, TM = BM / WM / 16, TN = BN / WN / 16, KS = BK / 64;
  constexpr int AB = BM * BK, BB = BN * BK, STAGE = AB + BB, LA = AB / 16 / NTH, LB = BB / 16 / NTH;
  static_assert(AB % (16 * NTH) == 0 && BB % (16 * NTH) == 0 && TN % 2 == 0 && i8_tile_lds(BM, BN, BK, ST) <= 160 * 1024, "tile shape");
  extern __shared__ __attribute__((aligned(16))) unsigned char i8_smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w / WN, wn = w % WN, lr = lane & 15, lg = lane >> 4;
  // tile order: workgroup L runs on XCD L % 8, whose L2 is its own: every XCD gets a contiguous run of tiles, four row tiles by all column tiles at a time
  int m0, n0;
  {
    const int c = blockIdx.x & 7, j = blockIdx.x >> 3, q = gridDim.x >> 3, r = gridDim.x & 7, id = c * q + min(c, r) + j;
    const int pieces = tl.subm * tl.subn, t = tl.first + id / pieces, piece = id % pieces;
    const int per = 4 * tl.nt, grp = t / per, top = grp * 4, gm = min(tl.mt - top, 4), in = t - grp * per;
    m0 = ((top + in % gm) * tl.subm + piece / tl.subn) * BM;
    n0 = ((in / gm) * tl.subn + piece % tl.subn) * BN;
    if (m0 >= M || n0 >= N) return;                          // (a piece of an edge tile with nothing in it; the whole workgroup)
  }
  // addresses: a uniform base and a 32-bit offset per lane (rows clamped: what lies past the last row or column is never stored)
  const int slabs = Kp / BK, k0 = SPLIT ? (int)((long long)slabs * blockIdx.y / gridDim.y) : 0;
  const int nk = SPLIT ? (int)((long long)slabs * (blockIdx.y + 1) / gridDim.y) - k0 : slabs;
  const int8_t* Ab = A + (size_t)m0 * Kp + (size_t)k0 * BK;
  const int8_t* Bb = B + (size_t)n0 * Kp + (size_t)k0 * BK;
  unsigned offA[LA], offB[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int sl = i * NTH + tid, row = sl / RCH, ch = (sl % RCH) ^ i8_swz_a<BK>(row);
    offA[i] = (unsigned)min(row, M - 1 - m0) * (unsigned)Kp + ch * 16;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int sl = i * NTH + tid, row = sl / RCH, ch = (sl % RCH) ^ i8_swz_b<BK>(row);
    offB[i] = (unsigned)min(row, N - 1 - n0) * (unsigned)Kp + ch * 16;
  }
  auto dma = [&](int slot, int kt) {
    unsigned char* base = i8_smem + slot * STAGE;
    const int8_t* ak = Ab + (size_t)kt * BK;
    const int8_t* bk = Bb + (size_t)kt * BK;
#pragma unroll
    for (int i = 0; i < LA; ++i) __builtin_amdgcn_global_load_lds((i8_gptr_t)(ak + offA[i]), (i8_lptr_t)(base + (i * NTH + w * 64) * 16), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < LB; ++i) __builtin_amdgcn_global_load_lds((i8_gptr_t)(bk + offB[i]), (i8_lptr_t)(base + AB + (i * NTH + w * 64) * 16), 16, 0, 0);
  };
  i32x4_t acc[TM][TN] = {};
  const int browl = (lr >> 2) * 8 + (lr & 3);                 // W rows of a pair of column tiles: + 4 for the second tile
  const int swa = i8_swz_a<BK>(lr), swb0 = i8_swz_b<BK>(browl), swb1 = i8_swz_b<BK>(browl + 4);
  const int arow = (wm * TM * 16 + lr) * BK, brow = (wn * TN * 16 + browl) * BK;
  auto frags = [&](int slot, int ks, i32x4_t (&bf)[TN], i32x4_t (&af)[TM]) {
    const unsigned char* as = i8_smem + slot * STAGE + arow;
    const unsigned char* bs = i8_smem + slot * STAGE + AB + brow;
    const int c = ks * 4 + lg;
#pragma unroll
    for (int j = 0; j < TN; ++j) bf[j] = *reinterpret_cast<const i32x4_t*>(bs + ((j >> 1) * 32 + (j & 1) * 4) * BK + (c ^ (j & 1 ? swb1 : swb0)) * 16);
#pragma unroll
    for (int i = 0; i < TM; ++i) af[i] = *reinterpret_cast<const i32x4_t*>(as + i * 16 * BK + (c ^ swa) * 16);
  };
  auto products = [&](const i32x4_t (&bf)[TN], const i32x4_t (&af)[TM]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af[i], acc[i][j], 0, 0, 0);
  };
  // slab kt has landed for this wave's own requests once only the ST - 2 younger slabs are outstanding; its own reads of the slab before are done
  auto ready = [&](int kt) {
    if (kt + ST - 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((ST - 2) * (LA + LB)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // scales and bias of the tile go to LDS under the first slabs: read at the end, they would stand in front of the stores of a short k
  float* const ep = reinterpret_cast<float*>(i8_smem + STAGE * ST);       // [BM] scales of x, [BN] scales of W, [BN] bias
  float ev[(BM + 2 * BN + NTH - 1) / NTH];
  if constexpr (!SPLIT) {
#pragma unroll
    for (int i = 0; i < (BM + 2 * BN + NTH - 1) / NTH; ++i) {
      const int j = i * NTH + tid;
      const float* src = j < BM ? sa + min(m0 + j, M - 1) : j < BM + BN ? sb + min(n0 + j - BM, N - 1) : (bias ? bias : sb) + min(n0 + j - BM - BN, N - 1);
      ev[i] = *src;
    }
  }
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) if (s < nk) dma(s, s);
  if constexpr (!SPLIT) {
#pragma unroll
    for (int i = 0; i < (BM + 2 * BN + NTH - 1) / NTH; ++i) {
      const int j = i * NTH + tid;
      if (j < BM + 2 * BN) ep[j] = j < BM + BN || bias ? ev[i] : 0.f;
    }
  }
  int slot = 0;
  if constexpr (KS == 2) {
    // the fragments of the next half slab are read under the products of the current one, across the barrier too
    i32x4_t bf[2][TN], af[2][TM];
    ready(0);
    if (ST - 1 < nk) dma(ST - 1, ST - 1);
    frags(0, 0, bf[0], af[0]);
    for (int kt = 0; kt < nk; ++kt) {
      frags(slot, 1, bf[1], af[1]);
      products(bf[0], af[0]);
      const int next = slot == ST - 1 ? 0 : slot + 1;
      if (kt + 1 < nk) {
        ready(kt + 1);
        if (kt + ST < nk) dma(slot, kt + ST);                 // the slot that slab kt has just left
        frags(next, 0, bf[0], af[0]);
      }
      products(bf[1], af[1]);
      slot = next;
    }
  } else {
    for (int kt = 0; kt < nk; ++kt) {
      ready(kt);
      if (kt + ST - 1 < nk) dma(slot == 0 ? ST - 1 : slot - 1, kt + ST - 1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        i32x4_t bf[TN], af[TM];
        frags(slot, ks, bf, af);
        products(bf, af);
      }
      slot = slot == ST - 1 ? 0 : slot + 1;
    }
  }
  // lane: row m0 + wm * TM * 16 + i * 16 + lr, columns n0 + wn * TN * 16 + jp * 32 + lg * 8 + (half * 4 + e)
  if constexpr (SPLIT) {                                      // integer partial sums, [split][M][N]
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = m0 + wm * TM * 16 + i * 16 + lr;
      if (row >= M) continue;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int col = n0 + wn * TN * 16 + (j >> 1) * 32 + lg * 8 + (j & 1) * 4;
        int* out = part + ((size_t)blockIdx.y * M + row) * N + col;
        if ((N & 3) == 0 && col < N) *reinterpret_cast<i32x4_t*>(out) = acc[i][j];
        else {
#pragma unroll
          for (int e = 0; e < 4; ++e) if (col + e < N) out[e] = acc[i][j][e];
        }
      }
    }
    return;
  }
  // y goes past the caches where its pieces of 64 bytes are whole; pieces that straddle need the cache to be put together. us of the layer, in brackets with a GELU
  // that reads y behind it, past the caches / through them:
  //   bf16  1568 x 512 -> 2048 (6.4 MB) 10.9 (17.8) / 11.3 (18.6)    3136 x 640 -> 2560 (16 MB) 17.4 (29.2) / 18.3 (30.4)    12544 x 512 -> 2048 (51 MB) 35.0 (58.5) / 35.1 (58.4)
  //         12544 x 1024 -> 4096 (103 MB) 77.4 (122) / 81.0 (125)    50176 x 512 -> 2048 (206 MB) 93.7 (185) / 101 (194)    200704 x 80 -> 320 (129 MB) 55.6 (108) / 53.0 (107)
  //   fp32  784 x 640 -> 2560 (8 MB) 10.7 (16.1) / 11.0 (17.2)       3136 x 320 -> 1280 (16 MB) 12.4 (22.4) / 13.0 (23.5)    12544 x 320 -> 1280 (64 MB) 28.8 (46.5) / 27.8 (46.7)
  //         50176 x 160 -> 640 (129 MB) 51.7 (84.0) / 41.6 (83.8): what a layer alone gains there, its reader pays
  const bool past = ((((uintptr_t)y) | ((uintptr_t)ldy * sizeof(T))) & 63) == 0;
#pragma unroll
  for (int jp = 0; jp < TN / 2; ++jp) {
    const int col = n0 + wn * TN * 16 + jp * 32 + lg * 8;
    float s[8], c[8];
    ld8(ep + BM + col - n0, s);
    ld8(ep + BM + BN + col - n0, c);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = m0 + wm * TM * 16 + i * 16 + lr;
      if (row >= M) continue;
      const float sr = ep[row - m0];
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i8_out(acc[i][2 * jp + (e >> 2)][e & 3], sr, s[e], c[e]);
      T* out = y + (size_t)row * ldy + col;
      if (past && col + 8 <= N) vec8_st<T, true>(out, v);
      else if (col + 8 <= N) vec8_st(out, v);
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (col + e < N) elem_st(out + e, v[e]);
      }
    }
  }
}

// sums of the splits -> y
template <typename T>
__global__ __launch_bounds__(256) void i8_join_kernel(const int* __restrict__ part, int splits, const float* __restrict__ sa, const float* __restrict__ sb,
                                                      const float* __restrict__ bias, T* __restrict__ y, long long ldy, int M, int N) {
  const long long all = (long long)M * N;
  for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < all; o += (long long)gridDim.x * 256) {
    int sum = 0;
    for (int s = 0; s < splits; ++s) sum += part[(size_t)s * all + o];
    const int m = (int)(o / N), n = (int)(o - (long long)m * N);
    elem_st(y + (size_t)m * ldy + n, i8_out(sum, sa[m], sb[n], bias ? bias[n] : 0.f));
  }
}
