// AdamW over many separate parameter tensors (fp32 / bf16 / fp16 each), moments in fp32 or in 8 bits, optional clip by the global gradient norm.
//
//   g' = g * min(1, max_norm / (|g| + 1e-6))         |g| over every tensor of the step
//   m  <- b1 m + (1 - b1) g'      v <- b2 v + (1 - b2) g'^2
//   p  <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments: blocks of 256 elements in storage order (a tensor starts a block of its own), per block
//   m = s_m k|k| / 127^2 (k int8),  v = s_v (k / 255)^4 (k uint8),  s_m = max|m|, s_v = max v (fp32)
// The square / fourth-power steps keep the relative step of |m| and sqrt(v) small near the top of a block (1.6 % / 0.8 %) and still reach down to
// 6e-5 / 1.5e-5 of it; a positive v never becomes code 0, so the denominator of the next step cannot vanish while m stays.
//
// Everything is bound by memory: 3 * sizeof(p) + 16 bytes per element (fp32 moments), 3 * sizeof(p) + 4 + 1/16 (8 bits), + sizeof(p) for the norm, whose pass
// over the gradients has to end before the first update. A large copy moves 4.8 TB/s on this card, a large sum reads 4.0.
//   660 M parameters, bf16, fp32 moments: 2.76 ms, 5.3 TB/s.   88.7 M fp32 with a clip: norm 101 us (3.5 TB/s) + 423 us (5.9 TB/s of addressed bytes).
//   660 M fp32, 8 bits: 1.94 ms, 5.5 TB/s.                     88.7 M bf16, 8 bits, with a clip: norm 56 us + 156 us (5.7 TB/s; vector units nine tenths busy).
//   3.7 M fp32 (144 tensors): 19 us (fp32 moments), 14 us (8 bits), next to 2.4 us for the step's records.
// A workgroup takes one piece of 2048 elements of one tensor, a thread one vector of eight: 4096-element pieces were 4 % slower, and the piece list (8 bytes per
// piece, made once) lets a launch cover tensors of one element and of 10^9 alike.
#pragma once
#include "vec8.cuh"

#define ADAMW_CHUNK 2048      // elements per workgroup of 256 threads: one vector of eight per thread
#define ADAMW_BLOCK 256       // elements per 8-bit block
#define ADAMW_MAX_GRADS 480   // tensors per launch: the gradients' addresses travel in the kernel arguments (4 KB at most)
#define ADAMW_MAX_GROUPS 48   // parameter groups per hyper launch (56 bytes each) and
#define ADAMW_MAX_HAS 512     // tensors per hyper launch (one bit each: has a gradient)

struct AdamwTensor {          // device table, one per parameter tensor (host mirror: MpmaeAdamwTensor)
  long long n, off;           // elements; first element in the flat moment buffers (a multiple of ADAMW_BLOCK)
  void* p;
  int group, dt;              // parameter group; 0 fp32, 1 bf16, 2 fp16
};
struct AdamwHyper {           // device table, one per parameter tensor, written by adamw_hyper_kernel for this step
  double b1, c1, b2, c2, coef;      // c = 1 - b; coef: the clip factor
  float decay, step, isbc2, eps;
};
struct AdamwGrads {
  const void* g[ADAMW_MAX_GRADS];
  int first;                  // index of the launch's first tensor
};
struct AdamwGroups {
  struct { double lr, b1, b2, eps, wd, ln_b1, ln_b2; } at[ADAMW_MAX_GROUPS];
  unsigned has[ADAMW_MAX_HAS / 32];
  int first, count, t0, t1;   // groups [first, first + count), tensors [t0, t1)
};

// block-uniform fp64 sum in a fixed order (wave butterflies, then the four waves in order)
__device__ __forceinline__ double adamw_block_sum(double x, double* red) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[w] = x;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < nw; ++i) s += red[i];
  return s;
}

// Eight consecutive elements from i on; those at or past n read as 0 and are not written. FULL: all inside. Loads are never behind a branch (one
// is waited for where the branch joins): a ragged tensor's come from clamped addresses.
template <typename T, bool FULL>
__device__ __forceinline__ void adamw_ld8(const T* p, long long i, long long n, float (&o)[8]) {
  if (FULL) { vec8_ld(p + i, o); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = elem_ld(p + min(i + e, n - 1));
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = i + e < n ? o[e] : 0.f;
}
template <typename T, bool FULL>
__device__ __forceinline__ void adamw_st8(T* p, long long i, long long n, const float (&o)[8]) {
  if (FULL) { vec8_st(p + i, o); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (i + e < n) elem_st(p + i + e, o[e]);
}
// a workgroup's chunk in the form that its tensor allows
#define ADAMW_BY_TYPE(...)                                                                        \
  if (t.dt == 0) { using T = float; __VA_ARGS__ }                                                 \
  else if (t.dt == 1) { using T = bf16_t; __VA_ARGS__ }                                           \
  else { using T = _Float16; __VA_ARGS__ }

// ---------------------------------------------------------------------------------
// Sum of squares of every gradient of the launch, in fp64 (a factor that went into 8-bit codes must not depend on the summation order): workgroup b
// walks chunks first + b, first + b + gridDim, ...; one partial per workgroup, no atomics.
// ---------------------------------------------------------------------------------
template <typename T, bool FULL>
__device__ __forceinline__ double adamw_sumsq_chunk(const T* g, long long n, long long base) {
  float x[8];
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  adamw_ld8<T, FULL>(g, base + threadIdx.x * 8, n, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e & 3] += (double)x[e] * (double)x[e];
  return (s[0] + s[1]) + (s[2] + s[3]);
}
__global__ __launch_bounds__(256) void adamw_norm_kernel(AdamwGrads grads, const AdamwTensor* __restrict__ tensors, const int2* __restrict__ chunks,
                                                         int nchunks, double* __restrict__ partials) {
  __shared__ double red[4];
  double s = 0.0;
  // the next piece's description is read under the sum of the current one: three dependent reads would stand in front of every piece
  int2 ch = chunks[blockIdx.x];
  AdamwTensor t = tensors[ch.x];
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const int2 ch_next = chunks[min(c + (int)gridDim.x, nchunks - 1)];
    const void* g = grads.g[ch.x - grads.first];
    const long long base = (long long)ch.y * ADAMW_CHUNK;
    if (g) {
      const bool full = base + ADAMW_CHUNK <= t.n;
      ADAMW_BY_TYPE(s += full ? adamw_sumsq_chunk<T, true>((const T*)g, t.n, base) : adamw_sumsq_chunk<T, false>((const T*)g, t.n, base);)
    }
    ch = ch_next;
    t = tensors[ch.x];
  }
  s = adamw_block_sum(s, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// ---------------------------------------------------------------------------------
// One workgroup: folds the norm's partials, decides on a skip (a non-finite norm leaves everything as it was, steps included), counts the steps of the
// tensors that have a gradient and writes their records. 1 - b^t in fp64: at t = 1 it is a difference of near-equal numbers.
// ---------------------------------------------------------------------------------
__global__ __launch_bounds__(512) void adamw_hyper_kernel(AdamwGroups groups, const AdamwTensor* __restrict__ tensors,
                                                          int* __restrict__ steps, AdamwHyper* __restrict__ hyper,
                                                          const double* __restrict__ partials, int npartials, double max_norm,
                                                          float* __restrict__ norm_skip) {
  __shared__ double red[8];
  float coef = 1.f;
  if (npartials > 0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < npartials; i += 512) s += partials[i];
    const double norm = sqrt(adamw_block_sum(s, red));
    const bool bad = !((float)norm < INFINITY);      // (as the norm is reported: one past fp32's range reads as infinity)
    if (threadIdx.x == 0) { norm_skip[0] = (float)norm; norm_skip[1] = bad ? 1.f : 0.f; }
    if (bad) return;
    coef = (float)fmin(1.0, max_norm / (norm + 1e-6));
  }
  for (int i = groups.t0 + threadIdx.x; i < groups.t1; i += 512) {
    const int g = tensors[i].group - groups.first;
    if (g < 0 || g >= groups.count || !(groups.has[(i - groups.t0) >> 5] >> ((i - groups.t0) & 31) & 1)) continue;
    const int t = steps[i] + 1;
    steps[i] = t;
    const double b1 = groups.at[g].b1, b2 = groups.at[g].b2, lr = groups.at[g].lr;
    AdamwHyper h;
    h.b1 = b1; h.b2 = b2;
    h.c1 = 1.0 - b1; h.c2 = 1.0 - b2; h.coef = (double)coef;
    h.decay = (float)(1.0 - lr * groups.at[g].wd);
    h.step = (float)(lr / -expm1((double)t * groups.at[g].ln_b1));
    h.isbc2 = (float)(1.0 / sqrt(-expm1((double)t * groups.at[g].ln_b2)));
    h.eps = (float)groups.at[g].eps;
    hyper[i] = h;
  }
}

// ---------------------------------------------------------------------------------
// fp32 moments
// ---------------------------------------------------------------------------------
template <typename T, bool FULL, bool CLIP>
__device__ __forceinline__ void adamw32_chunk(T* __restrict__ p, const T* __restrict__ g, float* __restrict__ m, float* __restrict__ v, long long n,
                                              long long base, AdamwHyper h, const AdamwHyper* hp) {
#pragma clang fp contract(off)      // (the same bits whichever form a chunk takes)
  const long long i = base + threadIdx.x * 8;
  if (!FULL && i >= n) return;
  float pv[8], gv[8], mv[8], vv[8];
  adamw_ld8<T, FULL>(p, i, n, pv);
  adamw_ld8<T, FULL>(g, i, n, gv);
  ld8(m + i, mv);                       // the flat moment buffers are padded to whole blocks: zero behind the tensor, and zero they stay
  ld8(v + i, vv);
  if (!CLIP) {
    asm volatile("" ::: "memory");
    h = *hp;
  }
  // (the clip factor meets the gradient first: its square alone leaves fp32's range at norms whose clipped gradients are ordinary numbers)
  const float b1 = (float)h.b1, c1 = (float)h.c1, b2 = (float)h.b2, c2 = (float)h.c2, coef = (float)h.coef;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float gc = CLIP ? gv[e] * coef : gv[e];
    mv[e] = __builtin_fmaf(b1, mv[e], c1 * gc);
    vv[e] = __builtin_fmaf(b2, vv[e], c2 * gc * gc);
    pv[e] = __builtin_fmaf(pv[e], h.decay, -(h.step * mv[e] / __builtin_fmaf(sqrtf(vv[e]), h.isbc2, h.eps)));
  }
  adamw_st8<T, FULL>(p, i, n, pv);
  st8(m + i, mv);
  st8(v + i, vv);
}
template <bool CLIP>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamwGrads grads, const AdamwTensor* __restrict__ tensors, const int2* __restrict__ chunks,
                                                      const AdamwHyper* __restrict__ hyper, float* __restrict__ m, float* __restrict__ v,
                                                      const float* __restrict__ norm_skip) {
  // behind a norm the pieces are walked backwards: the gradients read last are the ones the memory-side cache still holds
  const int2 ch = chunks[norm_skip ? gridDim.x - 1 - blockIdx.x : blockIdx.x];
  const AdamwTensor t = tensors[ch.x];
  void* p = t.p;
  const void* g = grads.g[ch.x - grads.first];
  if (!g || (norm_skip && norm_skip[1] != 0.f)) return;
  // The step's record: read behind the vector loads, it is not waited for before the first of them (660 M bf16: 2760 us, 2785 in front); behind a norm's check of the skip
  // in front of them is faster (88.7 M fp32: 529 us with the norm, 538 behind)
  AdamwHyper h;
  if (CLIP) h = hyper[ch.x];
  const long long base = (long long)ch.y * ADAMW_CHUNK;
  const bool full = base + ADAMW_CHUNK <= t.n;
  ADAMW_BY_TYPE(if (full) adamw32_chunk<T, true, CLIP>((T*)p, (const T*)g, m + t.off, v + t.off, t.n, base, h, hyper + ch.x);
                else adamw32_chunk<T, false, CLIP>((T*)p, (const T*)g, m + t.off, v + t.off, t.n, base, h, hyper + ch.x);)
}

// ---------------------------------------------------------------------------------
// 8-bit moments. A lane holds eight consecutive elements, 32 lanes a block: the block's maxima are five lane exchanges. The moments are formed in fp64
// (full rate on this machine) and the codes decided on them (adamw_codes_m / _v). Each fp64 operation rounds on its own, in the order of the formula (no
// contraction): a block's scale is often an exact tie between two fp32 numbers ((9 s + g) / 10), and the scale, and with it every code, must not depend on how
// a compiler groups the terms. 60 vector instructions per element; at 16 bit parameters (10 bytes per element) they and the memory take about as long.
// ---------------------------------------------------------------------------------
__device__ __forceinline__ unsigned adamw_max32(unsigned x) {      // maximum over the 32 lanes of a half wave (bit patterns of non-negative floats)
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));       // lanes 1 0 3 2
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));       // lanes 2 3 0 1
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true));      // 8 lanes mirrored
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true));      // 16 lanes mirrored
  const auto y = __builtin_amdgcn_permlane16_swap(x, x, false, false);                // rows of 16: {0 0 2 2}, {1 1 3 3}
  return max(y[0], y[1]);
}
// Codes of eight moments. Their fp32 estimates t = 127 sqrt(|m| / s), 255 (v / s)^(1/4) are off by less than 6e-5 (relative errors: 1.5 ulp of the quotient, halved
// by each root, 1 ulp of each root), so rounding one is certain unless it lies within 1e-4 of a half; then the whole vector is decided on the border above
// the estimate's whole part, in fp64: |m| >= (f + 1/2)^2 s / 127^2, v >= (f + 1/2)^4 s / 255^4 (the square is exact in fp32).
__device__ __forceinline__ void adamw_codes_m(const double (&m)[8], float s, float (&k)[8]) {       // |codes|, 0..127
  const float inv = 16129.f / s;
  float near = 1.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = __builtin_amdgcn_sqrtf(fabsf((float)m[e]) * inv);
    near = fminf(near, fabsf(__builtin_amdgcn_fractf(t) - 0.5f));
    k[e] = rintf(t);                              // (t <= 127 (1 + 1e-6))
  }
  if (near < 1e-4f) {
    const double border = (double)s * (1.0 / 16129.0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = floorf(__builtin_amdgcn_sqrtf(fabsf((float)m[e]) * inv)), b = f + 0.5f;
      k[e] = fminf(f + (fabs(m[e]) >= (double)(b * b) * border ? 1.f : 0.f), 127.f);
    }
  }
}
__device__ __forceinline__ void adamw_codes_v(const double (&v)[8], float s, float (&k)[8]) {       // 0..255, at least 1 where v > 0
  const float inv = 65025.f * 65025.f / s;
  float near = 1.f, least = 255.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)v[e] * inv));
    near = fminf(near, fabsf(__builtin_amdgcn_fractf(t) - 0.5f));
    k[e] = rintf(t);
    least = fminf(least, k[e]);
  }
  if (near < 1e-4f || least < 1.f) {
    const double border = (double)s * (1.0 / (65025.0 * 65025.0));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = floorf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)v[e] * inv))), b = f + 0.5f;
      const double b2 = (double)(b * b);
      k[e] = fmaxf(fminf(f + (v[e] >= b2 * b2 * border ? 1.f : 0.f), 255.f), v[e] > 0.0 ? 1.f : 0.f);
    }
  }
}
template <typename T, bool FULL>
__device__ __forceinline__ void adamw8_chunk(T* __restrict__ p, const T* __restrict__ g, uint8_t* __restrict__ mc, uint8_t* __restrict__ vc,
                                             float* __restrict__ ms, float* __restrict__ vs, long long n, long long base, const AdamwHyper& h) {
#pragma clang fp contract(off)
  const long long blk = base / ADAMW_BLOCK + (threadIdx.x >> 5);
  const long long i = blk * ADAMW_BLOCK + (threadIdx.x & 31) * 8;
  if (!FULL && blk * ADAMW_BLOCK >= n) return;     // (uniform over the block's 32 lanes)
  float pv[8], gv[8];
  adamw_ld8<T, FULL>(p, i, n, pv);
  adamw_ld8<T, FULL>(g, i, n, gv);
  uint2 mq = *reinterpret_cast<const uint2*>(mc + i), vq = *reinterpret_cast<const uint2*>(vc + i);
  const double am = (double)ms[blk] * (1.0 / 16129.0), av = (double)vs[blk] * (1.0 / (65025.0 * 65025.0));
  mq.x ^= 0x80808080u; mq.y ^= 0x80808080u;        // signed bytes + 128: the byte conversions are unsigned
  double m[8], v[8];
  unsigned mx = 0, vx = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float km = (float)((e < 4 ? mq.x : mq.y) >> (8 * (e & 3)) & 255u) - 128.f, kv = (float)((e < 4 ? vq.x : vq.y) >> (8 * (e & 3)) & 255u);
    const double gd = (double)gv[e] * h.coef, kv2 = (double)(kv * kv);
    m[e] = h.b1 * ((double)(km * fabsf(km)) * am) + h.c1 * gd;
    v[e] = h.b2 * (kv2 * kv2 * av) + h.c2 * gd * gd;
    mx = max(mx, __float_as_uint((float)m[e]) & 0x7fffffffu);
    vx = max(vx, __float_as_uint((float)v[e]) & 0x7fffffffu);
  }
  // one-instruction root and reciprocal (1 ulp each) unless eps is so small that a subnormal root would matter
  if (h.eps >= 1e-12f) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      pv[e] = __builtin_fmaf(-h.step * (float)m[e], __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_amdgcn_sqrtf((float)v[e]), h.isbc2, h.eps)), pv[e] * h.decay);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) pv[e] = pv[e] * h.decay - h.step * (float)m[e] / (sqrtf((float)v[e]) * h.isbc2 + h.eps);
  }
  adamw_st8<T, FULL>(p, i, n, pv);
  mx = adamw_max32(mx);
  vx = adamw_max32(vx);
  // a block with a non-finite moment gets a NaN scale (its moments read back as NaN, as fp32 moments would stay); an empty one the scale 0; codes 0 for both.
  // Scales whose reciprocal is out of fp32's range go through fp64.
  const bool mbad = mx >= 0x7f800000u, vbad = vx >= 0x7f800000u;
  const float sm = __uint_as_float(mx), sv = __uint_as_float(vx);
  float km[8], kv[8];
  if (!mbad && mx && sm < 1e-28f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) km[e] = fminf((float)floor(127.0 * sqrt(fabs(m[e]) / (double)sm) + 0.5), 127.f);
  } else {
    adamw_codes_m(m, sm, km);
  }
  if (!vbad && vx && sv < 1e-28f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) kv[e] = fmaxf(fminf((float)floor(255.0 * sqrt(sqrt(v[e] / (double)sv)) + 0.5), 255.f), v[e] > 0.0 ? 1.f : 0.f);
  } else {
    adamw_codes_v(v, sv, kv);
  }
  mq = vq = make_uint2(0, 0);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float biased = copysignf(km[e], (float)m[e]) + 128.f;
    if (e < 4) { mq.x = __builtin_amdgcn_cvt_pk_u8_f32(biased, e, mq.x); vq.x = __builtin_amdgcn_cvt_pk_u8_f32(kv[e], e, vq.x); }
    else { mq.y = __builtin_amdgcn_cvt_pk_u8_f32(biased, e - 4, mq.y); vq.y = __builtin_amdgcn_cvt_pk_u8_f32(kv[e], e - 4, vq.y); }
  }
  const bool mlive = !mbad && mx, vlive = !vbad && vx;
  mq.x = mlive ? mq.x ^ 0x80808080u : 0; mq.y = mlive ? mq.y ^ 0x80808080u : 0;
  vq.x = vlive ? vq.x : 0; vq.y = vlive ? vq.y : 0;
  *reinterpret_cast<uint2*>(mc + i) = mq;
  *reinterpret_cast<uint2*>(vc + i) = vq;
  if ((threadIdx.x & 31) == 0) { ms[blk] = mbad ? NAN : sm; vs[blk] = vbad ? NAN : sv; }
}
__global__ __launch_bounds__(256) void adamw8_kernel(AdamwGrads grads, const AdamwTensor* __restrict__ tensors, const int2* __restrict__ chunks,
                                                     const AdamwHyper* __restrict__ hyper, uint8_t* __restrict__ m, uint8_t* __restrict__ v,
                                                     float* __restrict__ ms, float* __restrict__ vs, const float* __restrict__ norm_skip) {
  // behind a norm the pieces are walked backwards: the gradients read last are the ones the memory-side cache still holds
  const int2 ch = chunks[norm_skip ? gridDim.x - 1 - blockIdx.x : blockIdx.x];
  const AdamwTensor t = tensors[ch.x];
  void* p = t.p;
  const void* g = grads.g[ch.x - grads.first];
  if (!g || (norm_skip && norm_skip[1] != 0.f)) return;
  const AdamwHyper h = hyper[ch.x];
  const long long base = (long long)ch.y * ADAMW_CHUNK, sb = t.off / ADAMW_BLOCK;
  const bool full = base + ADAMW_CHUNK <= t.n;
  ADAMW_BY_TYPE(if (full) adamw8_chunk<T, true>((T*)p, (const T*)g, m + t.off, v + t.off, ms + sb, vs + sb, t.n, base, h);
                else adamw8_chunk<T, false>((T*)p, (const T*)g, m + t.off, v + t.off, ms + sb, vs + sb, t.n, base, h);)
}

// the values the codes stand for, fp32: 2 + 1/32 bytes read and 8 written per element
__global__ __launch_bounds__(256) void adamw8_values_kernel(const uint8_t* __restrict__ mc, const uint8_t* __restrict__ vc, const float* __restrict__ ms,
                                                            const float* __restrict__ vs, float* __restrict__ m, float* __restrict__ v, long long n) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;      // n is a multiple of ADAMW_BLOCK
  if (i >= n) return;
  const uint2 mq = *reinterpret_cast<const uint2*>(mc + i), vq = *reinterpret_cast<const uint2*>(vc + i);
  const double am = (double)ms[i / ADAMW_BLOCK] * (1.0 / 16129.0), av = (double)vs[i / ADAMW_BLOCK] * (1.0 / (65025.0 * 65025.0));
  float mo[8], vo[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int km = (int)(int8_t)((e < 4 ? mq.x : mq.y) >> (8 * (e & 3)));
    const unsigned kv = ((e < 4 ? vq.x : vq.y) >> (8 * (e & 3))) & 255u;
    mo[e] = (float)((double)(km * abs(km)) * am);
    vo[e] = (float)((double)((kv * kv) * (kv * kv)) * av);
  }
  st8(m + i, mo);
  st8(v + i, vo);
}
