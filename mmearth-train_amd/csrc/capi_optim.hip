// extern "C" surface of libmpmae_hip.so, optimizer unit: AdamW over many separate tensors (optim.cuh). gfx950 only.
#include "capi_common.h"
#include "optim.cuh"
#include <cmath>

static_assert(sizeof(MpmaeAdamwTensor) == sizeof(AdamwTensor), "device table record");
static_assert(sizeof(AdamwHyper) == MPMAE_ADAMW_HYPER_BYTES, "device hyper record");
static_assert(sizeof(AdamwGrads) <= 3904 && sizeof(AdamwGroups) <= 3904, "kernel arguments hold at most 4 KB");

extern "C" {

int mpmae_adamw_multi(const MpmaeAdamwArgs* a, const void* const* grads, const double* groups, int ngroups, mpmae_stream_t s) {
  if (!a || !grads || !groups || ngroups < 1 || a->nt < 1 || !a->tensors || !a->chunks || !a->chunk_first || !a->steps || !a->hyper ||
      !a->m || !a->v || (a->bits != 8 && a->bits != 32) || (a->bits == 8 && (!a->ms || !a->vs)) || (a->max_norm > 0 && (!a->partials || !a->norm_skip)))
    return (int)hipErrorInvalidValue;
  for (int g = 0; g < ngroups; ++g) {
    const double* h = groups + 5 * (size_t)g;
    if (!(h[0] >= 0 && h[0] < INFINITY && h[1] >= 0 && h[1] < 1 && h[2] >= 0 && h[2] < 1 && h[3] >= 0 && h[3] < INFINITY && h[4] >= 0 && h[4] < INFINITY))
      return (int)hipErrorInvalidValue;      // (a beta of 1 divides by 1 - 1^t)
  }
  const AdamwTensor* tensors = reinterpret_cast<const AdamwTensor*>(a->tensors);
  const int2* chunks = reinterpret_cast<const int2*>(a->chunks);
  const bool clip = a->max_norm > 0;
  AdamwGrads q;
  const int nl = cdiv(a->nt, ADAMW_MAX_GRADS);
  auto take = [&](int l) {          // gradients of launch l's tensors -> its first and last chunk
    const int t0 = l * ADAMW_MAX_GRADS, t1 = a->nt < t0 + ADAMW_MAX_GRADS ? a->nt : t0 + ADAMW_MAX_GRADS;
    for (int t = t0; t < t1; ++t) q.g[t - t0] = grads[t];
    q.first = t0;
    return std::pair<int, int>(a->chunk_first[t0], a->chunk_first[t1]);
  };
  int npart = 0;
  if (clip) {
    for (int l = 0; l < nl; ++l) {
      const auto c = take(l);
      const int nc = c.second - c.first, nb = nc < MPMAE_ADAMW_NORM_BLOCKS ? nc : MPMAE_ADAMW_NORM_BLOCKS;
      if (nc < 1) continue;
      if (npart + nb > a->npartials) return (int)hipErrorInvalidValue;
      LAUNCH(adamw_norm_kernel, dim3(nb), dim3(256), 0, S_(s), q, tensors, chunks + c.first, nc, a->partials + npart);
      npart += nb;
    }
  }
  for (int g0 = 0; g0 < ngroups; g0 += ADAMW_MAX_GROUPS) {
    AdamwGroups gr;
    gr.first = g0; gr.count = ngroups - g0 < ADAMW_MAX_GROUPS ? ngroups - g0 : ADAMW_MAX_GROUPS;
    for (int g = 0; g < gr.count; ++g) {
      const double* h = groups + 5 * (size_t)(g0 + g);
      gr.at[g].lr = h[0]; gr.at[g].b1 = h[1]; gr.at[g].b2 = h[2]; gr.at[g].eps = h[3]; gr.at[g].wd = h[4];
      gr.at[g].ln_b1 = log(h[1]); gr.at[g].ln_b2 = log(h[2]);
    }
    for (gr.t0 = 0; gr.t0 < a->nt; gr.t0 = gr.t1) {
      gr.t1 = a->nt < gr.t0 + ADAMW_MAX_HAS ? a->nt : gr.t0 + ADAMW_MAX_HAS;
      for (unsigned& w : gr.has) w = 0;
      for (int t = gr.t0; t < gr.t1; ++t) if (grads[t]) gr.has[(t - gr.t0) >> 5] |= 1u << ((t - gr.t0) & 31);
      LAUNCH(adamw_hyper_kernel, dim3(1), dim3(512), 0, S_(s), gr, tensors, a->steps, reinterpret_cast<AdamwHyper*>(a->hyper),
             (const double*)a->partials, npart, a->max_norm, a->norm_skip);
    }
  }
  const float* skip = npart > 0 ? a->norm_skip : nullptr;
  for (int l = 0; l < nl; ++l) {
    const auto c = take(skip ? nl - 1 - l : l);
    const int nc = c.second - c.first;
    if (nc < 1) continue;
    if (a->bits == 32 && skip)
      LAUNCH(adamw32_kernel<true>, dim3(nc), dim3(256), 0, S_(s), q, tensors, chunks + c.first, (const AdamwHyper*)a->hyper, (float*)a->m, (float*)a->v, skip);
    else if (a->bits == 32)
      LAUNCH(adamw32_kernel<false>, dim3(nc), dim3(256), 0, S_(s), q, tensors, chunks + c.first, (const AdamwHyper*)a->hyper, (float*)a->m, (float*)a->v, skip);
    else
      LAUNCH(adamw8_kernel, dim3(nc), dim3(256), 0, S_(s), q, tensors, chunks + c.first, (const AdamwHyper*)a->hyper, (uint8_t*)a->m, (uint8_t*)a->v,
             a->ms, a->vs, skip);
  }
  RET();
}

int mpmae_adamw_values(const uint8_t* mc, const uint8_t* vc, const float* ms, const float* vs, float* m, float* v, long long n, mpmae_stream_t s) {
  if (!mc || !vc || !ms || !vs || !m || !v || n < 0 || n % ADAMW_BLOCK) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  LAUNCH(adamw8_values_kernel, dim3(cdiv(n, 2048)), dim3(256), 0, S_(s), mc, vc, ms, vs, m, v, n);
  RET();
}

}  // extern "C"
