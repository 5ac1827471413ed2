// What turns q.k into a score, and which keys a query sees: shared by the attention kernels.
//   s = scale q.k,  s = cap tanh(s / cap),  s -= slope |i - j|   (the last two where asked for)
// The keys that query i of a document of L keys sees are one run lo <= j < hi.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace bn {

constexpr float LOG2E = 1.4426950408889634f;

// Why a bn_scores cannot be used, or NULL. Caps from 2^-60 to 2^60: scores times or over them stay in fp32.
inline const char *scores_refusal(const bn_scores *s) {
  if (s->window < 0 || s->window > 0x3FFFFFFF) return "negative window, or one of 2^30 and more";
  if (!(s->softcap == 0.0f || (s->softcap >= 8.67361738e-19f && s->softcap <= 1.15292150e18f))) return "a cap is 0 (none) or lies in 2^-60 .. 2^60";
  if (!(s->scale >= -3.402823466e38f && s->scale <= 3.402823466e38f)) return "the scale has to be finite";
  return nullptr;
}

#ifdef __CUDACC__
// The run of keys that query i sees. With a window |i - j| < window; causal: no key behind the query, but
// for those of the document's prefix.
__device__ __forceinline__ void visible_keys(int i, int L, int prefix, int window, bool causal, int &lo, int &hi) {
  lo = 0, hi = L;
  if (causal) hi = min(L, max(i + 1, prefix));
  if (window > 0) {
    lo = max(0, i - window + 1);
    hi = (int)min((int64_t)hi, (int64_t)i + window);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap tanh(s / cap) times log2(e), for z = s / cap * 2 log2(e): tanh(x) = 1 - 2 / (e^2x + 1). Off by some
// 1e-7 of the cap everywhere (tanh.approx: 5e-4 of the cap, which for a cap of 50 is 2 % of a weight).
__device__ __forceinline__ float capped(float z, float cap_log2e) { return fmaf(-2.0f * cap_log2e, __fdividef(1.0f, ex2(z) + 1.0f), cap_log2e); }

// The same where 1e-7 of the cap would show in a weight: tanh(x) for |x| < 1 by Lambert's continued fraction, cut behind 9 (off by
// 6e-8 of itself at 1), so that a score far below the cap keeps its own precision.
constexpr float WIDE_CAP = 256.0f;  // (up to here scores are off by some 5e-5, a hundredth of what BF16 makes of a weight)
__device__ __forceinline__ float capped_wide(float z, float cap_log2e) {
  const float x = 0.5f / LOG2E * z, xx = x * x, up = fmaf(fmaf(xx, 1.0f, 105.0f), xx, 945.0f), down = fmaf(fmaf(xx, 15.0f, 420.0f), xx, 945.0f);
  return fabsf(x) < 1.0f ? cap_log2e * (x * __fdividef(up, down)) : capped(z, cap_log2e);
}

__device__ __forceinline__ float bf16_to_f32(uint32_t bits) { return __uint_as_float(bits << 16); }
#endif

}  // namespace bn
