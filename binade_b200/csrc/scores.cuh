// What turns q.k into a score, and which keys a query sees: shared by the attention kernels.
//   s = scale q.k,  s = cap tanh(s / cap),  s -= slope |i - j|   (the last two where asked for)
// The keys that query i of a document of L keys sees are one run lo <= j < hi.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace bn {

constexpr float LOG2E = 1.4426950408889634f;

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

__device__ __forceinline__ float bf16_to_f32(uint32_t bits) { return __uint_as_float(bits << 16); }
#endif

// The document of a packed batch that token t is in: true with its bounds [from, to), false when no
// document holds the token. Offsets that do not rise, or leave [0, T], name no token.
__device__ __forceinline__ bool document_of(const int32_t *__restrict__ offsets, int n, int T, int t, int &doc, int &from, int &to) {
  if (!offsets) {
    doc = 0, from = 0, to = T;
    return t < T;
  }
  int a = 0, b = n;  // the last i with offsets[i] <= t lies in [a, b], if there is one
  while (a < b) {
    const int m = (a + b + 1) >> 1;
    if (offsets[m] <= t) a = m;
    else b = m - 1;
  }
  if (a >= n) return false;
  doc = a, from = offsets[a], to = offsets[a + 1];
  return from >= 0 && from <= t && t < to && to <= T;
}

}  // namespace bn
