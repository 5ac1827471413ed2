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

}  // namespace bn
