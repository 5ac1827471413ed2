// Attention of prompts: packed documents, every query over the keys of its own document.
#include "scores.cuh"

namespace bn {
namespace {

struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;  // elements
  const int32_t *offsets, *prefix;
  const float *slopes;
  int T, docs, heads, kv_heads;
  int window, causal, zero_rest;
  float scale, cap;
};

template <int E>
__device__ __forceinline__ void load_row(const uint16_t *p, float (&x)[E]) {
  if constexpr (E == 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
    x[0] = bf16_to_f32(w & 0xFFFFu), x[1] = __uint_as_float(w & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const uint2 w = *reinterpret_cast<const uint2 *>(p + i);
      x[i] = bf16_to_f32(w.x & 0xFFFFu), x[i + 1] = __uint_as_float(w.x & 0xFFFF0000u);
      x[i + 2] = bf16_to_f32(w.y & 0xFFFFu), x[i + 3] = __uint_as_float(w.y & 0xFFFF0000u);
    }
  }
}

// One query of one head by a warp, keys one after the other; a lane has E = D / 32 neighbouring dimensions.
// Two passes, so that the values are weighted by shares of one: no sum of theirs can pass the largest of them.
template <int D>
__device__ void attend_row(const PromptArgs &a, int t, int head, int from, int to, int prefix) {
  constexpr int E = D / 32;
  const uint32_t lane = lane_id();
  const int kv = head / (a.heads / a.kv_heads), i = t - from;
  int lo, hi;
  visible_keys(i, to - from, prefix, a.window, a.causal, lo, hi);
  float q[E], o[E] = {}, m = -CUDART_INF_F, l = 0.0f;
  load_row<E>(a.q + t * a.q_token + head * a.q_head + lane * E, q);
  const float slope = a.slopes ? a.slopes[head] * LOG2E : 0.0f;
  auto score = [&](int j) {
    float x[E], dot = 0.0f;
    load_row<E>(a.k + (int64_t)(from + j) * a.k_token + kv * a.k_head + lane * E, x);
#pragma unroll
    for (int e = 0; e < E; e++) dot = fmaf(q[e], x[e], dot);
#pragma unroll
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(BN_FULL, dot, d);
    float s = dot * a.scale;
    s = a.cap > 0.0f ? capped(s * (2.0f * LOG2E / a.cap), a.cap * LOG2E) : s * LOG2E;
    return s - slope * (float)abs(i - j);
  };
  for (int j = lo; j < hi; j++) {
    const float s = score(j), top = fmaxf(m, s);
    l = fmaf(l, ex2(m - top), ex2(s - top));
    m = top;
  }
  const float inv = hi > lo ? 1.0f / l : 0.0f;
  for (int j = lo; j < hi; j++) {
    float x[E];
    const float p = ex2(score(j) - m) * inv;
    load_row<E>(a.v + (int64_t)(from + j) * a.v_token + kv * a.v_head + lane * E, x);
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = fmaf(p, x[e], o[e]);
  }
  uint16_t *const out = a.out + t * a.o_token + head * a.o_head + lane * E;
#pragma unroll
  for (int e = 0; e < E; e++) out[e] = f32_to_bf16_bits(o[e]);
}

template <int D>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const __grid_constant__ PromptArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.T * a.heads) return;
  const int t = (int)(row / a.heads), head = (int)(row % a.heads);
  int doc, from, to;
  if (document_of(a.offsets, a.docs, a.T, t, doc, from, to)) {
    attend_row<D>(a, t, head, from, to, a.prefix ? a.prefix[doc] : 0);
  } else if (a.zero_rest) {
    uint16_t *const out = a.out + t * a.o_token + head * a.o_head;
    for (int e = lane_id(); e < D; e += 32) out[e] = 0;
  }
}

}  // namespace
}  // namespace bn

extern "C" int bn_attention(const uint16_t *q, int64_t q_token, int64_t q_head, const uint16_t *k, int64_t k_token, int64_t k_head, const uint16_t *v, int64_t v_token, int64_t v_head, int64_t T, int64_t heads, int64_t kv_heads, int64_t D, const int32_t *offsets, int64_t docs, const int32_t *prefix, const bn_scores *scores, uint16_t *out, int64_t o_token, int64_t o_head, int zero_rest, void *stream) {
  if (T < 0 || T > 0x3FFFFFFF || heads < 1 || kv_heads < 1 || heads > 4096 || heads % kv_heads || docs < 0 || docs > 0x3FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_attention: bad size (query heads have to be a multiple of key heads)");
  if (D != 64 && D != 128 && D != 256) return bn::fail(BN_ERR_ARG, "bn_attention: a head has 64, 128 or 256 dimensions");
  if (!scores || (T && (!q || !k || !v || !out)) || (!offsets && docs != 1)) return bn::fail(BN_ERR_ARG, "bn_attention: null pointer, or no offsets for several documents");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15 || (q_token | q_head | k_token | k_head | v_token | v_head | o_token | o_head) & 7) return bn::fail(BN_ERR_ARG, "bn_attention: rows have to start on 16 bytes");
  if (scores->window < 0 || scores->window > 0x3FFFFFFF || !(scores->softcap >= 0.0f)) return bn::fail(BN_ERR_ARG, "bn_attention: negative window or cap");
  if (T == 0) return BN_OK;
  bn::PromptArgs a{q, k, v, out, q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head, offsets, prefix, scores->slopes, (int)T, (int)docs, (int)heads, (int)kv_heads, (int)scores->window, scores->causal, zero_rest, scores->scale, scores->softcap};
  const int64_t blocks = (T * heads + 3) / 4;
  if (blocks > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_attention: too many rows");
  auto kern = D == 64 ? bn::prompt_rows_kernel<64> : D == 128 ? bn::prompt_rows_kernel<128> : bn::prompt_rows_kernel<256>;
  kern<<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(a);
  return bn::launched("prompt_rows_kernel");
}
