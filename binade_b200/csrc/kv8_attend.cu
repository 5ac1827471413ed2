// Attention of new tokens over an 8-bit key/value cache (bn_kv8).
#include "kv8.cuh"

namespace bn {
namespace {

struct AttendArgs {
  bn_kv8 c;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_seq, q_token, q_head, o_seq, o_token, o_head;  // elements
  const int32_t *counts, *prefix;
  const float *slopes;
  int tokens, heads;
  int window, causal, zero_rest;
  float scale, cap;
};

// One query of one head by a warp, keys one after the other; a lane has E = D / 32 neighbouring dimensions.
template <int D, int KIND>
__global__ void __launch_bounds__(128) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int E = D / 32;
  const bn_kv8 &c = a.c;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= c.batch * a.tokens * a.heads) return;
  const int head = (int)(row % a.heads), t = (int)(row / a.heads % a.tokens);
  const int64_t b = row / a.heads / a.tokens;
  const uint32_t lane = lane_id();
  int held, brought;
  kv8_tokens(c, a.counts, a.tokens, b, held, brought);
  uint16_t *const out = a.out + b * a.o_seq + t * a.o_token + head * a.o_head + lane * E;
  if (t >= brought) {
    if (a.zero_rest)
      for (int e = 0; e < E; e++) out[e] = 0;
    return;
  }
  const int L = held + brought, i = held + t, kv = head / (a.heads / (int)c.kv_heads), full = L / c.block * c.block;
  const int64_t unit = b * c.kv_heads + kv;
  const int slot = kv8_slot(c, b, held, L / c.block);
  int lo, hi;
  visible_keys(i, L, a.prefix ? a.prefix[b] : 0, a.window, a.causal, lo, hi);
  float q[E], o[E] = {}, m = -CUDART_INF_F, l = 0.0f;
  for (int e = 0; e < E; e++) q[e] = bf16_to_f32(a.q[b * a.q_seq + t * a.q_token + head * a.q_head + lane * E + e]);
  const float slope = a.slopes ? a.slopes[head] * LOG2E : 0.0f;
  auto value = [&](const uint8_t *codes, const float *scales, const uint16_t *tail, int j, int e) {
    if (j < full) return kv8_code<KIND>(codes[(unit * c.rows + j) * D + lane * E + e]) * scales[unit * (c.rows / c.block) + j / c.block];
    return bf16_to_f32(tail[((unit * 2 + slot) * c.block + j - full) * D + lane * E + e]);
  };
  auto score = [&](int j) {
    float dot = 0.0f;
    for (int e = 0; e < E; e++) dot = fmaf(q[e], value(c.k, c.k_scale, c.k_tail, j, e), dot);
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
  const float inv = 1.0f / l;
  for (int j = lo; j < hi; j++) {
    const float p = ex2(score(j) - m) * inv;
    for (int e = 0; e < E; e++) o[e] = fmaf(p, value(c.v, c.v_scale, c.v_tail, j, e), o[e]);
  }
  for (int e = 0; e < E; e++) out[e] = f32_to_bf16_bits(o[e]);
}

}  // namespace
}  // namespace bn

extern "C" uint64_t bn_kv8_workspace(const bn_kv8 *, int64_t, int64_t) { return 0; }

extern "C" int bn_kv8_attend(const bn_kv8 *c, const uint16_t *q, int64_t q_seq, int64_t q_token, int64_t q_head, int64_t tokens, int64_t heads, const int32_t *counts, const int32_t *prefix, const bn_scores *scores, uint16_t *out, int64_t o_seq, int64_t o_token, int64_t o_head, int zero_rest, void *workspace, uint64_t workspace_bytes, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_attend", why);
  if (tokens < 0 || tokens > 0x3FFFFFFF || heads < 1 || heads > 4096 || heads % c->kv_heads) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: bad size (query heads have to be a multiple of the cache's heads)");
  if (!scores || (tokens && (!q || !out))) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: null pointer");
  if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_seq | q_token | q_head | o_seq | o_token | o_head) & 7) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: rows have to start on 16 bytes");
  if (scores->window < 0 || scores->window > 0x3FFFFFFF || !(scores->softcap >= 0.0f)) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: negative window or cap");
  (void)workspace, (void)workspace_bytes;
  if (tokens == 0) return BN_OK;
  bn::AttendArgs a{*c, q, out, q_seq, q_token, q_head, o_seq, o_token, o_head, counts, prefix, scores->slopes, (int)tokens, (int)heads, (int)scores->window, scores->causal, zero_rest, scores->scale, scores->softcap};
  const int64_t blocks = (c->batch * tokens * heads + 3) / 4;
  if (blocks > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: too many rows");
  auto pick = [&](auto kind) {
    constexpr int KIND = decltype(kind)::value;
    return c->D == 64 ? bn::attend_rows_kernel<64, KIND> : c->D == 128 ? bn::attend_rows_kernel<128, KIND> : bn::attend_rows_kernel<256, KIND>;
  };
  auto kern = c->kind == BN_KV8_INT8 ? pick(std::integral_constant<int, BN_KV8_INT8>()) : pick(std::integral_constant<int, BN_KV8_E4M3>());
  kern<<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(a);
  return bn::launched("attend_rows_kernel");
}
