// Attention of chunks of new tokens over an 8-bit cache: the host side of prompt.cuh for a cache.
#include "prompt.cuh"

namespace bn {
namespace {

template <int D, int KIND>
int chunk_launch(PromptArgs a, cudaStream_t stream) {
  const int log2 = block_group_log2(a.heads, a.kv_heads), group = 1 << log2;
  a.tiles = (int)(((int64_t)a.tokens * group + Tiles<D>::ROWS - 1) / Tiles<D>::ROWS);
  const int64_t blocks = a.c.batch * a.tiles * (a.heads / group);
  if (blocks > 0x7FFFFFFF || (int64_t)a.tokens * group > 0x3FFFFFFF) return fail(BN_ERR_ARG, "bn_kv8_attend: too many rows for one call");
  CUtensorMap q_map;
  if (!rows_map(&q_map, a.q, D, a.heads, a.tokens, a.c.batch, a.q_head, a.q_token, a.q_seq, group, 128 / group, 4)) return fail(BN_ERR_ARG, "bn_kv8_attend: no tensor map for these strides");
  return prompt_launch<D, KIND>(a, q_map, q_map, q_map, blocks, log2, stream);  // (K and V come by other ways)
}

template <int KIND>
int chunk_kind(const PromptArgs &a, cudaStream_t s) {
  return a.c.D == 64 ? chunk_launch<64, KIND>(a, s) : a.c.D == 128 ? chunk_launch<128, KIND>(a, s) : chunk_launch<256, KIND>(a, s);
}

}  // namespace

int kv8_chunk(const bn_kv8 *c, const uint16_t *q, int64_t q_seq, int64_t q_token, int64_t q_head, int64_t tokens, int64_t heads, const int32_t *counts, const int32_t *prefix, const bn_scores *scores, uint16_t *out, int64_t o_seq, int64_t o_token, int64_t o_head, int zero_rest, cudaStream_t stream) {
  PromptArgs a{};
  a.q = q, a.out = out, a.q_token = q_token, a.q_head = q_head, a.o_token = o_token, a.o_head = o_head, a.prefix = prefix, a.slopes = scores->slopes;
  a.heads = (int)heads, a.kv_heads = (int)c->kv_heads, a.window = (int)scores->window, a.causal = scores->causal, a.zero_rest = zero_rest, a.scale = scores->scale, a.cap = scores->softcap;
  a.c = *c, a.counts = counts, a.tokens = (int)tokens, a.q_seq = q_seq, a.o_seq = o_seq;
  return c->kind == BN_KV8_INT8 ? chunk_kind<BN_KV8_INT8>(a, stream) : chunk_kind<BN_KV8_E4M3>(a, stream);
}

int kv8_chunk_status(int *status) { return prompt_status(status); }
int kv8_chunk_status_reset() { return prompt_status_reset(); }

}  // namespace bn
