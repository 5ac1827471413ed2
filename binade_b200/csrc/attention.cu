// Attention of prompts: the host side of prompt.cuh for packed documents.
#include "prompt.cuh"

namespace bn {
namespace {

template <int D>
int attention_launch(const PromptArgs &a, cudaStream_t stream) {
  using G = Tiles<D>;
  const int log2 = block_group_log2(a.heads, a.kv_heads), group = 1 << log2;
  CUtensorMap q_map, k_map, v_map;
  if (!rows_map(&q_map, a.q, D, a.heads, a.T, 1, a.q_head, a.q_token, 0, group, 128 / group, 4) || !rows_map(&k_map, a.k, D, a.kv_heads, a.T, 1, a.k_head, a.k_token, 0, 1, G::BN, 3) || !rows_map(&v_map, a.v, D, a.kv_heads, a.T, 1, a.v_head, a.v_token, 0, 1, G::BN, 3))
    return fail(BN_ERR_ARG, "bn_attention: no tensor map for these strides");
  const int64_t blocks = ((int64_t)a.T * group / G::ROWS + a.docs + 1) * (a.heads / group);
  if (blocks > 0x7FFFFFFF || (int64_t)a.T * group > 0x3FFFFFFF) return fail(BN_ERR_ARG, "bn_attention: too many rows");
  return prompt_launch<D, FROM_BF16>(a, q_map, k_map, v_map, blocks, log2, stream);
}

}  // namespace

int attention_status(int *status) { return prompt_status(status); }
int attention_status_reset() { return prompt_status_reset(); }

}  // namespace bn

extern "C" int bn_attention(const uint16_t *q, int64_t q_token, int64_t q_head, const uint16_t *k, int64_t k_token, int64_t k_head, const uint16_t *v, int64_t v_token, int64_t v_head, int64_t T, int64_t heads, int64_t kv_heads, int64_t D, const int32_t *offsets, int64_t docs, const int32_t *prefix, const bn_scores *scores, uint16_t *out, int64_t o_token, int64_t o_head, int zero_rest, void *stream) {
  if (T < 0 || T > 0x3FFFFFFF || heads < 1 || kv_heads < 1 || heads > 4096 || heads % kv_heads || docs < 0 || docs > 0x3FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_attention: bad size (query heads have to be a multiple of key heads)");
  if (D != 64 && D != 128 && D != 256) return bn::fail(BN_ERR_ARG, "bn_attention: a head has 64, 128 or 256 dimensions");
  if (!scores || (T && (!q || !k || !v || !out)) || (!offsets && docs != 1)) return bn::fail(BN_ERR_ARG, "bn_attention: null pointer, or no offsets for several documents");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15 || (q_token | q_head | k_token | k_head | v_token | v_head | o_token | o_head) & 7) return bn::fail(BN_ERR_ARG, "bn_attention: rows have to start on 16 bytes");
  if (const char *why = bn::scores_refusal(scores)) return bn::refuse("bn_attention", why);
  if ((T > 1 && !(q_token && k_token && v_token && o_token)) || (heads > 1 && !(q_head && o_head)) || (kv_heads > 1 && !(k_head && v_head)) || (q_token | q_head | k_token | k_head | v_token | v_head) < 0) return bn::fail(BN_ERR_ARG, "bn_attention: rows have to lie apart");
  if (T == 0) return BN_OK;
  bn::PromptArgs a{q, k, v, out, q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head, offsets, prefix, scores->slopes, (int)T, (int)docs, (int)heads, (int)kv_heads, (int)scores->window, scores->causal, zero_rest, scores->scale, scores->softcap, {}, nullptr, 0, 0, 0, 0};
  const cudaStream_t s = (cudaStream_t)stream;
  return D == 64 ? bn::attention_launch<64>(a, s) : D == 128 ? bn::attention_launch<128>(a, s) : bn::attention_launch<256>(a, s);
}
