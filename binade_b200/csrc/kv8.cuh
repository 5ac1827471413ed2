// The 8-bit key/value cache of bn_kv8, as its kernels see it.
#pragma once

#include <cuda_fp8.h>

#include "scores.cuh"

namespace bn {

constexpr int KV8_INT8 = BN_KV8_INT8, KV8_E4M3 = BN_KV8_E4M3;

#ifdef __CUDACC__
// Tokens of sequence b: held before the call, brought by it (a call brings up to `most`, of which `counts`
// are real; what does not fit is not taken).
__device__ __forceinline__ void kv8_tokens(const bn_kv8 &c, const int32_t *__restrict__ counts, int most, int64_t b, int &held, int &brought) {
  held = min(max(c.length[b], 0), (int)c.max_seq);
  brought = counts ? min(max(counts[b], 0), most) : most;
  brought = min(brought, (int)c.max_seq - held);
}

// The slot of the tail that holds block j, for j the block open at `held` or the one that is open behind
// the tokens of the call.
__device__ __forceinline__ int kv8_slot(const bn_kv8 &c, int64_t b, int held, int j) { return (c.side[b] ^ (j != held / c.block)) & 1; }

// The value of a code, without its scale.
template <int KIND>
__device__ __forceinline__ float kv8_code(uint32_t byte) {
  if constexpr (KIND == KV8_INT8) {
    return (float)((int)byte - 128);
  } else {
    __nv_fp8_e4m3 f;
    f.__x = (__nv_fp8_storage_t)byte;
    return (float)f;
  }
}
#endif

int refuse(const char *who, const char *why);  // the two as the thread's last error (kv8.cu)

// Why a bn_kv8 cannot be used, or NULL.
inline const char *kv8_refusal(const bn_kv8 *c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !c->length || !c->side) return "null cache array";
  if (c->D != 64 && c->D != 128 && c->D != 256) return "a head has 64, 128 or 256 dimensions";
  if (c->block != 16 && c->block != 32 && c->block != 64) return "a block has 16, 32 or 64 tokens";
  if (c->kind != BN_KV8_INT8 && c->kind != BN_KV8_E4M3) return "unknown kind of codes";
  if (c->batch < 1 || c->kv_heads < 1 || c->batch > 65535 || c->kv_heads > 65535 || c->max_seq < 1 || c->max_seq > 0x3FFFFFFF || c->rows < c->max_seq || c->rows % 64) return "bad cache size (rows: max_seq rounded up to 64)";
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_tail | (uintptr_t)c->v_tail) & 15) return "cache arrays have to start on 16 bytes";
  return nullptr;
}

}  // namespace bn
