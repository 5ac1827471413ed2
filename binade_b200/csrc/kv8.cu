// Writing and reading back the 8-bit key/value cache (bn_kv8).
#include <stdio.h>

#include <type_traits>

#include "kv8.cuh"

namespace bn {

__device__ int g_kv8_error;  // 1: tokens were brought that the cache has no room for; 2: a length was asked for whose block is not held

namespace {

struct AppendArgs {
  bn_kv8 c;
  const uint16_t *k, *v;
  int64_t k_seq, k_token, k_head, v_seq, v_token, v_head;  // elements
  const int32_t *counts;
  int tokens, rel;  // tokens a sequence brings at most; blocks of the cache that those can touch
};

// A block per block of tokens, keys or values. 4 x 2000 tokens, 8 heads of 128 (49 MB): 23 us from DRAM, 15 where the tokens are
// in L2. Neither bytes (7.5 us) nor instructions (10.2 M, 9 us at full issue) bound it: a block's loads, maximum, codes and stores
// follow one another, and 2.3 rounds of blocks leave the SMs idle a third of the time.
template <int D, int CHUNKS>
__global__ void __launch_bounds__(128) append_kernel(const __grid_constant__ AppendArgs a) {
  const bn_kv8 &c = a.c;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what made the tokens, and what read the cache before
  const bool values = blockIdx.x & 1;
  const int rel = (int)(blockIdx.x >> 1), h = (int)blockIdx.y;
  const int64_t b = blockIdx.z;
  int held, brought;
  const bool all = kv8_tokens(c, a.counts, a.tokens, b, held, brought);
  if (!all && rel == 0 && h == 0 && !values && threadIdx.x == 0) atomicOr(&g_kv8_error, 1);
  if (brought && rel == 0 && h == 0 && !values && threadIdx.x == 0) kv8_note(c, b, held, held + brought);
  const int j = held / c.block + rel;
  if (brought == 0 || j > (held + brought - 1) / c.block) return;
  const bool v = values;
  append_block<D, CHUNKS>(c, v, b, h, j, held, held + brought, v ? a.v + b * a.v_seq + h * a.v_head : a.k + b * a.k_seq + h * a.k_head, v ? a.v_token : a.k_token);
}

__global__ void __launch_bounds__(256) advance_kernel(const __grid_constant__ bn_kv8 c, int n, const int32_t *__restrict__ counts) {
  const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b >= c.batch) return;
  const int held = min(max(c.length[b], 0), (int)c.max_seq);
  const int now = (int)min(max((int64_t)held + (counts ? counts[b] : n), (int64_t)0), c.max_seq);
  if (now != held) {
    const int block = now / c.block, slot = c.kept[2 * b] == block ? 0 : c.kept[2 * b + 1] == block ? 1 : -1;
    if (slot < 0 && now % c.block) {  // tokens of a block that went straight to codes, or whose rows are overwritten
      atomicOr(&g_kv8_error, 2);
      return;
    }
    if (slot >= 0) c.side[b] = slot;
    else if (block != held / c.block) c.side[b] ^= 1;
  }
  c.length[b] = now;
}

// Sixteen codes a thread at a time, as they lie: of keys sixteen dimensions of a token, of values four of four tokens. Tokens
// that the cache does not hold as zeros. Blocks: pieces of a sequence and head, those, and keys or values.
template <int KIND, int D>
__global__ void __launch_bounds__(256) dense_kernel(const __grid_constant__ bn_kv8 c, float *__restrict__ k, float *__restrict__ v) {
  const bool values = blockIdx.z;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t from_row = values ? at / (D / 4) * 4 : at / (D / 16);
  if (from_row >= c.max_seq) return;
  const int row = (int)from_row, col = (int)(values ? at % (D / 4) * 4 : at % (D / 16) * 16), block_log2 = 31 - __clz(c.block);
  const unsigned heads = (unsigned)c.kv_heads, units = (unsigned)c.batch * heads;
  for (unsigned unit = blockIdx.y; unit < units; unit += gridDim.y) {
    const unsigned b = unit / heads;
    const int length = min(max(c.length[b], 0), (int)c.max_seq), full = length >> block_log2 << block_log2;
    float x[16] = {};
    if (row < full) {  // (a block has whole rows of four)
      const float scale = (values ? c.v_scale : c.k_scale)[(int64_t)unit * (c.rows >> block_log2) + (row >> block_log2)];
      const uint4 w4 = *reinterpret_cast<const uint4 *>((values ? c.v : c.k) + ((int64_t)unit * c.rows + row) * D + (values ? 4 : 1) * col);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int e = 0; e < 16; e++) x[e] = kv8_code<KIND>((w[e >> 2] >> (8 * (e & 3))) & 0xFFu) * scale;
    } else if (row < length) {
      const uint16_t *const tail = (values ? c.v_tail : c.k_tail) + (((int64_t)unit * 2 + (c.side[b] & 1)) * c.block + row - full) * D + col;
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (row + (values ? e & 3 : 0) < length) x[e] = bf16_to_f32(tail[values ? (e & 3) * D + (e >> 2) : e]);
    }
    float *const out = (values ? v : k) + ((int64_t)unit * c.max_seq + row) * D + col;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (!values) *reinterpret_cast<float4 *>(out + 4 * e) = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
      else if (row + e < c.max_seq) *reinterpret_cast<float4 *>(out + e * D) = make_float4(x[e], x[4 + e], x[8 + e], x[12 + e]);
    }
  }
}

template <int KIND>
int dense_launch(const bn_kv8 &c, float *k, float *v, cudaStream_t s) {
  const int64_t units = c.batch * c.kv_heads, pieces = ((c.max_seq + 3) / 4 * 4 * (c.D / 16) + 255) / 256;
  const dim3 grid((unsigned)pieces, (unsigned)(units < 65535 ? units : 65535), 2);
  auto kern = c.D == 64 ? dense_kernel<KIND, 64> : c.D == 128 ? dense_kernel<KIND, 128> : dense_kernel<KIND, 256>;
  kern<<<grid, 256, 0, s>>>(c, k, v);
  return launched("dense_kernel");
}

}  // namespace

int kv8_status(int *status) {
  BN_CUDA(cudaMemcpyFromSymbol(status, g_kv8_error, sizeof(int)));
  return BN_OK;
}

int kv8_status_reset() {
  const int zero = 0;
  BN_CUDA(cudaMemcpyToSymbol(g_kv8_error, &zero, sizeof(int)));
  return BN_OK;
}

int refuse(const char *who, const char *why) {
  char msg[256];
  snprintf(msg, sizeof msg, "%s: %s", who, why);
  return fail(BN_ERR_ARG, msg);
}

}  // namespace bn

extern "C" int bn_kv8_append(const bn_kv8 *c, const uint16_t *k, int64_t k_seq, int64_t k_token, int64_t k_head, const uint16_t *v, int64_t v_seq, int64_t v_token, int64_t v_head, int64_t tokens, const int32_t *counts, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_append", why);
  if (tokens < 0 || tokens > 0x3FFFFFFF || (tokens && (!k || !v))) return bn::fail(BN_ERR_ARG, "bn_kv8_append: null pointer or bad number of tokens");
  if (((uintptr_t)k | (uintptr_t)v) & 15 || (k_seq | k_token | k_head | v_seq | v_token | v_head) & 7) return bn::fail(BN_ERR_ARG, "bn_kv8_append: rows have to start on 16 bytes");
  if (tokens == 0) return BN_OK;
  bn::AppendArgs a{*c, k, v, k_seq, k_token, k_head, v_seq, v_token, v_head, counts, (int)tokens, 0};
  a.rel = (int)((tokens + c->block - 1) / c->block) + 1;  // a run of tokens that starts inside a block touches one more
  auto pick = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return c->block == 16 ? bn::append_kernel<D, 16 * D / 1024> : c->block == 32 ? bn::append_kernel<D, 32 * D / 1024> : bn::append_kernel<D, 64 * D / 1024>;
  };
  auto kern = c->D == 64 ? pick(std::integral_constant<int, 64>()) : c->D == 128 ? pick(std::integral_constant<int, 128>()) : pick(std::integral_constant<int, 256>());
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)a.rel * 2, (unsigned)c->kv_heads, (unsigned)c->batch), cfg.blockDim = dim3(128), cfg.stream = (cudaStream_t)stream, cfg.attrs = attr, cfg.numAttrs = 1;
  BN_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  return bn::launched("append_kernel");
}

extern "C" int bn_kv8_advance(const bn_kv8 *c, int64_t n, const int32_t *counts, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_advance", why);
  if (n < -0x3FFFFFFF || n > 0x3FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_advance: bad number of tokens");
  if (!c->kept) return bn::refuse("bn_kv8_advance", "null cache array");
  bn::advance_kernel<<<(unsigned)((c->batch + 255) / 256), 256, 0, (cudaStream_t)stream>>>(*c, (int)n, counts);
  return bn::launched("advance_kernel");
}

extern "C" int bn_kv8_dense(const bn_kv8 *c, float *k, float *v, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_dense", why);
  if (!k || !v || ((uintptr_t)k | (uintptr_t)v) & 15) return bn::fail(BN_ERR_ARG, "bn_kv8_dense: outputs have to start on 16 bytes");
  if (c->batch * c->kv_heads > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_dense: the cache is too large for one call");
  return c->kind == BN_KV8_INT8 ? bn::dense_launch<BN_KV8_INT8>(*c, k, v, (cudaStream_t)stream) : bn::dense_launch<BN_KV8_E4M3>(*c, k, v, (cudaStream_t)stream);
}
