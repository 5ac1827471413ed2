// Writing and reading back the 8-bit key/value cache (bn_kv8).
#include <stdio.h>

#include "kv8.cuh"

namespace bn {

__device__ int g_kv8_error;  // 1: tokens were brought that the cache has no room for

namespace {

// The nearest code to x / scale, ties to the even one, for finite x; 0 for NaN, the largest code for an infinity.
// As stored, with 128 added. x times the inverse is off by at most 2^-15 in a quotient of up to 127: only next to the
// middle of two codes the real quotient decides, by the sign of x - middle * scale, which one rounding keeps.
__device__ __forceinline__ uint32_t int8_code(float x, float scale, float inv) {
  const float t = x * inv;
  int q = __float2int_rn(t);  // NaN: 0
  const float off = t - (float)q;
  if (fabsf(fabsf(off) - 0.5f) < 0.0005f) {
    const float middle = (float)q + (off > 0.0f ? 0.5f : -0.5f), side = fmaf(-middle, scale, x);
    const int below = (int)floorf(middle);
    q = side > 0.0f ? below + 1 : side < 0.0f ? below : below + (below & 1);
  }
  return (uint32_t)(min(max(q, -127), 127) + 128);
}

// Least power of two, at least 2^-100, times which 448 (the largest e4m3 value) is not below amax.
__device__ __forceinline__ float e4m3_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

__device__ __forceinline__ float finite_size(float x) {
  const float s = fabsf(x);
  return s <= 3.4028235e38f ? s : 0.0f;
}

struct AppendArgs {
  bn_kv8 c;
  const uint16_t *k, *v;
  int64_t k_seq, k_token, k_head, v_seq, v_token, v_head;  // elements
  const int32_t *counts;
  int tokens, rel;  // tokens a sequence brings at most; blocks of the cache that those can touch
};

// One block of tokens of one sequence and head, keys or values, by 128 threads: a full block is scaled, coded
// and stored; the tokens of the blocks that were open or stay open go to the tail in BF16. CHUNKS: pieces of
// eight values that a thread has: neighbours of one token, or for values two neighbours of four tokens, whose codes lie
// together. The read of the new rows and the write of the codes bound it; a block
// stays in registers between its maximum and its codes.
template <int CHUNKS>
__global__ void __launch_bounds__(128) append_kernel(const __grid_constant__ AppendArgs a) {
  const bn_kv8 &c = a.c;
  __shared__ float part_max[4];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what made the tokens, and what read the cache before
  uint32_t at = blockIdx.x;
  const bool values = at & 1;
  at >>= 1;
  const int rel = (int)(at % a.rel);
  at /= a.rel;
  const int h = (int)(at % (uint32_t)c.kv_heads);
  const int64_t b = at / (uint32_t)c.kv_heads, unit = b * c.kv_heads + h;
  int held, brought;
  kv8_tokens(c, a.counts, a.tokens, b, held, brought);
  if (rel == 0 && h == 0 && !values && threadIdx.x == 0) {
    const int asked = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
    if (asked > brought) atomicExch(&g_kv8_error, 1);
  }
  if (brought == 0) return;
  const int block = c.block, first = held / block, end = held + brought, last = (end - 1) / block;
  const int D = (int)c.D;
  const uint16_t *const in = values ? a.v + b * a.v_seq + h * a.v_head : a.k + b * a.k_seq + h * a.k_head;
  const int64_t step = values ? a.v_token : a.k_token;
  uint16_t *const tails = (values ? c.v_tail : c.k_tail) + unit * 2 * block * D;
  const int j = first + rel;
  if (j > last) return;
  {
    const bool full = (j + 1) * (int64_t)block <= end, open = j == first || !full;  // the first block goes to its slot, full or not
    uint16_t *const tail = tails + (open ? kv8_slot(c, b, held, j) : 0) * block * D;
    uint4 x[CHUNKS];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
      const int chunk = (int)threadIdx.x + 128 * i;
      if (values) {
        const int row = chunk / (D / 2) * 4, col = chunk % (D / 2) * 2;
        uint32_t w[4] = {};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int p = j * block + row + e;
          if (p < end && (full || p >= held)) w[e] = *reinterpret_cast<const uint32_t *>(p < held ? tail + (row + e) * D + col : in + (int64_t)(p - held) * step + col);
          if (open && p >= held && p < end) *reinterpret_cast<uint32_t *>(tail + (row + e) * D + col) = w[e];
        }
        // dimension by dimension: the order in which the codes lie
        x[i] = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
      } else {
        const int row = chunk / (D / 8), col = chunk % (D / 8) * 8, p = j * block + row;
        x[i] = make_uint4(0, 0, 0, 0);
        if (p < end && (full || p >= held)) x[i] = *reinterpret_cast<const uint4 *>(p < held ? tail + row * D + col : in + (int64_t)(p - held) * step + col);
        if (open && p >= held && p < end) *reinterpret_cast<uint4 *>(tail + row * D + col) = x[i];
      }
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int e = 0; e < 4; e++) amax = fmaxf(amax, fmaxf(finite_size(__uint_as_float(w[e] << 16)), finite_size(__uint_as_float(w[e] & 0xFFFF0000u))));
    }
    if (!full) return;
#pragma unroll
    for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(BN_FULL, amax, d));
    if (lane_id() == 0) part_max[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
    const float scale = c.kind == KV8_INT8 ? fmaxf(__fdiv_rn(amax, 127.0f), 7.888609052210118e-31f) : e4m3_scale(amax);
    const float inv = __frcp_rn(scale);  // (of a power of two: exact)
    uint8_t *const codes = (values ? c.v : c.k) + (unit * c.rows + (int64_t)j * block) * D;
    if (threadIdx.x == 0) (values ? c.v_scale : c.k_scale)[unit * (c.rows / block) + j] = scale;
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t out[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float f[4] = {__uint_as_float(w[2 * e] << 16), __uint_as_float(w[2 * e] & 0xFFFF0000u), __uint_as_float(w[2 * e + 1] << 16), __uint_as_float(w[2 * e + 1] & 0xFFFF0000u)};
        if (c.kind == KV8_INT8) {
          out[e] = int8_code(f[0], scale, inv) | int8_code(f[1], scale, inv) << 8 | int8_code(f[2], scale, inv) << 16 | int8_code(f[3], scale, inv) << 24;
        } else {
#pragma unroll
          for (int n = 0; n < 4; n++) f[n] = f[n] == f[n] ? f[n] * inv : 0.0f;
          out[e] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3) << 16;
        }
      }
      *reinterpret_cast<uint2 *>(codes + ((int64_t)threadIdx.x + 128 * i) * 8) = make_uint2(out[0], out[1]);
    }
  }
}

__global__ void __launch_bounds__(256) advance_kernel(const __grid_constant__ bn_kv8 c, int n, const int32_t *__restrict__ counts) {
  const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b >= c.batch) return;
  const int held = min(max(c.length[b], 0), (int)c.max_seq);
  const int now = (int)min(max((int64_t)held + (counts ? counts[b] : n), (int64_t)0), c.max_seq);
  c.length[b] = now;
  if (now / c.block != held / c.block) c.side[b] ^= 1;
}

// Eight values a thread, of keys eight of a token, of values two of four tokens, as the codes lie; tokens that the
// cache does not hold as zeros. Blocks: pieces of a sequence and head, those, and keys or values.
template <int KIND, int D>
__global__ void __launch_bounds__(256) dense_kernel(const __grid_constant__ bn_kv8 c, float *__restrict__ k, float *__restrict__ v) {
  const bool values = blockIdx.z;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, units = c.batch * c.kv_heads;
  const int row = (int)(values ? at / (D / 2) * 4 : at / (D / 8)), col = (int)(values ? at % (D / 2) * 2 : at % (D / 8) * 8);
  if (row >= c.max_seq) return;
  const int block_log2 = 31 - __clz(c.block);
  for (int64_t unit = blockIdx.y; unit < units; unit += gridDim.y) {
    const int64_t b = (int)unit / (int)c.kv_heads;
    const int length = min(max(c.length[b], 0), (int)c.max_seq), full = length >> block_log2 << block_log2;
    float x[8] = {};
    if (row < full) {  // (a block has whole rows of four)
      const float scale = (values ? c.v_scale : c.k_scale)[unit * (c.rows >> block_log2) + (row >> block_log2)];
      const uint2 w = *reinterpret_cast<const uint2 *>((values ? c.v : c.k) + (unit * c.rows + row) * D + (values ? 4 : 1) * col);
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = kv8_code<KIND>(((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 0xFFu) * scale;
    } else if (row < length) {
      const uint16_t *const tail = (values ? c.v_tail : c.k_tail) + ((unit * 2 + (c.side[b] & 1)) * c.block + row - full) * D + col;
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (row + (values ? e & 3 : 0) < length) x[e] = bf16_to_f32(tail[values ? (e & 3) * D + (e >> 2) : e]);
    }
    if (values) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (row + e < c.max_seq) *reinterpret_cast<float2 *>(v + (unit * c.max_seq + row + e) * D + col) = make_float2(x[e], x[4 + e]);
    } else {
      float4 *const out = reinterpret_cast<float4 *>(k + (unit * c.max_seq + row) * D + col);
      out[0] = make_float4(x[0], x[1], x[2], x[3]), out[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
  }
}

template <int KIND>
int dense_launch(const bn_kv8 &c, float *k, float *v, cudaStream_t s) {
  const int64_t units = c.batch * c.kv_heads, pieces = ((c.max_seq + 3) / 4 * 4 * (c.D / 8) + 255) / 256;
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
  const int64_t blocks = c->batch * c->kv_heads * a.rel * 2;
  if (blocks > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_append: too many tokens for one call");
  const int chunks = (int)(c->block * c->D / 1024);
  auto kern = chunks == 1 ? bn::append_kernel<1> : chunks == 2 ? bn::append_kernel<2> : chunks == 4 ? bn::append_kernel<4> : chunks == 8 ? bn::append_kernel<8> : bn::append_kernel<16>;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3(128), cfg.stream = (cudaStream_t)stream, cfg.attrs = attr, cfg.numAttrs = 1;
  BN_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  return bn::launched("append_kernel");
}

extern "C" int bn_kv8_advance(const bn_kv8 *c, int64_t n, const int32_t *counts, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_advance", why);
  if (n < -0x3FFFFFFF || n > 0x3FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_advance: bad number of tokens");
  bn::advance_kernel<<<(unsigned)((c->batch + 255) / 256), 256, 0, (cudaStream_t)stream>>>(*c, (int)n, counts);
  return bn::launched("advance_kernel");
}

extern "C" int bn_kv8_dense(const bn_kv8 *c, float *k, float *v, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_dense", why);
  if (!k || !v || ((uintptr_t)k | (uintptr_t)v) & 15) return bn::fail(BN_ERR_ARG, "bn_kv8_dense: outputs have to start on 16 bytes");
  if (c->batch * c->kv_heads > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_dense: the cache is too large for one call");
  return c->kind == BN_KV8_INT8 ? bn::dense_launch<BN_KV8_INT8>(*c, k, v, (cudaStream_t)stream) : bn::dense_launch<BN_KV8_E4M3>(*c, k, v, (cudaStream_t)stream);
}
