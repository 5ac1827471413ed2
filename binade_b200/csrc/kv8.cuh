// The 8-bit key/value cache of bn_kv8, as its kernels see it.
#pragma once

#include <cuda_fp8.h>

#include "scores.cuh"

namespace bn {

constexpr int KV8_INT8 = BN_KV8_INT8, KV8_E4M3 = BN_KV8_E4M3;

#ifdef __CUDACC__
// Tokens of sequence b: held before the call, brought by it (a call brings up to `most`, of which `counts`
// are real; what does not fit is not taken: false).
__device__ __forceinline__ bool kv8_tokens(const bn_kv8 &c, const int32_t *__restrict__ counts, int most, int64_t b, int &held, int &brought) {
  held = min(max(c.length[b], 0), (int)c.max_seq);
  const int asked = counts ? min(max(counts[b], 0), most) : most;
  brought = min(asked, (int)c.max_seq - held);
  return brought == asked;
}

// The slot of the tail that holds block j, for j the block open at `held` or the one that is open behind
// the tokens of the call.
__device__ __forceinline__ int kv8_slot(const bn_kv8 &c, int64_t b, int held, int j) { return (c.side[b] ^ (j != held / c.block)) & 1; }

// Notes, for advance, which blocks the tail's slots hold when the tokens held .. end - 1 are there: the block open at `held`, and the
// one open behind them or an earlier one, if its rows are still there.
__device__ __forceinline__ void kv8_note(const bn_kv8 &c, int64_t b, int held, int end) {
  if (!c.kept) return;
  const int first = held / c.block, last = end / c.block, slot = c.side[b] & 1;
  int32_t *const kept = c.kept + 2 * b;
  kept[slot] = first;
  if (last != first && end % c.block) kept[slot ^ 1] = last;
  else if (kept[slot ^ 1] >= first) kept[slot ^ 1] = -1;
}

// The value of a code, without its scale.
template <int KIND>
__device__ __forceinline__ float kv8_code(uint32_t byte) {
  if constexpr (KIND == KV8_INT8) {
    return __uint_as_float(0x4B000000u | byte) - 8388736.0f;  // 2^23 + code + 128, less both
  } else {
    __nv_fp8_e4m3 f;
    f.__x = (__nv_fp8_storage_t)byte;
    return (float)f;
  }
}
// The nearest code to x / scale, ties to the even one, for finite x; 0 for NaN, the largest code for an infinity.
// As stored, with 128 added. x times the inverse is off by at most 127 * 2^-23 in a quotient of up to 127: only next to the
// middle of two codes the real quotient decides, by the sign of x - middle * scale, which one rounding keeps.
__device__ __forceinline__ uint32_t int8_code(float x, float scale, float inv) {
  const float t = x * inv;
  int q = __float2int_rn(t);  // NaN: 0
  const float off = t - (float)q;
  if (fabsf(fabsf(off) - 0.5f) < 0.0001f) {
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

// Four finite values of a block (two words of BF16 pairs) as codes: the quotient is rounded by adding 1.5 x 2^23, whose last
// byte is then code + 128; `close` is set where a quotient lies next to the middle of two codes (int8_code decides there).
__device__ __forceinline__ uint32_t int8_codes(uint32_t lo, uint32_t hi, float inv, bool &close) {
  constexpr float MAGIC = 12582912.0f + 128.0f;
  const float x[4] = {__uint_as_float(lo << 16), __uint_as_float(lo & 0xFFFF0000u), __uint_as_float(hi << 16), __uint_as_float(hi & 0xFFFF0000u)};
  uint32_t r[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float t = x[e] * inv, sum = t + MAGIC, off = t - (sum - MAGIC);
    close |= fabsf(off) > 0.49998f;  // (the quotient is off by at most 127 * 2^-23)
    r[e] = __float_as_uint(sum);
  }
  return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

// Block j of one sequence and head, keys or values, by 128 threads: a full block is scaled, coded and stored; the
// tokens of the blocks that were open (the one at `held`) or stay open go to the tail in BF16. in: the new tokens'
// rows, `step` elements apart. CHUNKS: pieces of eight values that a thread has: neighbours of one token, or for values
// two neighbours of four tokens, whose codes lie together. A block stays in registers between its maximum and its
// codes.
template <int D, int CHUNKS>
__device__ __forceinline__ void append_block(const bn_kv8 &c, bool values, int64_t b, int h, int j, int held, int end, const uint16_t *__restrict__ in, int64_t step) {
  __shared__ uint32_t part_max[4];
  const int block = c.block;
  const int64_t unit = b * c.kv_heads + h;
  const bool full = (j + 1) * (int64_t)block <= end, open = j == held / block || !full;  // the first block goes to its slot, full or not
  uint16_t *const tail = (values ? c.v_tail : c.k_tail) + (unit * 2 + (open ? kv8_slot(c, b, held, j) : 0)) * block * D;
  uint4 x[CHUNKS];
  uint32_t most = 0;  // largest magnitudes, as pairs of 16 bits
  if (full && !open) {  // most blocks of a prompt: every token is new, and none goes to the tail
    in += (int64_t)(j * block - held) * step;
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
      const int chunk = (int)threadIdx.x + 128 * i;
      if (values) {
        const uint16_t *const at = in + (int64_t)(chunk / (D / 2) * 4) * step + chunk % (D / 2) * 2;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = *reinterpret_cast<const uint32_t *>(at + e * step);
        x[i] = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
      } else {
        x[i] = *reinterpret_cast<const uint4 *>(in + (int64_t)(chunk / (D / 8)) * step + chunk % (D / 8) * 8);
      }
    }
  } else {
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
    }
  }
#pragma unroll
  for (int i = 0; i < CHUNKS; i++)
    most = __vmaxu2(__vmaxu2(most, x[i].x & 0x7FFF7FFFu), __vmaxu2(x[i].y & 0x7FFF7FFFu, __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu)));
  if (!full) return;
#pragma unroll
  for (int d = 16; d; d >>= 1) most = __vmaxu2(most, __shfl_xor_sync(BN_FULL, most, d));
  __syncthreads();  // (another block's maxima may still be read)
  if (lane_id() == 0) part_max[threadIdx.x >> 5] = most;
  __syncthreads();
  most = __vmaxu2(__vmaxu2(part_max[0], part_max[1]), __vmaxu2(part_max[2], part_max[3]));
  float amax = __uint_as_float(max(most & 0xFFFFu, most >> 16) << 16);
  const bool odd = !(amax <= 3.4e38f);  // a value that is not finite: the largest of the others then
  if (odd) {
    amax = 0.0f;
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int e = 0; e < 4; e++) amax = fmaxf(amax, fmaxf(finite_size(__uint_as_float(w[e] << 16)), finite_size(__uint_as_float(w[e] & 0xFFFF0000u))));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(BN_FULL, amax, d));
    __syncthreads();
    if (lane_id() == 0) part_max[threadIdx.x >> 5] = __float_as_uint(amax);
    __syncthreads();
    amax = __uint_as_float(max(max(part_max[0], part_max[1]), max(part_max[2], part_max[3])));
  }
  const float scale = c.kind == KV8_INT8 ? fmaxf(__fdiv_rn(amax, 127.0f), 7.888609052210118e-31f) : e4m3_scale(amax);
  const float inv = __frcp_rn(scale);  // (of a power of two: exact)
  uint8_t *const codes = (values ? c.v : c.k) + (unit * c.rows + (int64_t)j * block) * D;
  if (threadIdx.x == 0) (values ? c.v_scale : c.k_scale)[unit * (c.rows / block) + j] = scale;
#pragma unroll
  for (int i = 0; i < CHUNKS; i++) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t out[2];
    bool slow = odd;
    if (c.kind == KV8_INT8 && !odd) out[0] = int8_codes(w[0], w[1], inv, slow), out[1] = int8_codes(w[2], w[3], inv, slow);
    if (c.kind != KV8_INT8 || slow) {
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
    }
    *reinterpret_cast<uint2 *>(codes + ((int64_t)threadIdx.x + 128 * i) * 8) = make_uint2(out[0], out[1]);
  }
}
#endif

int refuse(const char *who, const char *why);  // the two as the thread's last error (kv8.cu)

// Why a bn_kv8 cannot be used, or NULL.
inline const char *kv8_refusal(const bn_kv8 *c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !c->length || !c->side || !c->tickets) return "null cache array";
  if (c->D != 64 && c->D != 128 && c->D != 256) return "a head has 64, 128 or 256 dimensions";
  if (c->block != 16 && c->block != 32 && c->block != 64) return "a block has 16, 32 or 64 tokens";
  if (c->kind != BN_KV8_INT8 && c->kind != BN_KV8_E4M3) return "unknown kind of codes";
  if (c->batch < 1 || c->kv_heads < 1 || c->batch > 65535 || c->kv_heads > 65535 || c->max_seq < 1 || c->max_seq > 0x3FFFFFFF || c->rows < c->max_seq || c->rows % 64) return "bad cache size (rows: max_seq rounded up to 64)";
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_tail | (uintptr_t)c->v_tail) & 15) return "cache arrays have to start on 16 bytes";
  return nullptr;
}

}  // namespace bn
