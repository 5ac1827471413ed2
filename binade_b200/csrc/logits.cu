// What is done to the logits before a token is chosen: penalties for tokens that were said already, a bias,
// a grammar's mask, and the greedy choice.
#include <cooperative_groups.h>
#include <math_constants.h>

#include "common.cuh"

namespace bn {
namespace {

// A token sets its bit in `seen`; as part of the answer (not of the prompt) it is counted too. Sums of whole
// numbers: the order of the atomics does not show.
__global__ void __launch_bounds__(256) count_kernel(const void *__restrict__ tokens, int wide, int64_t row_step, int64_t n, const int32_t *__restrict__ lengths, int64_t V, int prompt, uint32_t *__restrict__ seen, int64_t seen_row, int32_t *__restrict__ counts, int64_t counts_row) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (i >= n || (lengths && i >= lengths[b])) return;
  const int64_t t = wide ? reinterpret_cast<const int64_t *>(tokens)[b * row_step + i] : reinterpret_cast<const int32_t *>(tokens)[b * row_step + i];
  if (t < 0 || t >= V) return;
  atomicOr(seen + b * seen_row + (t >> 5), 1u << (t & 31));
  if (!prompt) atomicAdd(counts + b * counts_row + t, 1);
}

struct LogitsArgs {
  const void *x;
  float *out;
  int64_t *token;
  int64_t x_row, out_row;  // elements
  int V;
  bn_logit_rules r;
};

struct Best {
  float value;
  int at;
};
__device__ __forceinline__ Best better(Best a, Best b) {  // the larger value, of equal ones the lower index; none: at < 0
  const bool take = b.at >= 0 && (a.at < 0 || b.value > a.value || (b.value == a.value && b.at < a.at));
  return take ? b : a;
}

// Bits t .. t + 3 of a row of 32-bit words that holds bits 0 .. V - 1; t may be negative.
__device__ __forceinline__ uint32_t four_bits(const uint32_t *__restrict__ words, int t, int V) {
  const int lo = max(t, 0) >> 5, hi = min(t + 3, V - 1) >> 5;
  const uint32_t a = __ldg(words + lo), b = hi == lo ? a : __ldg(words + hi);
  if (t < 0) return a << -t;
  return (t & 31) > 28 && hi > lo ? __funnelshift_r(a, b, t & 31) : a >> (t & 31);
}

// The cluster's barrier in two halves: a block's shared memory may be written from outside once that block is known
// to run, which its arrival tells. Arriving at the start and waiting before the store hides the barrier behind the pass.
// (Relaxed: no memory goes with it.)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// A cluster of blocks per row: the blocks take pieces of the vocabulary in turn, four tokens a thread, and the
// first of them joins their choices through distributed shared memory. One launch, whatever the batch: 6 us in a graph for
// one row of 128256 (the latency of a few loads in a row), 35 us for 64 rows of 151937 fp32 with penalties, bias and masks (2.3
// TB/s; 12 us of bytes, 17 of instructions at full issue: a thread's ten rounds each wait for their loads, then for the
// counts). Quads start where the output row
// has 16-byte boundaries (rows of an odd vocabulary start anywhere); the input is read in one piece
// where its row has them at the same places. Counts are read only where a token was said.
template <typename T, int THREADS, int U>
__global__ void __launch_bounds__(THREADS, U == 1 ? 4 : 2) logits_kernel(const __grid_constant__ LogitsArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster_arrive();
  const int64_t b = blockIdx.y;
  const T *const x = reinterpret_cast<const T *>(a.x) + b * a.x_row;
  float *const out = a.out + b * a.out_row;
  const bn_logit_rules &r = a.r;
  const uint32_t *const seen = r.seen ? r.seen + b * r.seen_row : nullptr, *const mask = r.mask ? r.mask + b * r.mask_row : nullptr;
  const int32_t *const counts = r.seen ? r.counts + b * r.counts_row : nullptr;
  const float *const bias = r.bias ? r.bias + b * r.bias_row : nullptr;
  const float repetition = r.repetition ? r.repetition[b] : r.repetition_all, presence = r.presence ? r.presence[b] : r.presence_all, frequency = r.frequency ? r.frequency[b] : r.frequency_all;
  const int shift = (int)(((uintptr_t)out >> 2) & 3);  // quad k: tokens 4k - shift ..
  const bool whole_x = (((uintptr_t)(x - shift)) & (4 * sizeof(T) - 1)) == 0, whole_bias = bias && ((uintptr_t)(bias - shift) & 15) == 0;
  const int V = a.V, quads = (V + shift + 3) / 4;
  Best best{-CUDART_INF_F, -1};
  // U quads a thread at a time, first all their loads, so that the few tokens that were said (whose counts are
  // a second load behind the first) wait once
  const int stride = (int)gridDim.x * THREADS;
  for (int k0 = blockIdx.x * THREADS + threadIdx.x; k0 < quads; k0 += U * stride) {
    float y[U][4], add[U][4];
    uint32_t said[U], open[U];
    int n[U];  // the count of the first token of the quad that was said
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = 4 * (k0 + u * stride) - shift;
      const bool inside = t >= 0 && t + 3 < V;
      said[u] = 0, open[u] = 15;
      if (k0 + u * stride >= quads) continue;
      if (inside && whole_x) {
        if constexpr (sizeof(T) == 2) {
          const uint2 w = *reinterpret_cast<const uint2 *>(x + t);
          y[u][0] = __uint_as_float(w.x << 16), y[u][1] = __uint_as_float(w.x & 0xFFFF0000u), y[u][2] = __uint_as_float(w.y << 16), y[u][3] = __uint_as_float(w.y & 0xFFFF0000u);
        } else {
          const float4 w = *reinterpret_cast<const float4 *>(x + t);
          y[u][0] = w.x, y[u][1] = w.y, y[u][2] = w.z, y[u][3] = w.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int at = min(max(t + e, 0), V - 1);
          if constexpr (sizeof(T) == 2) y[u][e] = __uint_as_float((uint32_t)x[at] << 16);
          else y[u][e] = x[at];
        }
      }
      if (seen) said[u] = four_bits(seen, t, V) & 15u;
      if (mask) open[u] = four_bits(mask, t, V) & 15u;
      if (bias) {
        if (inside && whole_bias) {
          const float4 w = *reinterpret_cast<const float4 *>(bias + t);
          add[u][0] = w.x, add[u][1] = w.y, add[u][2] = w.z, add[u][3] = w.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) add[u][e] = bias[min(max(t + e, 0), V - 1)];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = 4 * (k0 + u * stride) - shift;
      said[u] &= t < 0 ? 15u << -t : t + 3 >= V ? 15u >> (t + 4 - V) : 15u;
      n[u] = said[u] ? counts[t + __ffs((int)said[u]) - 1] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = 4 * (k0 + u * stride) - shift;
      if (k0 + u * stride >= quads) break;
      // every operation rounds by itself, in the order of the definition: a plain evaluation gives the same bits
      for (uint32_t left = said[u]; left; left &= left - 1) {  // few tokens are: a loop over those
        const int e = __ffs((int)left) - 1, count = left == said[u] ? n[u] : counts[t + e];
        float z = e & 2 ? (e & 1 ? y[u][3] : y[u][2]) : (e & 1 ? y[u][1] : y[u][0]);
        z = z > 0.0f ? __fdiv_rn(z, repetition) : __fmul_rn(z, repetition);
        if (count > 0) z = __fsub_rn(z, __fadd_rn(__fmul_rn(frequency, (float)count), presence));
#pragma unroll
        for (int i = 0; i < 4; i++) y[u][i] = i == e ? z : y[u][i];
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float &z = y[u][e];
        if (bias) z = __fadd_rn(z, add[u][e]);
        if (!((open[u] >> e) & 1u)) z = -CUDART_INF_F;
        if (z > best.value && t + e >= 0 && t + e < V) best = {z, t + e};  // (NaN is never chosen)
      }
      if (t >= 0 && t + 3 < V) {
        *reinterpret_cast<float4 *>(out + t) = make_float4(y[u][0], y[u][1], y[u][2], y[u][3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (t + e >= 0 && t + e < V) out[t + e] = y[u][e];
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) best = better(best, Best{__shfl_xor_sync(BN_FULL, best.value, d), __shfl_xor_sync(BN_FULL, best.at, d)});
  __shared__ Best warps[32], blocks[16];
  if (lane_id() == 0) warps[threadIdx.x >> 5] = best;
  __syncthreads();
  cluster_wait();
  if (threadIdx.x < 32) {
    best = threadIdx.x < THREADS / 32 ? warps[threadIdx.x] : Best{-CUDART_INF_F, -1};
#pragma unroll
    for (int d = 16; d; d >>= 1) best = better(best, Best{__shfl_xor_sync(BN_FULL, best.value, d), __shfl_xor_sync(BN_FULL, best.at, d)});
    if (threadIdx.x == 0) *cluster.map_shared_rank(blocks + cluster.block_rank(), 0) = best;
  }
  cluster.sync();
  if (cluster.block_rank() == 0 && threadIdx.x == 0) {
    for (unsigned i = 0; i < cluster.num_blocks(); i++) best = i ? better(best, blocks[i]) : blocks[0];
    a.token[b] = best.at;
  }
}

}  // namespace
}  // namespace bn

extern "C" int bn_token_counts(const void *tokens, int tokens64, int64_t row_step, int64_t batch, int64_t n, const int32_t *lengths, int64_t V, int prompt, uint32_t *seen, int64_t seen_row, int32_t *counts, int64_t counts_row, void *stream) {
  if (batch < 0 || batch > 65535 || n < 0 || V < 1 || V > 0x3FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_token_counts: bad size");
  if (n == 0 || batch == 0) return BN_OK;
  if (!tokens || !seen || !counts) return bn::fail(BN_ERR_ARG, "bn_token_counts: null pointer");
  if ((n + 255) / 256 > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_token_counts: too many tokens");
  bn::count_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)batch), 256, 0, (cudaStream_t)stream>>>(tokens, tokens64, row_step, n, lengths, V, prompt, seen, seen_row, counts, counts_row);
  return bn::launched("count_kernel");
}

extern "C" int bn_logits(const void *x, int fp32, int64_t x_row, int64_t batch, int64_t V, const bn_logit_rules *rules, float *out, int64_t out_row, int64_t *token, void *stream) {
  if (batch < 0 || batch > 65535 || V < 1 || V > 0x3FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_logits: bad size");
  if (!rules || (batch && (!x || !out || !token)) || (rules && rules->seen && !rules->counts)) return bn::fail(BN_ERR_ARG, "bn_logits: null pointer");
  if (batch == 0) return BN_OK;
  constexpr int threads = 512;
  const int quads = batch <= 8 ? 2 : 1;
  bn::LogitsArgs a{x, out, token, x_row, out_row, (int)V, *rules};
  // Blocks of a row: up to 8 (the portable cluster size), 16 where the rows are few; two quads a thread there, whose loads wait
  // together. us in a graph, 128256 tokens, penalties, one quad and 8 blocks / two and 16: 1 row 9.4 / 6.8, 8 rows 9.8 / 8.3, 16
  // rows 12.6 / 11.9, 32 rows 12.9 / 17.8, 64 rows 22 / 33.
  const int64_t need = (V + 4 * threads - 1) / (4 * threads);
  const unsigned most = batch <= 8 ? 16 : 8;
  unsigned blocks = 1;
  while (blocks < most && blocks < need) blocks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, (unsigned)batch), cfg.blockDim = dim3(threads), cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  auto kern = quads == 2 ? (fp32 ? bn::logits_kernel<float, threads, 2> : bn::logits_kernel<uint16_t, threads, 2>) : fp32 ? bn::logits_kernel<float, threads, 1> : bn::logits_kernel<uint16_t, threads, 1>;
  if (blocks > 8) BN_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  BN_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  return bn::launched("logits_kernel");
}
