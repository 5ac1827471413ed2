// Attention of new tokens over an 8-bit key/value cache (bn_kv8): for the few query rows that share a key head
// (a token or a short draft times the head's group), bound by reading the cache once.
//
// The rows are the M of mma.sync m16n8k16 (16 or 32 rows a block, f16 operands, fp32 sums): a
// decode step has 1 to 32 of them, which tcgen05's tiles of 64 and 128 rows would leave empty, and
// at one byte a value the legacy tensor path has the rate to spare.
//   codes -> f16   exact (8 bits fit f16's 11): int8 codes, stored as code + 128, become 1024 + byte by one byte
//                  permute and lose the 1152 by one subtraction; e4m3 converts in hardware
//   queries        to f16 after a power of two per row that puts its largest value in [1, 2): exact down to
//                  2^-24 of that value, below which a product does not show in an fp32 sum of scores
//   scores         K's scale multiplies the sum. A weight is p = 2^(s - m), m near the row's largest s, and goes to the sum
//                  of weights as it is; to the product with V's codes goes p' = p vscale 2^d in f16, d near m less
//                  the row's largest s + log2(vscale). Two maxima, since either sum must keep what weighs in it however
//                  far apart the blocks' scales lie: a block of zeros (scale 2^-100) weighs in the first alone
//   order of k     a dot product may take its dimensions, and the sum over keys its keys, in any order: each
//                  thread reads 16 neighbouring bytes of a key and calls them the elements that the
//                  fragments want. V's codes lie four keys at a time, dimension by dimension, since its fragments pair
//                  keys: a word is one dimension of the thread's four keys
//   rounding       of p' to f16, 2^-11 of it. A row's largest p' starts in 2^12 .. 2^13, so that this holds down to 2^-26 of the
//                  largest, and what is below 2^-37 of it is zero: where one key takes nearly all the weight and has no value,
//                  the others are the output
//   maxima         m and d move only when a p or a p' passes 2^15 (f16 ends at 2^16): a vote per 16 keys
//                  in place of shuffles and a rescaling of the sums
// A warp streams its own keys through a cp.async ring of its own: no barrier in the loop; the warps of a block
// are joined at the end. The work is the tiles of all sequences and heads in a row, cut into equal
// shares: sequences of unequal lengths load the SMs alike, and one long one spreads over all of them. A sequence and head
// that is cut leaves partial sums; the block that finishes last joins them (it takes the last of the tickets), or, where
// there may be many, a second kernel, always in the same order. The block with a sequence's last tile also appends the new tokens, reads them where they came from, and
// codes the block that they fill before it reads it: a decode step is one launch. Several groups of rows (more than
// 32, or 16 with heads of 256) read what an append kernel has written.
//
// Measured: 64 sequences of up to 8192 tokens, 8 key heads of 128, int8, 637 MB: 179 us, 3.6 TB/s, 55 % of the copy rate;
// one sequence of 131073, 269 MB: 71 us; one of 300: 21 us a call, 12 in a graph. What bounds the long ones: 68 M warp
// instructions (430 a piece of 16 keys; 45 % of the issue slots) at 12 warps an SM, fixed-latency waits first.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace bn {
namespace {

__device__ int g_attend_error;  // 1: tokens were brought that the cache has no room for
__device__ __forceinline__ void kv8_overflow() { atomicExch(&g_attend_error, 1); }

constexpr int WARPS = 4;
constexpr float MOST = 15.0f;  // p and p' may reach 2^15
constexpr float AIM = 13.0f;   // where a row's largest p' starts, in powers of two: that leaves 26 below it before f16 loses bits
constexpr float NOTHING = -3.402823466e38f;  // a row's m while no key was visible: finite, so that a masked score less m stays -inf

struct AttendArgs {
  bn_kv8 c;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_seq, q_token, q_head, o_seq, o_token, o_head;  // elements
  const int32_t *counts, *prefix;
  const float *slopes;
  const uint16_t *k, *v;  // new tokens to append, or NULL
  int64_t k_seq, k_token, k_head, v_seq, v_token, v_head;
  int tokens, heads, group;  // group: query heads of a key head
  int window, causal, zero_rest;
  float scale, cap;
  // workspace: tiles before each sequence [batch + 1], the share of a block; then partial results, two slots a block
  int64_t *plan;
  float *parts;
  int row_groups;
  int blocks;
  bool join_here;  // by the block that finishes last; else by the join kernel
};

template <int D, int MT>
struct Shape {
  static constexpr int ROWS = 16 * MT;                 // query rows of a block
  static constexpr int P = MT * D <= 128 ? 2 : 1;      // pieces of 16 keys that a warp takes at once, where registers allow two: their chains of dependent instructions overlap
  static constexpr int KS = 16 * P;                    // keys of a warp's stage
  static constexpr int TILE = KS * WARPS;              // keys of a block's step
  static constexpr int STAGES = D == 256 ? 3 : P == 2 && D == 128 ? 2 : 4;
  static constexpr int STAGE_BYTES = 2 * KS * D;
  static constexpr int NT = D / 8;                     // n8 tiles of the output
  static constexpr int RING = WARPS * STAGES * STAGE_BYTES;
  static constexpr int JOIN = WARPS * ROWS * (D + 4) * 4;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
  static constexpr int PART = ROWS * (D + 3);          // floats of a partial result: sums, then m, d and sums of weights
};

// Tiles of sequence b: of the blocks that are full before `split` from the first key on, then one of everything behind.
// split is the end of the blocks that were full before the call where the call appends, else of those that are full now.
struct Span {
  int held, brought, L, full, split, start, quant, tiles;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int64_t b, int tile) {
  Span s;
  kv8_tokens(a.c, a.counts, a.tokens, b, s.held, s.brought);
  const int log2 = 31 - __clz(a.c.block);
  s.L = s.held + s.brought, s.full = s.L >> log2 << log2, s.split = a.k ? s.held >> log2 << log2 : s.full, s.start = 0;
  if (s.brought == 0) {
    s.quant = s.tiles = 0;
    return s;
  }
  if (a.window > 0) s.start = min(max(0, s.held - a.window + 1) & ~15, s.split);  // the first query looks back furthest
  s.quant = (s.split - s.start + tile - 1) / tile;
  s.tiles = s.quant + (s.L > s.split);
  return s;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16x(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes, in the low or (HIGH) the high half of a word, as f16.
template <int KIND, bool HIGH>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
  uint32_t r;
  if constexpr (KIND == KV8_INT8) {
    r = __byte_perm(w, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));  // 1152
  } else if constexpr (HIGH) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  }
  return r;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
// Which 16-byte piece of a key's row in shared memory holds its piece `col`, and the same for a row of four keys of V:
// chosen so that the eight lanes of a 16-byte access meet no bank twice (K: four pieces of two neighbouring
// keys; V: two pieces of four rows).
template <int D>
__device__ __forceinline__ uint32_t k_piece(uint32_t key, uint32_t col) {
  return D == 64 ? col : col ^ ((key & 1u) << 2);
}
template <int D>
__device__ __forceinline__ uint32_t v_piece(uint32_t four, uint32_t col) {
  return D == 64 ? col ^ ((four & 1u) | ((four & 2u) << 1)) : col ^ (four & 3u);
}

// What a warp has so far of its lane's rows: sums of p' times codes, m and d (powers of two), sums of p.
template <int D, int MT>
struct State {
  float o[MT][Shape<D, MT>::NT][4];
  float m[MT][2], d[MT][2], l[MT][2];
};

// What a lane's rows need: positions (-1: no row), the factor from a sum of products to a score, the bias.
template <int MT>
struct Rows {
  int i[MT][2];
  float factor[MT][2], slope[MT][2];
  int L, prefix;
};

// What goes with a 16-key piece: its first key, the first key that is not its stage's, K's scale, V's and that as a power of
// two, whether some row does not see all of it.
struct PieceOf16 {
  int key0, end;
  float scale, vscale, vlog;
  bool masked;
};

// The scores of P pieces into weights: x holds the raw sums and gets p' (tile j, column 2c + e: key key0 + 4c + 2j + e).
// Updates the sum of weights; where a p or a p' would pass 2^MOST, moves m and d and rescales the sums.
template <int D, int MT, int P, bool PLAIN>
__device__ __forceinline__ void weigh(const AttendArgs &a, float (&x)[P][MT][2][4], const Rows<MT> &r, State<D, MT> &st, const PieceOf16 (&pc)[P]) {
  const int lane_key = 4 * (int)(lane_id() & 3u);
#pragma unroll
  for (int p = 0; p < P; p++) {
    const int first = pc[p].key0 + lane_key;
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float f = fmaxf(fminf(pc[p].scale * r.factor[mt][h], 3.0e38f), -3.0e38f);
        const bool wide = !PLAIN && a.cap > WIDE_CAP;
        if (wide) {
#pragma unroll
          for (int i = 0; i < 4; i++) x[p][mt][i >> 1][2 * h + (i & 1)] = capped_wide(x[p][mt][i >> 1][2 * h + (i & 1)] * f, a.cap * LOG2E);
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float &v = x[p][mt][j][2 * h + e];
            if (PLAIN || !wide) v *= f;
            if constexpr (!PLAIN) {
              if (a.cap > 0.0f && !wide) v = capped(v, a.cap * LOG2E);
              v = fmaf(-r.slope[mt][h], (float)abs(r.i[mt][h] - (first + 2 * j + e)), v);
            }
          }
      }
    if (pc[p].masked) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          int lo = 0, hi = 0;
          if (r.i[mt][h] >= 0) visible_keys(r.i[mt][h], r.L, r.prefix, a.window, a.causal, lo, hi);
          hi = min(hi, pc[p].end);
#pragma unroll
          for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int key = first + 2 * j + e;
              if (key < lo || key >= hi) x[p][mt][j][2 * h + e] = -CUDART_INF_F;
            }
        }
    }
  }
  float top[MT][2], top_v[MT][2];  // largest s and s + log2(vscale)
  bool over = false;
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      top[mt][h] = top_v[mt][h] = -CUDART_INF_F;
#pragma unroll
      for (int p = 0; p < P; p++) {
        const float t = fmaxf(fmaxf(x[p][mt][0][2 * h], x[p][mt][0][2 * h + 1]), fmaxf(x[p][mt][1][2 * h], x[p][mt][1][2 * h + 1]));
        top[mt][h] = fmaxf(top[mt][h], t), top_v[mt][h] = fmaxf(top_v[mt][h], t + pc[p].vlog);
      }
      over |= top[mt][h] - st.m[mt][h] > MOST || top_v[mt][h] - st.m[mt][h] + st.d[mt][h] > MOST;
    }
  if (__any_sync(BN_FULL, over)) {
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float t = top[mt][h], u = top_v[mt][h];
        t = fmaxf(t, __shfl_xor_sync(BN_FULL, t, 1)), u = fmaxf(u, __shfl_xor_sync(BN_FULL, u, 1));
        t = fmaxf(t, __shfl_xor_sync(BN_FULL, t, 2)), u = fmaxf(u, __shfl_xor_sync(BN_FULL, u, 2));
        t = fmaxf(t, st.m[mt][h]);
        const float rise = t - st.m[mt][h], d = fminf(st.d[mt][h] + rise, floorf(AIM - (u - t)));  // (m - d stays where it is unless a p' is too large)
        const float keep = ex2(-rise), keep_o = ex2(d - st.d[mt][h] - rise);
        st.m[mt][h] = t, st.d[mt][h] = d, st.l[mt][h] *= keep;
#pragma unroll
        for (int n = 0; n < Shape<D, MT>::NT; n++) st.o[mt][n][2 * h] *= keep_o, st.o[mt][n][2 * h + 1] *= keep_o;
      }
  }
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float to_v = ex2(st.d[mt][h]);
#pragma unroll
      for (int p = 0; p < P; p++) {
        const float g = fminf(pc[p].vscale * to_v, 3.0e38f);  // (where the product passes fp32, p is zero)
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float &v = x[p][mt][j][2 * h + e];
            v = ex2(v - st.m[mt][h]);
            sum += v;
            v *= g;
          }
        st.l[mt][h] += sum;
      }
    }
}

// The dimension of n8 tile t's column n.
template <int D>
__device__ __forceinline__ constexpr int dim_of(int t, int n) {
  return D == 64 ? 8 * n + t : 128 * (t / 16) + 16 * n + t % 16;
}

// Where the open block's tokens are read: from the tail, the new ones where they came from (if they come with the call).
struct OpenRows {
  const uint16_t *k_tail, *v_tail, *k, *v;  // tails less the block's first token; new ones less `from` tokens
  int64_t k_step, v_step;
  int D, from;
  __device__ __forceinline__ const uint16_t *key(int j) const { return j >= from ? k + j * k_step : k_tail + (int64_t)j * D; }
  __device__ __forceinline__ const uint16_t *value(int j) const { return j >= from ? v + j * v_step : v_tail + (int64_t)j * D; }
};

// New tokens of one sequence and head that fill a block, into the cache, by the block's 128 threads.
template <int D>
__device__ __noinline__ void append_filled(const AttendArgs &a, int64_t b, int h, int held, int L) {
  const int first = held / a.c.block, last = (L - 1) / a.c.block;
  for (int side = 0; side < 2; side++) {
    const uint16_t *const in = side ? a.v + b * a.v_seq + h * a.v_head : a.k + b * a.k_seq + h * a.k_head;
    const int64_t step = side ? a.v_token : a.k_token;
    for (int j = first; j <= last; j++) {
      if (a.c.block == 16) append_block<D, 16 * D / 1024>(a.c, side, b, h, j, held, L, in, step);
      else if (a.c.block == 32) append_block<D, 32 * D / 1024>(a.c, side, b, h, j, held, L, in, step);
      else append_block<D, 64 * D / 1024>(a.c, side, b, h, j, held, L, in, step);
    }
  }
  __syncthreads();
}

// The open block's 16 tokens from `key0` on, in BF16. Weights go in two BF16 halves (hi + lo: 2^-17), values over the power of two
// of the largest, which is V's scale then as a code's block has one: no sum passes fp32, and none is lost beside the codes' for a
// scale that is not theirs. Where a value is not finite, a weight of zero must not touch it: those go one by one.
template <int D, int MT, bool PLAIN>
__device__ void open_block(const AttendArgs &a, const uint16_t *const (&qrow)[MT][2], const OpenRows &rows, int L, int key0, const Rows<MT> &r, State<D, MT> &st) {
  const uint32_t lane = lane_id(), n = lane >> 2, c = lane & 3u;
  float x1[1][MT][2][4] = {};
  auto &x = x1[0];
  const uint16_t *k[2];
#pragma unroll
  for (int j = 0; j < 2; j++) k[j] = rows.key(min(key0 + 4 * (int)(n >> 1) + 2 * j + (int)(n & 1), L - 1)) + 16 * c;
#pragma unroll 1
  for (int g = 0; g < D / 64; g++)
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const uint2 k0 = *reinterpret_cast<const uint2 *>(k[0] + 64 * g + 4 * w), k1 = *reinterpret_cast<const uint2 *>(k[1] + 64 * g + 4 * w);
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        uint2 q[2] = {};
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (qrow[mt][h]) q[h] = *reinterpret_cast<const uint2 *>(qrow[mt][h] + 64 * g + 16 * c + 4 * w);
        const uint32_t f[4] = {q[0].x, q[1].x, q[0].y, q[1].y};
        mma_bf16x(x[mt][0], f, k0.x, k0.y);
        mma_bf16x(x[mt][1], f, k1.x, k1.y);
      }
    }
  Rows<MT> plain = r;  // the queries as they are: no power of two in the factor
#pragma unroll
  for (int mt = 0; mt < MT; mt++) plain.factor[mt][0] = plain.factor[mt][1] = a.cap > 0.0f ? a.scale * (2.0f * LOG2E / a.cap) : a.scale * LOG2E;
  const uint16_t *v[4];
  uint32_t most = 0;  // largest magnitudes, as pairs of 16 bits
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = rows.value(min(key0 + 4 * (int)c + i, L - 1));
#pragma unroll
  for (int t = 0; t < Shape<D, MT>::NT; t += 2)
#pragma unroll
    for (int i = 0; i < 4; i++) most = __vmaxu2(most, *reinterpret_cast<const uint32_t *>(v[i] + dim_of<D>(t, (int)n)) & 0x7FFF7FFFu);  // dims dim_of(t, n) and the next
  most = __reduce_max_sync(BN_FULL, max(most & 0xFFFFu, most >> 16));
  const bool odd = most >= 0x7F80u;
  if (odd) {  // the largest of the others
    most = 0;
#pragma unroll 1
    for (int t = 0; t < Shape<D, MT>::NT; t += 2)
#pragma unroll 1
      for (int i = 0; i < 4; i++) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(v[i] + dim_of<D>(t, (int)n)), lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
        most = max(most, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
      }
    most = __reduce_max_sync(BN_FULL, most);
  }
  const int exponent = min(max((int)(most >> 7), 27), 253);  // as it stands in fp32: 2^-100 .. 2^126
  const float vscale = __uint_as_float((uint32_t)exponent << 23), vinv = __uint_as_float((uint32_t)(254 - exponent) << 23);
  const PieceOf16 piece[1] = {{key0, L, 1.0f, vscale, (float)(exponent - 127), true}};
  weigh<D, MT, 1, PLAIN>(a, x1, plain, st, piece);
  uint32_t hi[MT][4], lo[MT][4];
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int f = 0; f < 4; f++) {
      const float p0 = x[mt][f >> 1][2 * (f & 1)], p1 = x[mt][f >> 1][2 * (f & 1) + 1];
      hi[mt][f] = pack_bf16(p0, p1);
      lo[mt][f] = pack_bf16(p0 - __uint_as_float(hi[mt][f] << 16), p1 - __uint_as_float(hi[mt][f] & 0xFFFF0000u));
    }
  if (!odd) {
    const uint32_t down = (__float_as_uint(vinv) >> 16) * 0x10001u;  // 2^-exponent twice, in BF16
#pragma unroll
    for (int t = 0; t < Shape<D, MT>::NT; t += 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        w[i] = *reinterpret_cast<const uint32_t *>(v[i] + dim_of<D>(t, (int)n));
        asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(down));
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const uint32_t b0 = __byte_perm(w[0], w[1], e ? 0x7632 : 0x5410), b1 = __byte_perm(w[2], w[3], e ? 0x7632 : 0x5410);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          mma_bf16x(st.o[mt][t + e], hi[mt], b0, b1);
          mma_bf16x(st.o[mt][t + e], lo[mt], b0, b1);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int key = 0; key < 16; key++) {
    const uint16_t *const row = rows.value(min(key0 + key, L - 1));
    const uint32_t from = (lane & ~3u) | (key >> 2);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float p = __shfl_sync(BN_FULL, x[mt][(key >> 1) & 1][2 * h + (key & 1)], from);
        if (p != 0.0f)
#pragma unroll
          for (int t = 0; t < Shape<D, MT>::NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) st.o[mt][t][2 * h + e] = fmaf(p, bf16_to_f32(row[dim_of<D>(t, 2 * (int)c + e)]) * vinv, st.o[mt][t][2 * h + e]);
      }
  }
}

// Four outputs of a row: sums of p' times codes by the sum of weights, without the 2^d that p' has more than p.
__device__ __forceinline__ uint2 quotients(float4 o, float l, float d) {
  const float inv = 1.0f / l, back = ex2(-d);  // (o / l first: it is never small where back is)
  return make_uint2(pack_bf16(o.x * inv * back, o.y * inv * back), pack_bf16(o.z * inv * back, o.w * inv * back));
}

// The parts of one sequence and head together, by the block that finished last: four dimensions a thread, sixteen parts
// at a time. Parts lie in the workspace, two slots a block of the grid; late: the first part is in its block's second slot.
template <int D, int MT>
__device__ __noinline__ void join_parts(const AttendArgs &a, int64_t b, int kv, int rows, int brought, int64_t first, int parts, bool late) {
  using S = Shape<D, MT>;
  constexpr int U = 16;
  for (int i = (int)threadIdx.x; i < rows * (D / 4); i += WARPS * 32) {
    const int row = i / (D / 4), col = i % (D / 4) * 4;
    float m = NOTHING, d = 0.0f, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p0 = 0; p0 < parts; p0 += U) {
      float pm[U], pd[U], pl[U];
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int p = min(p0 + u, parts - 1);
        const float *const part = a.parts + ((first + p) * 2 + (p == 0 && late ? 1 : 0)) * S::PART;
        pm[u] = __ldcg(part + S::ROWS * D + row), pd[u] = __ldcg(part + S::ROWS * (D + 1) + row), pl[u] = __ldcg(part + S::ROWS * (D + 2) + row);
        v[u] = __ldcg(reinterpret_cast<const float4 *>(part + row * D + col));
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < U; u++) top = fmaxf(top, pm[u]);
      const float had = (top - m) + d;
      d = had;
#pragma unroll
      for (int u = 0; u < U; u++) pd[u] += top - pm[u], d = fminf(d, pd[u]);  // (a part that stands for several here counts once)
      const float keep = ex2(d - had);
      l *= ex2(m - top), o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep;
      m = top;
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (p0 + u >= parts) break;
        const float f = ex2(d - pd[u]);
        l = fmaf(ex2(pm[u] - top), pl[u], l);
        o.x = fmaf(f, v[u].x, o.x), o.y = fmaf(f, v[u].y, o.y), o.z = fmaf(f, v[u].z, o.z), o.w = fmaf(f, v[u].w, o.w);
      }
    }
    const int t = row / a.group, head = kv * a.group + row % a.group;
    uint16_t *const out = a.out + b * a.o_seq + t * a.o_token + head * a.o_head + col;
    if (t < brought) *reinterpret_cast<uint2 *>(out) = quotients(o, l, d);
    else if (a.zero_rest) *reinterpret_cast<uint2 *>(out) = make_uint2(0, 0);
  }
}

template <int D, int KIND, int MT, bool PLAIN>
__global__ void __launch_bounds__(WARPS * 32, (D == 64 && MT == 1) ? 4 : (MT * D <= 128) ? 3 : 2) attend_kernel(const __grid_constant__ AttendArgs a) {
  using S = Shape<D, MT>;
  constexpr int NT = S::NT;
  extern __shared__ __align__(128) uint8_t attend_smem[];
  __shared__ int64_t found[2];
  __shared__ int64_t warp_tiles[WARPS];
  __shared__ bool last_ticket;
  __shared__ float join_m[WARPS][S::ROWS], join_d[WARPS][S::ROWS], join_l[WARPS][S::ROWS];
  __shared__ float scales[WARPS][S::STAGES][2][S::KS / 16];
  const uint32_t lane = lane_id(), warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3u;
  const bn_kv8 &cache = a.c;
  const int per_seq = (int)cache.kv_heads * a.row_groups;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this block's share of the tiles: every thread counts those of a run of sequences
  const int per_thread = (int)((cache.batch + WARPS * 32 - 1) / (WARPS * 32));
  const int64_t b_from = min((int64_t)threadIdx.x * per_thread, cache.batch), b_to = min(b_from + per_thread, cache.batch);
  int64_t mine = 0;
  bool nothing = false;
  for (int64_t b = b_from; b < b_to; b++) {
    const Span s = span_of(a, b, S::TILE);
    mine += s.tiles;
    nothing |= s.brought == 0;
    if (a.k && blockIdx.x == 0 && s.brought < (a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens)) kv8_overflow();
  }
  if (__syncthreads_or(nothing && a.zero_rest))  // sequences that bring nothing have no tiles: their rows are zeroed here
    for (int64_t b = blockIdx.x; b < cache.batch; b += gridDim.x)
      if (span_of(a, b, S::TILE).brought == 0)
        for (int i = (int)threadIdx.x; i < a.tokens * a.heads * (D / 8); i += WARPS * 32) {
          const int row = i / (D / 8);
          *reinterpret_cast<uint4 *>(a.out + b * a.o_seq + row / a.heads * a.o_token + row % a.heads * a.o_head + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
        }
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(BN_FULL, upto, d);
    if (lane >= (uint32_t)d) upto += o;
  }
  if (lane == 31) warp_tiles[warp] = upto;
  __syncthreads();
  int64_t before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    if (w < (int)warp) before += warp_tiles[w];
    total += warp_tiles[w];
  }
  const int64_t share = max((total * per_seq + a.blocks - 1) / a.blocks, (int64_t)1);
  int64_t x = (int64_t)blockIdx.x * share;
  const int64_t x_end = min(x + share, total * per_seq);
  for (int64_t b = b_from, at = before; b < b_to; b++) {
    const int tiles = span_of(a, b, S::TILE).tiles;
    if (blockIdx.x == 0) a.plan[b] = at;
    if (x >= at * per_seq && x < (at + tiles) * per_seq) found[0] = b, found[1] = at;
    at += tiles;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[cache.batch] = total, a.plan[cache.batch + 1] = share;
  __syncthreads();
  if (x >= x_end) return;
  int64_t b = found[0];
  Span s = span_of(a, b, S::TILE);
  int hr, tile;  // head and row group, tile inside it
  {
    const int64_t rest = x - found[1] * per_seq;
    hr = (int)(rest / s.tiles), tile = (int)(rest % s.tiles);
  }
  const uint32_t ring = smem_addr(attend_smem) + warp * (S::STAGES * S::STAGE_BYTES);
  const int block_log2 = 31 - __clz(cache.block);
  bool first = true;

  while (true) {
    const int kv = hr / a.row_groups, row0 = hr % a.row_groups * S::ROWS;
    const int rows = min(S::ROWS, a.group * a.tokens - row0);
    const int64_t unit = b * cache.kv_heads + kv;
    const int tile_end = (int)min((int64_t)s.tiles, tile + (x_end - x));
    const uint8_t *const codes[2] = {cache.k + unit * cache.rows * D, cache.v + unit * cache.rows * D};
    const int64_t scale_at = unit * (cache.rows / cache.block);

    // The block of the last tile appends: first, if the new tokens fill a block, which is then one more tile of codes
    // (from `split` on); else beside the copies.
    const bool appends = a.k && tile_end == s.tiles, fills = appends && s.full > s.split;
    const int codes_end = fills ? s.quant + 1 : min(tile_end, s.quant);
    auto key_of = [&](int t) { return (t < s.quant ? s.start + t * S::TILE : s.split) + (int)warp * S::KS; };
    // this warp's keys of tile t, 16 at a time: those of the full blocks come in whole pieces
    auto issue = [&](int t, int slot) {
      if (t < codes_end) {
        const int key0 = key_of(t), end = t < s.quant ? s.split : s.full;
        const uint32_t to = ring + slot * S::STAGE_BYTES;
#pragma unroll
        for (int sub = 0; sub < S::KS / 16; sub++) {
          if (key0 + 16 * sub >= end) {  // nothing there: zeros that the masks keep out
            for (int i = 0; sub && i < 2 * (D / 32); i++) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(to + (i & 1) * (S::KS * D) + sub * (16 * D) + (lane + 32 * (i >> 1)) * 16), "r"(0) : "memory");
            if (lane < 2) scales[warp][slot][lane][sub] = 1.0f;
            continue;
          }
#pragma unroll
          for (int side = 0; side < 2; side++) {
            const uint8_t *const from = codes[side] + (int64_t)(key0 + 16 * sub) * D + lane * 16;
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
              const uint32_t q = lane + 32 * i;
              const uint32_t at = side ? q / (D / 4) * (4 * D) + v_piece<D>(q / (D / 4), q % (D / 4)) * 16 : q / (D / 16) * D + k_piece<D>(q / (D / 16), q % (D / 16)) * 16;
              copy16(to + side * (S::KS * D) + sub * (16 * D) + at, from + i * 512);
            }
          }
          if (lane < 2) copy4(smem_addr(&scales[warp][slot][lane][sub]), (lane ? cache.v_scale : cache.k_scale) + scale_at + ((key0 + 16 * sub) >> block_log2));
        }
      }
      copies_commit();
    };
    if (appends && kv == 0 && threadIdx.x == 0) kv8_note(cache, b, s.held, s.L);
    if (fills) append_filled<D>(a, b, kv, s.held, s.L);
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; i++) issue(tile + i, i);
    if (appends && !fills) {  // rows of the open block, which nobody reads in this call: nothing waits for them
      const int64_t to = ((unit * 2 + kv8_slot(cache, b, s.held, s.held >> block_log2)) * cache.block + (s.held & (cache.block - 1))) * D;
      for (int i = (int)threadIdx.x; i < 2 * s.brought * (D / 8); i += WARPS * 32) {
        const int side = i & 1, row = (i >> 1) / (D / 8), col = (i >> 1) % (D / 8) * 8;
        const uint16_t *const from = side ? a.v + b * a.v_seq + row * a.v_token + kv * a.v_head : a.k + b * a.k_seq + row * a.k_token + kv * a.k_head;
        *reinterpret_cast<uint4 *>((side ? cache.v_tail : cache.k_tail) + to + row * D + col) = *reinterpret_cast<const uint4 *>(from + col);
      }
    }

    // ---- the rows of this lane: n and n + 8 of each 16
    const int t_first = row0 / a.group, t_last = min((row0 + rows - 1) / a.group, s.brought - 1);
    const int prefix = a.prefix ? a.prefix[b] : 0;
    int lo_most, hi_least, unused;
    visible_keys(s.held + t_last, s.L, prefix, a.window, a.causal, lo_most, unused);
    visible_keys(s.held + t_first, s.L, prefix, a.window, a.causal, unused, hi_least);
    Rows<MT> r;
    r.L = s.L, r.prefix = prefix;
    State<D, MT> st;
    uint32_t q[MT][D / 16][4];
    const uint16_t *qrow[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      uint4 raw[2][D / 64][2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = 16 * mt + 8 * h + (int)n, t = (row0 + row) / a.group, head = kv * a.group + (row0 + row) % a.group;
        const bool real = row < rows && t < s.brought;
        qrow[mt][h] = real ? a.q + b * a.q_seq + t * a.q_token + head * a.q_head : nullptr;
        r.i[mt][h] = real ? s.held + t : -1;
        r.slope[mt][h] = real && a.slopes ? a.slopes[head] * LOG2E : 0.0f;
        st.m[mt][h] = NOTHING, st.d[mt][h] = st.l[mt][h] = 0.0f;
        uint32_t most = 0;
#pragma unroll
        for (int g = 0; g < D / 64; g++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            raw[h][g][i] = real ? *reinterpret_cast<const uint4 *>(qrow[mt][h] + 64 * g + 16 * c + 8 * i) : make_uint4(0, 0, 0, 0);
            const uint32_t u[4] = {raw[h][g][i].x, raw[h][g][i].y, raw[h][g][i].z, raw[h][g][i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) most = max(most, max((u[e] << 16) & 0x7FFFFFFFu, u[e] & 0x7FFF0000u));
          }
        most = max(most, __shfl_xor_sync(BN_FULL, most, 1));
        most = max(most, __shfl_xor_sync(BN_FULL, most, 2));
        const int e = min(max((int)(most >> 23), 1), 253);  // exponent of the row's largest value
        const float down = __uint_as_float((uint32_t)(254 - e) << 23), up = __uint_as_float((uint32_t)e << 23);
        r.factor[mt][h] = (a.cap > 0.0f ? a.scale * (2.0f * LOG2E / a.cap) : a.scale * LOG2E) * up;
#pragma unroll
        for (int g = 0; g < D / 64; g++)
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const uint4 u = raw[h][g][w >> 1];
            const uint32_t p0 = w & 1 ? u.z : u.x, p1 = w & 1 ? u.w : u.y;
            q[mt][4 * g + w][h] = pack_f16(__uint_as_float(p0 << 16) * down, __uint_as_float(p0 & 0xFFFF0000u) * down);
            q[mt][4 * g + w][2 + h] = pack_f16(__uint_as_float(p1 << 16) * down, __uint_as_float(p1 & 0xFFFF0000u) * down);
          }
      }
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) st.o[mt][t][e] = 0.0f;
    }

    // ---- full blocks
    int slot = 0;
    for (int t = tile; t < codes_end; t++) {
      copies_wait<S::STAGES - 2>();
      __syncwarp();  // this tile's copies of all lanes are there, and the slot of the tile before is read
      issue(t + S::STAGES - 1, slot == 0 ? S::STAGES - 1 : slot - 1);
      const uint32_t at = ring + slot * S::STAGE_BYTES;
      const int first = key_of(t), end = t < s.quant ? s.split : s.full;
      if (first < end) {
        constexpr int P = S::P;
        float x[P][MT][2][4] = {};
        PieceOf16 piece[P];
#pragma unroll
        for (int g = 0; g < D / 64; g++)
#pragma unroll
          for (int sub = 0; sub < P; sub++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint32_t key = 16 * sub + 4 * (n >> 1) + 2 * j + (n & 1);
              const uint4 w4 = lds16(at + key * D + k_piece<D>(key, 4 * g + c) * 16);
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t b0 = codes_f16<KIND, false>(w[e]), b1 = codes_f16<KIND, true>(w[e]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) mma_f16(x[sub][mt][j], q[mt][4 * g + e], b0, b1);
              }
            }
#pragma unroll
        for (int sub = 0; sub < P; sub++) {
          const float vscale = scales[warp][slot][1][sub];
          float vlog;
          asm("lg2.approx.f32 %0, %1;" : "=f"(vlog) : "f"(vscale));
          const int key0 = first + 16 * sub;
          piece[sub] = {key0, end, scales[warp][slot][0][sub], vscale, vlog, key0 < lo_most || key0 + 16 > min(hi_least, end)};
        }
        weigh<D, MT, P, PLAIN>(a, x, r, st, piece);
#pragma unroll
        for (int sub = 0; sub < P; sub++) {
          uint32_t p[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int f = 0; f < 4; f++) p[mt][f] = pack_f16(x[sub][mt][f >> 1][2 * (f & 1)], x[sub][mt][f >> 1][2 * (f & 1) + 1]);
          const uint32_t vat = at + S::KS * D + (4 * sub + c) * (4 * D);
#pragma unroll
          for (int half = 0; half < (D + 127) / 128; half++)
#pragma unroll
            for (int i = 0; i < (D == 64 ? 2 : 4); i++) {
              const uint4 w4 = lds16(vat + v_piece<D>(c, 32 * half + (D == 64 ? 2 : 4) * n + i) * 16);
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t b0 = codes_f16<KIND, false>(w[e]), b1 = codes_f16<KIND, true>(w[e]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) mma_f16(st.o[mt][16 * half + 4 * i + e], p[mt], b0, b1);
              }
            }
        }
      }
      slot = slot + 1 == S::STAGES ? 0 : slot + 1;
    }
    // ---- the open block
    if (tile_end == s.tiles && s.L > s.full) {
      const int64_t tail_at = ((unit * 2 + kv8_slot(cache, b, s.held, s.full / cache.block)) * cache.block - s.full) * D;
      OpenRows rows{cache.k_tail + tail_at, cache.v_tail + tail_at, nullptr, nullptr, a.k_token, a.v_token, D, s.L};
      if (a.k) rows.from = s.held, rows.k = a.k + b * a.k_seq + kv * a.k_head - s.held * a.k_token, rows.v = a.v + b * a.v_seq + kv * a.v_head - s.held * a.v_token;
      for (int key0 = s.full + 16 * (int)warp; key0 < s.L; key0 += 16 * WARPS) open_block<D, MT, PLAIN>(a, qrow, rows, s.L, key0, r, st);
    }

    // ---- the warps' results together
    copies_wait<0>();
    __syncthreads();
    float *const join = reinterpret_cast<float *>(attend_smem);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float l = st.l[mt][h];
        l += __shfl_xor_sync(BN_FULL, l, 1);
        l += __shfl_xor_sync(BN_FULL, l, 2);
        const int row = 16 * mt + 8 * h + (int)n;
        if (c == 0) join_m[warp][row] = st.m[mt][h], join_d[warp][row] = st.d[mt][h], join_l[warp][row] = l;
        float *const to = join + (warp * S::ROWS + row) * (D + 4);
        constexpr int RUN = D == 64 ? 8 : 16;  // neighbouring dimensions of a column
#pragma unroll
        for (int t = 0; t < NT; t += 4)
#pragma unroll
          for (int e = 0; e < 2; e++) *reinterpret_cast<float4 *>(to + (t / RUN) * 128 + (2 * c + e) * RUN + t % RUN) = make_float4(st.o[mt][t][2 * h + e], st.o[mt][t + 1][2 * h + e], st.o[mt][t + 2][2 * h + e], st.o[mt][t + 3][2 * h + e]);
      }
    __syncthreads();
    const bool whole = tile == 0 && tile_end == s.tiles;
    float *const part = a.parts + ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * S::PART;
    for (int i = (int)threadIdx.x; i < rows * (D / 4); i += WARPS * 32) {
      const int row = i / (D / 4), col = i % (D / 4) * 4;
      float m = join_m[0][row], l = 0.0f, o[4] = {};
#pragma unroll
      for (int w = 1; w < WARPS; w++) m = fmaxf(m, join_m[w][row]);
      float d = (m - join_m[0][row]) + join_d[0][row];
#pragma unroll
      for (int w = 1; w < WARPS; w++) d = fminf(d, (m - join_m[w][row]) + join_d[w][row]);
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float f = ex2(d - ((m - join_m[w][row]) + join_d[w][row]));
        const float4 v = *reinterpret_cast<const float4 *>(join + (w * S::ROWS + row) * (D + 4) + col);
        l = fmaf(ex2(join_m[w][row] - m), join_l[w][row], l);
        o[0] = fmaf(f, v.x, o[0]), o[1] = fmaf(f, v.y, o[1]), o[2] = fmaf(f, v.z, o[2]), o[3] = fmaf(f, v.w, o[3]);
      }
      if (whole) {
        const int t = (row0 + row) / a.group, head = kv * a.group + (row0 + row) % a.group;
        if (t < s.brought) {
          *reinterpret_cast<uint2 *>(a.out + b * a.o_seq + t * a.o_token + head * a.o_head + col) = quotients(make_float4(o[0], o[1], o[2], o[3]), l, d);
        } else if (a.zero_rest) {
          *reinterpret_cast<uint2 *>(a.out + b * a.o_seq + t * a.o_token + head * a.o_head + col) = make_uint2(0, 0);
        }
      } else {
        *reinterpret_cast<float4 *>(part + row * D + col) = make_float4(o[0], o[1], o[2], o[3]);
        if (col == 0) part[S::ROWS * D + row] = m, part[S::ROWS * (D + 1) + row] = d, part[S::ROWS * (D + 2) + row] = l;
      }
    }
    if (!whole && a.join_here) {  // the last block of this sequence and head joins
      const int64_t from = x - tile;
      const int64_t left = from / share, right = (from + s.tiles - 1) / share;
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t ticket = atomicAdd(cache.tickets + unit, 1u);
        last_ticket = ticket == (uint32_t)(right - left);
        if (last_ticket) cache.tickets[unit] = 0, __threadfence();
      }
      __syncthreads();
      if (last_ticket) join_parts<D, MT>(a, b, kv, rows, s.brought, left, (int)(right - left) + 1, from != left * share);
    }
    x += tile_end - tile;
    if (x >= x_end) return;
    __syncthreads();  // the join's shared memory is the ring's
    first = false, tile = 0;
    if (++hr == per_seq) {
      hr = 0;
      do s = span_of(a, ++b, S::TILE);
      while (s.tiles == 0);
    }
  }
}

// Joins what blocks left of a sequence and head that was cut, where there are several groups of rows or may be many parts. A
// block per query row: a thread has four dimensions of every few parts.
constexpr int JOIN_THREADS = 256;

template <int D, int MT>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ AttendArgs a) {
  using S = Shape<D, MT>;
  constexpr int COLS = D / 4, GROUPS = JOIN_THREADS / COLS;
  __shared__ float tops[JOIN_THREADS / 32], least[JOIN_THREADS / 32], weights[16];
  __shared__ float4 sums[JOIN_THREADS];
  const int all_rows = a.group * a.tokens, per_seq = (int)a.c.kv_heads * a.row_groups;
  const int unit = (int)(blockIdx.x / (unsigned)all_rows), r = (int)(blockIdx.x % (unsigned)all_rows);
  const int64_t b = unit / (int)a.c.kv_heads;
  const int kv = unit % (int)a.c.kv_heads, hr = kv * a.row_groups + r / S::ROWS, row = r % S::ROWS;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t before = a.plan[b], tiles = a.plan[b + 1] - before, share = a.plan[a.c.batch + 1];
  const int64_t from = before * per_seq + hr * tiles, to = from + tiles;
  // (blocks and tiles of a launch both count to less than 2^53: doubles divide them, and the products check)
  int64_t first = (int64_t)((double)from / (double)share);
  if (first * share > from) first--;
  if ((first + 1) * share <= from) first++;
  const int t = r / a.group, head = kv * a.group + r % a.group;
  uint16_t *const out = a.out + b * a.o_seq + t * a.o_token + head * a.o_head;
  if (tiles == 0 || (first + 1) * share >= to) return;  // nothing, or one block's, which wrote the output
  int parts = 1;
  while ((first + parts) * share < to) parts += max(1, (int)((to - (first + parts) * share) / share));
  auto part_of = [&](int p) { return a.parts + ((first + p) * 2 + (p == 0 && from != first * share ? 1 : 0)) * S::PART; };
  float m = NOTHING;
  for (int p = (int)threadIdx.x; p < parts; p += JOIN_THREADS) m = fmaxf(m, part_of(p)[S::ROWS * D + row]);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(BN_FULL, m, d));
  if (lane_id() == 0) tops[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JOIN_THREADS / 32; w++) m = fmaxf(m, tops[w]);
  float d = CUDART_INF_F;
  for (int p = (int)threadIdx.x; p < parts; p += JOIN_THREADS) d = fminf(d, (m - part_of(p)[S::ROWS * D + row]) + part_of(p)[S::ROWS * (D + 1) + row]);
#pragma unroll
  for (int k = 16; k; k >>= 1) d = fminf(d, __shfl_xor_sync(BN_FULL, d, k));
  if (lane_id() == 0) least[threadIdx.x >> 5] = d;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JOIN_THREADS / 32; w++) d = fminf(d, least[w]);
  const int g = (int)threadIdx.x / COLS, col = (int)threadIdx.x % COLS * 4;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 4
  for (int p = g; p < parts; p += GROUPS) {
    const float *const part = part_of(p);
    const float pm = part[S::ROWS * D + row], f = ex2(d - ((m - pm) + part[S::ROWS * (D + 1) + row]));
    const float4 v = *reinterpret_cast<const float4 *>(part + row * D + col);
    l = fmaf(ex2(pm - m), part[S::ROWS * (D + 2) + row], l);
    o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
  }
  sums[threadIdx.x] = o;
  if (col == 0) weights[g] = l;
  static_assert(GROUPS <= 16, "");
  __syncthreads();
  if (g) return;
  for (int k = 1; k < GROUPS; k++) {
    const float4 v = sums[(int)threadIdx.x + k * COLS];
    o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w, l += weights[k];
  }
  int held, brought;
  kv8_tokens(a.c, a.counts, a.tokens, b, held, brought);
  if (t < brought) {
    *reinterpret_cast<uint2 *>(out + col) = quotients(o, l, d);
  } else if (a.zero_rest) {
    *reinterpret_cast<uint2 *>(out + col) = make_uint2(0, 0);
  }
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// Blocks of a launch, and bytes of its workspace.
struct Plan {
  int mt, row_groups, blocks;
  bool join_here;
  uint64_t plan_bytes, bytes;
};
template <int D>
Plan plan_of(const bn_kv8 *c, int64_t tokens, int64_t heads) {
  Plan p;
  const int64_t rows = heads / c->kv_heads * tokens;
  p.mt = D < 256 && rows > 16 ? 2 : 1;
  p.row_groups = (int)((rows + 16 * p.mt - 1) / (16 * p.mt));
  const int resident = (D == 64 && p.mt == 1) ? 4 : (p.mt * D <= 128) ? 3 : 2;
  const int tile = p.mt == 1 ? Shape<D, 1>::TILE : Shape<D, 2 - (D == 256)>::TILE;
  const int64_t most = c->batch * c->kv_heads * p.row_groups * ((c->max_seq + tile - 1) / tile + 1);
  const int64_t full = (int64_t)sm_count() * resident;
  p.blocks = (int)(most < full ? most : full);
  // A kernel for the join costs a launch, the block that finishes last a chain of loads that grows with the parts. One sequence
  // of 8 heads, here / kernel: 300 tokens, 6 parts at most, 13.5 / 15.4 us a call (the host's; 12.0 / 11.4 in a graph); in a graph
  // 1000 tokens 13.9 / 11.9, 130000, 55 parts, 93 / 71. 64 sequences: 300 tokens 30 / 35, 10000 258 / 262. Eight blocks a head: few
  // parts, or many heads, of which few are cut.
  p.join_here = p.row_groups == 1 && p.blocks <= 8 * c->batch * c->kv_heads;
  p.plan_bytes = ((uint64_t)(c->batch + 2) * 8 + 127) / 128 * 128;
  p.bytes = p.plan_bytes + (uint64_t)p.blocks * 2 * (16 * p.mt * (D + 3)) * 4;
  return p;
}
Plan plan_of(const bn_kv8 *c, int64_t tokens, int64_t heads) { return c->D == 64 ? plan_of<64>(c, tokens, heads) : c->D == 128 ? plan_of<128>(c, tokens, heads) : plan_of<256>(c, tokens, heads); }

template <int D, int KIND, int MT, bool PLAIN>
int attend_launch(const AttendArgs &a, cudaStream_t stream) {
  using S = Shape<D, MT>;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)a.blocks), cfg.blockDim = dim3(WARPS * 32), cfg.dynamicSmemBytes = S::SMEM, cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = 1;
  BN_CUDA(allow_smem(attend_kernel<D, KIND, MT, PLAIN>, S::SMEM));
  BN_CUDA(cudaLaunchKernelEx(&cfg, attend_kernel<D, KIND, MT, PLAIN>, a));
  if (a.join_here) return launched("attend_kernel");
  cfg.gridDim = dim3((unsigned)(a.c.batch * a.heads * a.tokens)), cfg.blockDim = dim3(JOIN_THREADS), cfg.dynamicSmemBytes = 0;
  BN_CUDA(cudaLaunchKernelEx(&cfg, join_kernel<D, MT>, a));
  return launched("attend_kernel");
}

template <int KIND, bool PLAIN>
int attend_kind(const AttendArgs &a, int mt, cudaStream_t s) {
  if (a.c.D == 64) return mt == 1 ? attend_launch<64, KIND, 1, PLAIN>(a, s) : attend_launch<64, KIND, 2, PLAIN>(a, s);
  if (a.c.D == 128) return mt == 1 ? attend_launch<128, KIND, 1, PLAIN>(a, s) : attend_launch<128, KIND, 2, PLAIN>(a, s);
  return attend_launch<256, KIND, 1, PLAIN>(a, s);
}

// Whether many rows go to the other kernel (kv8_chunk.cu), which reads a sequence's keys once for 256 rows (128 with heads
// of 256), but by one block from end to end: it wins where there are groups of 32 rows to fill the card several times over with
// this kernel's blocks. Where the two cross depends on the lengths, which the host does not know: near 50 groups at 500 keys,
// near 250 at 9000 and more; 100 lies between. us, this kernel / the other, 8 heads of 128 in groups of 4, by groups:
// 500 keys 64: 36 / 26, 128: 47 / 26; 9000 keys 64: 78 / 233, 128: 130 / 243, 256: 232 / 250, 504: 438 / 269.
bool chunk_wins(const bn_kv8 *c, int64_t tokens, int64_t heads) {
  const int64_t rows = heads / c->kv_heads * tokens, units = c->batch * c->kv_heads, per_block = c->D == 256 ? 128 : 256;
  const int64_t groups = (rows + 31) / 32, waves = (units * ((rows + per_block - 1) / per_block) + sm_count() - 1) / sm_count();
  return rows > 32 && units * groups > 100 * waves;
}

bool attend_sizes(const bn_kv8 *c, int64_t tokens, int64_t heads) { return tokens >= 0 && tokens <= 0x3FFFFFFF && heads >= 1 && heads <= 4096 && heads % c->kv_heads == 0; }

}  // namespace

int kv8_attend_status(int *status) {
  BN_CUDA(cudaMemcpyFromSymbol(status, g_attend_error, sizeof(int)));
  return BN_OK;
}

int kv8_attend_status_reset() {
  const int zero = 0;
  BN_CUDA(cudaMemcpyToSymbol(g_attend_error, &zero, sizeof(int)));
  return BN_OK;
}

}  // namespace bn

extern "C" uint64_t bn_kv8_workspace(const bn_kv8 *c, int64_t tokens, int64_t heads) {
  if (bn::kv8_refusal(c) || !bn::attend_sizes(c, tokens, heads) || tokens == 0) return 0;
  return bn::chunk_wins(c, tokens, heads) ? 0 : bn::plan_of(c, tokens, heads).bytes;
}

extern "C" int bn_kv8_attend(const bn_kv8 *c, const uint16_t *q, int64_t q_seq, int64_t q_token, int64_t q_head, const uint16_t *k, int64_t k_seq, int64_t k_token, int64_t k_head, const uint16_t *v, int64_t v_seq, int64_t v_token, int64_t v_head, int64_t tokens, int64_t heads, const int32_t *counts, const int32_t *prefix, const bn_scores *scores, uint16_t *out, int64_t o_seq, int64_t o_token, int64_t o_head, int zero_rest, void *workspace, uint64_t workspace_bytes, void *stream) {
  if (const char *why = bn::kv8_refusal(c)) return bn::refuse("bn_kv8_attend", why);
  if (!bn::attend_sizes(c, tokens, heads)) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: bad size (query heads have to be a multiple of the cache's heads)");
  if (!scores || (tokens && (!q || !out)) || !k != !v) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: null pointer");
  if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_seq | q_token | q_head | o_seq | o_token | o_head) & 7) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: rows have to start on 16 bytes");
  if (const char *why = bn::scores_refusal(scores)) return bn::refuse("bn_kv8_attend", why);
  if (tokens == 0) return BN_OK;
  const bool chunk = bn::chunk_wins(c, tokens, heads);
  const bn::Plan p = bn::plan_of(c, tokens, heads);
  if (chunk && ((tokens > 1 && !q_token) || (heads > 1 && !q_head) || (c->batch > 1 && !q_seq) || (q_seq | q_token | q_head) < 0)) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: query rows have to lie apart");
  if (chunk) {
    if (k)
      if (const int e = bn_kv8_append(c, k, k_seq, k_token, k_head, v, v_seq, v_token, v_head, tokens, counts, stream)) return e;
    return bn::kv8_chunk(c, q, q_seq, q_token, q_head, tokens, heads, counts, prefix, scores, out, o_seq, o_token, o_head, zero_rest, (cudaStream_t)stream);
  }
  if (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < p.bytes) return bn::fail(BN_ERR_CAPACITY, "bn_kv8_attend: the workspace is smaller than bn_kv8_workspace says, or not on 16 bytes");
  if (c->batch * heads * tokens > 0x7FFFFFFF) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: too many rows for one call");
  if (k && (((uintptr_t)k | (uintptr_t)v) & 15 || (k_seq | k_token | k_head | v_seq | v_token | v_head) & 7)) return bn::fail(BN_ERR_ARG, "bn_kv8_attend: rows have to start on 16 bytes");
  if (k && (p.row_groups > 1 || tokens > 16)) {  // (16 tokens fill one block at most)
    if (const int e = bn_kv8_append(c, k, k_seq, k_token, k_head, v, v_seq, v_token, v_head, tokens, counts, stream)) return e;
    k = v = nullptr;
  }
  bn::AttendArgs a{*c, q, out, q_seq, q_token, q_head, o_seq, o_token, o_head, counts, prefix, scores->slopes, k, v, k_seq, k_token, k_head, v_seq, v_token, v_head, (int)tokens, (int)heads, (int)(heads / c->kv_heads), (int)scores->window, scores->causal, zero_rest, scores->scale, scores->softcap, (int64_t *)workspace, (float *)((uint8_t *)workspace + p.plan_bytes), p.row_groups, p.blocks, p.join_here};
  const cudaStream_t s = (cudaStream_t)stream;
  if (scores->softcap == 0.0f && !scores->slopes) return c->kind == BN_KV8_INT8 ? bn::attend_kind<BN_KV8_INT8, true>(a, p.mt, s) : bn::attend_kind<BN_KV8_E4M3, true>(a, p.mt, s);
  return c->kind == BN_KV8_INT8 ? bn::attend_kind<BN_KV8_INT8, false>(a, p.mt, s) : bn::attend_kind<BN_KV8_E4M3, false>(a, p.mt, s);
}
