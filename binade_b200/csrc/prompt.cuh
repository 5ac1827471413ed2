// Attention of many query rows: of prompts (packed documents, every query over the keys of its own document: attention.cu)
// and of chunks of new tokens over an 8-bit cache (kv8_chunk.cu).
//
//   S = Q K^T, P = 2^(S scale log2(e) - m), O += P V, row sums of P; O / sum at the end, m a row's running maximum
//
// on the 5th-generation tensor cores (tcgen05): a block has 256 query rows as two tiles of 128 (one tile for heads of
// 256), S and O in tensor memory. Rows are (token, query head of the key head's group), so that a group shares
// the keys that a block reads. Warps by role:
//   a warp copies Q, K and V tiles by TMA (128-byte swizzle) into a ring
//   a warp issues the MMAs: for tile i in turn P_i V of the last keys, then Q_i K^T of the next, so that one
//     tile's softmax runs beside the other's products (heads of 256: two S buffers do the same for one tile)
//   four warps a tile do the softmax, a row a thread: S out of tensor memory, P back over it in BF16 (rounded by up
//     to 2^-8 of a weight; the sum takes it before that) as the second product's first operand
// m moves only when a row's maximum passes it by 8 (weights up to 2^8 are as good in BF16 and fp32): most
// tiles leave O where it is. V is the MMA's B by columns, as it lies in memory: nothing is transposed.
// Keys that no row of the block sees are not read. A row whose sums are not finite is computed again by one warp over its
// visible keys alone: 0 times a masked infinity or NaN is how it gets there, or the values themselves.
//
// Over a cache four more warps stand where the TMA of K and V was: they turn codes into BF16 (exact: both kinds
// fit its 8 bits) straight into the ring, the open block's tokens as they are. The scales stay apart: K's multiply
// the scores of their 16 keys or more, V's the weights, before these are rounded.
//
// Measured: 8192 tokens, 32 / 8 heads of 128, causal: 552 us a call among others (under the power cap), 1.00 PFLOP/s, 60 % of
// the measured cuBLAS rate; 481 us at full clocks. Tensor pipe 53 %, ex2's 53 %: a tile's S, softmax, P and O in a row are twice as
// long as either, and two tiles are what tensor memory holds. Chunk of 2 x 500 tokens over up to 9000, int8: 303 us a call, 260 at
// full clocks. 5003 tokens in 11 documents, heads of 256, cap, window: 76 us; 6001 in 7, heads of 64, bias: 58 us: blocks of a few
// key tiles, one an SM, whose start and end nothing hides (tensor pipe 20 and 13 %, ex2's 31 and 27 %).
//
// Every wait is bounded: a wait that gives up sets the device status, and the block still ends.
#pragma once

#include "kv8.cuh"
#include "tcgen05.cuh"

namespace bn {

namespace {

__device__ int g_prompt_error;  // 1: a bounded wait gave up; 2: the shared window did not fit

struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;  // elements
  const int32_t *offsets, *prefix;
  const float *slopes;
  int T, docs, heads, kv_heads;
  int window, causal, zero_rest;
  float scale, cap;
  // over a cache: its new tokens (up to `tokens` of each sequence); k and v above are not used
  bn_kv8 c;
  const int32_t *counts;
  int tokens, tiles;  // tiles: of a sequence's tokens
  int64_t q_seq, o_seq;
};

constexpr float NOTHING = -3.402823466e38f;  // m before the first visible key: finite, so that -inf (a masked score, or a key's own) less m stays that
constexpr int FROM_BF16 = -1;  // SRC: where keys and values come from; else the kind of a cache's codes

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

// Key or value row j of a sequence in the cache, as it stands for itself.
template <int E, int KIND>
__device__ __forceinline__ void load_cached(const bn_kv8 &c, bool values, int64_t unit, int j, int full, int slot, float (&x)[E]) {
  const int D = E * 32, d0 = (int)lane_id() * E;
  if (j >= full) {
    load_row<E>((values ? c.v_tail : c.k_tail) + ((unit * 2 + slot) * c.block + j - full) * D + d0, x);
    return;
  }
  const float scale = (values ? c.v_scale : c.k_scale)[unit * (c.rows / c.block) + j / c.block];
  const uint8_t *const at = values ? c.v + ((unit * c.rows + (j & ~3)) * D + 4 * d0 + (j & 3)) : c.k + (unit * c.rows + j) * D + d0;
#pragma unroll
  for (int e = 0; e < E; e++) x[e] = kv8_code<KIND>(at[values ? 4 * e : e]) * scale;
}

// What a block works on: rows row0 .. of a document's (or sequence's) n tokens times the group's heads, for one key head.
// The tokens are from .. of the packed ones (of sequence b's, over a cache); the first has position `held` of L.
struct Piece {
  int64_t b;
  int from, held, n, L, row0, prefix;
};

// One query of one head by a warp, keys one after the other; a lane has E = D / 32 neighbouring dimensions.
// Two passes, so that the values are weighted by shares of one: no sum of theirs can pass the largest of them. Writes
// dimensions from .. to - 1, which are the calling warp's: the row's other half may be another's.
template <int D, int SRC>
__device__ __noinline__ void attend_row(const PromptArgs &a, const Piece &p, int t, int head, int from, int to) {
  constexpr int E = D / 32;
  const uint32_t lane = lane_id();
  const int kv = head / (a.heads / a.kv_heads), i = p.held + t;
  const int64_t unit = p.b * a.kv_heads + kv;
  const int full = SRC == FROM_BF16 ? 0 : p.L / a.c.block * a.c.block, slot = SRC == FROM_BF16 ? 0 : kv8_slot(a.c, p.b, p.held, p.L / a.c.block);
  int lo, hi;
  visible_keys(i, p.L, p.prefix, a.window, a.causal, lo, hi);
  float q[E], o[E] = {}, m = NOTHING, l = 0.0f;
  load_row<E>(a.q + p.b * a.q_seq + (p.from + t) * a.q_token + head * a.q_head + lane * E, q);
  const float slope = a.slopes ? a.slopes[head] * LOG2E : 0.0f;
  auto row = [&](bool values, int j, float (&x)[E]) {
    if constexpr (SRC == FROM_BF16) load_row<E>(values ? a.v + (int64_t)(p.from + j) * a.v_token + kv * a.v_head + lane * E : a.k + (int64_t)(p.from + j) * a.k_token + kv * a.k_head + lane * E, x);
    else load_cached<E, SRC>(a.c, values, unit, j, full, slot, x);
  };
  auto score = [&](int j) {
    float x[E], dot = 0.0f;
    row(false, j, x);
#pragma unroll
    for (int e = 0; e < E; e++) dot = fmaf(q[e], x[e], dot);
#pragma unroll
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(BN_FULL, dot, d);
    float s = dot * a.scale;
    s = a.cap > 0.0f ? capped_wide(s * (2.0f * LOG2E / a.cap), a.cap * LOG2E) : s * LOG2E;
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
    const float w = ex2(score(j) - m) * inv;
    row(true, j, x);
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = fmaf(w, x[e], o[e]);
  }
  uint16_t *const out = a.out + p.b * a.o_seq + (p.from + t) * a.o_token + head * a.o_head + lane * E;
  if ((int)lane * E < from || (int)lane * E >= to) return;
#pragma unroll
  for (int e = 0; e < E; e++) out[e] = f32_to_bf16_bits(o[e]);
}

// Warps 0 .. 7 do the softmax; the next eight turn codes into BF16 where there are codes; then the warp that copies and
// the one that issues products, of a group of four. Registers move from the others to the softmax: the groups' shares add
// up to what the block was launched with (3 x 168 or 5 x 96).
template <int SRC>
struct Roles {
  static constexpr int WARPS = SRC == FROM_BF16 ? 12 : 20, TMA_WARP = WARPS - 4, MMA_WARP = WARPS - 3;
  static constexpr int SOFTMAX_REGS = SRC == FROM_BF16 ? 208 : 168, OTHER_REGS = SRC == FROM_BF16 ? 88 : 48;
};
constexpr int SOFTMAX_WARPS = 8, CODE_WARP = 8, CODE_WARPS = 8;
constexpr int SCALES_AHEAD = 8;  // key tiles whose scales the block holds: more than the ring can be ahead of the softmax
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr uint32_t PROMPT_SPINS = 1u << 22;
constexpr float RISE = 8.0f;                   // how far, in powers of two, a row's maximum may pass m

template <int D>
struct Tiles {
  static constexpr int NQ = D == 256 ? 1 : 2;        // query tiles of 128 rows
  static constexpr int ROWS = 128 * NQ;
  static constexpr int BN = D == 256 ? 64 : 128;     // keys of a step
  static constexpr int STAGES = D == 64 ? 8 : 4;     // ring slots of a K or V tile
  static constexpr uint32_t TILE_BYTES = BN * D * 2, Q_BYTES = 128 * D * 2;
  static constexpr uint32_t RAW_BYTES = BN * D;      // a tile of codes as they lie: two of them wait for the warps that turn them into BF16
  static constexpr uint32_t BARS = 384, SCALES = SCALES_AHEAD * 2 * (BN / 16) * 4;
  static constexpr uint32_t TOLD = NQ == 1 ? 2048 : 0;  // two halves' maxima, for two tiles
  static constexpr uint32_t WINDOW = NQ * Q_BYTES + STAGES * TILE_BYTES + BARS + SCALES + TOLD, WINDOW_CODES = WINDOW + 2 * RAW_BYTES;
  // with room to start on 1024 bytes; not where all of a block's shared memory is taken (the window starts on 1024
  // bytes when there is no static shared memory; a block whose window does not is refused)
  static constexpr uint32_t SMEM = WINDOW + 1024, SMEM_CODES = D == 256 ? WINDOW_CODES : WINDOW_CODES + 1024;
  static_assert(SMEM_CODES <= 227 * 1024, "a block's shared memory");
  static constexpr uint32_t S_AT = 0, O_AT = 2 * BN;  // tensor memory columns: two S buffers, then the sums
};

__device__ __forceinline__ bool prompt_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < PROMPT_SPINS; i++) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  atomicExch(&g_prompt_error, 1);
  return false;
}
__device__ __forceinline__ bool prompt_wait_warp(uint32_t bar, uint32_t parity) { return __all_sync(BN_FULL, prompt_wait(bar, parity)); }

// True in one lane of the warp, all of which has to get here: ahead of any wait.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// Slot s of the launch: document n owns slots floor(offsets[n] Gp / ROWS) + n and on, at least as many as it has
// tiles, so that no prefix sum over the documents is needed. False: the slot is empty.
template <int ROWS>
__device__ __forceinline__ bool piece_of(const PromptArgs &a, int group, int64_t slot, Piece &p) {
  int doc = 0;
  p.b = 0, p.from = 0, p.held = 0, p.n = p.L = a.T;
  int64_t first = 0;
  if (a.offsets) {
    auto start = [&](int n) { return (int64_t)min(max(a.offsets[n], 0), a.T) * group / ROWS + n; };
    int lo = 0, hi = a.docs;  // the last n with start(n) <= slot, by a warp's 32 looks at a time
    while (lo < hi) {
      const int step = (hi - lo + 31) / 32, look = lo + step * ((int)lane_id() + 1);
      const uint32_t below = __ballot_sync(BN_FULL, look <= hi && start(look) <= slot);
      const int some = __popc(below);
      hi = min(hi, lo + step * (some + 1) - 1), lo += step * some;
    }
    if (lo >= a.docs) return false;
    doc = lo, first = start(lo);
    p.from = min(max(a.offsets[doc], 0), a.T);
    p.n = p.L = min(max(a.offsets[doc + 1], 0), a.T) - p.from;
  }
  const int64_t row0 = (slot - first) * ROWS;
  if (slot < first || row0 >= (int64_t)p.L * group) return false;  // (a falling offset: L below 0)
  p.row0 = (int)row0;
  p.prefix = a.prefix ? a.prefix[doc] : 0;
  return true;
}

// The same over a cache: slots of a sequence's tokens, one sequence after the other. n: the real ones.
template <int ROWS>
__device__ __forceinline__ bool chunk_of(const PromptArgs &a, int group, int64_t slot, Piece &p) {
  p.b = slot / a.tiles, p.from = 0, p.row0 = (int)(slot % a.tiles) * ROWS;
  kv8_tokens(a.c, a.counts, a.tokens, p.b, p.held, p.n);
  p.L = p.held + p.n;
  p.prefix = a.prefix ? a.prefix[p.b] : 0;
  return p.row0 < (int64_t)p.n * group;
}

// Two codes, of the low or the HIGH half of a word, as BF16, exactly.
template <int KIND, bool HIGH>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
  uint32_t r;
  if constexpr (KIND == KV8_INT8) {  // byte u = code + 128: (128 + the low seven bits) less 128, or 256 where the code is below 0
    const uint32_t t = __byte_perm(w, 0x43434343u, HIGH ? 0x4342 : 0x4140);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t & 0xFF7FFF7Fu), "r"((t & 0x00800080u) ^ 0x43804380u));
  } else {  // sign, exponent and mantissa in BF16's places are the value times 2^-120
    const uint32_t t = __byte_perm(w, 0u, HIGH ? 0x3424 : 0x1404);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"((t & 0x80008000u) | ((t >> 4) & 0x07F007F0u)), "r"(0x7B807B80u));
  }
  return r;
}
__device__ __forceinline__ void sts8(uint32_t at, uint2 v) { asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(v.x), "r"(v.y) : "memory"); }
__device__ __forceinline__ void sts16(uint32_t at, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts_f32(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ float lds_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ uint64_t pair_f32(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split_f32(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// PLAIN: no cap, no bias, a positive scale. Else CAP: a cap, a WIDE one beyond WIDE_CAP (a kernel of its own: beside one another
// the two ways to cap spill 300 bytes a thread).
constexpr int NO_CAP = 0, USUAL = 1, WIDE = 2;
template <int D, bool PLAIN, int CAP, int SRC>
__global__ void __launch_bounds__(Roles<SRC>::WARPS * 32, 1) prompt_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ PromptArgs a, int group_log2, int head_groups) {
  using G = Tiles<D>;
  constexpr int NQ = G::NQ, BN = G::BN, ST = G::STAGES, TMA_WARP = Roles<SRC>::TMA_WARP, MMA_WARP = Roles<SRC>::MMA_WARP;
  constexpr bool CODES = SRC != FROM_BF16;
  // Weights to the sums in two halves: worth it where the softmax is what the products wait for (us, chunk of 2 x 500 tokens
  // over 9000: 263 / 280 in one piece; 6001 tokens with a bias: 55 / 57), not where the products of the other tile would
  // start instead (8192 tokens: 540 / 477). Key tiles of 64 with two S buffers a query tile instead: 734 there, since a product
  // of half the columns takes more than half the time.
  constexpr bool HALVES = NQ == 2 && (CODES || !PLAIN);
  extern __shared__ uint8_t prompt_smem[];
  const uint32_t lane = lane_id(), warp = threadIdx.x >> 5;
  const int group = 1 << group_log2;
  const uint32_t base = (smem_addr(prompt_smem) + 1023u) & ~1023u;
  const uint32_t q_at = base, ring_at = q_at + NQ * G::Q_BYTES, bars = ring_at + ST * G::TILE_BYTES;
  const uint32_t q_full = bars, s_full = bars + 16, p_full = bars + 32, o_done = bars + 48, ring_full = bars + 64, ring_empty = ring_full + 8 * ST, scale_full = ring_empty + 8 * ST, raw_full = scale_full + 8 * SCALES_AHEAD, raw_empty = raw_full + 16, p_half = raw_empty + 16, tmem_slot = p_half + 16, scales_at = bars + G::BARS, told_at = scales_at + G::SCALES, raw_at = told_at + G::TOLD;
  if (base + (CODES ? G::WINDOW_CODES : G::WINDOW) > smem_addr(prompt_smem) + (CODES ? G::SMEM_CODES : G::SMEM)) {
    if (threadIdx.x == 0) atomicExch(&g_prompt_error, 2);
    return;
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) mm_bar_init(q_full + 8 * i, 1), mm_bar_init(s_full + 8 * i, 1), mm_bar_init(p_full + 8 * i, NQ == 2 ? 128 : 256), mm_bar_init(p_half + 8 * i, 128), mm_bar_init(o_done + 8 * i, 1);
    for (int i = 0; i < ST; i++) mm_bar_init(ring_full + 8 * i, CODES ? CODE_WARPS : 1), mm_bar_init(ring_empty + 8 * i, 1);
    for (int i = 0; i < SCALES_AHEAD; i++) mm_bar_init(scale_full + 8 * i, CODE_WARPS);
    for (int i = 0; i < 2; i++) mm_bar_init(raw_full + 8 * i, 1), mm_bar_init(raw_empty + 8 * i, CODE_WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // Barriers of S, P and O: one per query tile; with one query tile one per S buffer, O's too, since the softmax may be
  // a tile ahead of the sums: a barrier's parity tells two phases apart, not three.

  // ---- the block's rows and the key tiles that they see; the last rows of a document, which see most, come first
  const int head_group = (int)(blockIdx.x % (unsigned)head_groups), head0 = head_group << group_log2, kv = head0 / (a.heads / a.kv_heads);
  const int64_t slot = (int64_t)(gridDim.x / (unsigned)head_groups) - 1 - blockIdx.x / (unsigned)head_groups;
  Piece p{};
  bool work;
  if constexpr (CODES) work = chunk_of<G::ROWS>(a, group, slot, p);
  else work = piece_of<G::ROWS>(a, group, slot, p);
  int j0[NQ], j1[NQ], J0 = 0x7FFFFFFF, J1 = 0;  // key tiles of each query tile, of both
#pragma unroll
  for (int i = 0; i < NQ; i++) {
    const int first = (p.row0 + 128 * i) >> group_log2, last = min((p.row0 + 128 * i + 127) >> group_log2, p.n - 1);
    j0[i] = j1[i] = 0;
    if (work && first < p.n) {
      int lo, hi, other;
      visible_keys(p.held + first, p.L, p.prefix, a.window, a.causal, lo, other);
      visible_keys(p.held + last, p.L, p.prefix, a.window, a.causal, other, hi);
      j0[i] = lo / BN, j1[i] = (hi + BN - 1) / BN;
      J0 = min(J0, j0[i]), J1 = max(J1, j1[i]);
    }
  }
  J0 = min(J0, J1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

  if (warp >= TMA_WARP) {
    fewer_registers<Roles<SRC>::OTHER_REGS>();  // (by whole groups of four warps)
    if (warp == TMA_WARP) {
    // ---------------------------------------------------------------- copies
    if (elect_one() && J1 > J0) {
#pragma unroll
      for (int i = 0; i < NQ; i++)
        if (j1[i] > j0[i]) {
          mm_bar_expect_tx(q_full + 8 * i, G::Q_BYTES);
          for (int x = 0; x < D / 64; x++) tma_load_4d(q_at + i * G::Q_BYTES + x * (128 * 128), &q_map, 64 * x, head0, p.from + ((p.row0 + 128 * i) >> group_log2), (int)p.b, q_full + 8 * i);
        }
      if constexpr (!CODES) {
        int at = 0;
        bool ok = true;
        auto fetch = [&](const CUtensorMap *map, int j) {
          const int s = at % ST;
          if (at >= ST && ok) ok = prompt_wait(ring_empty + 8 * s, ((at / ST) & 1) ^ 1);
          if (!ok) return;
          mm_bar_expect_tx(ring_full + 8 * s, G::TILE_BYTES);
          for (int x = 0; x < D / 64; x++) tma_load_3d(ring_at + s * G::TILE_BYTES + x * (BN * 128), map, 64 * x, kv, p.from + j * BN, ring_full + 8 * s);
          at++;
        };
        for (int j = J0; j <= J1 && ok; j++) {  // in the order of use
          if (j < J1) fetch(&k_map, j);
          if (j > J0) fetch(&v_map, j - 1);
        }
        for (int t = max(0, at - ST); t < at; t++) prompt_wait(ring_full + 8 * (t % ST), (t / ST) & 1);  // no copy outlives the block
      } else {
        const int full = p.L / a.c.block * a.c.block;
        const int64_t unit = p.b * a.kv_heads + kv;
        int at = 0;
        bool ok = true;
        auto fetch = [&](const uint8_t *codes, int j) {  // the tile's codes: one run of bytes, as far as its blocks are full
          const int s = at % 2, key0 = j * BN;
          if (at >= 2 && ok) ok = prompt_wait(raw_empty + 8 * s, ((at / 2) & 1) ^ 1);
          if (!ok) return;
          const uint32_t bytes = (uint32_t)(min(max(full - key0, 0), BN) * D);
          mm_bar_expect_tx(raw_full + 8 * s, bytes);
          if (bytes) asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(raw_at + s * G::RAW_BYTES), "l"(codes + (unit * a.c.rows + key0) * D), "r"(bytes), "r"(raw_full + 8 * s) : "memory");
          at++;
        };
        for (int j = J0; j <= J1 && ok; j++) {
          if (j < J1) fetch(a.c.k, j);
          if (j > J0) fetch(a.c.v, j - 1);
        }
        for (int t = max(0, at - 2); t < at; t++) prompt_wait(raw_full + 8 * (t % 2), (t / 2) & 1);
      }
#pragma unroll
      for (int i = 0; i < NQ; i++)
        if (j1[i] > j0[i]) prompt_wait(q_full + 8 * i, 0);
    }
    __syncwarp();
    } else if (warp == MMA_WARP) {
    // ---------------------------------------------------------------- products
    const bool lead = elect_one();
    constexpr uint32_t S_DESC = mma_idesc(128, BN), O_DESC = mma_idesc(128, D) | MMA_B_COLUMNS;
    bool ok = true;
    int at = 0;
    auto arrived = [&]() {  // the next tile of the ring
      const int s = at % ST;
      if (ok) ok = prompt_wait_warp(ring_full + 8 * s, (at / ST) & 1);
      at++;
      return ring_at + s * G::TILE_BYTES;
    };
    auto scores = [&](int i, int j, uint32_t k_tile) {
      const int n = j - j0[i], buf = NQ == 2 ? i : n & 1;
      if (n == 0 && ok) ok = prompt_wait_warp(q_full + 8 * i, 0);
      tc_fence_after();
      if (lead && ok) {
        const uint64_t dq = smem_desc(q_at + i * G::Q_BYTES), dk = smem_desc(k_tile);
#pragma unroll
        for (int s = 0; s < D / 16; s++) mma_bf16(tmem + G::S_AT + buf * BN, dq + (s >> 2) * (128 * 128 >> 4) + (s & 3) * 2, dk + (s >> 2) * (BN * 128 >> 4) + (s & 3) * 2, S_DESC, s != 0);
        mma_commit(s_full + 8 * buf);
      }
      __syncwarp();
    };
    auto sums = [&](int i, int j, uint32_t v_tile) {
      const int n = j - j0[i], buf = NQ == 2 ? i : n & 1;
      const uint64_t dv = smem_desc_columns(v_tile, BN * 128);
      auto steps = [&](int from, int to) {
#pragma unroll
        for (int s = from; s < to; s++) mma_bf16_tmem(tmem + G::O_AT + i * D, tmem + G::S_AT + buf * BN + 8 * s, dv + s * (2048 >> 4), O_DESC, (n | s) != 0);
      };
      if constexpr (HALVES) {  // the first half of the keys while the other half's weights are made
        if (ok) ok = prompt_wait_warp(p_half + 8 * buf, n & 1);
        tc_fence_after();
        if (lead && ok) steps(0, BN / 32);
        __syncwarp();
      }
      if (ok) ok = prompt_wait_warp(p_full + 8 * buf, NQ == 2 ? n & 1 : (n >> 1) & 1);
      tc_fence_after();
      if (lead && ok) {
        steps(HALVES ? BN / 32 : 0, BN / 16);
        mma_commit(o_done + 8 * buf);
      }
      __syncwarp();
    };
    for (int j = J0; j <= J1; j++) {
      uint32_t k_tile = 0, v_tile = 0;
      const int k_slot = at % ST;
      if (j < J1) k_tile = arrived();
      if constexpr (NQ == 1) {
        if (j < J1) scores(0, j, k_tile);
      }
      const int v_slot = at % ST;
      if (j > J0) v_tile = arrived();
#pragma unroll
      for (int i = 0; i < NQ; i++) {
        if (j > j0[i] && j <= j1[i]) sums(i, j - 1, v_tile);
        if constexpr (NQ == 2) {
          if (j >= j0[i] && j < j1[i]) scores(i, j, k_tile);
        }
      }
      if (lead && ok) {  // both tiles are free when these products are done
        if (j < J1) mma_commit(ring_empty + 8 * k_slot);
        if (j > J0) mma_commit(ring_empty + 8 * v_slot);
      }
      __syncwarp();
    }
    for (int t = max(0, at - ST); t < at && ok; t++) ok = prompt_wait_warp(ring_empty + 8 * (t % ST), (t / ST) & 1);  // nor does a product
    }
  } else if (CODES && warp >= CODE_WARP) {
    fewer_registers<Roles<SRC>::OTHER_REGS>();
    // ---------------------------------------------------------------- codes to BF16
    if constexpr (CODES) {
        constexpr int THREADS = CODE_WARPS * 32, PIECES = BN * D / 16 / THREADS;  // 16-byte pieces of a tile's codes that a thread has
      const int tid = (int)threadIdx.x - CODE_WARP * 32, full = p.L / a.c.block * a.c.block;
      const int64_t unit = p.b * a.kv_heads + kv;
      const uint16_t *const k_tail = a.c.k_tail + (unit * 2 + (work ? kv8_slot(a.c, p.b, p.held, p.L / a.c.block) : 0)) * a.c.block * D, *const v_tail = a.c.v_tail + (k_tail - a.c.k_tail);
      // Where a thread's first piece lies: K sixteen dimensions of a key, V four dimensions of four keys. The next pieces lie
      // K_STEP or V_STEP keys on, a multiple of eight: the swizzle is the same.
      constexpr int K_STEP = THREADS * 16 / D, V_STEP = THREADS * 16 / D;
      static_assert(K_STEP % 8 == 0, "");
      const int k_key = tid / (D / 16), k_dim = tid % (D / 16) * 16, v_key = tid / (D / 4) * 4, v_dim = tid % (D / 4) * 4;
      const uint32_t k_to = (k_dim / 64) * (BN * 128), k_lo = k_to + swz(k_key, k_dim % 64 / 8), k_hi = k_to + swz(k_key, k_dim % 64 / 8 + 1);
      const bool k_swap = D > 64 && (tid & 4);  // lanes of the next 64 dimensions store their second half first: other banks
      uint32_t v_to[4];
#pragma unroll
      for (int r = 0; r < 4; r++) v_to[r] = (v_dim / 64) * (BN * 128) + (v_dim % 8) * 2 + swz(v_key + r, v_dim % 64 / 8);
      int at = 0;
      bool ok = true;
      auto scale_of = [&](int j) {  // of both sides, for 16 keys a thread; 1 in the open block
        const int side = tid / (BN / 16), key = j * BN + tid % (BN / 16) * 16;
        return tid < 2 * (BN / 16) && key < full ? (side ? a.c.v_scale : a.c.k_scale)[unit * (a.c.rows / a.c.block) + key / a.c.block] : 1.0f;
      };
      float scale = J0 < J1 ? scale_of(J0) : 1.0f;
      auto fetch = [&](bool values, int j) {
        const int s = at % ST, key0 = j * BN;
        const uint32_t to = ring_at + s * G::TILE_BYTES, raw = raw_at + (at % 2) * G::RAW_BYTES + tid * 16;
        const bool whole = key0 + BN <= full;
        if (ok) ok = prompt_wait_warp(raw_full + 8 * (at % 2), (at / 2) & 1);
        if (at >= ST && ok) ok = prompt_wait_warp(ring_empty + 8 * s, ((at / ST) & 1) ^ 1);
        if (!ok) return;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
          const uint32_t dst = to + i * (K_STEP * 128);
          const uint4 w = lds16(raw + i * (THREADS * 16));
          if (values) {
            const int key = key0 + v_key + i * V_STEP;
            if (whole || key < full) {  // (blocks have whole rows of four)
              const uint32_t a01 = __byte_perm(w.x, w.y, 0x5140), b01 = __byte_perm(w.x, w.y, 0x7362), a23 = __byte_perm(w.z, w.w, 0x5140), b23 = __byte_perm(w.z, w.w, 0x7362);
              sts8(dst + v_to[0], make_uint2(codes_bf16<SRC, false>(a01), codes_bf16<SRC, false>(a23)));
              sts8(dst + v_to[1], make_uint2(codes_bf16<SRC, true>(a01), codes_bf16<SRC, true>(a23)));
              sts8(dst + v_to[2], make_uint2(codes_bf16<SRC, false>(b01), codes_bf16<SRC, false>(b23)));
              sts8(dst + v_to[3], make_uint2(codes_bf16<SRC, true>(b01), codes_bf16<SRC, true>(b23)));
            } else {
#pragma unroll 1
              for (int r = 0; r < 4; r++) sts8(dst + (v_dim / 64) * (BN * 128) + (v_dim % 8) * 2 + swz(v_key + r, v_dim % 64 / 8), key + r < p.L ? *reinterpret_cast<const uint2 *>(v_tail + (int64_t)(key + r - full) * D + v_dim) : make_uint2(0, 0));
            }
          } else {
            const int key = key0 + k_key + i * K_STEP;
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (whole || key < full) {
              lo = make_uint4(codes_bf16<SRC, false>(w.x), codes_bf16<SRC, true>(w.x), codes_bf16<SRC, false>(w.y), codes_bf16<SRC, true>(w.y));
              hi = make_uint4(codes_bf16<SRC, false>(w.z), codes_bf16<SRC, true>(w.z), codes_bf16<SRC, false>(w.w), codes_bf16<SRC, true>(w.w));
            } else if (key < p.L) {
              const uint4 *const row = reinterpret_cast<const uint4 *>(k_tail + (int64_t)(key - full) * D + k_dim);
              lo = row[0], hi = row[1];
            }
            sts16(dst + (k_swap ? k_hi : k_lo), k_swap ? hi : lo), sts16(dst + (k_swap ? k_lo : k_hi), k_swap ? lo : hi);
          }
        }
        if (!values) {  // both scales of the tile's keys, 16 at a time
          const int idx = (j - J0) % SCALES_AHEAD;
          if (tid < 2 * (BN / 16)) sts_f32(scales_at + (uint32_t)(idx * 2 * (BN / 16) + tid) * 4u, scale);
          __syncwarp();
          if (lane == 0) mm_bar_arrive(scale_full + 8 * idx);
          scale = scale_of(j + 1);  // (past the last full block: 1)
        }
        fence_async_smem();  // the tensor core reads shared memory through the async proxy
        __syncwarp();
        if (lane == 0) mm_bar_arrive(ring_full + 8 * s), mm_bar_arrive(raw_empty + 8 * (at % 2));
        at++;
      };
      for (int j = J0; j <= J1 && ok; j++) {
        if (j < J1) fetch(false, j);
        if (j > J0) fetch(true, j - 1);
      }
    }
  } else {
    more_registers<Roles<SRC>::SOFTMAX_REGS>();
    // ---------------------------------------------------------------- softmax
    // Two query tiles: four warps each. One: two warps share 32 rows, each with half the columns; they tell one another
    // their maxima, and in the end their weights, through shared memory.
    constexpr int CN = NQ == 2 ? BN : BN / 2, OD = NQ == 2 ? D : D / 2;
    const int i = NQ == 2 ? (int)warp >> 2 : 0, part = NQ == 2 ? 0 : (int)warp >> 2, row = (int)((warp & 3) * 32 + lane);
    const int col0 = part * CN;
    auto told = [&](int n, int half) { return told_at + (uint32_t)(((n & 1) * 2 + half) * 128 + row) * 4u; };
    auto both_halves = [&]() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    const uint32_t lanes = ((warp & 3) * 32u) << 16;
    const int at_row = p.row0 + 128 * i + row, tok = at_row >> group_log2, head = head0 + (at_row & (group - 1));
    const bool real = j1[i] > j0[i] && tok < p.n;
    const int pos = p.held + tok, first_pos = p.held + ((p.row0 + 128 * i) >> group_log2);
    int lo, hi, lo_most, hi_least, other;
    visible_keys(pos, p.L, p.prefix, a.window, a.causal, lo, hi);
    visible_keys(p.held + min((p.row0 + 128 * i + 127) >> group_log2, p.n - 1), p.L, p.prefix, a.window, a.causal, lo_most, other);
    visible_keys(first_pos, p.L, p.prefix, a.window, a.causal, other, hi_least);
    const float slope = !PLAIN && a.slopes && real ? a.slopes[head] * LOG2E : 0.0f;
    const float c = a.scale * LOG2E;
    const uint32_t o_at = tmem + G::O_AT + i * D + part * OD + lanes;
    float m = NOTHING, l = 0.0f;
    bool ok = true;
    for (int j = j0[i]; j < j1[i]; j++) {
      const int n = j - j0[i], buf = NQ == 2 ? i : n & 1;
      const uint32_t s_at = tmem + G::S_AT + buf * BN + lanes;  // (P: half the columns)
      if (ok) ok = prompt_wait_warp(s_full + 8 * buf, NQ == 2 ? n & 1 : (n >> 1) & 1);
      if (CODES && ok) ok = prompt_wait_warp(scale_full + 8 * ((j - J0) % SCALES_AHEAD), ((j - J0) / SCALES_AHEAD) & 1);
      if (!ok) {  // (no half waits for one that gave up)
        if constexpr (NQ == 1) both_halves();
        continue;
      }
      tc_fence_after();
      uint32_t s[CN];
#pragma unroll
      for (int x = 0; x < CN; x += 32) tmem_load32(s_at + col0 + x, s + x);
      tmem_wait_loads();
      const int key0 = j * BN + col0;
      const uint32_t scales = scales_at + (uint32_t)(((j - J0) % SCALES_AHEAD) * 2 * (BN / 16) + col0 / 16) * 4u;
      if constexpr (CODES && !PLAIN) {
#pragma unroll
        for (int x = 0; x < CN; x += 16) {
          const float ks = lds_f32(scales + x / 4);
          const uint64_t f = pair_f32(ks, ks);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float v0, v1;
            split_f32(mul_f32x2(pair_f32(__uint_as_float(s[x + e]), __uint_as_float(s[x + e + 1])), f), v0, v1);
            s[x + e] = __float_as_uint(v0), s[x + e + 1] = __float_as_uint(v1);
          }
        }
      }
      if constexpr (CAP) {
        const uint64_t f = pair_f32(a.scale * (2.0f * LOG2E / a.cap), a.scale * (2.0f * LOG2E / a.cap));
#pragma unroll
        for (int x = 0; x < CN; x += 2) {
          float z0, z1;
          split_f32(mul_f32x2(pair_f32(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), f), z0, z1);
          s[x] = __float_as_uint(CAP == WIDE ? capped_wide(z0, a.cap * LOG2E) : capped(z0, a.cap * LOG2E));
          s[x + 1] = __float_as_uint(CAP == WIDE ? capped_wide(z1, a.cap * LOG2E) : capped(z1, a.cap * LOG2E));
        }
      }
      if constexpr (!PLAIN) {  // s c - slope |i - j|; the bias is a line where all keys lie before the queries
        const uint64_t f = pair_f32(CAP ? 1.0f : c, CAP ? 1.0f : c);
        const float gap = (float)(pos - key0);
        if (key0 + CN <= first_pos) {
          const uint64_t up = pair_f32(slope, slope), from = pair_f32(-slope * gap, -slope * gap);
#pragma unroll
          for (int x = 0; x < CN; x += 2) {
            float v0, v1;
            split_f32(fma_f32x2(pair_f32(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), f, fma_f32x2(up, pair_f32((float)x, (float)(x + 1)), from)), v0, v1);
            s[x] = __float_as_uint(v0), s[x + 1] = __float_as_uint(v1);
          }
        } else {
#pragma unroll
          for (int x = 0; x < CN; x++) s[x] = __float_as_uint(fmaf(-slope, fabsf(gap - (float)x), __uint_as_float(s[x]) * (CAP ? 1.0f : c)));
        }
      }
      if (key0 < lo_most || key0 + CN > hi_least) {
        const uint32_t from = (uint32_t)(lo - key0), count = (uint32_t)(hi - lo);
#pragma unroll
        for (int x = 0; x < CN; x++)
          if ((uint32_t)x - from >= count) s[x] = 0xFF800000u;  // -inf
      }
      float top = -CUDART_INF_F, factor[CODES && PLAIN ? CN / 16 : 1];  // PLAIN over a cache: K's scale goes with c
      if constexpr (CODES && PLAIN) {
#pragma unroll
        for (int x = 0; x < CN; x += 16) {
          factor[x / 16] = c * lds_f32(scales + x / 4);
          float most = __uint_as_float(s[x]), most2 = __uint_as_float(s[x + 1]);
#pragma unroll
          for (int e = 2; e < 16; e += 2) most = fmaxf(most, __uint_as_float(s[x + e])), most2 = fmaxf(most2, __uint_as_float(s[x + e + 1]));
          top = fmaxf(top, fmaxf(most, most2) * factor[x / 16]);
        }
      } else {
        float top2 = __uint_as_float(s[1]);
        top = __uint_as_float(s[0]);
#pragma unroll
        for (int x = 2; x < CN; x += 2) top = fmaxf(top, __uint_as_float(s[x])), top2 = fmaxf(top2, __uint_as_float(s[x + 1]));
        top = fmaxf(top, top2);
        if constexpr (PLAIN) top *= c;
      }
      if constexpr (NQ == 1) {
        sts_f32(told(n, part), top);
        tc_fence_before();  // the other half's scores have been read when its weights are written over them
        both_halves();
        tc_fence_after();
        top = fmaxf(top, lds_f32(told(n, part ^ 1)));
      }
      if (__any_sync(BN_FULL, top > m + RISE)) {
        const bool rise = top > m + RISE;
        const float keep = rise ? ex2(m - top) : 1.0f;
        if (rise) m = top;
        l *= keep;
        if (n) {  // the sums so far, once the product before is done
          if (ok) ok = prompt_wait_warp(o_done + 8 * (NQ == 2 ? i : (n - 1) & 1), NQ == 2 ? (n - 1) & 1 : ((n - 1) >> 1) & 1);
          tc_fence_after();
#pragma unroll 1
          for (int x = 0; x < OD; x += 32) {
            uint32_t o[32];
            tmem_load32(o_at + x, o);
            tmem_wait_loads();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_store32(o_at + x, o);
          }
        }
      }
      uint64_t cc = pair_f32(PLAIN ? c : 1.0f, PLAIN ? c : 1.0f), vv = 0;
      const uint64_t mm = pair_f32(-m, -m);
      uint64_t sum = 0, sum2 = 0;
#pragma unroll
      for (int x = 0; x < CN; x += 4) {
        if (CODES && x % 16 == 0) {
          if constexpr (PLAIN) cc = pair_f32(factor[CODES ? x / 16 : 0], factor[CODES ? x / 16 : 0]);
          const float vs = lds_f32(scales + (BN / 16 + x / 16) * 4);
          vv = pair_f32(vs, vs);
        }
        float e0, e1, e2, e3;
        split_f32(fma_f32x2(pair_f32(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), cc, mm), e0, e1);
        split_f32(fma_f32x2(pair_f32(__uint_as_float(s[x + 2]), __uint_as_float(s[x + 3])), cc, mm), e2, e3);
        uint64_t p01 = pair_f32(ex2(e0), ex2(e1)), p23 = pair_f32(ex2(e2), ex2(e3));
        sum = add_f32x2(sum, p01), sum2 = add_f32x2(sum2, p23);
        if constexpr (CODES) p01 = mul_f32x2(p01, vv), p23 = mul_f32x2(p23, vv);
        split_f32(p01, e0, e1), split_f32(p23, e2, e3);
        s[x / 2] = bf16_pair(e0, e1), s[x / 2 + 1] = bf16_pair(e2, e3);
        if (HALVES && x == CN / 2 - 4) {  // half of the keys
          tmem_store32(s_at, s);
          tmem_wait_stores();
          tc_fence_before();
          mm_bar_arrive(p_half + 8 * buf);
        }
      }
      if constexpr (NQ == 2 && !HALVES) tmem_store32(s_at, s);
      if constexpr (NQ == 2) tmem_store32(s_at + CN / 4, s + CN / 4);
      else tmem_store16(s_at + col0 / 2, s);
      float s0, s1;
      split_f32(add_f32x2(sum, sum2), s0, s1);
      l += s0 + s1;
      tmem_wait_stores();
      tc_fence_before();
      mm_bar_arrive(p_full + 8 * buf);
    }
    // ---- the rows' outputs
    if (j1[i] > j0[i]) {
      const int n = j1[i] - j0[i] - 1;
      if (ok) ok = prompt_wait_warp(o_done + 8 * (NQ == 2 ? i : n & 1), NQ == 2 ? n & 1 : (n >> 1) & 1);
      tc_fence_after();
      if constexpr (NQ == 1) {
        sts_f32(told(0, part), l);  // (the last tile's maxima have been read by both halves: its product is done)
        both_halves();
        l += lds_f32(told(0, part ^ 1));
      }
      bool odd = !(l > 0.0f && l <= 3.0e38f);
      const float inv = 1.0f / l;
      uint16_t *const out = a.out + p.b * a.o_seq + (int64_t)(p.from + tok) * a.o_token + head * a.o_head + part * OD;
      if (ok) {
#pragma unroll 1
        for (int x = 0; x < OD; x += 32) {
          uint32_t o[32];
          tmem_load32(o_at + x, o);
          tmem_wait_loads();
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float u = __uint_as_float(o[e + 2 * k]), v = __uint_as_float(o[e + 2 * k + 1]);
              odd |= !(fabsf(u) <= 3.0e38f) || !(fabsf(v) <= 3.0e38f);
              w[k] = bf16_pair(u * inv, v * inv);
            }
            if (real) *reinterpret_cast<uint4 *>(out + x + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        uint32_t again = __ballot_sync(BN_FULL, odd && real);
        __syncwarp();  // what is written again comes behind what the row's own lane wrote
        for (; again; again &= again - 1) {
          const int other_row = p.row0 + 128 * i + (int)(warp & 3) * 32 + __ffs((int)again) - 1;
          attend_row<D, SRC>(a, p, other_row >> group_log2, head0 + (other_row & (group - 1)), part * OD, part * OD + OD);
        }
      }
    }
  }
  if (CODES && a.zero_rest && warp < SOFTMAX_WARPS) {  // rows of this block whose tokens are not real
    const int end = min(p.row0 + G::ROWS, a.tokens << group_log2);
    for (int r = max(p.row0, p.n << group_log2) + (int)warp; r < end; r += SOFTMAX_WARPS) {
      uint16_t *const out = a.out + p.b * a.o_seq + (int64_t)(r >> group_log2) * a.o_token + (head0 + (r & (group - 1))) * a.o_head;
      if (lane < D / 8) *reinterpret_cast<uint4 *>(out + 8 * lane) = make_uint4(0, 0, 0, 0);
    }
  }
  if (!CODES && a.offsets && a.zero_rest && warp < SOFTMAX_WARPS) {  // tokens of no document, a share of them a block
    const int begin = min(max(a.offsets[0], 0), a.T), end = max(begin, min(max(a.offsets[a.docs], 0), a.T));
    const int64_t rest = (int64_t)(begin + a.T - end) * a.heads;
    for (int64_t r = (int64_t)blockIdx.x * SOFTMAX_WARPS + warp; r < rest; r += (int64_t)gridDim.x * SOFTMAX_WARPS) {
      const int t = (int)(r / a.heads);
      uint16_t *const out = a.out + (int64_t)(t < begin ? t : t - begin + end) * a.o_token + r % a.heads * a.o_head;
      if (lane < D / 8) *reinterpret_cast<uint4 *>(out + 8 * lane) = make_uint4(0, 0, 0, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// A tensor map of BF16 rows [sequences, tokens, heads, D] in pieces of 64 dimensions; tokens past the last read as zeros.
inline bool rows_map(CUtensorMap *m, const uint16_t *p, int D, int64_t heads, int64_t tokens, int64_t seqs, int64_t head, int64_t token, int64_t seq, int box_heads, int box_tokens, int dims_used) {
  TensorMapEncodeFn encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)seqs}, steps[3] = {(cuuint64_t)(heads > 1 ? head : D) * 2, (cuuint64_t)(tokens > 1 ? token : D) * 2, (cuuint64_t)(seqs > 1 ? seq : D) * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens, 1}, unit[4] = {1, 1, 1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)dims_used, const_cast<uint16_t *>(p), dims, steps, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query heads of a block: the largest power of two that divides the key head's group, up to 64.
inline int block_group_log2(int64_t heads, int64_t kv_heads) {
  int log2 = 0;
  while (log2 < 6 && (heads / kv_heads) % (2 << log2) == 0) log2++;
  return log2;
}

template <int D, int SRC>
int prompt_launch(const PromptArgs &a, const CUtensorMap &q_map, const CUtensorMap &k_map, const CUtensorMap &v_map, int64_t blocks, int log2, cudaStream_t stream) {
  auto kern = a.cap > WIDE_CAP ? prompt_kernel<D, false, WIDE, SRC> : a.cap > 0.0f ? prompt_kernel<D, false, USUAL, SRC> : !a.slopes && a.scale > 0.0f ? prompt_kernel<D, true, NO_CAP, SRC> : prompt_kernel<D, false, NO_CAP, SRC>;
  const uint32_t smem = SRC == FROM_BF16 ? Tiles<D>::SMEM : Tiles<D>::SMEM_CODES;
  BN_CUDA(allow_smem(kern, smem));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3(Roles<SRC>::WARPS * 32), cfg.dynamicSmemBytes = smem, cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = 1;
  BN_CUDA(cudaLaunchKernelEx(&cfg, kern, q_map, k_map, v_map, a, log2, a.heads >> log2));
  return launched("prompt_kernel");
}

int prompt_status(int *status) {
  BN_CUDA(cudaMemcpyFromSymbol(status, g_prompt_error, sizeof(int)));
  return BN_OK;
}

int prompt_status_reset() {
  const int zero = 0;
  BN_CUDA(cudaMemcpyToSymbol(g_prompt_error, &zero, sizeof(int)));
  return BN_OK;
}

}  // namespace
}  // namespace bn
