// Causal attention over a cache held in 4 bits (kv4.h has the format), on the half-precision matrix cores: they take every
// number of the cache exactly, so nothing is rounded on the way from the cache into a product.
//
// Queries go there as half precision too, scaled by a power of two that brings a row's largest to 2^14 .. 2^15 (the score's
// factor takes it back): bfloat16's eight bits fit with room, float32's 24 are three terms, each the rounding of what the ones before
// it left, and three products.  The softmax's weights 2^(s - ref + 7), ref the column's largest score or up to 8 below it, are rounded to half
// precision, eleven bits (bfloat16 build: 2^-11 of a weight, an eighth of the output's own 2^-8), or are three such terms
// (float32 build).  Scores, maxima, sums and outputs are 32 bits.
//
// What they measure on an MI355X, of 28 query and 4 key heads of 128 dims in bfloat16 (a copy reaches 5.0 TB/s there, a product of 8,192^3 1.23
// PFLOP/s): 8 tokens at 131,072 positions 124 us + 8 for the join, 605 MB at 4.9 TB/s; 8 at 32,768 36 + 5, 151 MB; one at 2,100 5.8 + 3.3,
// by waits (a launch that does nothing takes 2.9, and each dependent trip to memory half a microsecond).  A prompt of 8,192 tokens 590 to
// 670 us with the clock that the card's power allows, 0.72 to 0.82 PFLOP/s; one of 2,048 63 + 9; 512 tokens behind 1,536 39 + 6.
#include <math.h>

#include "api.h"
#include "common.h"
#include "kv4.h"

#define KV4_BLOCK 64               // positions of a block: one pass of products
#define KV4_WAVES 4                // waves that share a chunk, the unit of the decoding kernel's work list
#define KV4_MOST_ROUNDS 4          // blocks of a chunk that each of them takes, at most
#define KV4_ITEM_FACTOR 1024       // the most chunks of a token; the factor of the token's slot in an item
#define KV4_COLUMNS 16             // query heads of a key head that a wave takes at a time
#define KV4_RAISE 8.0f             // how far (log2) scores may pass the reference before it is raised
#define KV4_WEIGHT 7.0f            // log2 of a weight at the reference: at most 2^15 goes to half precision
#define KV4_FAR 4096.0f            // references (log2) beyond which scores have theirs taken off before their factor (kv4_refer)
#define LOG2E 1.4426950408889634f

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// Terms of a number's split into half precision (its bits, eleven at a time).
constexpr int TERMS = AXON_BF16 ? 1 : 3;

__device__ __forceinline__ f32x4 kv4_mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Eight numbers as TERMS operands.
__device__ __forceinline__ void kv4_split(const float (&x)[8], u32x4 (&out)[TERMS]) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int n = 0; n < TERMS; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2_t h = {(_Float16)rest[2 * i], (_Float16)rest[2 * i + 1]};
      unsigned pair = __builtin_bit_cast(unsigned, h);
      if (n + 1 < TERMS) {
        // what is left of each, exactly, out of the pair in one instruction (from h the compiler rounds each number once more alone: 256 for
        // 32 numbers in place of 112; 1,000 tokens of 14 heads of 64 dims in a window of 700 42 -> 38 us)
        float left;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(left) : "v"(pair), "v"(rest[2 * i]));
        rest[2 * i] = left;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(left) : "v"(pair), "v"(rest[2 * i + 1]));
        rest[2 * i + 1] = left;
      }
      out[n][i] = pair;
    }
  }
}

// The power of two that brings `largest` (of a row of queries) to 2^14 .. 2^15; 0 for a row of zeros or of what is not finite.
__device__ __forceinline__ int kv4_query_shift(float largest) {
  return largest > 0.0f && largest < INFINITY ? 14 - ilogbf(largest) : 0;
}

// A score's factor to log2, which takes the query's power of two back.  Of the smallest queries it is below all numbers, and would be 0, which is
// not a number with what a masked place holds: 2^-126 in its place leaves scores (up to 2^38 before it) that are nothing to 32 bits either.
__device__ __forceinline__ float kv4_score_factor(float scale, int shift) { return fmaxf(ldexpf(scale * LOG2E, -shift), 0x1p-126f); }

// Positions of a chunk of a token that sees `seen` positions: by the token alone, so that its result does not depend on what else a
// step holds.  Up to 8,192 positions every wave has one block, which spreads a token over the chip; a longer one pays for
// its partial results.  28 heads over 4 of 128, us, attention + join, one block a wave / up to four: 1 token at 8,192 5.9 + 3.4 / 11.4 + 3.0, at
// 32,768 9.8 + 5.4 / 12.6 + 3.9; 8 tokens at 8,192 15.0 + 3.9 / 16.7 + 3.8, at 32,768 39.8 + 6.6 / 36.4 + 4.6, at 131,072 144 + 26 / 124 + 7.6.
__host__ __device__ inline int kv4_chunk(int seen) {
  int rounds = 1;
  while (rounds < KV4_MOST_ROUNDS && seen > 8192 * rounds) rounds *= 2;
  return rounds * KV4_WAVES * KV4_BLOCK;
}

// The weights are taken relative to a reference, which is raised to a block's maximum only where that is KV4_RAISE or more above it
// (the first block's always): what was summed before is then scaled by the factor returned, 1 for a column whose
// reference stays.  A column's arithmetic depends on its own scores alone.
struct Kv4Reference {
  float score = -INFINITY;         // as the products leave it; times c its log2
  float add = 0.0f;                // what a score times c has added to it for its weight's log2
  bool far = false;                // a column of the wave has its reference taken off its scores
};
__device__ __forceinline__ float kv4_raise(Kv4Reference& ref, float block_max, float c) {
  const bool up = __fmul_rn(__fsub_rn(block_max, ref.score), c) > KV4_RAISE;  // (nothing seen yet, and nothing now: not a number, so no)
  const float before = ref.score;
  ref.score = up ? block_max : before;
  return up ? __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(before, ref.score), c)) : 1.0f;
}

// The rest of it, where one of the wave's was raised.  score c rounded and KV4_WEIGHT less that rounded are off by 2^-13 each up to KV4_FAR,
// for all of a reference's weights alike.  At 2^25 they would be off by more than KV4_WEIGHT, and weights out of half precision's range:
// a column beyond KV4_FAR has its reference taken off its scores before their factor, exactly where it matters, near the largest.
__device__ __forceinline__ bool kv4_far(float score, float c) { return fabsf(__fmul_rn(score, c)) > KV4_FAR && fabsf(score) < INFINITY; }
__device__ __forceinline__ void kv4_refer(Kv4Reference& ref, float c) {
  const bool far = kv4_far(ref.score, c);
  ref.far = __any(far);
  ref.add = ref.score == -INFINITY ? 0.0f : __fsub_rn(KV4_WEIGHT, far ? 0.0f : __fmul_rn(ref.score, c));
}

// ============================================================================ single tokens
// The query heads of a key head are the columns of S^T = K Q^T (sixteen at a time), positions its rows; what a lane then holds of
// the weights are the operands of O^T = V^T P^T.  Lane (l16, h), h = lane / 16:
// * K: row l16 of tile t = 2 u + v is position 32 u + 8 (l16 / 4) + 4 v + l16 % 4 of the block, so that the lane ends with the
//   scores of positions 32 u + 8 h + {0 .. 7}, its operand of step u of O^T; its dims are h HD/4 .. + HD/4, one piece of
//   its row, of one group: a scale a row.
// * V^T: row l16 of tile dt is dim HD/16 l16 + dt, so that the lane reads HD/4 neighbouring bytes of an octet, all of one group, and
//   ends with neighbouring dims of its column.
template <int HD>
struct Kv4Keys {                   // a block's bytes on their way: nothing of it is unpacked
  unsigned words[4][HD / 32], scale[4];
};
template <int HD>
struct Kv4Values {
  uint4 words[2][HD / 64], scale[2];
};

// Where a wave reads.  An octet of slots lies at the same place in both caches: its words at `words`, its scales at `scales`, in
// units of 32 bytes from the cache's start (so 32 bits count 128 GB), each octet's in a lane.
struct Kv4Place {
  const unsigned char *k_words, *k_scales, *v_words, *v_scales;        // the caches' starts and the lane's part of an octet
  unsigned words, scales;
};

template <int HD>
__device__ __forceinline__ Kv4Place kv4_place_of(const unsigned char* k_cache, const unsigned char* v_cache, const int32_t* table_row, int c0,
                                                 int pos, int wave, int kvh, int n_kv_heads, int page_size, int lane) {
  static_assert(8 * KV4_MOST_ROUNDS <= 64, "an octet of the wave's blocks a lane");
  const int l16 = lane & 15, h = lane >> 4;
  const int p = min(c0 + KV4_BLOCK * (KV4_WAVES * (lane >> 3) + wave) + 8 * (lane & 7), pos);      // (past the token: its own last page)
  const unsigned page = table_row[p >> __builtin_ctz(page_size)], octet = (p & (page_size - 1)) >> 3;
  const unsigned head = (page * n_kv_heads + kvh) * (unsigned)(page_size * kv4_row_bytes(HD) / 32);
  Kv4Place at;
  at.words = head + octet * (HD / 8);
  at.scales = head + page_size * (HD / 64) + octet * (HD / 64);
  at.k_words = k_cache + ((l16 & 3) * (HD / 2) + h * (HD / 8));
  at.k_scales = k_cache + ((l16 & 3) * (HD / 16) + h * (HD / 4) / 32 * 2);
  at.v_words = v_cache + l16 * (HD / 4);
  at.v_scales = v_cache + l16 * (HD / 16) / 32 * 16;
  return at;
}

__device__ __forceinline__ const unsigned char* kv4_at(const unsigned char* base, unsigned units) { return base + ((size_t)units << 5); }

// The wave's b-th block.
template <int HD>
__device__ __forceinline__ void kv4_load(Kv4Keys<HD>& out, const Kv4Place& at, int b, int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int octet = 8 * b + 4 * u + ((lane & 15) >> 2);
    const unsigned char* words = kv4_at(at.k_words, __shfl(at.words, octet, AXON_WAVE));
    const unsigned char* scales = kv4_at(at.k_scales, __shfl(at.scales, octet, AXON_WAVE));
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      unsigned(&w)[HD / 32] = out.words[2 * u + v];
      if constexpr (HD == 128) {
        const uint4 four = *reinterpret_cast<const uint4*>(words + v * 4 * (HD / 2));
        w[0] = four.x; w[1] = four.y; w[2] = four.z; w[3] = four.w;
      } else {
        const uint2 two = *reinterpret_cast<const uint2*>(words + v * 4 * (HD / 2));
        w[0] = two.x; w[1] = two.y;
      }
      out.scale[2 * u + v] = *reinterpret_cast<const uint16_t*>(scales + v * 4 * (HD / 16));
    }
  }
}

template <int HD>
__device__ __forceinline__ void kv4_load(Kv4Values<HD>& out, const Kv4Place& at, int b, int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int octet = 8 * b + 4 * u + (lane >> 4);
    const uint4* words = reinterpret_cast<const uint4*>(kv4_at(at.v_words, __shfl(at.words, octet, AXON_WAVE)));
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) out.words[u][i] = words[i];
    out.scale[u] = *reinterpret_cast<const uint4*>(kv4_at(at.v_scales, __shfl(at.scales, octet, AXON_WAVE)));
  }
}

// S^T of a block: s[2 u + v][r] is position 32 u + 8 h + 4 v + r of column l16, unscaled.
template <int HD>
__device__ __forceinline__ void kv4_scores(const Kv4Keys<HD>& keys, const u32x4 (&qf)[HD / 32][TERMS], const Kv4Masks& masks, f32x4 (&s)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    half2_t sc[4], cc[4];
    kv4_pair_scale(keys.scale[t] | keys.scale[t] << 16, sc[0], cc[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) { sc[i] = sc[0]; cc[i] = cc[0]; }
    s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
      const u32x4 a = kv4_operand(keys.words[t][j], sc, cc, masks);
#pragma unroll
      for (int n = TERMS - 1; n >= 0; --n) s[t] = kv4_mma(a, qf[j][n], s[t]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// From a block's scores: its weights 2^(s c - ref + KV4_WEIGHT) as operands of O^T, added to the column's sum l.  whole: every position is
// seen (the same for the wave); else those of lo .. pos are, and the block begins at p0.  rescale(factor) is called where a reference of
// the wave is raised.
template <typename Rescale>
__device__ __forceinline__ void kv4_weights(f32x4 (&s)[4], bool whole, int p0, int lo, int pos, float c, int lane, Kv4Reference& ref, float& l,
                                            u32x4 (&pf)[2][TERMS], Rescale rescale) {
  if (!whole) {
    int first = p0 + 8 * (lane >> 4);
    asm volatile("" : "+v"(first));            // a branch of its own: whole blocks pay nothing for the mask
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = first + 32 * (t >> 1) + 4 * (t & 1) + r;
        s[t][r] = p >= lo && p <= pos ? s[t][r] : -INFINITY;
      }
  }
  float mx = -INFINITY;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[t][r]);
  mx = fmaxf(mx, __shfl_xor(mx, 16, AXON_WAVE));
  mx = fmaxf(mx, __shfl_xor(mx, 32, AXON_WAVE));
  const float factor = kv4_raise(ref, mx, c);
  if (__any(factor != 1.0f)) {
    l = __fmul_rn(l, factor);
    rescale(factor);
    kv4_refer(ref, c);
  }
  if (__builtin_expect(ref.far, 0)) {
    const float off = kv4_far(ref.score, c) ? ref.score : 0.0f;                // (0 leaves a score as it is)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][r] = __fsub_rn(s[t][r], off);
  }
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * u + (i >> 2)][i & 3], c, ref.add));
      sum = __fadd_rn(sum, w[i]);
    }
    kv4_split(w, pf[u]);
  }
  l = __fadd_rn(l, sum);                       // (the lane's own sixteen positions of each block; the column's four lanes join at the end)
}

// The block's values, weighted, added to the column's output: o[dt][r] is dim HD/16 (4 h + r) + dt of column l16.
template <int HD>
__device__ __forceinline__ void kv4_values(const Kv4Values<HD>& values, const u32x4 (&pf)[2][TERMS], bool whole, int p0, int lo, int pos,
                                           int lane, const Kv4Masks& masks, f32x4 (&o)[HD / 16]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    unsigned metas[4] = {values.scale[u].x, values.scale[u].y, values.scale[u].z, values.scale[u].w};
    if (!whole) {
      // a weight of zero times what an unseen place holds has to be zero, whatever that is
      int first = p0 + 32 * u + 8 * (lane >> 4);
      asm volatile("" : "+v"(first));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = first + 2 * i;
        metas[i] &= (p >= lo && p <= pos ? 0x0000ffffu : 0u) | (p + 1 >= lo && p + 1 <= pos ? 0xffff0000u : 0u);
      }
    }
    half2_t sc[4], cc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) kv4_pair_scale(metas[i], sc[i], cc[i]);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) {
      const uint4 four = values.words[u][dt / 4];
      const unsigned word = dt % 4 == 0 ? four.x : dt % 4 == 1 ? four.y : dt % 4 == 2 ? four.z : four.w;
      const u32x4 a = kv4_operand(word, sc, cc, masks);
#pragma unroll
      for (int n = TERMS - 1; n >= 0; --n) o[dt] = kv4_mma(a, pf[u][n], o[dt]);
      if (dt % 2) __builtin_amdgcn_sched_barrier(0);       // (else every tile is unpacked before the first product)
    }
  }
}

// The wave's queries: column l16 (the last one again past `columns`), dims h HD/4 + 8 j + {0 .. 7}.
template <int HD>
struct Kv4Queries {
  float x[HD / 32][8];
};

template <int HD>
__device__ __forceinline__ void kv4_load(Kv4Queries<HD>& out, const elem_t* row, int columns, int lane) {
  const elem_t* src = row + (size_t)min(lane & 15, columns - 1) * HD + (lane >> 4) * (HD / 4);
#pragma unroll
  for (int j = 0; j < HD / 32; ++j) {
    float a[4], b[4];
    load4_guarded(src + 8 * j, 4, true, a);
    load4_guarded(src + 8 * j + 4, 4, true, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out.x[j][i] = a[i];
      out.x[j][4 + i] = b[i];
    }
  }
}

// As operands of S^T.  Returns the score's factor, which takes their power of two back.
template <int HD>
__device__ __forceinline__ float kv4_operands(Kv4Queries<HD>& q, float scale, u32x4 (&qf)[HD / 32][TERMS]) {
  float largest = 0.0f;
#pragma unroll
  for (int j = 0; j < HD / 32; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(q.x[j][i]));
  largest = fmaxf(largest, __shfl_xor(largest, 16, AXON_WAVE));
  largest = fmaxf(largest, __shfl_xor(largest, 32, AXON_WAVE));
  const int shift = kv4_query_shift(largest);
  const float up = ldexpf(1.0f, shift / 2), up2 = ldexpf(1.0f, shift - shift / 2);      // (2^shift alone may be out of range)
#pragma unroll
  for (int j = 0; j < HD / 32; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q.x[j][i] = q.x[j][i] * up * up2;
    kv4_split(q.x[j], qf[j]);
  }
  return kv4_score_factor(scale, shift);
}

// A workgroup has a chunk of a token and a set of up to sixteen query heads of a key head: grid (key heads x sets, work items).  Each of its
// waves takes every KV4_WAVES-th block; what they sum is joined through LDS, in the order of the waves.  Of a token of one chunk the output
// is stored at once; else output, reference and sum go to `partial` ([slot][head][chunk][HD], then [slot][head][chunk][2]).
// Bound by the cache's bytes where there is work for the chip (three workgroups of 12 waves a CU have 110 KB of it on their way), by
// dependent trips to memory where there is not.
template <int HD>
__global__ void __launch_bounds__(64 * KV4_WAVES, TERMS == 1 ? 3 : 2)
kv4_decode_kernel(const elem_t* __restrict__ q, int q_stride, const unsigned char* __restrict__ k_cache,
                  const unsigned char* __restrict__ v_cache, const int32_t* __restrict__ block_table, int table_stride,
                  const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows, elem_t* __restrict__ out,
                  const int32_t* __restrict__ token_index, int n_tokens, const int32_t* __restrict__ work, int n_work,
                  float* __restrict__ partial, int max_chunks, int n_heads, int n_kv_heads, int sets, int page_size, int window, float scale) {
  constexpr int DT = HD / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, h = lane >> 4;
  const int at_item = blockIdx.z * 65535 + blockIdx.y;
  if (at_item >= n_work) return;
  const int item = work[at_item];
  if (item < 0) return;                              // padding of the list
  const int slot = item / KV4_ITEM_FACTOR, chunk = item % KV4_ITEM_FACTOR;
  if (slot >= n_tokens || chunk >= max_chunks) return;
  const int kvh = sets == 1 ? blockIdx.x : blockIdx.x / sets, set = blockIdx.x - kvh * sets;
  const int group = n_heads / n_kv_heads, head0 = kvh * group + set * KV4_COLUMNS, columns = min(KV4_COLUMNS, group - set * KV4_COLUMNS);
  const int t = token_index ? token_index[slot] : slot, pos = positions[t];
  elem_t* out_row = out + ((size_t)t * n_heads + head0) * HD;
  if (pos < 0) {                                     // padding of the batch: zeros
    if (chunk == 0)
      for (int i = threadIdx.x; i < columns * HD; i += 64 * KV4_WAVES) out_row[i] = from_float(0.0f);
    return;
  }
  const int lo = window > 0 ? max(0, pos + 1 - window) : 0, size = kv4_chunk(pos + 1 - lo);
  const int first_chunk = lo / size, n_chunks = pos / size - first_chunk + 1;
  if (chunk >= n_chunks) return;
  const int c0 = (first_chunk + chunk) * size;
  // the wave's blocks: chunk blocks wave, wave + KV4_WAVES, ..., of which those from the first one that is seen to the token's own
  const int first_block = max(0, lo - c0) / KV4_BLOCK, last_block = min(size - 1, pos - c0) / KV4_BLOCK;
  const int b_first = max(0, first_block - wave + KV4_WAVES - 1) / KV4_WAVES, b_last = last_block < wave ? -1 : (last_block - wave) / KV4_WAVES;
  Kv4Queries<HD> queries;
  kv4_load<HD>(queries, q + (size_t)t * q_stride + (size_t)head0 * HD, columns, lane);
  const Kv4Place at = kv4_place_of<HD>(k_cache, v_cache, block_table + (size_t)seq_rows[t] * table_stride, c0, pos, wave, kvh, n_kv_heads,
                                       page_size, lane);
  __shared__ __align__(16) float o_of[KV4_WAVES][KV4_COLUMNS][HD + 4];
  __shared__ float ref_of[KV4_WAVES][KV4_COLUMNS], l_of[KV4_WAVES][KV4_COLUMNS];
  Kv4Reference ref;
  float top_log2 = -INFINITY, l = 0.0f;              // (what is joined is compared as log2)
  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (b_first <= b_last) {
    Kv4Masks masks = kv4_masks();
    Kv4Keys<HD> keys;
    Kv4Values<HD> values;
    kv4_load<HD>(keys, at, b_first, lane);
    kv4_load<HD>(values, at, b_first, lane);
    u32x4 qf[HD / 32][TERMS];
    const float c = kv4_operands<HD>(queries, scale, qf);
    for (int b = b_first; b <= b_last; ++b) {
      // the next block's keys are asked for when this one's are used up, its values likewise: each has the other's work to arrive in
      const int p0 = c0 + (b * KV4_WAVES + wave) * KV4_BLOCK;
      const bool whole = p0 >= lo && p0 + KV4_BLOCK - 1 <= pos;
      f32x4 s[4];
      u32x4 pf[2][TERMS];
      kv4_scores<HD>(keys, qf, masks, s);
      __builtin_amdgcn_sched_barrier(0);
      if (b < b_last) kv4_load<HD>(keys, at, b + 1, lane);
      __builtin_amdgcn_sched_barrier(0);
      kv4_weights(s, whole, p0, lo, pos, c, lane, ref, l, pf, [&](float factor) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[dt][r] = __fmul_rn(o[dt][r], factor);
      });
      kv4_values<HD>(values, pf, whole, p0, lo, pos, lane, masks, o);
      __builtin_amdgcn_sched_barrier(0);
      if (b < b_last) kv4_load<HD>(values, at, b + 1, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
    l = __fadd_rn(l, __shfl_xor(l, 16, AXON_WAVE));
    l = __fadd_rn(l, __shfl_xor(l, 32, AXON_WAVE));
    top_log2 = __fmul_rn(ref.score, c);
  }
  if (l16 < columns) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int dt = 0; dt < DT; dt += 4)
        *reinterpret_cast<float4*>(&o_of[wave][l16][DT * (4 * h + r) + dt]) = make_float4(o[dt][r], o[dt + 1][r], o[dt + 2][r], o[dt + 3][r]);
    if (h == 0) {
      ref_of[wave][l16] = top_log2;
      l_of[wave][l16] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < columns * (HD / 4); i += 64 * KV4_WAVES) {
    const int col = i / (HD / 4), d = i % (HD / 4) * 4;
    float top = ref_of[0][col];
#pragma unroll
    for (int w = 1; w < KV4_WAVES; ++w) top = fmaxf(top, ref_of[w][col]);
    const float base = top == -INFINITY ? 0.0f : top;
    float weight = 0.0f;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < KV4_WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(__fsub_rn(ref_of[w][col], base));
      const f32x4 v = *reinterpret_cast<const f32x4*>(&o_of[w][col][d]);
      weight = __builtin_fmaf(l_of[w][col], f, weight);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(v[e], f, sum[e]);
    }
    if (n_chunks == 1) {
      const float inv = __fdiv_rn(1.0f, weight);
#pragma unroll
      for (int e = 0; e < 4; ++e) out_row[col * HD + d + e] = from_float(__fmul_rn(sum[e], inv));
    } else {
      const size_t row = ((size_t)slot * n_heads + head0 + col) * max_chunks + chunk;
      *reinterpret_cast<f32x4*>(partial + row * HD + d) = sum;
      if (d == 0) *reinterpret_cast<float2*>(partial + (size_t)n_tokens * n_heads * max_chunks * HD + 2 * row) = make_float2(top, weight);
    }
  }
}

// A token's chunks joined: with M the largest of their maxima, out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M); JOIN_SUMS sums side
// by side over every JOIN_SUMS-th chunk, ascending, added in order.  grid (tokens, heads); a thread has four dims of one of the sums. 
// Bound by its launch: 3.3 us for one token of 9 chunks, 4.0 for 64, 7.6 for 8 of 128 chunks.
#define JOIN_SUMS 8
template <int HD>
__global__ void __launch_bounds__(JOIN_SUMS * HD / 4)
kv4_join_kernel(const float* __restrict__ partial, const int32_t* __restrict__ positions, const int32_t* __restrict__ token_index,
                elem_t* __restrict__ out, int n_tokens, int max_chunks, int n_heads, int window) {
  constexpr int THREADS = JOIN_SUMS * HD / 4, AHEAD = 4;
  __shared__ float factor[KV4_ITEM_FACTOR], l_sums[JOIN_SUMS], wave_max[THREADS / 64];
  __shared__ __align__(16) float sums[JOIN_SUMS][HD];
  const int slot = blockIdx.x, head = blockIdx.y, t = token_index ? token_index[slot] : slot, pos = positions[t];
  if (pos < 0) return;
  const int lo = window > 0 ? max(0, pos + 1 - window) : 0, size = kv4_chunk(pos + 1 - lo), n = min(pos / size - lo / size + 1, max_chunks);
  if (n == 1) return;                                // stored by the chunk's own block
  const size_t row = ((size_t)slot * n_heads + head) * max_chunks;
  const float* ml = partial + (size_t)n_tokens * n_heads * max_chunks * HD + 2 * row;
  const int d = threadIdx.x % (HD / 4) * 4, part = threadIdx.x / (HD / 4);
  const float* src = partial + row * HD + d;
  // the first chunks' outputs are asked for beside the maxima (of a chunk that is not there the last one's)
  float4 ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) ahead[j] = *reinterpret_cast<const float4*>(src + (size_t)min(part + j * JOIN_SUMS, n - 1) * HD);
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < n; i += THREADS) mx = fmaxf(mx, ml[2 * i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, AXON_WAVE));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x / 64] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) mx = fmaxf(mx, wave_max[w]);
  const float ref = mx == -INFINITY ? 0.0f : mx;
  for (int i = threadIdx.x; i < n; i += THREADS) factor[i] = __builtin_amdgcn_exp2f(__fsub_rn(ml[2 * i], ref));
  __syncthreads();
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  float l = 0.0f;
  auto add = [&](int i, const float4& v) {
    const float f = factor[i];
    o = f32x4{__builtin_fmaf(v.x, f, o[0]), __builtin_fmaf(v.y, f, o[1]), __builtin_fmaf(v.z, f, o[2]), __builtin_fmaf(v.w, f, o[3])};
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (part + j * JOIN_SUMS < n) add(part + j * JOIN_SUMS, ahead[j]);
  int i = part + AHEAD * JOIN_SUMS;
  for (; i + (AHEAD - 1) * JOIN_SUMS < n; i += AHEAD * JOIN_SUMS) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ahead[j] = *reinterpret_cast<const float4*>(src + (size_t)(i + j * JOIN_SUMS) * HD);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) add(i + j * JOIN_SUMS, ahead[j]);
  }
  for (; i < n; i += JOIN_SUMS) add(i, *reinterpret_cast<const float4*>(src + (size_t)i * HD));
  if (d == 0) {
    for (int c = part; c < n; c += JOIN_SUMS) l = __builtin_fmaf(ml[2 * c + 1], factor[c], l);
    l_sums[part] = l;
  }
  *reinterpret_cast<f32x4*>(&sums[part][d]) = o;
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float total = 0.0f, weight = 0.0f;
#pragma unroll
  for (int s = 0; s < JOIN_SUMS; ++s) {
    total = __fadd_rn(total, sums[s][threadIdx.x]);
    weight = __fadd_rn(weight, l_sums[s]);
  }
  out[((size_t)t * n_heads + head) * HD + threadIdx.x] = from_float(__fmul_rn(total, __fdiv_rn(1.0f, weight)));
}

// ============================================================================ prompt portions
// A workgroup has a tile of up to 128 consecutive tokens of one request and HPB query heads of a key head, four waves a head, 32 rows each;
// grid (key heads x sets of HPB heads, tiles), tiles with the most work first, so that the shortest are left for the end.  A block of 64
// positions is unpacked once a workgroup, an octet of slots a wave, into half precision in LDS, where all waves read it: K [64][HD] and V^T
// [HD][64], 16-byte pieces of a row permuted so that sixteen neighbouring rows' pieces lie in different banks.  Two stages: block b + 1 is
// unpacked, and block b + 2 on its way in registers (four and a half bits a number, so few), beside the products of block b. S^T = K Q^T
// and O^T = V^T P^T by 32x32x16 products: what a lane holds of the first is its operand of the second.  Row r of a tile of S^T is position
// pi(r) of it, pi swapping bits 2 and 3, so that register e of tile pt is position 32 pt + 16 (e / 8) + 8 half + e % 8. Of a block a wave
// has 32 products (1,024 cycles of its matrix core), 235 vector instructions, 32 of them exponentials, and 32 KB of LDS to read: of a
// prompt of 8,192 tokens the matrix cores are at work for 42 % of the cycles, the vector units for 57 %, LDS for some 55 %, at the 1.8 GHz
// that the card's power allows then.  A tile alone takes 1.5 us a block.
typedef __attribute__((ext_vector_type(16))) float f32x16;
#define KV4_ROWS 128               // tokens of a tile
// Positions lie in segments that end at 1,024, 2,048, 4,096, 8,192 and every 8,192 behind.  What a row sums is closed at a segment's end
// and folded, in order, into what the segments before gave, whether one workgroup takes them all (its sums then wait in the workspace) or
// one each, which kv4_fold_kernel joins: the same bits, so a row's result does not depend on how many tiles a step has.  Workgroups that
// began together get to a segment's end together, and their 128 KB each take 6 us there and 6 back.  With ends at 2,048 and 8,192 alone /
// these, 28 heads over 4 of 128 dims: 512 tokens behind 1,536 60 / 39 + 6 us, 980 in ragged portions up to 4,400 positions 81 + 5 / 68 + 9,
// a prompt of 2,048 69 / 63 + 9, of 4,096 179 / 183, of 8,192 660 / 675 (without ends 650; with one every 2,048 700).
__host__ __device__ inline int kv4_segment_of(int p) { return p < 1024 ? 0 : p < 2048 ? 1 : p < 4096 ? 2 : p < 8192 ? 3 : 3 + p / 8192; }
__host__ __device__ inline int kv4_segment_start(int s) { return s < 3 ? s * 1024 : s == 3 ? 4096 : s > 262146 ? 0x7fffffff : (s - 3) * 8192; }

__device__ __forceinline__ f32x16 kv4_mma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int HD>
struct Kv4Stage {
  static constexpr int BYTES = KV4_BLOCK * HD * 2, NANS = HD / 4;     // of a block's keys or values, of its values that are not numbers
  // two blocks' keys, V blocks' values and what is not a number among them
  static constexpr int all(int v) { return 2 * BYTES + v * (BYTES + NANS); }
  // a row's pieces are permuted by this
  __device__ static __forceinline__ int k_swizzle(int row) { return HD == 128 ? row & 15 : (row >> 1) & 7; }
  __device__ static __forceinline__ int v_swizzle(int dim) { return (dim >> 1) & 7; }
  // where the 16 bytes of dims 8 chunk .. of a row of K, of positions 8 octet .. of a dim's row of V^T lie
  __device__ static __forceinline__ int k_at(int row, int chunk) {
    return row * (HD * 2) + ((chunk ^ k_swizzle(row)) << 4);
  }
  __device__ static __forceinline__ int v_at(int dim, int octet) { return dim * 128 + ((octet ^ v_swizzle(dim)) << 4); }
};

// An octet of slots of one head on its way: a lane has HD/64 words of a row of K (eight lanes a row) and of V^T (neighbouring dims).
template <int HD>
struct Kv4Octet {
  unsigned k[HD / 64], v[HD / 64], k_scale;
  uint4 v_scale;
};

template <int HD>
__device__ __forceinline__ void kv4_load(Kv4Octet<HD>& out, const unsigned char* k_cache, const unsigned char* v_cache, int page, int p,
                                         size_t page_bytes, size_t head_at, int page_size, int lane) {
  const int octet = (p & (page_size - 1)) >> 3;
  const size_t base = page * page_bytes + head_at;                 // (all of it the wave's)
  const unsigned words = octet * (4 * HD), scales = page_size * (HD / 2) + octet * (HD / 2);
  const unsigned char *k = k_cache + base, *v = v_cache + base;
  if constexpr (HD == 128) {
    const uint2 a = *reinterpret_cast<const uint2*>(k + (words + lane * 8)), b = *reinterpret_cast<const uint2*>(v + (words + lane * 8));
    out.k[0] = a.x; out.k[1] = a.y; out.v[0] = b.x; out.v[1] = b.y;
  } else {
    out.k[0] = *reinterpret_cast<const unsigned*>(k + (words + lane * 4));
    out.v[0] = *reinterpret_cast<const unsigned*>(v + (words + lane * 4));
  }
  // row lane / 8, group (lane % 8) / 2 of four (HD 128) or (lane % 8) / 4 of two; of V^T the group of dim HD/64 lane
  out.k_scale = *reinterpret_cast<const uint16_t*>(k + (scales + (lane >> 3) * (HD / 16) + (lane & 7) * (HD / 64) / 4 * 2));
  out.v_scale = *reinterpret_cast<const uint4*>(v + (scales + lane * (HD / 64) / 32 * 16));
}

// For a block of which a row of the tile sees only some positions: the values' scales of those that no row sees (outside first .. last) become
// zero, and so do those of values that are not numbers: a row that does not see them has a weight of zero for them, and
// zero times them has to be zero.  Where such values are is left in `nans` [group][octet], a bit a slot.
template <int HD>
__device__ __forceinline__ void kv4_edge(Kv4Octet<HD>& in, int octet, int p, int first, int last, unsigned char* nans, int lane) {
  unsigned metas[4] = {in.v_scale.x, in.v_scale.y, in.v_scale.z, in.v_scale.w}, mask = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool nan = (metas[i >> 1] >> (16 * (i & 1)) & 0x7C00) == 0x7C00;
    const bool seen = p + i >= first && p + i <= last;
    if (nan || !seen) metas[i >> 1] &= ~(0xffffu << (16 * (i & 1)));
    if (nan && seen) mask |= 1u << i;
  }
  if (lane * (HD / 64) % 32 == 0) nans[lane * (HD / 64) / 32 * 8 + octet] = (unsigned char)mask;
  in.v_scale = make_uint4(metas[0], metas[1], metas[2], metas[3]);
}

// Unpacked into its stages, as octet `octet` of its block, in PIECES pieces (0, 1: keys, 2, 3: values).
#define KV4_PIECES 4
template <int HD>
__device__ __forceinline__ void kv4_unpack(const Kv4Octet<HD>& in, unsigned char* k_stage, unsigned char* v_stage, int octet, int piece,
                                           const Kv4Masks& masks, int lane) {
  half2_t sc[4], cc[4];
  const int w = piece & 1;
  if (w >= HD / 64) return;
  if (piece < 2) {
    kv4_pair_scale(in.k_scale | in.k_scale << 16, sc[0], cc[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) { sc[i] = sc[0]; cc[i] = cc[0]; }
    *reinterpret_cast<u32x4*>(k_stage + Kv4Stage<HD>::k_at(8 * octet + (lane >> 3), (lane & 7) * (HD / 64) + w)) =
        kv4_operand(in.k[w], sc, cc, masks);
  } else {
    const unsigned metas[4] = {in.v_scale.x, in.v_scale.y, in.v_scale.z, in.v_scale.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) kv4_pair_scale(metas[i], sc[i], cc[i]);
    *reinterpret_cast<u32x4*>(v_stage + Kv4Stage<HD>::v_at(lane * (HD / 64) + w, octet)) = kv4_operand(in.v[w], sc, cc, masks);
  }
}

__device__ __forceinline__ void kv4_meet() {       // everyone's part of the stage is written, everyone has read the other
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A wave's state of a segment: its rows' outputs, references (in the workspace their log2) and (each half of the wave its own) sums.  Kept as the
// lanes hold it.
template <int HD>
struct Kv4State {
  f32x16 o[HD / 32];
  float ref, l;
  static constexpr int FLOATS = KV4_ROWS * HD + 2 * 256;              // of a tile and head
};

template <int HD>
__device__ __forceinline__ void kv4_store(const Kv4State<HD>& st, float* at, int wave, int lane, unsigned nan_groups) {
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt) {
    const bool nan = nan_groups >> dt & 1;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(at + (((wave * (HD / 32) + dt) * 4 + g) * 64 + lane) * 4) =
          nan ? make_float4(NAN, NAN, NAN, NAN) : make_float4(st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]);
  }
  *reinterpret_cast<float2*>(at + KV4_ROWS * HD + (wave * 64 + lane) * 2) = make_float2(st.ref, st.l);
}

// Two states in order, one in the lanes (LATER: the second), one in memory, into the lanes: of a tile of heads of HD dims, the groups of 32 dims
// from dt0 on that the lanes have.
template <int HD, bool LATER, int DIMS>
__device__ __forceinline__ void kv4_fold(Kv4State<DIMS>& st, const float* at, int wave, int lane, int dt0) {
  const float2 other = *reinterpret_cast<const float2*>(at + KV4_ROWS * HD + (wave * 64 + lane) * 2);
  const float top = fmaxf(other.x, st.ref), base = top == -INFINITY ? 0.0f : top;
  const float f_other = __builtin_amdgcn_exp2f(__fsub_rn(other.x, base)), f_mine = __builtin_amdgcn_exp2f(__fsub_rn(st.ref, base));
  auto join = [&](float mine, float theirs) {
    return LATER ? __builtin_fmaf(theirs, f_other, __fmul_rn(mine, f_mine)) : __builtin_fmaf(mine, f_mine, __fmul_rn(theirs, f_other));
  };
#pragma unroll
  for (int dt = 0; dt < DIMS / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 v = *reinterpret_cast<const float4*>(at + (((wave * (HD / 32) + dt0 + dt) * 4 + g) * 64 + lane) * 4);
      st.o[dt][4 * g] = join(st.o[dt][4 * g], v.x);
      st.o[dt][4 * g + 1] = join(st.o[dt][4 * g + 1], v.y);
      st.o[dt][4 * g + 2] = join(st.o[dt][4 * g + 2], v.z);
      st.o[dt][4 * g + 3] = join(st.o[dt][4 * g + 3], v.w);
    }
  st.l = join(st.l, other.y);
  st.ref = top;
}

template <int HD>
__device__ __forceinline__ void kv4_store_row(const Kv4State<HD>& st, elem_t* out_row, int lane, unsigned nan_groups) {
  const float all = __fdiv_rn(1.0f, __fadd_rn(st.l, __shfl_xor(st.l, 32, AXON_WAVE)));
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt) {
    const float inv = nan_groups >> dt & 1 ? NAN : all;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      elem_t* dst = out_row + dt * 32 + g * 8 + (lane >> 5) * 4;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __fmul_rn(st.o[dt][4 * g + e], inv);
#if AXON_BF16
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
#else
      *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
#endif
    }
  }
}

template <int HD, int HPB>
__device__ __forceinline__ void kv4_prefill_tile(unsigned char* smem, int t0, int count, const elem_t* __restrict__ q, int q_stride,
                                                 const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache,
                                                 const int32_t* __restrict__ block_table, int table_stride,
                                                 const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows,
                                                 elem_t* __restrict__ out, int segment, int slot, float* __restrict__ partial, int n_slots,
                                                 int n_heads, int n_kv_heads, int page_size, int window, float scale) {
  using S = Kv4Stage<HD>;
  constexpr int WAVES = 4 * HPB, OCTETS = 8 / WAVES, DT = HD / 32, KS = HD / 16, V_STAGES = 1 + HPB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
  const int group = n_heads / n_kv_heads, sets = (group + HPB - 1) / HPB, kvh = blockIdx.x / sets;
  const int in_group = (blockIdx.x % sets) * HPB + (wave >> 2), head = kvh * group + min(in_group, group - 1);
  const int pos0 = __builtin_amdgcn_readfirstlane(positions[t0]);
  const int my_row = (wave & 3) * 32 + l32, row = min(my_row, count - 1);
  const bool live = in_group < group && (wave & 3) * 32 < count;             // the wave has rows of its own
  elem_t* out_row = out + ((size_t)(t0 + row) * n_heads + head) * HD;
  if (pos0 < 0) {                                  // padding: zeros
    if (live && my_row < count)
      for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); ++d) out_row[d] = from_float(0.0f);
    return;
  }
  const int last = pos0 + count - 1, first = window > 0 ? max(0, pos0 + 1 - window) : 0;        // what any row sees
  const int my_pos = pos0 + row, my_lo = window > 0 ? max(0, my_pos + 1 - window) : 0;
  const int seg_first = kv4_segment_of(first), seg_last = kv4_segment_of(last);
  if (segment >= 0 && (segment < seg_first || segment > seg_last)) return;
  if ((segment >= 0 || seg_first < seg_last) && (slot < 0 || slot >= n_slots)) return;        // (no room for what has to be kept)
  float* state_at = partial + ((size_t)max(slot, 0) * n_heads + head) * Kv4State<HD>::FLOATS;
  const int base = max(first, segment >= 0 ? kv4_segment_start(segment) : 0) / KV4_BLOCK * KV4_BLOCK;
  const int end = segment >= 0 ? min(last, kv4_segment_start(segment + 1) - 1) : last, n_blocks = (end - base) / KV4_BLOCK + 1;
  // what all rows of the tile, of the wave, see
  const int tile_lo = window > 0 ? max(0, last + 1 - window) : 0;
  const int wave_hi = pos0 + (wave & 3) * 32, wave_last = min(wave_hi + 31, last), wave_lo = window > 0 ? max(0, wave_last + 1 - window) : 0;
  const int wave_first = window > 0 ? max(0, wave_hi + 1 - window) : 0;

  const int32_t* table_row = block_table + (size_t)__builtin_amdgcn_readfirstlane(seq_rows[t0]) * table_stride;
  const size_t head_bytes = (size_t)page_size * kv4_row_bytes(HD), page_bytes = head_bytes * n_kv_heads, head_at = head_bytes * kvh;
  const int shift = __builtin_ctz(page_size);
  Kv4Masks masks = kv4_masks();
  auto k_at = [](int b) { return (b & 1) * S::BYTES; };
  auto v_at = [](int b) { return 2 * S::BYTES + (int)((unsigned)b % V_STAGES) * S::BYTES; };
  auto nans_of = [&](int b) { return smem + (2 + V_STAGES) * S::BYTES + (unsigned)b % V_STAGES * S::NANS; };
  // an octet past the tile's last position: its page's
  auto place = [&](int b, int n) { return min(base + b * KV4_BLOCK + 8 * (n * WAVES + wave), last); };
  auto edge = [&](int b) { return base + b * KV4_BLOCK < tile_lo || base + b * KV4_BLOCK + KV4_BLOCK - 1 > pos0; };
  int page[OCTETS];
  Kv4Octet<HD> octets[OCTETS];
  auto look_up = [&](int b) {
#pragma unroll
    for (int n = 0; n < OCTETS; ++n) page[n] = table_row[place(b, n) >> shift];
  };
  auto ask = [&](int b) {
#pragma unroll
    for (int n = 0; n < OCTETS; ++n) kv4_load<HD>(octets[n], k_cache, v_cache, page[n], place(b, n), page_bytes, head_at, page_size, lane);
  };
  auto mend = [&](int b) {
    if (edge(b))
#pragma unroll
      for (int n = 0; n < OCTETS; ++n)
        kv4_edge<HD>(octets[n], n * WAVES + wave, base + b * KV4_BLOCK + 8 * (n * WAVES + wave), first, last, nans_of(b), lane);
  };
  auto unpack = [&](int b, int piece) {
#pragma unroll
    for (int n = 0; n < OCTETS; ++n) kv4_unpack<HD>(octets[n], smem + k_at(b), smem + v_at(b), n * WAVES + wave, piece, masks, lane);
  };
  auto unpack_all = [&](int b) {
#pragma unroll
    for (int piece = 0; piece < KV4_PIECES; ++piece) unpack(b, piece);
  };
  look_up(0);
  ask(0);
  look_up(1);

  u32x4 qf[KS][TERMS];
  float c;
  {
    const elem_t* src = q + (size_t)(t0 + row) * q_stride + (size_t)head * HD + half * 8;
    float x[KS][8], largest = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float a[4], b[4];
      load4_guarded(src + ks * 16, 4, true, a);
      load4_guarded(src + ks * 16 + 4, 4, true, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[ks][i] = a[i];
        x[ks][4 + i] = b[i];
        largest = fmaxf(largest, fmaxf(fabsf(a[i]), fabsf(b[i])));
      }
    }
    largest = fmaxf(largest, __shfl_xor(largest, 32, AXON_WAVE));
    const int by = kv4_query_shift(largest);
    const float up = ldexpf(1.0f, by / 2), up2 = ldexpf(1.0f, by - by / 2);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[ks][i] = x[ks][i] * up * up2;
      kv4_split(x[ks], qf[ks]);
    }
    c = kv4_score_factor(scale, by);
  }
  Kv4State<HD> st;
  f32x16(&o)[DT] = st.o;
  float& l = st.l;
  Kv4Reference ref;
  auto clear = [&]() {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    ref = Kv4Reference{};
    l = 0.0f;
  };

  // (what is asked for past the last block is of the last page, and is not used)
  mend(0);
  unpack_all(0);
  ask(1);
  look_up(2);
  kv4_meet();
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem;
  const int k_row = (l32 & 0x13) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);      // pi
  // the wave's part of a block that none of its rows sees
  auto pass = [&](int b) {
    mend(b + 1);
    unpack_all(b + 1);
    ask(b + 2);
    look_up(b + 3);
    kv4_meet();
  };
  const int from = live ? max(0, wave_first - base) / KV4_BLOCK : n_blocks, to = live ? min((wave_last - base) / KV4_BLOCK, n_blocks - 1) : -1;
  // The second head's waves meet the others between a block's scores and its weights: the matrix cores have the products of the one head's
  // scores while the vector unit has the weights of the other's block before.  (So its values are read while those two blocks on are
  // unpacked.)  Prompts of 3,600 tokens 160 -> 155 us, of 6,000 412 -> 398; of 8,192, where the card's power bounds it, within 1 %.
  const bool late = HPB == 2 && wave >= 4;
  unsigned nan_groups = 0;                         // groups of 32 dims in which the lane's row sees a value that is not a number
  bool kept = false;                               // segments before this one wait in the workspace
  for (int b = 0, seg_end; b < n_blocks; b = seg_end) {
  seg_end = min(n_blocks, (kv4_segment_start(kv4_segment_of(base + b * KV4_BLOCK) + 1) - base) / KV4_BLOCK);
  clear();
  for (; b < min(from, seg_end); ++b) pass(b);
  for (; b <= min(to, seg_end - 1); ++b) {
    const int p0 = base + b * KV4_BLOCK;
    mend(b + 1);
    {
      // A row begins at a multiple of its size, and piece 2 n + half of it is piece `half` with n's bits exclusive-ored in: one instruction
      // from a base each.  The bases are opaque, or the compiler keeps every address in a register across the loop.
      unsigned k_base = lds0 + k_at(b) + k_row * (HD * 2) + ((half ^ S::k_swizzle(k_row)) << 4);
      unsigned v_base = lds0 + v_at(b) + l32 * 128 + ((half ^ S::v_swizzle(l32)) << 4);
      asm volatile("" : "+v"(k_base), "+v"(v_base));
      // The scores, fragments read two groups of products ahead, and the next block unpacked a piece behind each group: the matrix cores
      // work on the group meanwhile.
      constexpr int GROUPS = KS / 2;
      f32x16 s[2];
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[pt][e] = 0.0f;
      u32x4 kf[3][4];
      auto read_k = [&](int g) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const unsigned at = k_base ^ ((2 * g + kk) << 5);
          lds_read16<0>(kf[g % 3][2 * kk], at);
          lds_read16<32 * HD * 2>(kf[g % 3][2 * kk + 1], at);
        }
      };
      read_k(0);
      read_k(1);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        if (g + 2 < GROUPS) read_k(g + 2);
        if (g + 2 < GROUPS) wait_lgkmcnt<8>();
        else if (g + 1 < GROUPS) wait_lgkmcnt<4>();
        else wait_lgkmcnt<0>();
        use_frags<4>(kf[g % 3]);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int n = TERMS - 1; n >= 0; --n)
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) s[pt] = kv4_mma32(kf[g % 3][2 * kk + pt], qf[2 * g + kk][n], s[pt]);
#pragma unroll
        for (int piece = 0; piece < KV4_PIECES / GROUPS; ++piece) unpack(b + 1, g * (KV4_PIECES / GROUPS) + piece);
      }
      ask(b + 2);
      look_up(b + 3);
      if (late) kv4_meet();
      const bool whole = p0 + KV4_BLOCK - 1 <= wave_hi && p0 >= wave_lo;
      if (!whole) {
        int from = p0 + 8 * half;
        asm volatile("" : "+v"(from));
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int p = from + 32 * pt + 16 * (e >> 3) + (e & 7);
            s[pt][e] = p >= my_lo && p <= my_pos ? s[pt][e] : -INFINITY;
          }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx[pt] = fmaxf(mx[pt], s[pt][e]);
      float top = fmaxf(mx[0], mx[1]);
      top = fmaxf(top, __shfl_xor(top, 32, AXON_WAVE));
      const float factor = kv4_raise(ref, top, c);
      if (__any(factor != 1.0f)) {
        l = __fmul_rn(l, factor);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] = __fmul_rn(o[dt][e], factor);
        kv4_refer(ref, c);
      }
      if (__builtin_expect(ref.far, 0)) {
        const float off = kv4_far(ref.score, c) ? ref.score : 0.0f;
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[pt][e] = __fsub_rn(s[pt][e], off);
      }
      // The weights of sixteen positions, then their products with all dims: on those the matrix cores work while the vector unit has the
      // weights of the next sixteen.
      float sum[2] = {0.0f, 0.0f};
      u32x4 vf[2][DT];
      auto read_v = [&](int st) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) lds_read16_step<32 * 128, DT>(vf[st & 1][dt], v_base ^ (st << 5), dt);
      };
      read_v(0);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (st + 1 < 4) read_v(st + 1);
        float w[8];
        u32x4 pf[TERMS];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[st >> 1][8 * (st & 1) + i], c, ref.add));
          sum[i & 1] = __fadd_rn(sum[i & 1], w[i]);
        }
        asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));       // (added here, beside products: else behind the last of them, 1 to 2 % later)
        kv4_split(w, pf);
        if (st + 1 < 4) wait_lgkmcnt<DT>();
        else wait_lgkmcnt<0>();
        use_frags<DT>(vf[st & 1]);
#pragma unroll
        for (int n = TERMS - 1; n >= 0; --n)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] = kv4_mma32(vf[st & 1][dt], pf[n], o[dt]);
      }
      l = __fadd_rn(l, __fadd_rn(sum[0], sum[1]));
      if (edge(b)) {
        const uint64_t low = my_lo <= p0 ? ~0ull : my_lo - p0 > 63 ? 0ull : ~0ull << (my_lo - p0),
                       high = my_pos >= p0 + 63 ? ~0ull : ~(~0ull << max(my_pos - p0 + 1, 0));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          if (*reinterpret_cast<const uint64_t*>(nans_of(b) + 8 * dt) & low & high) nan_groups |= 1u << dt;
      }
    }
    if (!late) kv4_meet();
  }
  for (; b < seg_end; ++b) pass(b);
  if (!live || (segment < 0 && seg_first == seg_last)) continue;
  st.ref = __fmul_rn(ref.score, c);                // (what is folded is compared as log2)
  if (kept) kv4_fold<HD, true>(st, state_at, wave & 3, lane, 0);
  if (seg_end < n_blocks || segment >= 0) {
    kv4_store<HD>(st, state_at, wave & 3, lane, nan_groups);
    nan_groups = 0;
    kept = true;
  }
  }
  if (!live || my_row >= count || segment >= 0) return;
  kv4_store_row<HD>(st, out_row, lane, nan_groups);
}

// tiles [n][columns] = (first token, count, segment or -1 for all that the tile sees, slot of the workspace, kv4_fold_kernel's).
template <int HD, int HPB>
__global__ void __launch_bounds__(256 * HPB, TERMS == 1 || HD == 64 ? 2 : 1)
kv4_prefill_kernel(const elem_t* __restrict__ q, int q_stride, const unsigned char* __restrict__ k_cache,
                   const unsigned char* __restrict__ v_cache, const int32_t* __restrict__ block_table, int table_stride,
                   const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows, elem_t* __restrict__ out,
                   const int32_t* __restrict__ tiles, int columns, float* __restrict__ partial, int n_slots, int n_heads, int n_kv_heads,
                   int page_size, int window, float scale) {
  extern __shared__ __align__(256) unsigned char smem[];
  const int32_t* mine = tiles + columns * blockIdx.y;
  const int t0 = mine[0], count = mine[1], segment = mine[2], slot = mine[3];
  if (count <= 0 || count > KV4_ROWS || segment < -1) return;
  kv4_prefill_tile<HD, HPB>(smem, t0, count, q, q_stride, k_cache, v_cache, block_table, table_stride, positions, seq_rows, out, segment, slot,
                            partial, n_slots, n_heads, n_kv_heads, page_size, window, scale);
}

// The segments of the tiles whose segments had a workgroup each, folded in order: rows of five whose last says how many there are, which lie
// in as many slots from theirs on.  grid (heads, groups of 32 dims, KV4_FOLDS that share the rows); a thread has sixteen dims of a row of the tile,
// half of the group, as kv4_store left them.  Bound by its launch (2.9 us of one that does nothing) and two trips to memory: 5.6 us for
// four tiles of two segments of 28 heads of 128 dims, 13 for eight of up to four.
#define KV4_FOLDS 8
template <int HD>
__global__ void __launch_bounds__(256)
kv4_fold_kernel(elem_t* __restrict__ out, const int32_t* __restrict__ tiles, int n_tiles, const float* __restrict__ partial, int n_slots,
                int n_heads) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, head = blockIdx.x, dt = blockIdx.y, my_row = wave * 32 + (lane & 31);
  const size_t tile = (size_t)n_heads * Kv4State<HD>::FLOATS;
  for (int first = 0, seen = 0; first < n_tiles; first += 64) {
    uint64_t folds = __ballot(first + lane < n_tiles && tiles[5 * (first + lane) + 4] > 0);
    for (; folds != 0; folds &= folds - 1) {
      if (seen++ % KV4_FOLDS != (int)blockIdx.z) continue;
      const int32_t* mine = tiles + 5 * (first + __builtin_ctzll(folds));
      const int t0 = mine[0], count = mine[1], slot = mine[3], segments = mine[4];
      if (count <= 0 || count > KV4_ROWS || slot < 0 || slot > n_slots - segments || wave * 32 >= count) continue;
      const float* at = partial + slot * tile + (size_t)head * Kv4State<HD>::FLOATS;
      Kv4State<32> st;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 v = *reinterpret_cast<const float4*>(at + (((wave * (HD / 32) + dt) * 4 + g) * 64 + lane) * 4);
        st.o[0][4 * g] = v.x; st.o[0][4 * g + 1] = v.y; st.o[0][4 * g + 2] = v.z; st.o[0][4 * g + 3] = v.w;
      }
      const float2 own = *reinterpret_cast<const float2*>(at + KV4_ROWS * HD + (wave * 64 + lane) * 2);
      st.ref = own.x;
      st.l = own.y;
      for (int s = 1; s < segments; ++s) kv4_fold<HD, false>(st, at + s * tile, wave, lane, dt);
      if (my_row < count) kv4_store_row<32>(st, out + ((size_t)(t0 + my_row) * n_heads + head) * HD + dt * 32, lane, 0);
    }
  }
}

// ============================================================================ entry points
// Positions of a chunk of a token that sees `seen` positions.
extern "C" int axk_kv4_decode_chunk(int seen) { return kv4_chunk(seen); }
extern "C" int axk_kv4_decode_item_factor(void) { return KV4_ITEM_FACTOR; }
extern "C" int axk_kv4_prefill_tile(void) { return KV4_ROWS; }

extern "C" long axk_kv4_decode_workspace(int n_tokens, int n_heads, int head_dim, int max_chunks) {
  return (long)n_tokens * n_heads * max_chunks * (head_dim + 2);
}

static int kv4_attention_args(const char* name, const void* q, int q_stride, const void* k_cache, const void* v_cache, const void* out,
                              int n_heads, int n_kv_heads, int head_dim, int page_size, int window, float scale) {
  AXK_REQUIRE(kv4_takes(head_dim, page_size) && n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads <= 65535,
              "%s: head_dim %d, page size %d, %d/%d heads are not taken", name, head_dim, page_size, n_heads, n_kv_heads);
  AXK_REQUIRE(window >= 0 && scale > 0.0f && scale < INFINITY, "%s: window %d, scale %g", name, window, scale);
  AXK_REQUIRE((uintptr_t)q % 16 == 0 && q_stride >= 0 && q_stride * sizeof(elem_t) % 16 == 0 && (uintptr_t)k_cache % 16 == 0 &&
                  (uintptr_t)v_cache % 16 == 0 && (uintptr_t)out % 16 == 0,
              "%s: q (rows %d apart), the caches and out must be 16-byte aligned", name, q_stride);
  return 0;
}

extern "C" int axk_kv4_attention_decode(const void* q, int q_stride, const void* k_cache, const void* v_cache,
                                        const int32_t* block_table, int table_stride, const int32_t* positions,
                                        const int32_t* seq_rows, void* out, const int32_t* token_index, int n_tokens,
                                        const int32_t* work, int n_work, float* partial, int max_chunks, int n_heads, int n_kv_heads,
                                        int head_dim, int page_size, int window, float scale, void* stream) {
  const int rc = kv4_attention_args("kv4_attention_decode", q, q_stride, k_cache, v_cache, out, n_heads, n_kv_heads, head_dim, page_size,
                                    window, scale);
  if (rc != 0) return rc;
  const int sets = ceil_div(n_heads / n_kv_heads, KV4_COLUMNS);
  AXK_REQUIRE(n_tokens >= 0 && n_tokens <= 1 << 20, "kv4_attention_decode: %d tokens", n_tokens);
  AXK_REQUIRE(max_chunks >= 1 && max_chunks <= KV4_ITEM_FACTOR, "kv4_attention_decode: %d chunks of a token (at most %d)", max_chunks,
              KV4_ITEM_FACTOR);
  AXK_REQUIRE(n_work >= 0 && (n_work == 0 || work != nullptr), "kv4_attention_decode: a work list of %d items", n_work);
  if (n_tokens == 0 || n_work == 0) return 0;
  AXK_REQUIRE(partial != nullptr && (uintptr_t)partial % 16 == 0, "kv4_attention_decode: needs its workspace, 16-byte aligned");
  const dim3 units(n_kv_heads * sets, n_work < 65535 ? n_work : 65535, (n_work + 65534) / 65535);
#define LAUNCH(HD)                                                                                                              \
  {                                                                                                                             \
    kv4_decode_kernel<HD><<<units, 64 * KV4_WAVES, 0, (hipStream_t)stream>>>(                                                               \
        (const elem_t*)q, q_stride, (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride,    \
        positions, seq_rows, (elem_t*)out, token_index, n_tokens, work, n_work, partial, max_chunks, n_heads, n_kv_heads, sets, \
        page_size, window, scale);                                                                                              \
  }
  if (head_dim == 64) LAUNCH(64) else LAUNCH(128)
#undef LAUNCH
  AXK_LAUNCH_CHECK("kv4_attention_decode");
  if (max_chunks > 1) {
    const dim3 rows(n_tokens, n_heads);
#define JOIN(HD)                                                                                                                \
  kv4_join_kernel<HD><<<rows, JOIN_SUMS * HD / 4, 0, (hipStream_t)stream>>>(partial, positions, token_index, (elem_t*)out,      \
                                                                            n_tokens, max_chunks, n_heads, window)
    if (head_dim == 64) JOIN(64);
    else JOIN(128);
#undef JOIN
    AXK_LAUNCH_CHECK("kv4_attention_decode");
  }
  return 0;
}

extern "C" int axk_kv4_prefill_segment(int position) { return kv4_segment_of(position); }
extern "C" int axk_kv4_prefill_segment_start(int segment) { return kv4_segment_start(segment); }

// Floats that a slot of the tiles' workspace has.
extern "C" long axk_kv4_prefill_workspace(int n_slots, int n_heads, int head_dim) {
  return (long)n_slots * n_heads * (head_dim == 64 ? Kv4State<64>::FLOATS : Kv4State<128>::FLOATS);
}

// One query head a workgroup while there are up to three a CU, which spread better; beyond that two, which share what is unpacked: 672
// tiles and heads in ragged portions 68 against 73 us, 616 of a prompt of 2,800 tokens 103 against 110, 896 of one of 4,096 199 against
// 190 (28 heads over 4 of 128 dims, the only ones that were timed).  The float32 build has no registers for two.
extern "C" int axk_kv4_prefill_heads(int n_tiles, int n_heads, int n_kv_heads) {
  return AXON_BF16 && n_kv_heads > 0 && n_heads / n_kv_heads >= 2 && (long)n_tiles * n_heads > 768 ? 2 : 1;
}

extern "C" int axk_kv4_attention_prefill(const void* q, int q_stride, const void* k_cache, const void* v_cache,
                                         const int32_t* block_table, int table_stride, const int32_t* positions,
                                         const int32_t* seq_rows, void* out, const int32_t* tiles, int n_tiles, int columns,
                                         float* partial, long partial_floats, int n_heads, int n_kv_heads, int head_dim, int page_size, int window,
                                         float scale, void* stream) {
  const int rc = kv4_attention_args("kv4_attention_prefill", q, q_stride, k_cache, v_cache, out, n_heads, n_kv_heads, head_dim,
                                    page_size, window, scale);
  if (rc != 0) return rc;
  AXK_REQUIRE(n_tiles >= 0 && n_tiles <= 65535 && (n_tiles == 0 || tiles != nullptr), "kv4_attention_prefill: %d tiles (at most 65535)", n_tiles);
  AXK_REQUIRE(columns == 4 || columns == 5, "kv4_attention_prefill: tiles of %d numbers (4, or 5 where some are cut)", columns);
  AXK_REQUIRE(partial_floats >= 0 && (uintptr_t)partial % 16 == 0 && (partial_floats == 0 || partial != nullptr),
              "kv4_attention_prefill: a workspace of %ld floats, 16-byte aligned", partial_floats);
  if (n_tiles == 0) return 0;
  const int group = n_heads / n_kv_heads;
  const long slots = partial_floats / axk_kv4_prefill_workspace(1, n_heads, head_dim);
  const int n_slots = (int)(slots < 1 << 30 ? slots : 1 << 30);
#define LAUNCH(HD, HPB)                                                                                                         \
  {                                                                                                                             \
    constexpr int lds = Kv4Stage<HD>::all(1 + HPB);                                                                                      \
    static uint64_t configured = 0;                                                            /* a bit for each device */      \
    int device = 0;                                                                                                             \
    hipError_t e = hipGetDevice(&device);                                                                                       \
    if (e == hipSuccess && !(configured >> (device & 63) & 1))                                                                  \
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_prefill_kernel<HD, HPB>),                                      \
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);                                                 \
    if (e != hipSuccess) {                                                                                                      \
      axk_set_error("kv4_attention_prefill: cannot reserve %d bytes of LDS: %s", lds, hipGetErrorString(e));                    \
      return -2;                                                                                                                \
    }                                                                                                                           \
    configured |= 1ull << (device & 63);                                                                                        \
    kv4_prefill_kernel<HD, HPB><<<dim3(n_kv_heads * ((group + HPB - 1) / HPB), n_tiles), 256 * HPB, lds, (hipStream_t)stream>>>( \
        (const elem_t*)q, q_stride, (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride,    \
        positions, seq_rows, (elem_t*)out, tiles, columns, partial, n_slots, n_heads, n_kv_heads, page_size, window, scale);    \
  }
#if AXON_BF16
  if (axk_kv4_prefill_heads(n_tiles, n_heads, n_kv_heads) == 2) {
    if (head_dim == 64) LAUNCH(64, 2) else LAUNCH(128, 2)
  } else
#endif
  {
    if (head_dim == 64) LAUNCH(64, 1) else LAUNCH(128, 1)
  }
#undef LAUNCH
  AXK_LAUNCH_CHECK("kv4_attention_prefill");
  if (columns == 5 && n_slots > 0) {
    const dim3 folds(n_heads, head_dim / 32, KV4_FOLDS);
    if (head_dim == 64) kv4_fold_kernel<64><<<folds, 256, 0, (hipStream_t)stream>>>((elem_t*)out, tiles, n_tiles, partial, n_slots, n_heads);
    else kv4_fold_kernel<128><<<folds, 256, 0, (hipStream_t)stream>>>((elem_t*)out, tiles, n_tiles, partial, n_slots, n_heads);
    AXK_LAUNCH_CHECK("kv4_attention_prefill");
  }
  return 0;
}
