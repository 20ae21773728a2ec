// Causal attention over a cache held in 4 bits (kv4.h has the format), on the half-precision matrix cores: they take every
// number of the cache exactly, so nothing is rounded on the way from the cache into a product.
//
// Queries go there as half precision too, scaled by a power of two that brings a row's largest to 2^14 .. 2^15 (the score's
// factor takes it back): bfloat16's eight bits fit with room, float32's 24 are three terms, each the rounding of what the ones before
// it left, and three products.  The softmax's weights 2^(s - m + 14) are rounded to half precision, eleven bits (bfloat16
// build; 2^-12 of a weight, an eighth of what the output's rounding takes), or are three such terms (float32 build).
// Scores, maxima, sums and outputs are 32 bits.
#include <math.h>

#include "api.h"
#include "common.h"
#include "instances.h"
#include "kv4.h"

#define KV4_BLOCK 64               // positions of a block: one pass of products, one maximum
#define KV4_CHUNK 256              // positions of one item of the decoding kernel's work list
#define KV4_ITEM_FACTOR 1024       // the most chunks of a token; the factor of the token's slot in an item
#define KV4_COLUMNS 16             // query heads of a key head that a wave takes at a time
#define KV4_SIDE_UNITS 2048        // fewer units than this: a wave a block
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
      out[n][i] = __builtin_bit_cast(unsigned, h);
      if (n + 1 < TERMS) {
        rest[2 * i] = __fsub_rn(rest[2 * i], (float)h[0]);
        rest[2 * i + 1] = __fsub_rn(rest[2 * i + 1], (float)h[1]);
      }
    }
  }
}

// The power of two that brings `largest` (of a row of queries) to 2^14 .. 2^15; 0 for a row of zeros or of what is not finite.
__device__ __forceinline__ int kv4_query_shift(float largest) {
  return largest > 0.0f && largest < INFINITY ? 14 - ilogbf(largest) : 0;
}

// A chunk's largest score (log2), sum of weights and output, folded into what its blocks before gave.
__device__ __forceinline__ void kv4_fold(float& m, float& l, float m_b, float l_b, float& a, float& b) {
  const float mn = fmaxf(m, m_b), ref = mn == -INFINITY ? 0.0f : mn;
  a = __builtin_amdgcn_exp2f(__fsub_rn(m, ref));
  b = __builtin_amdgcn_exp2f(__fsub_rn(m_b, ref));
  l = __builtin_fmaf(l, a, __fmul_rn(l_b, b));
  m = mn;
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
struct Kv4Block {                  // a block's bytes on their way: nothing of it is unpacked
  static constexpr int KW = HD / 32, VW = HD / 64;      // words of K a row, sixteens of bytes of V^T an octet
  unsigned k[4][KW];
  unsigned k_scale[4];
  uint4 v[2][VW];
  uint4 v_scale[2];
};

template <int HD>
__device__ __forceinline__ void kv4_load(Kv4Block<HD>& blk, const unsigned char* k_cache, const unsigned char* v_cache, int pages, int c0, int b,
                                         size_t page_bytes, size_t head_at, int page_size, int lane) {
  constexpr int KW = HD / 32, VW = HD / 64;
  const int l16 = lane & 15, h = lane >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int ko = 8 * b + 4 * u + (l16 >> 2), vo = 8 * b + 4 * u + h;      // octets of the chunk
    const unsigned char* kp = k_cache + __shfl(pages, ko, AXON_WAVE) * page_bytes + head_at;
    const unsigned char* vp = v_cache + __shfl(pages, vo, AXON_WAVE) * page_bytes + head_at;
    const int k_slot = (c0 + 8 * ko) & (page_size - 1), v_octet = ((c0 + 8 * vo) & (page_size - 1)) >> 3;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int slot = k_slot + 4 * v + (l16 & 3);
      const unsigned char* at = kp + slot * (HD / 2) + h * (HD / 8);
      if constexpr (KW == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(at);
        blk.k[2 * u + v][0] = w.x; blk.k[2 * u + v][1] = w.y; blk.k[2 * u + v][2] = w.z; blk.k[2 * u + v][3] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(at);
        blk.k[2 * u + v][0] = w.x; blk.k[2 * u + v][1] = w.y;
      }
      blk.k_scale[2 * u + v] = reinterpret_cast<const uint16_t*>(kp + page_size * (HD / 2))[slot * (HD / 32) + h * (HD / 4) / 32];
    }
    const uint4* words = reinterpret_cast<const uint4*>(vp + ((size_t)v_octet * HD + l16 * (HD / 16)) * 4);
#pragma unroll
    for (int i = 0; i < VW; ++i) blk.v[u][i] = words[i];
    blk.v_scale[u] = *reinterpret_cast<const uint4*>(vp + page_size * (HD / 2) + (v_octet * (HD / 32) + l16 * (HD / 16) / 32) * 16);
  }
}

// A block's (m, l, o): o[dt][r] is dim HD/16 (4 h + r) + dt of column l16.  p0: its first position; positions lo .. pos are seen.
template <int HD>
__device__ __forceinline__ void kv4_block(const Kv4Block<HD>& blk, const u32x4 (&qf)[HD / 32][TERMS], int p0, int lo, int pos, float c,
                                          int lane, float& m_b, float& l_b, f32x4 (&o)[HD / 16]) {
  constexpr int KW = HD / 32, DT = HD / 16;
  const int h = lane >> 4;
  f32x4 s[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    half2_t sc[4], cc[4];
    kv4_pair_scale(blk.k_scale[t] | blk.k_scale[t] << 16, sc[0], cc[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) { sc[i] = sc[0]; cc[i] = cc[0]; }
    s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const u32x4 a = kv4_operand(blk.k[t][j], sc, cc);
#pragma unroll
      for (int n = TERMS - 1; n >= 0; --n) s[t] = kv4_mma(a, qf[j][n], s[t]);
    }
  }
  const bool whole = p0 >= lo && p0 + KV4_BLOCK - 1 <= pos;          // the same for the wave
  if (!whole) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = p0 + 32 * (t >> 1) + 8 * h + 4 * (t & 1) + r;
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
  m_b = __fmul_rn(mx, c);
  const float ref = m_b == -INFINITY ? 0.0f : __fsub_rn(14.0f, m_b);
  float sum = 0.0f;
  u32x4 pf[2][TERMS];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * u + (i >> 2)][i & 3], c, ref));
      sum = __fadd_rn(sum, w[i]);
    }
    kv4_split(w, pf[u]);
  }
  sum = __fadd_rn(sum, __shfl_xor(sum, 16, AXON_WAVE));
  l_b = __fadd_rn(sum, __shfl_xor(sum, 32, AXON_WAVE));
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const unsigned metas[4] = {blk.v_scale[u].x, blk.v_scale[u].y, blk.v_scale[u].z, blk.v_scale[u].w};
    half2_t sc[4], cc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned keep = 0xffffffffu;
      if (!whole) {
        // a weight of zero times what an unseen place holds has to be zero, whatever that is
        const int p = p0 + 32 * u + 8 * h + 2 * i;
        keep = (p >= lo && p <= pos ? 0x0000ffffu : 0u) | (p + 1 >= lo && p + 1 <= pos ? 0xffff0000u : 0u);
      }
      kv4_pair_scale(metas[i] & keep, sc[i], cc[i]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const uint4 four = blk.v[u][dt / 4];
      const unsigned word = dt % 4 == 0 ? four.x : dt % 4 == 1 ? four.y : dt % 4 == 2 ? four.z : four.w;
      const u32x4 a = kv4_operand(word, sc, cc);
#pragma unroll
      for (int n = TERMS - 1; n >= 0; --n) o[dt] = kv4_mma(a, pf[u][n], o[dt]);
    }
  }
}

// The wave's queries as operands: column l16 (zeros past `columns`), dims h HD/4 + 8 j + {0 .. 7}.  Returns the score's factor.
template <int HD>
__device__ __forceinline__ float kv4_queries(const elem_t* row, int columns, float scale, int lane, u32x4 (&qf)[HD / 32][TERMS]) {
  constexpr int KW = HD / 32;
  const int l16 = lane & 15, h = lane >> 4;
  float x[KW][8], largest = 0.0f;
#pragma unroll
  for (int j = 0; j < KW; ++j) {
    const elem_t* src = row + (size_t)min(l16, columns - 1) * HD + h * (HD / 4) + 8 * j;
    float a[4], b[4];
    load4_guarded(src, 4, true, a);
    load4_guarded(src + 4, 4, true, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[j][i] = a[i];
      x[j][4 + i] = b[i];
      largest = fmaxf(largest, fmaxf(fabsf(a[i]), fabsf(b[i])));
    }
  }
  largest = fmaxf(largest, __shfl_xor(largest, 16, AXON_WAVE));
  largest = fmaxf(largest, __shfl_xor(largest, 32, AXON_WAVE));
  const int shift = kv4_query_shift(largest);
#pragma unroll
  for (int j = 0; j < KW; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[j][i] = l16 < columns ? ldexpf(x[j][i], shift) : 0.0f;
    kv4_split(x[j], qf[j]);
  }
  return ldexpf(scale * LOG2E, -shift);
}

// A unit is a chunk of a token and a set of up to sixteen query heads of a key head.  SIDE 1: a wave a unit, its four blocks one
// after the other; 4: a wave a block, folded in the same order through LDS: the same bits.  Of a token of one chunk the
// output is stored at once; else (o, m, l) go to `partial` ([slot][head][chunk][HD], then [slot][head][chunk][2]).
template <int HD, int SIDE>
__global__ void __launch_bounds__(64 * SIDE)
kv4_decode_kernel(const elem_t* __restrict__ q, int q_stride, const unsigned char* __restrict__ k_cache,
                  const unsigned char* __restrict__ v_cache, const int32_t* __restrict__ block_table, int table_stride,
                  const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows, elem_t* __restrict__ out,
                  const int32_t* __restrict__ token_index, int n_tokens, const int32_t* __restrict__ work, float* __restrict__ partial,
                  int max_chunks, int n_heads, int n_kv_heads, int sets, int page_size, int window, float scale) {
  constexpr int DT = HD / 16;
  const int lane = threadIdx.x & 63, wave = SIDE == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_item = n_kv_heads * sets, item = work[blockIdx.x / per_item];
  if (item < 0) return;                              // padding of the list
  const int slot = item / KV4_ITEM_FACTOR, chunk = item % KV4_ITEM_FACTOR;
  if (slot >= n_tokens || chunk >= max_chunks) return;
  const int kvh = blockIdx.x % per_item / sets, set = blockIdx.x % sets;
  const int group = n_heads / n_kv_heads, head0 = kvh * group + set * KV4_COLUMNS, columns = min(KV4_COLUMNS, group - set * KV4_COLUMNS);
  const int t = token_index ? token_index[slot] : slot, pos = positions[t];
  elem_t* out_row = out + ((size_t)t * n_heads + head0) * HD;
  if (pos < 0) {                                     // padding of the batch: zeros
    if (chunk == 0)
      for (int i = threadIdx.x; i < columns * HD; i += 64 * SIDE) out_row[i] = from_float(0.0f);
    return;
  }
  const int lo = window > 0 ? max(0, pos + 1 - window) : 0;
  const int first_chunk = lo / KV4_CHUNK, n_chunks = pos / KV4_CHUNK - first_chunk + 1;
  if (chunk >= n_chunks) return;
  const int c0 = (first_chunk + chunk) * KV4_CHUNK;
  // the pages of the chunk's 32 octets, looked up once (places past the token: its own last page)
  const int32_t* table_row = block_table + (size_t)seq_rows[t] * table_stride;
  const int pages = table_row[min(c0 + 8 * (lane & 31), pos) / page_size];
  const size_t head_bytes = (size_t)page_size * kv4_row_bytes(HD), page_bytes = head_bytes * n_kv_heads, head_at = head_bytes * kvh;
  const int b_first = max(0, lo - c0) / KV4_BLOCK, b_last = min(KV4_CHUNK - 1, pos - c0) / KV4_BLOCK;

  Kv4Block<HD> blk;
  const int b0 = SIDE == 1 ? b_first : wave;
  if (b0 <= b_last) kv4_load<HD>(blk, k_cache, v_cache, pages, c0, b0, page_bytes, head_at, page_size, lane);
  u32x4 qf[HD / 32][TERMS];
  const float c = kv4_queries<HD>(q + (size_t)t * q_stride + (size_t)head0 * HD, columns, scale, lane, qf);
  const int l16 = lane & 15, h = lane >> 4;
  const bool alone = n_chunks == 1;
  const size_t row = ((size_t)slot * n_heads + head0) * max_chunks + chunk;      // of column 0; a column further: max_chunks
  float* ml = partial + (size_t)n_tokens * n_heads * max_chunks * HD;
  if constexpr (SIDE == 1) {
    float m = -INFINITY, l = 0.0f;
    f32x4 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = b0; b <= b_last; ++b) {
      Kv4Block<HD> next = blk;
      if (b < b_last) kv4_load<HD>(next, k_cache, v_cache, pages, c0, b + 1, page_bytes, head_at, page_size, lane);
      float m_b, l_b, fa, fb;
      f32x4 o[DT];
      kv4_block<HD>(blk, qf, c0 + b * KV4_BLOCK, lo, pos, c, lane, m_b, l_b, o);
      kv4_fold(m, l, m_b, l_b, fa, fb);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[dt][r] = __builtin_fmaf(acc[dt][r], fa, __fmul_rn(o[dt][r], fb));
      blk = next;
    }
    if (l16 >= columns) return;
    if (alone) {
      const float inv = __fdiv_rn(1.0f, l);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) out_row[l16 * HD + DT * (4 * h + r) + dt] = from_float(__fmul_rn(acc[dt][r], inv));
      return;
    }
    float* dst = partial + (row + (size_t)l16 * max_chunks) * HD + DT * 4 * h;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int dt = 0; dt < DT; dt += 4)
        *reinterpret_cast<float4*>(dst + DT * r + dt) = make_float4(acc[dt][r], acc[dt + 1][r], acc[dt + 2][r], acc[dt + 3][r]);
    if (h == 0) *reinterpret_cast<float2*>(ml + 2 * (row + (size_t)l16 * max_chunks)) = make_float2(m, l);
  } else {
    __shared__ __align__(16) float o_of[SIDE][KV4_COLUMNS][HD + 4];
    __shared__ float m_of[SIDE][KV4_COLUMNS], l_of[SIDE][KV4_COLUMNS];
    if (wave >= b_first && wave <= b_last) {
      float m_b, l_b;
      f32x4 o[DT];
      kv4_block<HD>(blk, qf, c0 + wave * KV4_BLOCK, lo, pos, c, lane, m_b, l_b, o);
      if (l16 < columns) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int dt = 0; dt < DT; dt += 4)
            *reinterpret_cast<float4*>(&o_of[wave][l16][DT * (4 * h + r) + dt]) = make_float4(o[dt][r], o[dt + 1][r], o[dt + 2][r], o[dt + 3][r]);
        if (h == 0) {
          m_of[wave][l16] = m_b;
          l_of[wave][l16] = l_b;
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns * (HD / 4); i += 64 * SIDE) {
      const int col = i / (HD / 4), d = i % (HD / 4) * 4;
      float m = -INFINITY, l = 0.0f;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int b = b_first; b <= b_last; ++b) {
        float fa, fb;
        kv4_fold(m, l, m_of[b][col], l_of[b][col], fa, fb);
        const float4 o4 = *reinterpret_cast<const float4*>(&o_of[b][col][d]);
        acc = f32x4{__builtin_fmaf(acc[0], fa, __fmul_rn(o4.x, fb)), __builtin_fmaf(acc[1], fa, __fmul_rn(o4.y, fb)),
                    __builtin_fmaf(acc[2], fa, __fmul_rn(o4.z, fb)), __builtin_fmaf(acc[3], fa, __fmul_rn(o4.w, fb))};
      }
      if (alone) {
        const float inv = __fdiv_rn(1.0f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) out_row[col * HD + d + e] = from_float(__fmul_rn(acc[e], inv));
      } else {
        *reinterpret_cast<float4*>(partial + (row + (size_t)col * max_chunks) * HD + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) *reinterpret_cast<float2*>(ml + 2 * (row + (size_t)col * max_chunks)) = make_float2(m, l);
      }
    }
  }
}

// A token's chunks joined: with M the largest of their maxima, out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M), four sums side by
// side over every fourth chunk, ascending, added in order.  grid (tokens, heads), 4 HD threads.
template <int HD>
__global__ void __launch_bounds__(4 * HD)
kv4_join_kernel(const float* __restrict__ partial, const int32_t* __restrict__ positions, const int32_t* __restrict__ token_index,
                elem_t* __restrict__ out, int n_tokens, int max_chunks, int n_heads, int window) {
  __shared__ float factor[KV4_ITEM_FACTOR], sums[4][HD], l_sums[4], wave_max[4 * HD / 64];
  const int slot = blockIdx.x, head = blockIdx.y, t = token_index ? token_index[slot] : slot, pos = positions[t];
  if (pos < 0) return;
  const int lo = window > 0 ? max(0, pos + 1 - window) : 0, n = min(pos / KV4_CHUNK - lo / KV4_CHUNK + 1, max_chunks);
  if (n == 1) return;                                // stored by the chunk's own block
  const size_t row = ((size_t)slot * n_heads + head) * max_chunks;
  const float* ml = partial + (size_t)n_tokens * n_heads * max_chunks * HD + 2 * row;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < n; i += 4 * HD) mx = fmaxf(mx, ml[2 * i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, AXON_WAVE));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x / 64] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4 * HD / 64; ++w) mx = fmaxf(mx, wave_max[w]);
  const float ref = mx == -INFINITY ? 0.0f : mx;
  for (int i = threadIdx.x; i < n; i += 4 * HD) factor[i] = __builtin_amdgcn_exp2f(__fsub_rn(ml[2 * i], ref));
  __syncthreads();
  const int d = threadIdx.x % HD, part = threadIdx.x / HD;
  float o = 0.0f, l = 0.0f;
  for (int i = part; i < n; i += 4) o = __builtin_fmaf(partial[(row + i) * HD + d], factor[i], o);
  if (d == 0)
    for (int i = part; i < n; i += 4) l = __builtin_fmaf(ml[2 * i + 1], factor[i], l);
  sums[part][d] = o;
  if (d == 0) l_sums[part] = l;
  __syncthreads();
  if (part != 0) return;
  const float total = __fadd_rn(__fadd_rn(sums[0][d], sums[1][d]), __fadd_rn(sums[2][d], sums[3][d]));
  const float weight = __fadd_rn(__fadd_rn(l_sums[0], l_sums[1]), __fadd_rn(l_sums[2], l_sums[3]));
  out[((size_t)t * n_heads + head) * HD + d] = from_float(__fmul_rn(total, __fdiv_rn(1.0f, weight)));
}

// ============================================================================ prompt portions
__device__ inline void kv4_attend(const elem_t* q, long q_stride, const unsigned char* k_cache, const unsigned char* v_cache,
                                  const int32_t* block_table, int table_stride, const int32_t* positions, const int32_t* seq_rows,
                                  elem_t* out, int t, int qh, int n_heads, int n_kv_heads, int head_dim, int page_size, int window,
                                  float scale, float* qs, float* es) {
  const int lane = threadIdx.x, kvh = qh / (n_heads / n_kv_heads), pos = positions[t];
  elem_t* orow = out + ((size_t)t * n_heads + qh) * head_dim;
  if (pos < 0) {
    for (int d = lane; d < head_dim; d += AXON_WAVE) orow[d] = from_float(0.0f);
    return;
  }
  const int lo = window > 0 ? max(0, pos + 1 - window) : 0;
  const int32_t* table_row = block_table + (size_t)seq_rows[t] * table_stride;
  for (int d = lane; d < head_dim; d += AXON_WAVE) qs[d] = to_float(q[t * q_stride + (size_t)qh * head_dim + d]);
  __syncthreads();
  const size_t head_bytes = (size_t)page_size * kv4_row_bytes(head_dim);
  float M = -INFINITY, L = 0.0f, O[2] = {0.0f, 0.0f};
  for (int b0 = lo / 64 * 64; b0 <= pos; b0 += 64) {
    const int p = b0 + lane;
    const bool live = p >= lo && p <= pos;
    float s = -INFINITY;
    if (live) {
      const unsigned char* base = k_cache + ((size_t)table_row[p / page_size] * n_kv_heads + kvh) * head_bytes;
      const int slot = p % page_size;
      float dot = 0.0f;
      for (int w = 0; w < head_dim / 8; ++w) {
        const unsigned word = reinterpret_cast<const unsigned*>(base)[slot * (head_dim / 8) + w];
        const unsigned meta = reinterpret_cast<const uint16_t*>(base + page_size * head_dim / 2)[slot * (head_dim / 32) + w / 4];
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = fmaf(qs[8 * w + i], kv4_value(__builtin_rotateright32(word, kv4_place(i)) & 15u, meta), dot);
      }
      s = dot * scale;
    }
    const float mn = fmaxf(M, wave_max(s));
    const float e = live ? expf(s - mn) : 0.0f, a = M == -INFINITY ? 0.0f : expf(M - mn);
    L = fmaf(L, a, wave_sum(e));
    M = mn;
    es[lane] = e;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = lane + i * AXON_WAVE;
      if (d >= head_dim) continue;
      O[i] *= a;
      for (int j = max(lo - b0, 0); j <= min(pos - b0, 63); ++j) {
        const int pj = b0 + j, slot = pj % page_size;
        const unsigned char* base = v_cache + ((size_t)table_row[pj / page_size] * n_kv_heads + kvh) * head_bytes;
        const unsigned word = reinterpret_cast<const unsigned*>(base)[(slot / 8) * head_dim + d];
        const unsigned meta =
            reinterpret_cast<const uint16_t*>(base + page_size * head_dim / 2)[((slot / 8) * (head_dim / 32) + d / 32) * 8 + slot % 8];
        O[i] = fmaf(es[j], kv4_value(__builtin_rotateright32(word, kv4_place(slot & 7)) & 15u, meta), O[i]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + i * AXON_WAVE < head_dim) orow[lane + i * AXON_WAVE] = from_float(__fdiv_rn(O[i], L));
}

__global__ void __launch_bounds__(AXON_WAVE)
kv4_attention_kernel(const elem_t* __restrict__ q, long q_stride, const unsigned char* __restrict__ k_cache,
                     const unsigned char* __restrict__ v_cache, const int32_t* __restrict__ block_table, int table_stride,
                     const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows, elem_t* __restrict__ out,
                     const int32_t* __restrict__ token_index, const int32_t* __restrict__ tiles, int n_heads, int n_kv_heads,
                     int head_dim, int page_size, int window, float scale) {
  __shared__ float qs[128], es[AXON_WAVE];
  int t = blockIdx.x;
  if (tiles) {
    const int32_t* mine = tiles + 4 * (blockIdx.x / 256) + 2 * (blockIdx.x / 128 % 2);
    if ((int)(blockIdx.x % 128) >= mine[1]) return;
    t = mine[0] + blockIdx.x % 128;
  } 
  kv4_attend(q, q_stride, k_cache, v_cache, block_table, table_stride, positions, seq_rows, out, t, blockIdx.y, n_heads, n_kv_heads,
             head_dim, page_size, window, scale, qs, es);
}

// ============================================================================ entry points
extern "C" int axk_kv4_decode_chunk(void) { return KV4_CHUNK; }
extern "C" int axk_kv4_decode_item_factor(void) { return KV4_ITEM_FACTOR; }
extern "C" int axk_kv4_prefill_tile(void) { return 128; }

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
  AXK_REQUIRE(max_chunks >= 1 && max_chunks <= KV4_ITEM_FACTOR, "kv4_attention_decode: %d chunks of %d positions (at most %d)", max_chunks,
              KV4_CHUNK, KV4_ITEM_FACTOR);
  AXK_REQUIRE(n_work >= 0 && (n_work == 0 || work != nullptr) && (long)n_work * n_kv_heads * sets < (1l << 31),
              "kv4_attention_decode: a work list of %d items", n_work);
  AXK_REQUIRE(partial != nullptr && (uintptr_t)partial % 16 == 0, "kv4_attention_decode: needs its workspace, 16-byte aligned");
  if (n_tokens == 0 || n_work == 0) return 0;
  const unsigned units = (unsigned)n_work * n_kv_heads * sets;
  const bool side = units < KV4_SIDE_UNITS;
#define LAUNCH(HD, SIDE)                                                                                                        \
  {                                                                                                                             \
    AXK_INSTANCE(INST_KV4_DECODE, HD, SIDE);                                                                                    \
    kv4_decode_kernel<HD, SIDE><<<units, 64 * SIDE, 0, (hipStream_t)stream>>>(                                                  \
        (const elem_t*)q, q_stride, (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride,    \
        positions, seq_rows, (elem_t*)out, token_index, n_tokens, work, partial, max_chunks, n_heads, n_kv_heads, sets,         \
        page_size, window, scale);                                                                                              \
  }
  if (head_dim == 64) { if (side) LAUNCH(64, 4) else LAUNCH(64, 1) }
  else { if (side) LAUNCH(128, 4) else LAUNCH(128, 1) }
#undef LAUNCH
  AXK_LAUNCH_CHECK("kv4_attention_decode");
  if (max_chunks > 1) {
    if (head_dim == 64)
      kv4_join_kernel<64><<<dim3(n_tokens, n_heads), 256, 0, (hipStream_t)stream>>>(partial, positions, token_index, (elem_t*)out, n_tokens,
                                                                                    max_chunks, n_heads, window);
    else
      kv4_join_kernel<128><<<dim3(n_tokens, n_heads), 512, 0, (hipStream_t)stream>>>(partial, positions, token_index, (elem_t*)out,
                                                                                     n_tokens, max_chunks, n_heads, window);
    AXK_LAUNCH_CHECK("kv4_attention_decode");
  }
  return 0;
}

extern "C" int axk_kv4_attention_prefill(const void* q, int q_stride, const void* k_cache, const void* v_cache,
                                         const int32_t* block_table, int table_stride, const int32_t* positions,
                                         const int32_t* seq_rows, void* out, const int32_t* tiles, int n_tiles, int n_heads,
                                         int n_kv_heads, int head_dim, int page_size, int window, float scale, void* stream) {
  const int rc = kv4_attention_args("kv4_attention_prefill", q, q_stride, k_cache, v_cache, out, n_heads, n_kv_heads, head_dim,
                                    page_size, window, scale);
  if (rc != 0) return rc;
  AXK_REQUIRE(n_tiles >= 0 && n_tiles < (1 << 22), "kv4_attention_prefill: %d tiles", n_tiles);
  if (n_tiles == 0) return 0;
  kv4_attention_kernel<<<dim3(n_tiles * 256, n_heads), AXON_WAVE, 0, (hipStream_t)stream>>>(
      (const elem_t*)q, q_stride, (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride, positions,
      seq_rows, (elem_t*)out, nullptr, tiles, n_heads, n_kv_heads, head_dim, page_size, window, scale);
  AXK_LAUNCH_CHECK("kv4_attention_prefill");
  return 0;
}
