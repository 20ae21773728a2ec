// Causal attention over a cache held in 4 bits (kv4.h has the format): a wave a (token, query head), positions in blocks of 64
// with a running maximum and sum.
#include <math.h>

#include "api.h"
#include "common.h"
#include "kv4.h"

#define KV4_CHUNK 256              // positions of one item of the decoding kernel's work list
#define KV4_ITEM_FACTOR 1024       // the most chunks of a token; the factor of the token's slot in an item

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
  } else if (token_index) {
    t = token_index[t];
  }
  kv4_attend(q, q_stride, k_cache, v_cache, block_table, table_stride, positions, seq_rows, out, t, blockIdx.y, n_heads, n_kv_heads,
             head_dim, page_size, window, scale, qs, es);
}

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
  AXK_REQUIRE(n_tokens >= 0 && n_tokens <= 65535, "kv4_attention_decode: %d tokens", n_tokens);
  if (n_tokens == 0) return 0;
  kv4_attention_kernel<<<dim3(n_tokens, n_heads), AXON_WAVE, 0, (hipStream_t)stream>>>(
      (const elem_t*)q, q_stride, (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride, positions,
      seq_rows, (elem_t*)out, token_index, nullptr, n_heads, n_kv_heads, head_dim, page_size, window, scale);
  AXK_LAUNCH_CHECK("kv4_attention_decode");
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
