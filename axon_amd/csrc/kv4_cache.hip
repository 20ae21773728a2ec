// Writing the 4-bit cache (with the rotary encoding of the rows that are stored) and reading rows of it back.  The format and
// its arithmetic are in kv4.h.
#include <math.h>

#include "api.h"
#include "common.h"
#include "kv4.h"

// Eight neighbouring numbers of a row, 16-byte aligned (bfloat16) or 32 (float32).
__device__ inline void load8(const elem_t* p, float (&v)[8]) {
  load4_guarded(p, 4, true, v);
  float w[4];
  load4_guarded(p + 4, 4, true, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[4 + i] = w[i];
}

__device__ inline void store8(elem_t* p, const float (&v)[8]) {
#if AXON_BF16
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
#else
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
#endif
}

// The tokens from t on that lie in one octet of slots of one request, one position behind the other: 0 if t continues such a
// run (its first token's thread has it), or is padding (a negative position).
__device__ inline int octet_run(const int32_t* positions, const int32_t* seq_rows, int t, int n_tokens) {
  const int pos = positions[t], row = seq_rows[t];
  if (pos < 0) return 0;
  if ((pos & 7) != 0 && t > 0 && positions[t - 1] == pos - 1 && seq_rows[t - 1] == row) return 0;
  int n = 1;
  while (n < 8 - (pos & 7) && t + n < n_tokens && positions[t + n] == pos + n && seq_rows[t + n] == row) ++n;
  return n;
}

// The scale word of a group of 32 dims, eight of them in each of four neighbouring lanes, and the lane's eight numbers.
__device__ inline unsigned kv4_quantise8(const float (&x)[8], unsigned (&n)[8]) {
  float lo = 0.0f, hi = 0.0f;
  int bad = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad |= !(fabsf(x[i]) < INFINITY);
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, off, AXON_WAVE));
    hi = fmaxf(hi, __shfl_xor(hi, off, AXON_WAVE));
    bad |= __shfl_xor(bad, off, AXON_WAVE);
  }
  const int bits = kv4_scale_bits(__fsub_rn(hi, lo));
  const float s = kv4_scale_of(bits);
  if (bad || bits == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = 0;
    return bad ? KV4_NAN : 0;
  }
  const float z = fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.0f), 15.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = (unsigned)fminf(fmaxf(__fadd_rn(rintf(__fdiv_rn(x[i], s)), z), 0.0f), 15.0f);
  return bits | (unsigned)z;
}

// Dims c0 .. c0 + 7 of a head's row behind the rotation (rotate-half on the first rotary_dim dims; half a multiple of 8).
__device__ inline void rotated8(const elem_t* head, const float* tab, int c0, int rotary_dim, float (&out)[8]) {
  load8(head + c0, out);
  if (c0 >= rotary_dim) return;
  const int half = rotary_dim / 2;
  const bool upper = c0 >= half;
  const int i0 = upper ? c0 - half : c0;
  float other[8];
  load8(head + (upper ? c0 - half : c0 + half), other);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = tab[2 * (i0 + i)], c = tab[2 * (i0 + i) + 1];
    out[i] = upper ? __fadd_rn(__fmul_rn(other[i], s), __fmul_rn(out[i], c)) : __fsub_rn(__fmul_rn(out[i], c), __fmul_rn(other[i], s));
  }
}

// A block a token: its queries (a thread the eight pairs of dims i .. i + 7 and i + half .., or eight dims behind the rotated
// ones), its keys (a thread a word) and, at the first token of an octet of slots, the values of all tokens of the octet that
// the step brings (a thread eight dims of up to eight positions).
__global__ void __launch_bounds__(256)
rope_kv4_write_kernel(const elem_t* qkv, long qkv_stride, elem_t* q_out, long q_stride, const float* __restrict__ table,
                      const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows,
                      const int32_t* __restrict__ block_table, int table_stride, unsigned char* __restrict__ k_cache,
                      unsigned char* __restrict__ v_cache, int n_tokens, int n_heads, int n_kv_heads, int head_dim, int rotary_dim,
                      int page_size, int write_kv) {
  const int t = blockIdx.x, half = rotary_dim / 2;
  const elem_t* row = qkv + (size_t)t * qkv_stride;
  const float* tab = table + (size_t)t * half * 2;
  const int q_units = half / 8 + (head_dim - rotary_dim) / 8;
  for (int u = threadIdx.x; u < n_heads * q_units; u += 256) {
    const int head = u / q_units, c = u % q_units;
    const elem_t* src = row + head * head_dim;
    elem_t* dst = q_out + (size_t)t * q_stride + head * head_dim;
    if (c < half / 8) {
      float a[8], b[8];
      load8(src + 8 * c, a);
      load8(src + half + 8 * c, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = tab[2 * (8 * c + i)], co = tab[2 * (8 * c + i) + 1], x = a[i];
        a[i] = __fsub_rn(__fmul_rn(x, co), __fmul_rn(b[i], s));
        b[i] = __fadd_rn(__fmul_rn(x, s), __fmul_rn(b[i], co));
      }
      store8(dst + 8 * c, a);
      store8(dst + half + 8 * c, b);
    } else {
      float a[8];
      const int d = rotary_dim + 8 * (c - half / 8);
      load8(src + d, a);
      store8(dst + d, a);
    }
  }
  if (!write_kv) return;
  const int pos = positions[t];
  if (pos < 0) return;                                       // padding
  const int words = head_dim / 8, kv_units = n_kv_heads * words;
  const size_t head_bytes = (size_t)page_size * kv4_row_bytes(head_dim);
  const int page = block_table[(size_t)seq_rows[t] * table_stride + pos / page_size], slot = pos % page_size;
  const int run = octet_run(positions, seq_rows, t, n_tokens);
  for (int u = threadIdx.x; u < 2 * kv_units; u += 256) {      // (a group's four lanes are in it together: words come in fours)
    const bool is_v = u >= kv_units;
    if (is_v && run == 0) break;
    const int w = is_v ? u - kv_units : u, kvh = w / words, c0 = w % words * 8;
    if (!is_v) {
      float x[8];
      unsigned n[8];
      rotated8(row + (n_heads + kvh) * head_dim, tab, c0, rotary_dim, x);
      const unsigned meta = kv4_quantise8(x, n);
      unsigned word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) word |= __builtin_rotateleft32(n[i], kv4_place(i));
      unsigned char* base = k_cache + ((size_t)page * n_kv_heads + kvh) * head_bytes;
      reinterpret_cast<unsigned*>(base)[slot * words + c0 / 8] = word;
      if (c0 % 32 == 0)
        reinterpret_cast<uint16_t*>(base + page_size * head_dim / 2)[slot * (head_dim / 32) + c0 / 32] = (uint16_t)meta;
      continue;
    }
    unsigned char* base = v_cache + ((size_t)page * n_kv_heads + kvh) * head_bytes;
    uint16_t* scales = reinterpret_cast<uint16_t*>(base + page_size * head_dim / 2) + ((slot / 8) * (head_dim / 32) + c0 / 32) * 8;
    unsigned word[8], mask = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word[i] = 0;
    for (int j = 0; j < run; ++j) {
      float x[8];
      unsigned n[8];
      load8(row + (size_t)j * qkv_stride + (n_heads + n_kv_heads + kvh) * head_dim + c0, x);
      const unsigned meta = kv4_quantise8(x, n);
      const int e = (slot & 7) + j, at = kv4_place(e);
      auto turned = [&](unsigned v) { return __builtin_rotateleft32(v, at); };
      mask |= turned(15u);
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] |= turned(n[i]);
      if (c0 % 32 == 0) scales[e] = (uint16_t)meta;
    }
    unsigned* dst = reinterpret_cast<unsigned*>(base) + (slot / 8) * head_dim + c0;
    if (run == 8) {
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(word[0], word[1], word[2], word[3]);
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(word[4], word[5], word[6], word[7]);
    } else {
      // a part of the octet: its own bits alone, so that runs of one octet that lie apart in a step do not undo each other
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __hip_atomic_fetch_and(dst + i, ~mask, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_fetch_or(dst + i, word[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
}

extern "C" int axk_kv4_ok(int head_dim, int page_size) { return kv4_takes(head_dim, page_size) ? 1 : 0; }
extern "C" int axk_kv4_row_bytes(int head_dim) { return kv4_row_bytes(head_dim); }

extern "C" int axk_rope_kv4_write(const void* qkv, long qkv_stride, void* q_out, long q_stride, const float* table,
                                  const int32_t* positions, const int32_t* seq_rows, const int32_t* block_table, int table_stride,
                                  void* k_cache, void* v_cache, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                  int rotary_dim, int page_size, int write_kv, void* stream) {
  AXK_REQUIRE(n_tokens >= 0 && n_heads > 0 && n_kv_heads > 0 && kv4_takes(head_dim, page_size),
              "rope_kv4_write: T=%d nh=%d nkv=%d head_dim %d page size %d are not taken", n_tokens, n_heads, n_kv_heads, head_dim,
              page_size);
  AXK_REQUIRE(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 16 == 0,
              "rope_kv4_write: rotary_dim %d must be a multiple of 16 and at most head_dim %d", rotary_dim, head_dim);
  AXK_REQUIRE((uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0 && qkv_stride * sizeof(elem_t) % 16 == 0 &&
                  q_stride * sizeof(elem_t) % 16 == 0,
              "rope_kv4_write: rows must be 16-byte aligned (strides %ld and %ld)", qkv_stride, q_stride);
  AXK_REQUIRE(!write_kv || ((uintptr_t)k_cache % 16 == 0 && (uintptr_t)v_cache % 16 == 0), "rope_kv4_write: caches must be 16-byte aligned");
  if (n_tokens == 0) return 0;
  rope_kv4_write_kernel<<<n_tokens, 256, 0, (hipStream_t)stream>>>(
      (const elem_t*)qkv, qkv_stride, (elem_t*)q_out, q_stride, table, positions, seq_rows, block_table, table_stride,
      (unsigned char*)k_cache, (unsigned char*)v_cache, n_tokens, n_heads, n_kv_heads, head_dim, rotary_dim, page_size, write_kv);
  AXK_LAUNCH_CHECK("rope_kv4_write");
  return 0;
}

// Rows (seq_rows[i], positions[i]) of the cache as plain rows [n][kv heads][head_dim] of the compute dtype, each number rounded
// once (bfloat16 holds eight of its up to ten bits).  A thread has eight dims: of a key's row one word, of the values the eight
// words that hold them for all rows of an octet that lie side by side in the list.
__global__ void __launch_bounds__(256)
kv4_read_kernel(const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache,
                const int32_t* __restrict__ block_table, int table_stride, const int32_t* __restrict__ positions,
                const int32_t* __restrict__ seq_rows, elem_t* __restrict__ k_out, elem_t* __restrict__ v_out, int n_rows,
                int n_kv_heads, int head_dim, int page_size) {
  const int words = head_dim / 8, kv_units = n_kv_heads * words;
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(at / (2 * kv_units)), u = (int)(at % (2 * kv_units));
  if (r >= n_rows) return;
  const bool is_v = u >= kv_units;
  const int w = is_v ? u - kv_units : u, kvh = w / words, c0 = w % words * 8;
  const int pos = positions[r];
  const size_t out_row = (size_t)n_kv_heads * head_dim;
  elem_t* dst = (is_v ? v_out : k_out) + (size_t)r * out_row + kvh * head_dim + c0;
  float v[8];
  if (pos < 0) {                                             // padding: a row of zeros
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    store8(dst, v);
    return;
  }
  const int run = is_v ? octet_run(positions, seq_rows, r, n_rows) : 1;
  if (run == 0) return;
  const int page = block_table[(size_t)seq_rows[r] * table_stride + pos / page_size], slot = pos % page_size;
  const unsigned char* base = (is_v ? v_cache : k_cache) + ((size_t)page * n_kv_heads + kvh) * page_size * kv4_row_bytes(head_dim);
  const uint16_t* scales = reinterpret_cast<const uint16_t*>(base + page_size * head_dim / 2);
  if (!is_v) {
    const unsigned word = reinterpret_cast<const unsigned*>(base)[slot * words + c0 / 8];
    const unsigned meta = scales[slot * (head_dim / 32) + c0 / 32];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = kv4_value(__builtin_rotateright32(word, kv4_place(i)) & 15u, meta);
    store8(dst, v);
    return;
  }
  const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned*>(base) + (slot / 8) * head_dim + c0);
  const uint4 w0 = src[0], w1 = src[1];
  const unsigned word[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
  for (int j = 0; j < run; ++j) {
    const int e = (slot & 7) + j;
    const unsigned meta = scales[((slot / 8) * (head_dim / 32) + c0 / 32) * 8 + e];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = kv4_value(__builtin_rotateright32(word[i], kv4_place(e)) & 15u, meta);
    store8(dst + j * out_row, v);
  }
}

extern "C" int axk_kv4_read(const void* k_cache, const void* v_cache, const int32_t* block_table, int table_stride,
                            const int32_t* positions, const int32_t* seq_rows, void* k_out, void* v_out, int n_rows, int n_kv_heads,
                            int head_dim, int page_size, void* stream) {
  AXK_REQUIRE(n_rows >= 0 && n_kv_heads > 0 && kv4_takes(head_dim, page_size),
              "kv4_read: n=%d nkv=%d head_dim %d page size %d are not taken", n_rows, n_kv_heads, head_dim, page_size);
  AXK_REQUIRE((uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0 && (uintptr_t)k_cache % 16 == 0 && (uintptr_t)v_cache % 16 == 0,
              "kv4_read: caches and rows must be 16-byte aligned");
  const long units = (long)n_rows * 2 * n_kv_heads * (head_dim / 8);
  AXK_REQUIRE(units / 256 < (1l << 31) - 1, "kv4_read: %d rows are too many", n_rows);
  if (n_rows == 0) return 0;
  kv4_read_kernel<<<(unsigned)((units + 255) / 256), 256, 0, (hipStream_t)stream>>>(
      (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride, positions, seq_rows, (elem_t*)k_out,
      (elem_t*)v_out, n_rows, n_kv_heads, head_dim, page_size);
  AXK_LAUNCH_CHECK("kv4_read");
  return 0;
}
