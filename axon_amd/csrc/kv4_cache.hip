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

// Up to LIST_ROWS neighbouring tokens (or rows that are read) of a block: where each lies, and the runs that begin among them, rows that
// lie one position behind the other in one octet of slots of one request.  A run that goes on behind them is the block's all the
// same, and one that began before them is not: an octet's words are stored by one block, once, where a step has the whole of it.
#define LIST_ROWS 16
struct RowList {
  int pos[LIST_ROWS], page[LIST_ROWS], run_first[LIST_ROWS], run_rows[LIST_ROWS], runs;
};

__device__ inline void list_rows(RowList& list, const int32_t* positions, const int32_t* seq_rows, const int32_t* block_table, int table_stride,
                                 int first, int n, int n_tokens, int page_size) {
  if (threadIdx.x < AXON_WAVE) {
    const int i = threadIdx.x, t = first - 1 + i;                // lane 0: the row before them
    const bool there = t >= 0 && t < n_tokens && i <= n + 7;
    const int pos = there ? positions[t] : -1, row = there ? seq_rows[t] : -1;
    if (i >= 1 && i <= n) {
      list.pos[i - 1] = pos;
      list.page[i - 1] = pos < 0 ? 0 : block_table[(size_t)row * table_stride + pos / page_size];        // (padding has no place)
    }
    const int pos_before = __shfl_up(pos, 1, AXON_WAVE), row_before = __shfl_up(row, 1, AXON_WAVE);       // (of every lane: none is left out)
    const bool follows = i > 0 && pos >= 0 && (pos & 7) != 0 && pos_before == pos - 1 && row_before == row;
    const uint64_t stops = __ballot(!follows), starts = stops & __ballot(i >= 1 && i <= n && pos >= 0);
    if (starts >> i & 1) {                                       // (a run has eight rows at most: lane n + 8 follows nothing)
      const int at = __popcll(starts & ((1ull << i) - 1));
      list.run_first[at] = i - 1;
      list.run_rows[at] = __builtin_ctzll(stops >> (i + 1)) + 1;
    }
    if (i == 0) list.runs = __popcll(starts);
  }
  __syncthreads();
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
  // x / s, correctly rounded, by the scale's reciprocal and what the product leaves: q = x r is within two units of its last place, the rest
  // x - q s is exact, and q + rest r is off by 2^-23 units before it is rounded, while a quotient by a scale of six bits
  // is 2^-7 units or more away from the middle between two numbers, where the rounding would turn.
  const float r = __fdiv_rn(1.0f, s);
  auto quotient = [&](float v) {
    const float q = __fmul_rn(v, r);
    return __builtin_fmaf(__builtin_fmaf(-q, s, v), r, q);
  };
  const float z = fminf(fmaxf(rintf(quotient(-lo)), 0.0f), 15.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = (unsigned)fminf(fmaxf(__fadd_rn(rintf(quotient(x[i])), z), 0.0f), 15.0f);
  return bits | (unsigned)z;
}

// Dims c0 .. c0 + 7 of a head's row behind the rotation (rotate-half on the first rotary_dim dims; half a multiple of 8).  All loads are
// without a branch, so that they are under way together: dims that do not turn read themselves and the table's first 64 bytes, which have
// to be there also where nothing turns.
__device__ inline void rotated8(const elem_t* head, const float* tab, int c0, int rotary_dim, float (&out)[8]) {
  const int half = rotary_dim / 2, to = c0 >= half ? -half : half;
  const bool turn = c0 < rotary_dim, upper = c0 >= half;
  const float4* at = reinterpret_cast<const float4*>(tab + (turn ? 2 * min(c0, c0 + to) : 0));
  float x[8], y[8];
  float4 sin_cos[4];
  load8(head + c0, x);
  load8(head + (c0 + (turn ? to : 0)), y);
#pragma unroll
  for (int i = 0; i < 4; ++i) sin_cos[i] = at[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = i % 2 ? sin_cos[i / 2].z : sin_cos[i / 2].x, c = i % 2 ? sin_cos[i / 2].w : sin_cos[i / 2].y;
    const float turned = upper ? __fadd_rn(__fmul_rn(y[i], s), __fmul_rn(x[i], c)) : __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y[i], s));
    out[i] = turn ? turned : x[i];
  }
}

// The blocks behind the first kv_blocks have the queries of Q_TOKENS tokens each: a thread the eight pairs of dims i .. i + 7 and i + half
// .. (or sixteen dims behind the rotated ones) of several heads of a token, whose sines and cosines it reads once.  The first, which take
// longer, have the keys and values of up to `rows` tokens: a thread a word of keys, or eight dims of a run's values, whose words hold up to
// eight positions. Bound by its bytes in prompts (qkv in, q and the cache out: 8192 tokens of 28 and 4 heads of 128 dims take 25 us, 143 MB
// at 5.7 TB/s), by its waits in steps of few tokens (8: 4.8 us; a launch of the queries' blocks alone 2.9).
template <int Q_TOKENS>
__global__ void __launch_bounds__(256)
rope_kv4_write_kernel(const elem_t* qkv, long qkv_stride, elem_t* q_out, long q_stride, const float* __restrict__ table,
                      const int32_t* __restrict__ positions, const int32_t* __restrict__ seq_rows,
                      const int32_t* __restrict__ block_table, int table_stride, unsigned char* __restrict__ k_cache,
                      unsigned char* __restrict__ v_cache, int n_tokens, int n_heads, int n_kv_heads, int head_dim, int rotary_dim,
                      int page_size, int kv_blocks, int rows) {
  __shared__ RowList list;
  const int half = rotary_dim / 2;
  if ((int)blockIdx.x >= kv_blocks) {
    const int units = head_dim / 16, lanes = 256 / units / Q_TOKENS;           // lanes that share a token's heads
    const int c = threadIdx.x % units, slot = threadIdx.x / units, t = (blockIdx.x - kv_blocks) * Q_TOKENS + slot / lanes;
    if (t >= n_tokens) return;
    const bool turn = c < half / 8;
    const int d0 = turn ? 8 * c : rotary_dim + 16 * (c - half / 8), d1 = turn ? d0 + half : d0 + 8;
    float sin_cos[16];
    if (turn) {
      const float4* tab = reinterpret_cast<const float4*>(table + ((size_t)t * half + d0) * 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = tab[i];
        sin_cos[4 * i] = v.x; sin_cos[4 * i + 1] = v.y; sin_cos[4 * i + 2] = v.z; sin_cos[4 * i + 3] = v.w;
      }
    }
    const elem_t* src = qkv + (size_t)t * qkv_stride;
    elem_t* dst = q_out + (size_t)t * q_stride;
    constexpr int AHEAD = AXON_BF16 ? 4 : 2;                   // heads asked for before the first is stored (the rows may be the same)
    for (int head = slot % lanes; head < n_heads; head += AHEAD * lanes) {
      float a[AHEAD][8], b[AHEAD][8];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int at = min(head + n * lanes, n_heads - 1) * head_dim;
        load8(src + at + d0, a[n]);
        load8(src + at + d1, b[n]);
      }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        if (head + n * lanes >= n_heads) break;
        if (turn)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float s = sin_cos[2 * i], co = sin_cos[2 * i + 1], x = a[n][i];
            a[n][i] = __fsub_rn(__fmul_rn(x, co), __fmul_rn(b[n][i], s));
            b[n][i] = __fadd_rn(__fmul_rn(x, s), __fmul_rn(b[n][i], co));
          }
        const int at = (head + n * lanes) * head_dim;
        store8(dst + at + d0, a[n]);
        store8(dst + at + d1, b[n]);
      }
    }
    return;
  }
  const int first = blockIdx.x * rows, n = min(rows, n_tokens - first), words = head_dim / 8, kv_units = n_kv_heads * words, slots = page_size - 1;
  const size_t head_bytes = (size_t)page_size * kv4_row_bytes(head_dim);
  // keys: token i, word w of its keys; values: the same, of a run's first token (units come in fours, a group's lanes, and so do threads)
  auto keys = [&](int i, int w, float(&x)[8]) {
    rotated8(qkv + (size_t)(first + i) * qkv_stride + (n_heads + w / words) * head_dim, table + (size_t)(first + i) * half * 2, w % words * 8,
             rotary_dim, x);
  };
  auto values = [&](int i, int w, float(&x)[8]) {
    load8(qkv + (size_t)(first + i) * qkv_stride + (n_heads + n_kv_heads) * head_dim + w * 8, x);
  };
  // a thread's first unit is asked for before anything is known of the tokens' places
  float ahead[8];
  bool fresh = true;
  int u = threadIdx.x;
  if (u < n * kv_units) keys(u / kv_units, u % kv_units, ahead);
  else if (u < (n + 1) * kv_units) values(0, u - n * kv_units, ahead);
  list_rows(list, positions, seq_rows, block_table, table_stride, first, n, n_tokens, page_size);
  for (; u < n * kv_units; u += 256, fresh = false) {
    const int i = u / kv_units, w = u % kv_units, kvh = w / words, c0 = w % words * 8, pos = list.pos[i];
    if (!fresh) keys(i, w, ahead);
    if (pos < 0) continue;
    unsigned numbers[8];
    const unsigned meta = kv4_quantise8(ahead, numbers);
    unsigned word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= __builtin_rotateleft32(numbers[e], kv4_place(e));
    unsigned char* base = k_cache + ((size_t)list.page[i] * n_kv_heads + kvh) * head_bytes;
    const int slot = pos & slots;
    reinterpret_cast<unsigned*>(base)[slot * words + c0 / 8] = word;
    if (c0 % 32 == 0) reinterpret_cast<uint16_t*>(base + page_size * head_dim / 2)[slot * (head_dim / 32) + c0 / 32] = (uint16_t)meta;
  }
  for (u -= n * kv_units; u < list.runs * kv_units; u += 256, fresh = false) {
    const int run = u / kv_units, w = u % kv_units, kvh = w / words, c0 = w % words * 8, i0 = list.run_first[run], run_rows = list.run_rows[run];
    const int slot = list.pos[i0] & slots;
    unsigned char* base = v_cache + ((size_t)list.page[i0] * n_kv_heads + kvh) * head_bytes;
    uint16_t* scales = reinterpret_cast<uint16_t*>(base + page_size * head_dim / 2) + ((slot / 8) * (head_dim / 32) + c0 / 32) * 8;
    unsigned word[8], mask = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word[e] = 0;
    auto take = [&](int e, const float(&x)[8]) {
      unsigned numbers[8];
      const unsigned meta = kv4_quantise8(x, numbers);
      const int at = kv4_place(e);
      mask |= __builtin_rotateleft32(15u, at);
#pragma unroll
      for (int d = 0; d < 8; ++d) word[d] |= __builtin_rotateleft32(numbers[d], at);
      if (c0 % 32 == 0) scales[e] = (uint16_t)meta;
    };
    unsigned* dst = reinterpret_cast<unsigned*>(base) + (slot / 8) * head_dim + c0;
    if (run_rows == 8) {
      float x[8][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) values(i0 + e, w, x[e]);
#pragma unroll
      for (int e = 0; e < 8; ++e) take(e, x[e]);
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(word[0], word[1], word[2], word[3]);
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(word[4], word[5], word[6], word[7]);
    } else {
      for (int e = 0; e < run_rows; ++e) {
        if (e > 0 || i0 > 0 || !fresh) values(i0 + e, w, ahead); // (the first token's: asked for already)
        take((slot & 7) + e, ahead);
      }
      // a part of the octet: its own bits alone, so that the octet's other runs, which may lie elsewhere in the step, are not undone
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        __hip_atomic_fetch_and(dst + d, ~mask, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_fetch_or(dst + d, word[d], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
  AXK_REQUIRE((uintptr_t)table % 16 == 0, "rope_kv4_write: the table must be 16-byte aligned");
  if (n_tokens == 0) return 0;
  // Few tokens: a block each for its queries and for its keys and values.  Of 28 query and 4 key/value heads of 128 dims, so or in blocks
  // of four and eight tokens: 8 single tokens 4.7 and 9.4 us, 128 7.7 and 12.9, 512 17.9 and 21.1; a portion of 64 tokens 7.2 and 9.1, of
  // 1024 9.6 and 10.9, of 2048 16.6 and 13.2.  Blocks of sixteen tokens: 1024 13.4, 4096 17.4 against 17.1 by eight, 8192 24.8 against
  // 26.7.
  const bool few = n_tokens <= 1024;
  const int rows = few ? 1 : n_tokens <= 4096 ? 8 : LIST_ROWS, q_blocks = few ? n_tokens : ceil_div(n_tokens, 4);
  const int kv_blocks = write_kv ? ceil_div(n_tokens, rows) : 0;
  const unsigned blocks = q_blocks + kv_blocks;
#define LAUNCH(Q_TOKENS)                                                                                                          \
  rope_kv4_write_kernel<Q_TOKENS><<<blocks, 256, 0, (hipStream_t)stream>>>(                                                       \
      (const elem_t*)qkv, qkv_stride, (elem_t*)q_out, q_stride, rotary_dim > 0 ? table : (const float*)qkv, positions, seq_rows,  \
      block_table, table_stride, (unsigned char*)k_cache, (unsigned char*)v_cache, n_tokens, n_heads, n_kv_heads, head_dim,       \
      rotary_dim, page_size, kv_blocks, rows)
  if (few) LAUNCH(1);
  else LAUNCH(4);
#undef LAUNCH
  AXK_LAUNCH_CHECK("rope_kv4_write");
  return 0;
}

// Rows (seq_rows[i], positions[i]) of the cache as plain rows [n][kv heads][head_dim] of the compute dtype, each number rounded
// once (bfloat16 holds eight of its up to ten bits).  grid (lists of LIST_ROWS rows, keys | values): a thread a word of keys, or the words of
// eight dims of a run's values, which it unpacks as the products' operands are.  A run of whole octets is its
// first block's; no words are read twice.  Bound by the rows that it stores: eight requests' 16384 positions of 4 heads of 128 dims take 76
// us, 344 MB at 4.5 TB/s; by its waits for few (301 rows: 4.5 us).
__global__ void __launch_bounds__(256)
kv4_read_kernel(const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache,
                const int32_t* __restrict__ block_table, int table_stride, const int32_t* __restrict__ positions,
                const int32_t* __restrict__ seq_rows, elem_t* __restrict__ k_out, elem_t* __restrict__ v_out, int n_rows,
                int n_kv_heads, int head_dim, int page_size) {
  __shared__ RowList list;
  const int first = blockIdx.x * LIST_ROWS, n = min(LIST_ROWS, n_rows - first);
  list_rows(list, positions, seq_rows, block_table, table_stride, first, n, n_rows, page_size);
  const int words = head_dim / 8, kv_units = n_kv_heads * words, slots = page_size - 1;
  const size_t out_row = (size_t)n_kv_heads * head_dim, head_bytes = (size_t)page_size * kv4_row_bytes(head_dim);
  const Kv4Masks masks = kv4_masks();
  if (blockIdx.y == 0) {
    for (int u = threadIdx.x; u < n * kv_units; u += 256) {
      const int i = u / kv_units, w = u % kv_units, kvh = w / words, c0 = w % words * 8, pos = list.pos[i], slot = pos & slots;
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};               // (padding)
      if (pos >= 0) {
        const unsigned char* base = k_cache + ((size_t)list.page[i] * n_kv_heads + kvh) * head_bytes;
        const unsigned word = reinterpret_cast<const unsigned*>(base)[slot * words + c0 / 8];
        const unsigned meta = reinterpret_cast<const uint16_t*>(base + page_size * head_dim / 2)[slot * (head_dim / 32) + c0 / 32];
        half2_t sc[4], cc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) kv4_pair_scale(meta | meta << 16, sc[e], cc[e]);
        const u32x4 pairs = kv4_operand(word, sc, cc, masks);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = kv4_half(pairs[e / 2], e % 2);
      }
      store8(k_out + (size_t)(first + i) * out_row + kvh * head_dim + c0, v);
    }
    return;
  }
  for (int u = threadIdx.x; u < n * kv_units; u += 256) {                          // padding's values
    const int i = u / kv_units, w = u % kv_units;
    const float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (list.pos[i] < 0) store8(v_out + (size_t)(first + i) * out_row + w * 8, v);
  }
  for (int u = threadIdx.x; u < list.runs * kv_units; u += 256) {
    const int run = u / kv_units, w = u % kv_units, kvh = w / words, c0 = w % words * 8, i0 = list.run_first[run];
    const int slot = list.pos[i0] & slots, low = slot & 7, high = low + list.run_rows[run];
    const unsigned char* base = v_cache + ((size_t)list.page[i0] * n_kv_heads + kvh) * head_bytes;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned*>(base) + (slot / 8) * head_dim + c0);
    const uint4 metas = *reinterpret_cast<const uint4*>(base + page_size * head_dim / 2 + ((slot / 8) * (head_dim / 32) + c0 / 32) * 16);
    const uint4 w0 = src[0], w1 = src[1];
    const unsigned word[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w}, meta[4] = {metas.x, metas.y, metas.z, metas.w};
    half2_t sc[4], cc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) kv4_pair_scale(meta[e], sc[e], cc[e]);
    u32x4 pairs[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) pairs[d] = kv4_operand(word[d], sc, cc, masks);
    elem_t* dst = v_out + (size_t)(first + i0) * out_row + kvh * head_dim + c0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e < low || e >= high) continue;
      float v[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) v[d] = kv4_half(pairs[d][e / 2], e % 2);
      store8(dst + (size_t)(e - low) * out_row, v);
    }
  }
}

extern "C" int axk_kv4_read(const void* k_cache, const void* v_cache, const int32_t* block_table, int table_stride,
                            const int32_t* positions, const int32_t* seq_rows, void* k_out, void* v_out, int n_rows, int n_kv_heads,
                            int head_dim, int page_size, void* stream) {
  AXK_REQUIRE(n_rows >= 0 && n_kv_heads > 0 && kv4_takes(head_dim, page_size),
              "kv4_read: n=%d nkv=%d head_dim %d page size %d are not taken", n_rows, n_kv_heads, head_dim, page_size);
  AXK_REQUIRE((uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0 && (uintptr_t)k_cache % 16 == 0 && (uintptr_t)v_cache % 16 == 0,
              "kv4_read: caches and rows must be 16-byte aligned");
  if (n_rows == 0) return 0;
  kv4_read_kernel<<<dim3(ceil_div(n_rows, LIST_ROWS), 2), 256, 0, (hipStream_t)stream>>>(
      (const unsigned char*)k_cache, (const unsigned char*)v_cache, block_table, table_stride, positions, seq_rows, (elem_t*)k_out,
      (elem_t*)v_out, n_rows, n_kv_heads, head_dim, page_size);
  AXK_LAUNCH_CHECK("kv4_read");
  return 0;
}
