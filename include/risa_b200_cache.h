/*
 * C-ABI of the serving operators of librisa_b200.so: rotary positions, a paged key/value cache,
 * attention of new tokens over it, the attention its keys receive, and eviction.  The reference
 * project has no counterpart (it attends whole sequences and keeps nothing between calls).
 *
 * Conventions are those of risa_b200.h: device pointers, element strides, the caller's stream, a
 * status code with risa_b200_last_error(), no allocation, no host synchronisation.  Everything that
 * changes from step to step (lengths, offsets, page table) is read on the device, so a captured
 * graph replays with new contents.
 * dtype codes: 0 = float32, 1 = float16, 2 = bfloat16, 4 = int8 codes with a scale per token and head.
 */
#ifndef RISA_B200_CACHE_H
#define RISA_B200_CACHE_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Pages of keys and values: [pages, kv_heads, page_size, head_dim] contiguous, 16-byte aligned;
 * scales f32 [pages, kv_heads, page_size] (int8 only, else NULL).  page_size: 16, 32, 64 or 128;
 * head_dim: 64, 128 or 256; dtype_code: 1, 2 or 4. */
typedef struct {
  void* keys;
  void* values;
  float* key_scales;
  float* value_scales;
  int pages, kv_heads, page_size, head_dim, dtype_code;
} risa_b200_cache;

/* A row of a page table leads to fewer slots than this: kernels count them in 32 bits and step past
 * the last one by what a block of threads or a ring of tiles covers. */
#define RISA_B200_CACHE_MOST_SLOTS (((int64_t)1 << 31) - 8192)

/* One step of a batch.  The tokens of sequence s are rows query_offsets[s] .. query_offsets[s+1]-1
 * of the packed tensors (NULL: row s alone) and the last ones of the lengths[s] tokens that its row
 * of page_table [batch, table_width] leads to.  Entries of the table behind a sequence's length are
 * not read.  A page outside the pool is never read or written: its keys are hidden, and
 * risa_b200_device_status() reports it. */
typedef struct {
  const int32_t* page_table;
  const int32_t* lengths;
  const int32_t* query_offsets;
  int batch, table_width, tokens;
} risa_b200_step;

/* Angles: pair i at position p turns by p * turns[i] / 2^64 of a full turn; cosines and sines are
 * multiplied by magnitude.  interleaved 0: pair i = channels (i, i + rotary_dim / 2); 1: channels
 * (2 i, 2 i + 1).  Channels from rotary_dim on are copied. */
typedef struct {
  const uint64_t* turns;
  int rotary_dim;
  float magnitude;
  int interleaved;
} risa_b200_rotary;

/* out = x with every [batch, heads, tokens] row of head_dim channels rotated by its position, or by
 * the transposed rotation (the gradient).  out may be x.  positions: int32 or int64 at
 * b * position_stride_b + n * position_stride_n.  Strides of the channel axis are 1. */
int risa_b200_rotate(const void* x, void* out, int dtype_code, int batch, int heads, int tokens,
                     int head_dim, const int64_t x_strides[3], const int64_t out_strides[3],
                     const void* positions, int positions_64, int64_t position_stride_b,
                     int64_t position_stride_n, const risa_b200_rotary* rotary, int transposed,
                     void* stream);

/* Writes one step's keys and values [tokens, kv_heads, head_dim] to their pages, the keys rotated
 * where rotary is given (its angle: positions[token], or the token's place in the cache where
 * positions is NULL), and q [tokens, q_heads, head_dim] rotated to q_out (both NULL: none; rows
 * behind the last sequence give 0).  Strides are of (token, head) in elements, multiples of 8; pointers are 16-byte aligned. */
int risa_b200_cache_append(const risa_b200_cache* cache, const risa_b200_step* step, const void* k,
                           const int64_t k_strides[2], const void* v, const int64_t v_strides[2],
                           const void* q, const int64_t q_strides[2], void* q_out,
                           const int64_t q_out_strides[2], int q_heads, int dtype_code,
                           const risa_b200_rotary* rotary, const void* positions, int positions_64,
                           void* stream);

/* softmax(scale * q K^T) V of every packed token over its sequence's cached keys; with is_causal the
 * token at place p of its sequence sees keys max(0, p - window + 1) .. p (window 0: from the start),
 * without it all of them.  q, out: dtype_code 1 or 2 (the cache's own unless that is int8).  lse: f32
 * [tokens, q_heads] or NULL.  Rows that see no key give 0 and -inf.  clear_rest: rows of no
 * sequence are written the same way, bit 0 those of out, bit 1 those of lse, else left as they were. */
size_t risa_b200_paged_attention_scratch_size(const risa_b200_cache* cache,
                                              const risa_b200_step* step, int q_heads);
int risa_b200_paged_attention(const risa_b200_cache* cache, const risa_b200_step* step,
                              const void* q, const int64_t q_strides[2], int q_heads,
                              int dtype_code, void* out, const int64_t out_strides[2], float* lse,
                              float scale, int is_causal, int window, int clear_rest,
                              void* scratch, size_t scratch_bytes, void* stream);

/* weights[b, h, j] = previous[b, h, j] + sum over the sequence's new tokens and the query heads of
 * key head h of exp(scale * q . k_j - lse): the attention that key j received.  weights, previous
 * (NULL: zeros; may be weights): f32 [batch, kv_heads, table_width * page_size] contiguous.  Hidden
 * keys and rows whose lse is -inf add nothing. */
size_t risa_b200_key_weights_scratch_size(const risa_b200_cache* cache, const risa_b200_step* step,
                                          int q_heads);
int risa_b200_key_weights(const risa_b200_cache* cache, const risa_b200_step* step, const void* q,
                          const int64_t q_strides[2], int q_heads, int dtype_code,
                          const float* lse, float scale, int is_causal, int window,
                          const float* previous, float* weights, void* scratch,
                          size_t scratch_bytes, void* stream);

/* Keeps min(length, budget) tokens of every (sequence, key head): the `recent` last ones and those of
 * the largest weights among the others (equal weights: lowest index first; NaN counts as largest),
 * and copies them in their order to the pages of target_table [batch, target_width], which must hold
 * the budget and share no page with what is read.  step->query_offsets and tokens are not used.
 * weights: f32 [batch, kv_heads, table_width * page_size].  kept: int32 [batch, kv_heads, budget],
 * -1 behind the last; new_lengths: int32 [batch]; new_weights: f32 [batch, kv_heads,
 * target_width * page_size], 0 behind the last. */
int risa_b200_cache_evict(const risa_b200_cache* cache, const risa_b200_step* step,
                          const float* weights, const int32_t* target_table, int target_width,
                          int budget, int recent, int32_t* kept, int32_t* new_lengths,
                          float* new_weights, void* stream);

#ifdef __cplusplus
}
#endif
#endif
