/*
 * C-ABI of the serving operators of librisa_b200.so: rotary positions, a paged key/value cache,
 * attention of new tokens over it, the attention its keys receive, and eviction.  The reference
 * project has no counterpart (it attends whole sequences and keeps nothing between calls).
 *
 * Conventions are those of risa_b200.h: device pointers, element strides, the caller's stream, a
 * status code with risa_b200_last_error(), no allocation, no host synchronisation.  Everything that
 * changes from step to step (lengths, offsets, page table) is read on the device, so a captured
 * graph replays with new contents.
 * What a call writes lies apart from all that it reads, unless it is said below that it may be one
 * of its inputs itself: CTAs write while others still read, and addresses are not compared.
 * dtype codes: 0 = float32, 1 = float16, 2 = bfloat16, 4 = int8 codes with a scale per token and head,
 * 5 = 4-bit codes with a scale per token and head and one per 16 channels.
 */
#ifndef RISA_B200_CACHE_H
#define RISA_B200_CACHE_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Pages of keys and values: [pages, kv_heads, page_size, head_dim] contiguous, 16-byte aligned;
 * scales f32 [pages, kv_heads, page_size] (int8; NULL for 16-bit values).  page_size: 16, 32, 64 or
 * 128; head_dim: 64, 128 or 256; dtype_code: 1, 2, 4 or 5.
 * 4-bit codes: a value is code * group scale * token scale.  Rows of head_dim / 2 bytes; channel
 * 8 w + 2 i + j as code + 8 (codes -7..7) in bits 16 j + 4 i of the row's 32-bit word w.  The scale
 * pointers lead to bytes [pages, kv_heads, page_size * (1 + head_dim / 16)], 16-byte aligned: of each
 * page and head first the token scales, powers of two as the exponent field of a float (0: a scale of
 * zero, 255: a row that is not finite), then for each token the scales of its groups of 16 channels,
 * e4m3 numbers from 0 to 448: neither a sign bit nor e4m3's NaN, which are read by their bits and
 * not checked (append writes none). */
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

/* Positions of several axes (time, height, width): pair i follows axis axes[i] (bytes on the device;
 * those from `count` on count as the last axis), whose positions lie `position_stride` elements
 * behind those of the axis before it (0: all axes have the same).  count: 1 to 8. */
typedef struct {
  const uint8_t* axes;
  int count;
  int64_t position_stride;
} risa_b200_rotary_axes;
#define RISA_B200_MOST_AXES 8

/* out = x with every [batch, heads, tokens] row of head_dim channels rotated by its position, or by
 * the transposed rotation (the gradient).  out may be x.  positions: int32 or int64 at
 * b * position_stride_b + n * position_stride_n.  Strides of the channel axis are 1. */
int risa_b200_rotate(const void* x, void* out, int dtype_code, int batch, int heads, int tokens,
                     int head_dim, const int64_t x_strides[3], const int64_t out_strides[3],
                     const void* positions, int positions_64, int64_t position_stride_b,
                     int64_t position_stride_n, const risa_b200_rotary* rotary, int transposed,
                     void* stream);
/* The same by positions of several axes (NULL: of one). */
int risa_b200_rotate_axes(const void* x, void* out, int dtype_code, int batch, int heads, int tokens,
                          int head_dim, const int64_t x_strides[3], const int64_t out_strides[3],
                          const void* positions, int positions_64, int64_t position_stride_b,
                          int64_t position_stride_n, const risa_b200_rotary* rotary,
                          const risa_b200_rotary_axes* axes, int transposed, void* stream);

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
/* The same by positions of several axes (NULL: of one); without positions every axis has the token's
 * place in the cache. */
int risa_b200_cache_append_axes(const risa_b200_cache* cache, const risa_b200_step* step,
                                const void* k, const int64_t k_strides[2], const void* v,
                                const int64_t v_strides[2], const void* q,
                                const int64_t q_strides[2], void* q_out,
                                const int64_t q_out_strides[2], int q_heads, int dtype_code,
                                const risa_b200_rotary* rotary, const risa_b200_rotary_axes* axes,
                                const void* positions, int positions_64, void* stream);

/* The step's keys and values [tokens, kv_heads, head_dim] as they lie in the cache, codes as the values
 * that they stand for, rounded to dtype_code (1 or 2; a 16-bit cache's own).  Rows of no sequence, or
 * whose sequence is too short for them, give 0.  Strides are of (token, head) in elements, multiples of 8;
 * pointers are 16-byte aligned. */
int risa_b200_cache_read(const risa_b200_cache* cache, const risa_b200_step* step, void* k,
                         const int64_t k_strides[2], void* v, const int64_t v_strides[2],
                         int dtype_code, void* stream);

/* softmax(scale * q K^T) V of every packed token over its sequence's cached keys; with is_causal the
 * token at place p of its sequence sees keys max(0, p - window + 1) .. p (window 0: from the start),
 * without it all of them.  q, out: dtype_code 1 or 2 (the cache's own unless that holds codes); out
 * may be q itself, with its strides.  lse: f32
 * [tokens, q_heads] or NULL.  Rows that see no key give 0 and -inf.  clear_rest: rows of no
 * sequence are written the same way, bit 0 those of out, bit 1 those of lse, else left as they were. */
size_t risa_b200_paged_attention_scratch_size(const risa_b200_cache* cache,
                                              const risa_b200_step* step, int q_heads);
int risa_b200_paged_attention(const risa_b200_cache* cache, const risa_b200_step* step,
                              const void* q, const int64_t q_strides[2], int q_heads,
                              int dtype_code, void* out, const int64_t out_strides[2], float* lse,
                              float scale, int is_causal, int window, int clear_rest,
                              void* scratch, size_t scratch_bytes, void* stream);
/* With a window, keys 0 .. sinks-1 of the sequence stay visible in front of it (those up to the
 * token's own place). */
int risa_b200_paged_attention_sinks(const risa_b200_cache* cache, const risa_b200_step* step,
                                    const void* q, const int64_t q_strides[2], int q_heads,
                                    int dtype_code, void* out, const int64_t out_strides[2],
                                    float* lse, float scale, int is_causal, int window, int sinks,
                                    int clear_rest, void* scratch, size_t scratch_bytes,
                                    void* stream);

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
int risa_b200_key_weights_sinks(const risa_b200_cache* cache, const risa_b200_step* step,
                                const void* q, const int64_t q_strides[2], int q_heads,
                                int dtype_code, const float* lse, float scale, int is_causal,
                                int window, int sinks, const float* previous, float* weights,
                                void* scratch, size_t scratch_bytes, void* stream);

/* Keeps min(length, budget) tokens of every (sequence, key head): the `recent` last ones and those of
 * the largest weights among the others (equal weights: lowest index first; NaN counts as largest),
 * and copies them in their order to the pages of target_table [batch, target_width], which must hold
 * the budget and share no page with what is read.  step->query_offsets and tokens are not used.
 * weights: f32 [batch, kv_heads, table_width * page_size].  kept: int32 [batch, kv_heads, budget],
 * -1 behind the last; new_lengths: int32 [batch], may be the step's lengths; new_weights: f32
 * [batch, kv_heads, target_width * page_size], 0 behind the last. */
int risa_b200_cache_evict(const risa_b200_cache* cache, const risa_b200_step* step,
                          const float* weights, const int32_t* target_table, int target_width,
                          int budget, int recent, int32_t* kept, int32_t* new_lengths,
                          float* new_weights, void* stream);

/* ---- pages shared, handed out, given back and moved ----------------------------------------------
 * references: int32 [pages], how many entries of page tables lead to each page; 0: the page is free.
 * Entries behind a sequence's length are not read; one that leads outside the pool is not counted, and
 * risa_b200_device_status() reports it.  Tables and lengths that fork returns are others than the
 * step's, and compact's target_references others than references; compact's table may be the
 * step's page_table itself. */

/* Row c of table [children, table_width] and lengths[c] become those of sequence parents[c] of the
 * step, -1 behind the length (a parent outside 0..batch-1: an empty sequence); references counts the
 * new entries.  step->query_offsets and tokens are not used here and in compact. */
int risa_b200_fork_sequences(const risa_b200_cache* cache, int32_t* references,
                             const risa_b200_step* step, const int32_t* parents, int children,
                             int32_t* table, int32_t* lengths, void* stream);

/* Brings every sequence from lengths[s] to new_lengths[s] tokens (at most what its row of the table
 * holds).  A longer one gets pages: the lowest that were free, in the order of the sequences; where its
 * last page is not full and has more than one reference it first gets a page in place of that, with a
 * copy of its tokens (each sequence that shares it, also where all of them grow in one call).  A
 * shorter one gives back the pages behind its length (their entries become -1); they are handed out
 * from the next call on.  granted[s]: the length that the pages found allow
 * (a sequence whose shared page could not be replaced keeps its length); it may be lengths or
 * new_lengths itself. */
size_t risa_b200_resize_scratch_size(const risa_b200_cache* cache, int batch);
int risa_b200_resize_sequences(const risa_b200_cache* cache, int32_t* references,
                               int32_t* page_table, int table_width, const int32_t* lengths,
                               const int32_t* new_lengths, int batch, int32_t* granted,
                               void* scratch, size_t scratch_bytes, void* stream);

/* Copies the pages in use (references > 0), in their order, to the first pages of another pool whose
 * pages are of the same kind; table: the step's page table for that pool (-1 behind the lengths),
 * target_references its counts, used[0] the number of pages in use.  Pages that the target has no room for are
 * not copied, and their entries become -1. */
size_t risa_b200_compact_scratch_size(const risa_b200_cache* cache, const risa_b200_cache* target);
int risa_b200_cache_compact(const risa_b200_cache* cache, const int32_t* references,
                            const risa_b200_step* step, const risa_b200_cache* target,
                            int32_t* table, int32_t* target_references, int32_t* used,
                            void* scratch, size_t scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
