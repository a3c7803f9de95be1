/*
 * nve_b200_kv.h — paged cache of key / value rows: the second kind of cache of this library.
 *
 * The set-associative cache (nve_c_api.h, nve_b200_ops.h) holds embedding rows and answers insert, lookup + pool
 * and replacement by accumulated counters.  This one holds the key and value rows of the tokens a model has seen
 * and answers the same three requests: append (rotate and store new rows), attend (one new token per sequence
 * reads every row of its sequence: a lookup pooled with softmax weights) and evict (the rows that drew the least
 * attention leave).  nve_b200_rotary is the rotation alone, forward and backward, for training.
 *
 * Conventions are those of nve_b200_ops.h: plain DEVICE pointers, byte strides, a cudaStream_t cast to void*; every
 * entry returns an nve_status_t and leaves its message for nve_get_last_error().  Nothing here allocates or
 * synchronises, every call can be captured into a CUDA graph, kernels run on the current device.  Results do not
 * depend on the order in which blocks run: no floating-point atomics.
 *
 * A sequence is a row of a page table (int32 page ids) and a length: its row i lives in page table[i / page_size]
 * at slot i % page_size.  Entries of the table behind the last row are never read.  A page may be shared by
 * sequences as long as none of them writes it (append, accumulated weights).
 *
 * Page ids and lengths are data on the device, so the kernels check them: a row on a page outside [0, num_pages)
 * is treated as absent, a length outside [0, capacity] is clamped, and the event is OR-ed into *status
 * (NVE_B200_KV_BAD_*) for the host to read when it likes.
 */
#ifndef NVE_B200_KV_H
#define NVE_B200_KV_H

#include <stddef.h>

#include "nve_c_api.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
  NVE_B200_KV_BAD_PAGE = 1,   /* a page id outside [0, num_pages): the row was left out */
  NVE_B200_KV_BAD_LENGTH = 2, /* a length below 0 or above the capacity: clamped; an appended row without a place */
  NVE_B200_KV_BAD_AXIS = 4,   /* a pair_axis outside [0, num_axes): the pair was not turned */
  NVE_B200_KV_TIMED_OUT = 8   /* a wait inside a kernel ran into its limit: the outputs of that call are not complete */
};

/* A paged cache.  Rows are head_width values of one head of one token; the last dimension is dense. */
typedef struct {
  void* keys;                /* [num_pages][page_size][num_heads] rows at these strides */
  void* values;
  int64_t key_strides[3];    /* bytes: page, slot, head; multiples of 16, any order in memory */
  int64_t value_strides[3];
  float* weights;            /* [num_pages][num_heads][page_size] dense: attention each row drew; NULL = not kept */
  const float* key_scale;    /* E4M3 rows, [num_heads]: value = scale * stored, positive and not subnormal; NULL = 1 */
  const float* value_scale;
  nve_data_type_t dtype;     /* FLOAT16, BFLOAT16 or E4M3 */
  int64_t num_pages;
  int32_t page_size;         /* any size from 1 */
  int32_t num_heads;
  int32_t head_width;        /* row bytes a multiple of 16, at most 256 values */
  int32_t* status;           /* one device word, may be NULL */
} nve_b200_kv_cache_t;

/* Rows of `num_heads` heads per token.  Strides in bytes, multiples of the value size. */
typedef struct {
  const void* in;
  void* out; /* may equal in, with the same strides; must not overlap it in another way */
  int64_t in_token_stride, in_head_stride;
  int64_t out_token_stride, out_head_stride;
  int32_t num_heads;
} nve_b200_head_rows_t;

/*
 * Rotary positions with several axes.  Pair i of a row is turned by
 *   angle(i, t) = positions[pair_axis[i]][t] * inv_freq[i]
 * (computed and reduced in 64 bits), (a, b) -> (a cos - b sin, b cos + a sin).  Pairs are values (i, i + num_pairs),
 * or (2i, 2i + 1) when `interleaved`; values from 2 * num_pairs on are copied.
 */
typedef struct {
  const int32_t* positions; /* [num_axes][tokens] */
  int64_t axis_stride, token_stride; /* elements */
  int32_t num_axes;
  const float* inv_freq;     /* [num_pairs] */
  const int32_t* pair_axis;  /* [num_pairs]; NULL = axis 0 */
  int32_t num_pairs;
  int32_t interleaved;
  int32_t* status;           /* one device word for BAD_AXIS, may be NULL */
} nve_b200_rotary_t;

/*
 * Turns the rows of one or two groups (queries, keys) of `num_tokens` tokens.  dtype FLOAT32, FLOAT16 or BFLOAT16.
 * backward != 0 turns by the negated angles: the gradient of the inputs from the gradient of the outputs.
 */
NVE_C_API nve_status_t nve_b200_rotary(const nve_b200_rotary_t* rotary, nve_data_type_t dtype, int32_t head_width,
                                       int64_t num_tokens, const nve_b200_head_rows_t* groups, int32_t num_groups,
                                       int32_t backward, void* stream);

/*
 * Append.  Token t of sequence b (csr_offsets[b] <= t < csr_offsets[b + 1], or num_tokens / num_sequences tokens
 * each when csr_offsets is NULL) becomes row lengths[b] + t - csr_offsets[b] of its sequence: its keys, turned by
 * `rotary`, and its values are stored, in E4M3 caches divided by their head's scale and saturated; the weight of
 * the row starts at 0; its queries, turned, go to q.out.  Tokens outside [csr_offsets[0], csr_offsets[n]) are
 * padding: nothing of theirs is written, but zeros to q.out with zero_padding.  A row behind the page table's end is not stored (BAD_LENGTH).
 * new_lengths[b] = min(lengths[b] + new rows, capacity); it must not be `lengths` itself.
 */
typedef struct {
  nve_data_type_t dtype;      /* of q, k and v: the cache's type, or FLOAT16 / BFLOAT16 for an E4M3 cache */
  int64_t num_tokens;
  nve_b200_head_rows_t q;     /* q.in NULL: no queries */
  nve_b200_head_rows_t k, v;  /* `out` unused */
  const nve_b200_rotary_t* rotary; /* host pointer; NULL: nothing is turned */
  const int32_t* page_table;  /* [num_sequences][pages_per_sequence], rows page_table_stride elements apart */
  int64_t page_table_stride;
  int32_t pages_per_sequence;
  int32_t num_sequences;
  const int32_t* lengths;
  const int32_t* csr_offsets;
  int32_t* new_lengths;
  int32_t zero_padding;
} nve_b200_kv_append_t;

NVE_C_API nve_status_t nve_b200_kv_append(const nve_b200_kv_cache_t* cache, const nve_b200_kv_append_t* args,
                                          void* stream);

/*
 * Attention of one new token per sequence.  Query head i reads key head i / (num_q_heads / num_heads):
 *   s_j = scale * q . k_j,  lse = log(sum_j exp s_j),  out = sum_j exp(s_j - lse) v_j   over the sequence's rows.
 * With accumulate_weights every row's weight grows by the exp(s_j - lse) of the query heads that read it.  A
 * sequence without rows (or whose scores are all -inf) gives out = 0 and lse = -inf.  What lies in a page behind the
 * last row (NaN included) has no influence.
 *
 * Scratch, the protocol of nve_b200_gather_rows_sorted: scratch == NULL writes the size for these sizes to
 * *scratch_bytes (it depends on no device data); a second call with a 256-byte aligned device buffer of that size
 * runs.  Calls that may overlap in time need buffers of their own.
 */
typedef struct {
  nve_data_type_t dtype;      /* of q and out: the cache's type, or FLOAT16 / BFLOAT16 for an E4M3 cache */
  int32_t num_sequences;
  int32_t num_q_heads;        /* a multiple of the cache's num_heads */
  const void* q;              /* [num_sequences][num_q_heads] rows; address and strides multiples of 16 bytes */
  int64_t q_sequence_stride, q_head_stride;
  void* out;                  /* address and strides multiples of the value size */
  int64_t out_sequence_stride, out_head_stride;
  float* lse;                 /* [num_sequences][num_q_heads] dense, may be NULL */
  const int32_t* page_table;
  int64_t page_table_stride;
  int32_t pages_per_sequence;
  const int32_t* lengths;
  int32_t max_length;         /* no length is above this; at most pages_per_sequence * page_size */
  float scale;
  int32_t accumulate_weights;
} nve_b200_kv_attend_t;

NVE_C_API nve_status_t nve_b200_kv_attend(const nve_b200_kv_cache_t* cache, const nve_b200_kv_attend_t* args,
                                          void* scratch, size_t* scratch_bytes, void* stream);

/*
 * Eviction by accumulated weight, for every (sequence, head) on its own.  A sequence of more than `budget` rows
 * keeps its first `sinks` and last `recent` rows and, of the others, those with the largest weight (equal weights:
 * the earliest; NaN counts as -inf), `budget` in all; a shorter one keeps every row.  The kept rows, in their old
 * order, with their weights, are written to the pages of new_page_table, which must be other pages than those read
 * (pages shared with other sequences stay as they are; the old pages are the caller's to free).
 * kept[b][h][j] = old row of new row j, -1 behind the last; new_lengths[b] = min(lengths[b], budget).
 */
typedef struct {
  int32_t num_sequences;
  const int32_t* page_table;
  int64_t page_table_stride;
  int32_t pages_per_sequence;
  const int32_t* lengths;
  int32_t max_length;         /* no length is above this; at most pages_per_sequence * page_size */
  const int32_t* new_page_table;
  int64_t new_page_table_stride;
  int32_t new_pages_per_sequence; /* at least min(budget, max_length) rows */
  int32_t budget, sinks, recent;  /* sinks + recent <= budget */
  int32_t* kept;              /* [num_sequences][num_heads][budget] dense */
  int32_t* new_lengths;
} nve_b200_kv_evict_t;

NVE_C_API nve_status_t nve_b200_kv_evict(const nve_b200_kv_cache_t* cache, const nve_b200_kv_evict_t* args,
                                         void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NVE_B200_KV_H */
