/*
 * cacheir_b200_serving.h -- C ABI of libcacheir_b200_serving.so: the operators that a step of a batch needs whose requests share
 * prompts. Pages and page slots for new tokens, rotary positions with the append to the page pool, decode attention that reads a
 * common prefix once for all of its requests, and log probabilities of tokens.
 *
 * The conventions of cacheir_b200.h hold: device pointers, nothing is allocated or synchronised, 0 / cudaError_t / CACHEIR_B200_E*,
 * non-positive extents return 0 without launching.
 */
#ifndef CACHEIR_B200_SERVING_H_
#define CACHEIR_B200_SERVING_H_

#include "cacheir_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Page tables of a batch, kept on the device.
 *
 * The page walk is the reference's `_extend_pages` (cacheir/runtime/kv_cache.py:111-123, cacheir/runtime/cuda.py:395-406): a page is
 * opened where a token's position is a multiple of page_size. `free_pages` [capacity] is a stack of page ids, `free_count` its height;
 * pages are taken from its top in the order of the sequences and, within one, of their tokens.
 *
 * extend: sequence b gets new_lens[b] more tokens (<= 0: none). Its new pages enter page_table[b] ([sequences][max_pages]), seq_lens[b]
 *   grows (a length below 0 counts as 0). cu_rows [sequences + 1] receives the first row of every sequence, and row r of sequence b, in
 *   order, its position, row_seq = b and slots = page * page_size + position % page_size. Rows behind the last token get position 0,
 *   row_seq -1 and slot -1. (Pages come from the caller: slots are meant for pools of fewer than 2^31 rows.)
 * shrink: sequence b keeps its first min(keep_lens[b], seq_lens[b]) tokens (below 0: none). The pages behind them return to the stack,
 *   the first one of the call on top, so that the same tokens would get the same pages again; page_table keeps its entries. The first
 *   held_pages[b] pages of a row (held_pages may be NULL) belong to somebody else and never return. (A sequence that keeps fewer tokens than
 *   those pages hold has let go of them: extending opens pages of its own in their place, which held_pages must not count any more.)
 *
 * Each is all or nothing. A call that cannot be done changes nothing but `status` (and, for extend, the outputs: no rows, all slots
 * -1); status[0] keeps the first such reason until the caller sets it to 0:
 *   > 0  so many pages are missing            -1  more tokens than `rows`
 *   -2   a sequence is longer than its table  -3  the stack's height is below 0 or (would be) above its capacity
 * At most CACHEIR_B200_MAX_SEQUENCES sequences, tables of fewer than 2^31 tokens (CACHEIR_B200_ELIMIT). */
#define CACHEIR_B200_MAX_SEQUENCES 16384
typedef struct {
  int32_t* page_table;
  int32_t* seq_lens;
  const int32_t* change;      /* extend: new_lens; shrink: keep_lens */
  const int32_t* held_pages;  /* shrink */
  int32_t* free_pages;        /* extend reads them only */
  int32_t* free_count;
  int32_t* positions;         /* this one and the next three: extend */
  int32_t* row_seq;
  int32_t* slots;
  int32_t* cu_rows;
  int32_t* status;
  int sequences, max_pages, page_size, capacity;
  int rows;                   /* extend */
} cacheir_b200_tables_args;
int cacheir_b200_extend_page_tables(const cacheir_b200_tables_args* args, void* stream);
int cacheir_b200_shrink_page_tables(const cacheir_b200_tables_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Rotary positions of q and k rows and, with slots, the append of k and v to the page pool.
 *
 * Beside cacheir_b200_rope_append (the reference's interleaved rotation of whole heads, cacheir/runtime/cuda.py:1072-1102): both pair
 * layouts, the first `rot` of `dim` values only, and any frequencies. `turns` [rot/2] holds the frequency of every pair in turns per
 * position as a 64-bit binary fraction (freq / 2 pi * 2^64, modulo 2^64): position times that is exact modulo one turn, so the angle of
 * a far position is as good as that of a near one.
 *   (a, b) -> factor * (a cos - b sin, a sin + b cos), the pair (2i, 2i+1) (layout 0) or (i, i + rot/2) (layout 1)
 * q [rows][heads][dim], k, v [rows][kv_heads][dim], rows q_stride / k_stride / v_stride elements apart, heads dense. q_out, k_out (either
 * may be NULL, or its input) are dense or have their own row strides. With slots (else NULL, and no pools): row r's k and v go to row
 * slots[r] % page_size of page slots[r] / page_size of k_cache, v_cache [num_slots][kv_heads][page_size][dim]; a row whose slot is
 * outside the pool is left out altogether, q_out and k_out included. Rows with one slot: each value there is of one of them, any. */
#define CACHEIR_B200_ROTARY_INTERLEAVED 0
#define CACHEIR_B200_ROTARY_HALF 1
typedef struct {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* k_cache;
  void* v_cache;
  const int32_t* positions;
  const int32_t* slots;
  const uint64_t* turns;
  long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  int rows, heads, kv_heads, dim, rot, layout, num_slots, page_size, dtype;
  float factor;
} cacheir_b200_rotary_args;
int cacheir_b200_rotary_append(const cacheir_b200_rotary_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Decode attention of groups of sequences with a common prefix.
 *
 * The results of cacheir_b200_paged_attention_decode_batch (the reference's `paged_attention_decode_batch_kernel`,
 * cacheir/backends/triton_kernels.py:174-217) for batches in which neighbouring sequences open with the same tokens: the keys and values
 * of the common part are read once for a group and multiplied with the queries of all of its rows together.
 *   group_rows int32 [groups + 1], ascending: the rows of group g are group_rows[g] .. group_rows[g + 1] - 1 (a group may be empty, but there
 *   are no more groups than rows)
 *   prefix_lens int32 [groups]: common tokens of the group; prefix_table int32 [groups][prefix_pages]: the pages that hold them
 * Row b attends to tokens t < seq_lens[b]; those below its group's prefix are read through prefix_table, the others through
 * page_table[b] (entries of pages that lie wholly in the prefix are not read). A prefix may end inside a page. A prefix longer than
 * prefix_pages * page_size counts as that long; rows outside every group have no prefix. seq_lens[b] <= 0 gives zeros.
 * A key with a score of -inf has no weight (a row of such keys alone gives zeros); NaN among a row's scores gives NaN. What stands behind a
 * row's end, in its last page or in the rest of its group's prefix, may hold anything. A row that ends inside its group's prefix reads its
 * keys for itself, through prefix_table.
 * Up to 65535 rows and as many key/value heads, tables of up to 2^30 tokens (CACHEIR_B200_ELIMIT), heads of up to 512
 * (CACHEIR_B200_EUNSUPPORTED).
 *   num_slots: slots of the pools; page ids outside them read as zeros.
 *   workspace: cacheir_b200_shared_prefix_workspace_bytes(...) bytes, 16-byte aligned, used by this call's kernels only: calls that may
 *   overlap need one each.
 * Partial results are joined in a fixed order: the same bits for the same arguments. */
typedef struct {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* out;
  const int32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* group_rows;
  const int32_t* prefix_table;
  const int32_t* prefix_lens;
  void* workspace;
  size_t workspace_bytes;
  long long q_stride, out_stride;
  int batch, heads, kv_heads, dim, page_size, num_slots, max_pages, groups, prefix_pages, dtype;
  float softmax_scale;
} cacheir_b200_prefix_args;
size_t cacheir_b200_shared_prefix_workspace_bytes(int batch, int heads, int dim);
/* Kernels that one call launches for these extents (aligned, dense q): 2 on CUDA cores (any type and size, slower than
 * cacheir_b200_paged_attention_decode_batch on the same batch); on tensor cores (fp16 and bf16, dim 64 and 128,
 * pages of a multiple of 16 tokens, up to 64 query heads per key/value head) 2 without groups, 3 with up to 64 of them, 4 with more. */
int cacheir_b200_shared_prefix_launches(int batch, int heads, int kv_heads, int dim, int page_size, int groups, int dtype);
int cacheir_b200_shared_prefix_attention(const cacheir_b200_prefix_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Log probabilities of tokens, entropies and the likeliest alternatives of rows of logits [rows][vocab] (row_stride elements apart).
 *   y = logits / temperature; logprobs[r] = y[tokens[r]] - log sum exp y; entropy[r] = -sum p log p (nats)
 *   top_ids, top_logprobs [rows][top]: the `top` largest values in falling order, equal ones by rising index
 * Stands beside cacheir_b200_argmax_rows (`argmax` of the reference's scheduler, cacheir/runtime/scheduler.py:456-478).
 * -inf is a masked value (probability 0). A row of nothing else has logprobs -inf and entropy 0. A row with NaN or +inf has NaN for both
 * and for top_logprobs; NaN is the largest value for top_ids. tokens[r] < 0: no token, logprobs 0; tokens[r] >= vocab: NaN.
 * logprobs (with tokens), entropy and the top pair may be NULL. 1e-6 <= temperature <= 1e6. top <= CACHEIR_B200_MAX_TOP and <= vocab, and
 * with it rows of up to 4 MB (CACHEIR_B200_ELIMIT). */
#define CACHEIR_B200_MAX_TOP 32
typedef struct {
  const void* logits;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  long long row_stride;       /* 0: vocab */
  double temperature;
  int rows, vocab, top, dtype;
} cacheir_b200_logprobs_args;
int cacheir_b200_token_logprobs(const cacheir_b200_logprobs_args* args, void* stream);

/* First bounded wait of a kernel of this library that gave up on the current device (0: none); synchronises. */
int cacheir_b200_serving_device_status(int reset);

#ifdef __cplusplus
}
#endif
#endif
