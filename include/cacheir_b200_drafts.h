/*
 * cacheir_b200_drafts.h -- C ABI of libcacheir_b200_drafts.so: the operators of a step that verifies drafted tokens. Every sequence brings
 * rows, a token each: row 0 is its last certain token, the others follow an earlier row of it (a tree, or a chain) and take the places
 * behind it in the sequence's pages. Norms of query and key heads with rotary positions and the append, attention under the tree's
 * mask, logits with penalties, biases and masks, the rows' positions and masks, the accepted path and its keys and values moved together.
 *
 * The conventions of cacheir_b200.h hold: device pointers, nothing is allocated or synchronised, 0 / cudaError_t / CACHEIR_B200_E*,
 * non-positive extents return 0 without launching.
 */
#ifndef CACHEIR_B200_DRAFTS_H_
#define CACHEIR_B200_DRAFTS_H_

#include "cacheir_b200_serving.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of a sequence: cu_rows int32 [sequences + 1], ascending; sequence b has the rows cu_rows[b] .. cu_rows[b + 1] - 1 (what lies outside
 * 0 .. rows counts as its end). They are the last tokens of seq_lens[b]: row i of n stands at place seq_lens[b] - n + i of its pages. */

/* ------------------------------------------------------------------------
 * Norms of the heads of q and k, rotary positions, and with slots the append of k and v to the page pool.
 *   x -> x / sqrt(mean x^2 + eps) * (weight + offset), then as cacheir_b200_rotary_append, of which this is the form with norms: `rotary`
 * holds its arguments. q_weight, k_weight [dim], both of weight_dtype: that of q, or float32; either may be NULL (weight + offset = 1).
 * Everything is worked out in 32 bits and rounded once. eps >= 0. */
typedef struct {
  cacheir_b200_rotary_args rotary;
  const void* q_weight;
  const void* k_weight;
  int weight_dtype;
  float eps, offset;
} cacheir_b200_norm_rotary_args;
int cacheir_b200_norm_rotary_append(const cacheir_b200_norm_rotary_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Attention of the rows of drafted tokens over their sequence's pages.
 *
 * Beside cacheir_b200_paged_attention_decode_batch (the reference's `paged_attention_decode_batch_kernel`,
 * cacheir/backends/triton_kernels.py:174-217), which has one row per sequence. Row i of sequence b, with n rows and c = seq_lens[b] - n
 * tokens in front of them, sees the tokens t < c and of its sequence's rows
 *   those j whose bit j % 32 of visible[row][j / 32] is set (visible int32 [rows][words]; rows j >= 32 words are seen by none), or
 *   visible NULL: the rows j <= i (a chain).
 * A row that sees nothing gives zeros; rows behind the last sequence are left as they were in out. What a row does not see may hold
 * anything, also numbers that are none. A key with a score of -inf has no weight (in front of the rows, weight 0: its value has to be a number); NaN among a row's
 * scores gives NaN.
 * q, out [rows][heads][dim], rows q_stride / out_stride elements apart; pools [num_slots][kv_heads][page_size][dim]; page_table
 * [sequences][max_pages], page ids outside the pool read as zeros; tokens behind max_pages * page_size are not there.
 * Up to 65535 sequences, 2^24 rows, as many key/value heads as 65535, tables of up to 2^30 tokens, words <= 32 (CACHEIR_B200_ELIMIT), heads
 * of up to 512 (CACHEIR_B200_EUNSUPPORTED).
 *   workspace: cacheir_b200_tree_attention_workspace_bytes(...) bytes (enough for whatever kernel serves the call, 68 MB at most with heads of 128; 0: NULL will do),
 *   16-byte aligned, used by this call's kernels only: calls that may overlap need one each.
 * Scores, sums and outputs are in 32 bits. 16-bit types with heads of 64 or 128 and pages of a multiple of 16 tokens go to the tensor cores, which take the softmax's
 * probabilities rounded to the element type; in all other calls these have 32 bits too.
 * Partial results are joined in a fixed order: the same bits for the same arguments. */
#define CACHEIR_B200_MAX_DRAFT_WORDS 32
typedef struct {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* out;
  const int32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* cu_rows;
  const int32_t* visible;
  void* workspace;
  size_t workspace_bytes;
  long long q_stride, out_stride;
  int rows, sequences, heads, kv_heads, dim, page_size, num_slots, max_pages, words, dtype;
  float softmax_scale;        /* <= 0: 1 / sqrt(dim) */
} cacheir_b200_tree_args;
size_t cacheir_b200_tree_attention_workspace_bytes(int rows, int heads, int dim);
int cacheir_b200_tree_attention(const cacheir_b200_tree_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Logits as the next token is to be picked from: for token t of a row of sequence b,
 *   c = times that t stands in the generated part of the sequence's history (places prompt_lens[b] .. history_lens[b] - 1), and among the
 *       drafted tokens that the row sees, itself among them (with draft_ids)
 *   x = logits; where c > 0 or t stands in the prompt: x > 0 ? x / repetition : x * repetition
 *   x -= frequency * c;  c > 0: x -= presence;  x += bias of t;  t not allowed: x = -inf
 * worked out in 32 bits and rounded once. Stands beside cacheir_b200_argmax_rows and cacheir_b200_token_logprobs, which follow it.
 *   row_seq int32 [rows] (NULL: row r is of sequence r): rows whose sequence is outside 0 .. sequences - 1 are left as they were in out
 *   history int32 [sequences][history_width], history_lens, prompt_lens int32 [sequences] (prompt_lens NULL: no prompt); NULL: no history
 *   draft_ids int64 [rows] with cu_rows (see above) and visible int32 [rows][words] (as in cacheir_b200_tree_attention); NULL: none.
 *     Row 0, a sequence's last certain token, is among what its rows see. So either the history ends in front of it, and it counts as generated through its
 *     draft_ids; or the history holds it, as generated or, in the first step behind a prompt, as the prompt's last token, and its draft_ids is -1. With both it
 *     counts twice. (cacheir_b200_accept_drafts does not look at draft_ids of row 0.)
 *   repetition (> 0), frequency, presence float [sequences]; each NULL: without
 *   bias_ids int32 [sequences][biases], bias_values float: of several entries with one token the last counts
 *   allowed int32 [rows][ceil(vocab / 32)]: bit t % 32 of word t / 32, 1 where the token may come
 * Tokens outside the vocabulary are left out. out has the same type or is float32. It may be logits, with the same type and row stride; other rows of it that lie over
 * rows of logits are refused (CACHEIR_B200_EINVAL). Up to 524280 rows, vocabularies of up to 2^28,
 * histories of fewer than 2^29 tokens, words <= 32 (CACHEIR_B200_ELIMIT). */
typedef struct {
  const void* logits;
  void* out;
  const int32_t* row_seq;
  const int32_t* history;
  const int32_t* history_lens;
  const int32_t* prompt_lens;
  const int64_t* draft_ids;
  const int32_t* cu_rows;
  const int32_t* visible;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int32_t* bias_ids;
  const float* bias_values;
  const int32_t* allowed;
  long long row_stride, out_stride;
  int rows, sequences, vocab, history_width, words, biases, dtype, out_dtype;
} cacheir_b200_logits_args;
int cacheir_b200_adjust_logits(const cacheir_b200_logits_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Drafted tokens as rows. parents int32 [rows]: of a row its parent's number inside the sequence; -1, or anything but an earlier row,
 * means none. Up to 65535 sequences (CACHEIR_B200_ELIMIT).
 *
 * map: positions[r] = tokens in front of the sequence's rows + number of rows that r follows; visible[r][words] = the rows that it
 *   follows and itself, as bits. Rows behind the last sequence: position 0, no bits. A sequence of more than 32 words rows has bits for the
 *   first 32 words of them only; status[0] then becomes its number of rows (the largest of several) and stays until the caller sets it to 0.
 * accept: the path that was picked. It begins with row 0 and goes on, while there is one, with the first row whose parent is the row it has
 *   come to and whose draft_ids is what was picked there (chosen int64 [rows]); up to `depth` rows.
 *   counts[b] = rows of the path (0: the sequence has none), path int32 [sequences][depth] = their row numbers, -1 behind them,
 *   next_ids[b] = what was picked at the last of them (-1: no rows), keep_lens[b] = seq_lens[b] - n + counts[b].
 * keep: keys and values of the i-th row of every path to the slot of its sequence's i-th row, in `pools` pools [num_slots][kv_heads]
 *   [page_size][dim] whose addresses lie in an array on the host. slots [rows] as from cacheir_b200_extend_page_tables; what would read or
 *   write outside the pools is left out. Paths are such that row numbers rise (accept's do). */
typedef struct {
  const int32_t* parents;
  const int32_t* cu_rows;
  const int32_t* seq_lens;
  int32_t* positions;
  int32_t* visible;
  int32_t* status;
  int rows, sequences, words;
} cacheir_b200_draft_map_args;
int cacheir_b200_map_drafts(const cacheir_b200_draft_map_args* args, void* stream);

typedef struct {
  const int64_t* chosen;
  const int64_t* draft_ids;
  const int32_t* parents;
  const int32_t* cu_rows;
  const int32_t* seq_lens;
  int32_t* counts;
  int32_t* path;
  int64_t* next_ids;
  int32_t* keep_lens;
  int rows, sequences, depth;
} cacheir_b200_accept_args;
int cacheir_b200_accept_drafts(const cacheir_b200_accept_args* args, void* stream);

typedef struct {
  void* const* pools;         /* on the host */
  const int32_t* slots;
  const int32_t* cu_rows;
  const int32_t* counts;
  const int32_t* path;
  int pool_count, rows, sequences, depth, num_slots, kv_heads, page_size, dim, dtype;
} cacheir_b200_keep_args;
int cacheir_b200_keep_accepted(const cacheir_b200_keep_args* args, void* stream);

/* First bounded wait of a kernel of this library that gave up on the current device (0: none); synchronises. */
int cacheir_b200_drafts_device_status(int reset);

#ifdef __cplusplus
}
#endif
#endif
