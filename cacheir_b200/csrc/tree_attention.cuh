// Shared by the kernels of attention over drafted tokens.
#pragma once

#include "cacheir_b200_drafts.h"
#include "common.cuh"
#include "serving_status.h"

namespace cb200 {

// A sequence's part of a call: its rows, the tokens in front of them, and all its tokens that the table has room for.
struct TreeSequence {
  int row, rows;              // first row, number of rows
  int front;                  // token t of the sequence is its row t - front (below 0 where it has more rows than tokens)
  int keys;
};
__device__ __forceinline__ TreeSequence tree_sequence(const cacheir_b200_tree_args& a, int b) {
  TreeSequence s;
  s.row = min(max(a.cu_rows[b], 0), a.rows);
  s.rows = max(min(max(a.cu_rows[b + 1], 0), a.rows) - s.row, 0);
  const int len = max(a.seq_lens[b], 0);
  s.front = len - s.rows;
  s.keys = min(len, a.max_pages * a.page_size);
  return s;
}
// 32 of the sequence's rows that row i sees, those from 32 q on, as bits.
__device__ __forceinline__ uint32_t tree_word(const cacheir_b200_tree_args& a, const TreeSequence& s, int i, int q) {
  if (q < 0 || 32 * q >= s.rows) return 0u;
  uint32_t bits;
  if (!a.visible) bits = i >= 32 * q + 31 ? 0xffffffffu : i < 32 * q ? 0u : (2u << (i & 31)) - 1u;
  else bits = q < a.words ? static_cast<uint32_t>(a.visible[static_cast<size_t>(s.row + i) * a.words + q]) : 0u;
  return s.rows - 32 * q < 32 ? bits & ((1u << (s.rows - 32 * q)) - 1u) : bits;
}

// Partial results of the general kernel, where keys are cut into pieces: for every (piece, row, head) a maximum (log2 domain) and a denominator, and the unnormalised
// output. As many pieces as 64 MB of outputs hold; rows that fill more than half of that are not cut and need no scratch, which so does not grow with the batch.
constexpr int kMaxTreePieces = 64;
inline int tree_pieces(int rows, int heads, int dim) {
  const size_t one = static_cast<size_t>(rows) * heads * dim * 4, n = (static_cast<size_t>(64) << 20) / (one > 0 ? one : 1);
  return n < 1 ? 1 : n > kMaxTreePieces ? kMaxTreePieces : static_cast<int>(n);
}

// Tensor-core kernels (tree_attention_mma.cu): 16-bit types, head sizes 64 and 128, pages of a multiple of 16 tokens.
size_t tree_fast_bytes(int dim);
bool tree_fast_supported(const cacheir_b200_tree_args& a);
int launch_tree_fast(const cacheir_b200_tree_args& a, cudaStream_t stream);
int tree_device_status(bool reset);

}  // namespace cb200
