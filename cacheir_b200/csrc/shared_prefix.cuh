// Shared by the kernels of decode attention over common prefixes.
#pragma once

#include "cacheir_b200_serving.h"
#include "common.cuh"

namespace cb200 {

// Where partial results go: for every (piece, row, head) a maximum (log2 domain) and a denominator, and the unnormalised output.
struct PrefixParts {
  float* ml;       // [pieces][batch][heads][2]
  float* acc;      // [pieces][batch][heads][dim]
  int pieces;
};

// First row of group g, inside the batch whatever the caller's array holds.
__device__ __forceinline__ int group_start(const cacheir_b200_prefix_args& a, int g) { return min(max(a.group_rows[g], 0), a.batch); }

// The group of a row (group_rows is ascending); -1 outside every group.
__device__ __forceinline__ int group_of_row(const cacheir_b200_prefix_args& a, int row) {
  if (a.groups <= 0 || row < a.group_rows[0] || row >= a.group_rows[a.groups]) return -1;
  int lo = 0, hi = a.groups;               // last g with group_rows[g] <= row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.group_rows[mid] <= row) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int prefix_of_group(const cacheir_b200_prefix_args& a, int g) {
  const long long room = static_cast<long long>(a.prefix_pages) * a.page_size;
  return static_cast<int>(min(static_cast<long long>(max(a.prefix_lens[g], 0)), room));
}

constexpr int kMaxPieces = 64;
// Pieces per row that the scratch holds: 64 MB of them, but 4 at least.
inline int prefix_pieces(int batch, int heads, int dim) {
  const size_t one = static_cast<size_t>(batch) * heads * dim * 4;
  const size_t n = one > 0 ? (static_cast<size_t>(64) << 20) / one : 4;
  return n < 4 ? 4 : n > kMaxPieces ? kMaxPieces : static_cast<int>(n);
}
inline size_t prefix_ml_bytes(int batch, int heads, int pieces) {
  return (static_cast<size_t>(pieces) * batch * heads * 2 * 4 + 255) / 256 * 256;
}

}  // namespace cb200
