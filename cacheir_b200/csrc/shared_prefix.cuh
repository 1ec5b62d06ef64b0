// Shared by the kernels of decode attention over common prefixes.
#pragma once

#include "cacheir_b200_serving.h"
#include "common.cuh"
#include "serving_status.h"

namespace cb200 {

// What the kernel of the common parts leaves for the one that joins: how its work was cut (see shared_prefix_mma.cu).
struct PlanGroup {
  int start;                  // its first unit
  int row, rows;              // its rows
  int prefix;                 // its common tokens
};
struct PrefixPlan {
  int units;                  // of all items
  int ctas;                   // blocks that share them
  int unused[2];
  PlanGroup group[1];         // [groups], and the end of the last one's units
};

// The scratch: plan, then for every (piece, row, head) a maximum (log2 domain) and a denominator, and the unnormalised output. Up to `pieces`
// of them come from the common parts (general kernels: from either), up to `own` from a row's own keys.
struct PrefixParts {
  PrefixPlan* plan;
  float* ml;       // [pieces + own][batch][heads][2]
  float* acc;      // [pieces + own][batch][heads][dim]
  int pieces, own;
};

// First row of group g, inside the batch whatever the caller's array holds.
__device__ __forceinline__ int group_start(const cacheir_b200_prefix_args& a, int g) { return min(max(a.group_rows[g], 0), a.batch); }

// The group of a row (group_rows is ascending), -1 outside every group, and its common tokens; a whole warp. Up to 32 groups are looked at
// in one round of loads.
__device__ __forceinline__ int prefix_of_group(const cacheir_b200_prefix_args& a, int g) {
  const long long room = static_cast<long long>(a.prefix_pages) * a.page_size;
  return static_cast<int>(min(static_cast<long long>(max(a.prefix_lens[g], 0)), room));
}
__device__ __forceinline__ int group_of_row(const cacheir_b200_prefix_args& a, int row, int* prefix) {
  *prefix = 0;
  if (a.groups <= 0) return -1;
  const int lane = threadIdx.x & 31;
  if (a.groups <= 32) {
    bool mine = false;
    int len = 0;
    if (lane < a.groups) {
      mine = a.group_rows[lane] <= row && row < a.group_rows[lane + 1];
      len = prefix_of_group(a, lane);
    }
    const uint32_t found = __ballot_sync(0xffffffffu, mine);
    if (found == 0) return -1;
    const int g = 31 - __clz(found);
    *prefix = __shfl_sync(0xffffffffu, len, g);
    return g;
  }
  int lo = 0, hi = a.groups + 1;           // the number of starts up to `row` is in lo .. hi; 32 of them are looked at at a time
  while (hi > lo) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const int below = __popc(__ballot_sync(0xffffffffu, at < hi && a.group_rows[at] <= row));
    if (below == 0) break;
    const int first = lo + (below - 1) * step;        // its start is at or below the row
    hi = min(hi, first + step);
    lo = first + 1;
  }
  if (lo == 0 || lo == a.groups + 1) return -1;
  *prefix = prefix_of_group(a, lo - 1);
  return lo - 1;
}

constexpr int kMaxPieces = 64;
constexpr int kMinPieces = 4;
// Pieces per row that the scratch holds: 64 MB of them, but 4 at least.
inline int prefix_pieces(int batch, int heads, int dim) {
  const size_t one = static_cast<size_t>(batch) * heads * dim * 4;
  const size_t n = one > 0 ? (static_cast<size_t>(64) << 20) / one : kMinPieces;
  return n < kMinPieces ? kMinPieces : n > kMaxPieces ? kMaxPieces : static_cast<int>(n);
}
// Parts of a row's own keys: more than one where there are few rows.
constexpr int kMaxOwnParts = 8;
inline int own_parts(int batch) {
  int n = 1;
  while (n < kMaxOwnParts && 2 * n * batch <= kNumSMs) n *= 2;
  return n;
}
inline size_t round_up_256(size_t n) { return (n + 255) / 256 * 256; }
inline size_t prefix_plan_bytes(int batch) { return round_up_256(sizeof(PrefixPlan) + static_cast<size_t>(batch) * sizeof(PlanGroup)); }
inline size_t prefix_ml_bytes(int batch, int heads, int pieces) { return round_up_256(static_cast<size_t>(pieces) * batch * heads * 2 * 4); }

// Tensor-core kernels (shared_prefix_mma.cu): 16-bit types, head sizes 64 and 128, pages of a multiple of 16 tokens.
bool prefix_fast_supported(const cacheir_b200_prefix_args& a);
int prefix_fast_launches(int groups);
int launch_prefix_fast(const cacheir_b200_prefix_args& a, const PrefixParts& parts, cudaStream_t stream);

}  // namespace cb200
