// Drafted tokens as rows: their positions and the rows that they see, the accepted path, and its keys and values moved together.
//
// All three are bound by latency: positions and paths are a few thousand numbers, and the first value that is moved is known after three loads that depend on one another. 128
// sequences of 33 to 64 rows, 32 layers of 8 heads of 128 in fp16: 2.2, 2.7 and 15.0 us one by one (the 63 MB that are moved take 9.7), 22.6 us together; 4 sequences of 6 to 8
// rows, 4 layers: 5.4 us together.
#include "cacheir_b200_drafts.h"
#include "common.cuh"

namespace cb200 {
namespace {

// The rows of sequence b, inside the arrays whatever cu_rows holds.
__device__ __forceinline__ int2 rows_of(const int32_t* cu_rows, int rows, int b) {
  const int lo = min(max(cu_rows[b], 0), rows);
  return make_int2(lo, max(min(max(cu_rows[b + 1], 0), rows) - lo, 0));
}

// ---- map: a block a sequence, a thread a row, which walks up among the rows of its round and goes on from what the rounds before have written ----
constexpr int kMapThreads = 64;
static_assert(kMapThreads == 64, "a round's rows are the bits of a 64-bit word");

__global__ void __launch_bounds__(kMapThreads)
map_drafts_kernel(const cacheir_b200_draft_map_args a) {
  chain_enter();
  __shared__ int s_parent[kMapThreads];
  const int b = blockIdx.x;
  if (b == a.sequences) {                     // rows behind the last sequence
    const int2 last = rows_of(a.cu_rows, a.rows, a.sequences - 1);
    for (int r = last.x + last.y + threadIdx.x; r < a.rows; r += kMapThreads) {
      a.positions[r] = 0;
      for (int w = 0; w < a.words; ++w) a.visible[static_cast<size_t>(r) * a.words + w] = 0;
    }
    return;
  }
  const int2 mine = rows_of(a.cu_rows, a.rows, b);
  const int n = mine.y, first = a.seq_lens[b] - n;
  if (n > 32 * a.words && threadIdx.x == 0) atomicMax(a.status, n);
  const int32_t* parents = a.parents + mine.x;
  const int tid = threadIdx.x;
  int next = tid < n ? parents[tid] : -1;
  for (int base = 0; base < n; base += kMapThreads) {
    const int i = base + tid;
    __syncthreads();                          // (what the round before wrote is there, and its parents are not looked at any more)
    s_parent[tid] = next;
    next = i + kMapThreads < n ? parents[i + kMapThreads] : -1;
    __syncthreads();
    if (i >= n) continue;
    int at = i, depth = -1;
    uint64_t bits = 0;
    while (at >= base) {
      ++depth;
      bits |= 1ull << (at - base);
      const int up = s_parent[at - base];
      at = up < at ? max(up, -1) : -1;
    }
    // (numbers fall on the way up: what is left of it lies in earlier rounds)
    if (at >= 0) depth += a.positions[mine.x + at] - first + 1;
    const int32_t* above = a.visible + static_cast<size_t>(mine.x + max(at, 0)) * a.words;
    int32_t* line = a.visible + static_cast<size_t>(mine.x + i) * a.words;
    const int here = base >> 5;               // word of the round's first row
    for (int w = 0; w < a.words; ++w)         // (rows behind the words' bits have none)
      line[w] = w < here ? (at >= 0 ? above[w] : 0) : w == here ? static_cast<int32_t>(bits) : w == here + 1 ? static_cast<int32_t>(bits >> 32) : 0;
    a.positions[mine.x + i] = first + depth;
  }
}

// ---- accept: a warp a sequence, which walks down ----
__global__ void __launch_bounds__(32)
accept_drafts_kernel(const cacheir_b200_accept_args a) {
  chain_enter();
  const int b = blockIdx.x, lane = threadIdx.x;
  const int2 mine = rows_of(a.cu_rows, a.rows, b);
  const int n = mine.y;
  const int32_t* parents = a.parents + mine.x;
  const int64_t* ids = a.draft_ids + mine.x;
  int32_t* path = a.path + static_cast<size_t>(b) * a.depth;
  // a lane has every 32nd row: of the first ones parents and tokens stay in registers
  constexpr int kHeld = 4;
  int parent[kHeld];
  int64_t id[kHeld], pick[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int r = i * 32 + lane;
    parent[i] = r < n ? parents[r] : -1;
    id[i] = r < n ? ids[r] : -1;
    pick[i] = r < n ? a.chosen[mine.x + r] : -1;
  }
  auto picked = [&](int row) {
    int64_t v = -1;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (row >> 5 == i) v = __shfl_sync(0xffffffffu, pick[i], row & 31);
    return row < kHeld * 32 ? v : a.chosen[mine.x + row];
  };
  int at = 0, count = n > 0 ? 1 : 0;
  int64_t next = n > 0 ? picked(0) : -1;
  if (lane == 0 && n > 0) path[0] = mine.x;
  bool found = n > 0;
  while (found && count < a.depth) {
    found = false;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (found) break;
      const int r = i * 32 + lane;
      const uint32_t hit = __ballot_sync(0xffffffffu, r > at && r < n && parent[i] == at && id[i] == next);
      if (hit) {
        found = true;
        at = i * 32 + __ffs(hit) - 1;
      }
    }
    for (int r0 = max(kHeld * 32, at & ~31); !found && r0 < n; r0 += 32) {          // (a row follows an earlier one: a path takes one look at every row)
      const int r = r0 + lane;
      const uint32_t hit = __ballot_sync(0xffffffffu, r > at && r < n && parents[min(r, n - 1)] == at && ids[min(r, n - 1)] == next);
      if (hit) {
        found = true;
        at = r0 + __ffs(hit) - 1;
      }
    }
    if (found) {
      if (lane == 0) path[count] = mine.x + at;
      ++count;
      next = picked(at);
    }
  }
  for (int i = count + lane; i < a.depth; i += 32) path[i] = -1;
  if (lane == 0) {
    a.counts[b] = count;
    a.next_ids[b] = next;
    a.keep_lens[b] = a.seq_lens[b] - n + count;
  }
}

// ---- keep: a block a sequence and some pools, a thread a column, which it moves in the order of the path ----
constexpr int kKeepThreads = 128;
constexpr int kKeepPools = 128;               // of a launch
constexpr int kKeepShare = 4;                 // pools of a block, which a thread has under way together (16 took 18.3 us, 8 15.9) ..
constexpr int kKeepDeep = 3;                  // .. with so many rows of each
constexpr int kKeepMoves = 64;                // moves that a block looks up together
static_assert(kKeepMoves <= kKeepThreads, "a thread a move");

struct KeepParams {
  cacheir_b200_keep_args a;
  int pools;
  void* pool[kKeepPools];
};

// A row's source is never a target before it, as row numbers rise along a path: all that is written before it is read lies in front of it.
// What takes time is the way from the path over slots to the values, three dependent loads (rows are looked up before it is known how many count); so it is
// gone once for several pools.
template <typename V>
__global__ void __launch_bounds__(kKeepThreads)
keep_accepted_kernel(const __grid_constant__ KeepParams p) {
  chain_enter();
  __shared__ int s_from[kKeepMoves], s_to[kKeepMoves];         // slots; -1: none
  const cacheir_b200_keep_args& a = p.a;
  const int b = blockIdx.x;
  const int32_t* path = a.path + static_cast<size_t>(b) * a.depth;
  const int width = a.dim * (a.dtype == CACHEIR_B200_F32 ? 4 : 2) / static_cast<int>(sizeof(V));          // units of a line
  const long long outside = static_cast<long long>(a.num_slots) * a.page_size;
  int row = static_cast<int>(threadIdx.x) < kKeepMoves && static_cast<int>(threadIdx.x) + 1 < a.depth ? path[threadIdx.x + 1] : -1;
  const int2 mine = rows_of(a.cu_rows, a.rows, b);
  const int count = min(min(a.counts[b], a.depth), mine.y);
  auto line_of = [&](int r) {
    const int slot = r >= 0 && r < a.rows ? a.slots[r] : -1;
    return slot < 0 || slot >= outside ? -1 : slot;
  };
  const int first_pool = blockIdx.y * kKeepShare, pools = min(kKeepShare, p.pools - first_pool);
  for (int i0 = 1; i0 < count; i0 += kKeepMoves) {             // (rows of one round are read after those before it were written, in any thread)
    const int moves = min(kKeepMoves, count - i0);
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < moves) {
      if (i0 > 1) row = path[i0 + threadIdx.x];
      const int to = mine.x + i0 + threadIdx.x;
      s_from[threadIdx.x] = row == to ? -1 : line_of(row);
      s_to[threadIdx.x] = line_of(to);
    }
    __syncthreads();
    for (int c = blockIdx.z * kKeepThreads + threadIdx.x; c < a.kv_heads * width; c += gridDim.z * kKeepThreads) {
      const int head = c / width, at = c - head * width;
      auto place = [&](int slot) {
        return ((static_cast<long long>(slot / a.page_size) * a.kv_heads + head) * a.page_size + slot % a.page_size) * width + at;
      };
      for (int j0 = 0; j0 < moves; j0 += kKeepDeep) {
        V v[kKeepShare][kKeepDeep];
#pragma unroll
        for (int e = 0; e < kKeepDeep; ++e) {
          const int j = min(j0 + e, moves - 1), from = s_from[j];
          if (j0 + e < moves && from >= 0 && s_to[j] >= 0) {
            const long long x = place(from);
#pragma unroll
            for (int k = 0; k < kKeepShare; ++k)
              if (k < pools) v[k][e] = static_cast<const V*>(p.pool[first_pool + k])[x];
          }
        }
#pragma unroll
        for (int e = 0; e < kKeepDeep; ++e) {
          const int j = min(j0 + e, moves - 1), to = s_to[j];
          if (j0 + e < moves && to >= 0 && s_from[j] >= 0) {
            const long long x = place(to);
#pragma unroll
            for (int k = 0; k < kKeepShare; ++k)
              if (k < pools) static_cast<V*>(p.pool[first_pool + k])[x] = v[k][e];
          }
        }
      }
    }
  }
}

template <typename V>
int launch_keep(const cacheir_b200_keep_args& a, cudaStream_t stream) {
  const long long columns = static_cast<long long>(a.kv_heads) * a.dim * dtype_size(a.dtype) / static_cast<long long>(sizeof(V));
  const long long chunks = (columns + kKeepThreads - 1) / kKeepThreads;
  for (int first = 0; first < a.pool_count; first += kKeepPools) {
    KeepParams p;
    p.a = a;
    p.pools = a.pool_count - first < kKeepPools ? a.pool_count - first : kKeepPools;
    for (int i = 0; i < p.pools; ++i) p.pool[i] = a.pools[first + i];
    const dim3 grid(a.sequences, (p.pools + kKeepShare - 1) / kKeepShare, static_cast<unsigned>(chunks < 64 ? chunks : 64));
    const cudaError_t e = launch_chained(keep_accepted_kernel<V>, grid, dim3(kKeepThreads), 0, stream, p);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_map_drafts(const cacheir_b200_draft_map_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_draft_map_args a = *args;
  if (a.rows <= 0 || a.sequences <= 0) return 0;
  if (!a.parents || !a.cu_rows || !a.seq_lens || !a.positions || !a.visible || !a.status || a.words <= 0) return CACHEIR_B200_EINVAL;
  if (a.sequences > 65535 || a.words > CACHEIR_B200_MAX_DRAFT_WORDS) return CACHEIR_B200_ELIMIT;
  const cudaError_t e = launch_chained(map_drafts_kernel, dim3(a.sequences + 1), dim3(kMapThreads), 0, as_stream(stream), a);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

extern "C" int cacheir_b200_accept_drafts(const cacheir_b200_accept_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_accept_args a = *args;
  if (a.rows <= 0 || a.sequences <= 0) return 0;
  if (!a.chosen || !a.draft_ids || !a.parents || !a.cu_rows || !a.seq_lens || !a.counts || !a.path || !a.next_ids || !a.keep_lens || a.depth <= 0)
    return CACHEIR_B200_EINVAL;
  if (a.sequences > 65535) return CACHEIR_B200_ELIMIT;
  const cudaError_t e = launch_chained(accept_drafts_kernel, dim3(a.sequences), dim3(32), 0, as_stream(stream), a);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

extern "C" int cacheir_b200_keep_accepted(const cacheir_b200_keep_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_keep_args a = *args;
  if (a.pool_count <= 0 || a.rows <= 0 || a.sequences <= 0) return 0;
  if (!a.pools || !a.slots || !a.cu_rows || !a.counts || !a.path || a.depth <= 0 || a.num_slots <= 0 || a.kv_heads <= 0 || a.page_size <= 0 || a.dim <= 0 ||
      dtype_size(a.dtype) == 0)
    return CACHEIR_B200_EINVAL;
  bool wide = a.dim * dtype_size(a.dtype) % 16 == 0;
  for (int i = 0; i < a.pool_count; ++i) {
    if (!a.pools[i]) return CACHEIR_B200_EINVAL;
    wide = wide && aligned_to(a.pools[i], 16);
  }
  if (a.sequences > 65535 || static_cast<long long>(a.kv_heads) * a.dim > 1LL << 24) return CACHEIR_B200_ELIMIT;
  if (wide) return launch_keep<uint4>(a, as_stream(stream));
  return dtype_size(a.dtype) == 4 ? launch_keep<uint32_t>(a, as_stream(stream)) : launch_keep<uint16_t>(a, as_stream(stream));
}
