// Page tables of a batch, kept on the device: pages for new tokens off a stack of free ones, the map from the rows of a step to page
// slots, and the way back.
//
// With P tokens to a page, sequence b of len tokens that gets n more needs ceil((len + n) / P) - ceil(len / P) new pages. Two running
// sums over the sequences, of rows and of pages, say where its rows stand and which pages of the stack are its own; everything else is
// then independent: a page goes to its place in a table, a row finds its sequence by bisection in the row sums.
//
// Little data (12 bytes a row, 8 a page, 12 a sequence) and much latency: read lengths, sum, look up, write. So it is one launch, of one block
// where there is little to do. A call changes what it reads (lengths, stack height), so all reads of those come before all writes: the
// blocks are one thread-block cluster, each of which sums all sequences by itself, and meet once in between. Many rows (above 2048) are left
// to a second kernel on all SMs, which needs only what the first one leaves: 1024 sequences with 0 to 255 new tokens each in 140001
// rows and the way back took 40.6 us with the rows in one cluster of eight blocks and the way back in one block, 15.7 us like this (from a graph).
#include "cacheir_b200_serving.h"
#include "common.cuh"
#include "serving_status.h"
#include "tc_ptx.cuh"

namespace cb200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kClusterBlocks = 8;
constexpr int kOwnRows = 2048;              // rows that the first kernel takes itself
constexpr int kRowsPerWarp = 128;

struct TableArgs : cacheir_b200_tables_args {
  int fills;                  // extend: the rows are filled in here
};

__device__ __forceinline__ int pages_of(long long tokens, int page_size) { return static_cast<int>((tokens + page_size - 1) / page_size); }

// Exclusive sums over the block of two numbers per thread, and their totals.
__device__ __forceinline__ void block_scan(long long (&v)[2], long long (&total)[2]) {
  __shared__ long long s_warp[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long own[2] = {v[0], v[1]};
#pragma unroll
  for (int off = 1; off < 32; off <<= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long up = __shfl_up_sync(0xffffffffu, v[i], off);
      if (lane >= off) v[i] += up;
    }
  if (lane == 31) { s_warp[0][warp] = v[0]; s_warp[1][warp] = v[1]; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    long long w = lane < static_cast<int>(blockDim.x >> 5) ? s_warp[i][lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += up;
    }
    total[i] = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    v[i] = v[i] - own[i] + (warp > 0 ? before : 0);
  }
}

// Last index i with starts[i] <= at (starts[0] = 0, n entries).
__device__ __forceinline__ int owner(const int32_t* starts, int n, int at) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= at) lo = mid; else hi = mid;
  }
  return lo;
}

template <bool EXTEND>
__global__ void __launch_bounds__(kThreads)
page_tables_kernel(const TableArgs p) {
  chain_enter();
  extern __shared__ int32_t smem[];
  int32_t* s_len = smem;                                    // [sequences] tokens before
  int32_t* s_page = s_len + p.sequences;                    // [sequences] first page of the call that is this sequence's
  int32_t* s_row = s_page + p.sequences;                    // extend: [sequences] first row
  const int rank = blockIdx.x, ranks = gridDim.x, n = p.sequences;
  const int per = (n + blockDim.x - 1) / blockDim.x;        // neighbouring sequences of a thread
  const int lo = min(n, static_cast<int>(threadIdx.x) * per), hi = min(n, lo + per);
  const int count = *p.free_count;

  // ---- what every sequence needs ----
  long long sum[2] = {0, 0}, total[2];
  bool bad = false;
  const long long room = static_cast<long long>(p.max_pages) * p.page_size;
  auto need = [&](int b, int len, int* tokens) {            // pages that come or go
    if constexpr (EXTEND) {
      *tokens = max(p.change[b], 0);
      return pages_of(static_cast<long long>(len) + *tokens, p.page_size) - pages_of(len, p.page_size);
    } else {
      *tokens = min(max(p.change[b], 0), len);
      const int first = max(pages_of(*tokens, p.page_size), p.held_pages ? p.held_pages[b] : 0);
      return max(0, pages_of(len, p.page_size) - first);
    }
  };
  for (int b = lo; b < hi; ++b) {
    const int len = max(p.seq_lens[b], 0);
    int tokens;
    const int pages = need(b, len, &tokens);
    bad = bad || static_cast<long long>(len) + (EXTEND ? tokens : 0) > room;
    s_len[b] = len;
    sum[0] += tokens;
    sum[1] += pages;
  }
  block_scan(sum, total);
  const bool too_long = __syncthreads_or(bad ? 1 : 0) != 0;
  int why = 0;
  if (too_long) why = -2;
  else if (count < 0 || count > p.capacity || (!EXTEND && count + total[1] > p.capacity)) why = -3;
  else if (EXTEND && total[0] > p.rows) why = -1;
  else if (EXTEND && total[1] > count) why = static_cast<int>(min(total[1] - count, 0x7fffffffLL));
  // (sums that are used below fit in 32 bits: rows <= p.rows, pages <= capacity)
  if (why == 0) {
    long long row = sum[0], page = sum[1];
    for (int b = lo; b < hi; ++b) {
      int tokens;
      const int pages = need(b, s_len[b], &tokens);
      s_page[b] = static_cast<int32_t>(page);
      if constexpr (EXTEND) s_row[b] = static_cast<int32_t>(row);
      row += tokens;
      page += pages;
    }
  }
  __syncthreads();
  if (ranks > 1) ptx::cluster_sync_release();               // everybody has read what the call changes
  const int pages = why == 0 ? static_cast<int>(total[1]) : 0;

  // ---- lengths, heights, row starts ----
  if (rank == 0) {
    if (why != 0) {
      if (threadIdx.x == 0 && *p.status == 0) *p.status = why;
      if constexpr (EXTEND)
        for (int b = threadIdx.x; b <= n; b += blockDim.x) p.cu_rows[b] = 0;
    } else {
      for (int b = threadIdx.x; b < n; b += blockDim.x) {
        const int len = s_len[b];
        if constexpr (EXTEND) {
          const int first = s_row[b], end = b + 1 < n ? s_row[b + 1] : static_cast<int>(total[0]);
          p.cu_rows[b] = first;
          p.seq_lens[b] = len + end - first;
        } else {
          p.seq_lens[b] = min(max(p.change[b], 0), len);
        }
      }
      if (threadIdx.x == 0) {
        if constexpr (EXTEND) p.cu_rows[n] = static_cast<int32_t>(total[0]);
        *p.free_count = EXTEND ? count - pages : count + pages;
      }
    }
  }
  // ---- pages ----
  const int thread = rank * blockDim.x + threadIdx.x, threads = ranks * blockDim.x;
  for (int i = thread; i < pages; i += threads) {
    const int b = owner(s_page, n, i);
    int32_t* row = p.page_table + static_cast<size_t>(b) * p.max_pages;
    if constexpr (EXTEND) {
      row[pages_of(s_len[b], p.page_size) + i - s_page[b]] = p.free_pages[count - 1 - i];
    } else {
      const int after = b + 1 < n ? s_page[b + 1] : pages;  // the sequence's pages are its last ones
      p.free_pages[count + pages - 1 - i] = row[pages_of(s_len[b], p.page_size) - (after - i)];
    }
  }
  // ---- rows ----
  if constexpr (EXTEND) {
    const int used = why == 0 ? static_cast<int>(total[0]) : 0;
    for (int r = thread; r < (p.fills ? p.rows : 0); r += threads) {
      int pos = 0, b = -1, slot = -1;
      if (r < used) {
        b = owner(s_row, n, r);
        pos = s_len[b] + r - s_row[b];
        const int page = pos / p.page_size, opened = page - pages_of(s_len[b], p.page_size);
        const int id = opened < 0 ? p.page_table[static_cast<size_t>(b) * p.max_pages + page] : p.free_pages[count - 1 - (s_page[b] + opened)];
        slot = id * p.page_size + pos % p.page_size;
      }
      p.positions[r] = pos;
      p.row_seq[r] = b;
      p.slots[r] = slot;
    }
  }
}

// The rows of a call whose sequences have been dealt with: 128 neighbours a warp, four a lane.
__global__ void __launch_bounds__(256)
token_rows_kernel(const TableArgs p) {
  chain_enter();
  const int lane = threadIdx.x & 31, first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kRowsPerWarp, r0 = first + lane * 4;
  if (first >= p.rows) return;
  const int n = p.sequences, used = p.cu_rows[n];
  int pos[4] = {0, 0, 0, 0}, seq[4] = {-1, -1, -1, -1}, slot[4] = {-1, -1, -1, -1};
  if (first < used) {
    // The sequence of the warp's first row: the starts up to it are counted, 32 of them looked at at a time.
    int lo = 0, hi = n;
    while (hi > lo) {
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const int below = __popc(__ballot_sync(0xffffffffu, at < hi && p.cu_rows[at] <= first));
      if (below == 0) break;
      const int found = lo + (below - 1) * step;
      hi = min(hi, found + step);
      lo = found + 1;
    }
    const int base = lo - 1, last = min(first + kRowsPerWarp, used) - 1;
    int count[4] = {base, base, base, base};
    for (int b = base + 1; b < n; b += 32) {               // .. and of the others: the starts behind that
      const int start = b + lane < n ? p.cu_rows[b + lane] : 0x7fffffff;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int s = __shfl_sync(0xffffffffu, start, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) count[j] += s <= r0 + j ? 1 : 0;
      }
      if (__shfl_sync(0xffffffffu, start, 31) > last) break;
    }
    int end[4], len[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      end[j] = r0 + j < used ? p.cu_rows[count[j] + 1] : 0;
      len[j] = r0 + j < used ? p.seq_lens[count[j]] : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r0 + j < used) {
        seq[j] = count[j];
        pos[j] = len[j] - (end[j] - (r0 + j));
        slot[j] = p.page_table[static_cast<size_t>(seq[j]) * p.max_pages + pos[j] / p.page_size] * p.page_size + pos[j] % p.page_size;
      }
  }
  const bool wide = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.row_seq) | reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
  if (wide && r0 + 4 <= p.rows) {
    *reinterpret_cast<int4*>(p.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    *reinterpret_cast<int4*>(p.row_seq + r0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
    *reinterpret_cast<int4*>(p.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r0 + j < p.rows) {
        p.positions[r0 + j] = pos[j];
        p.row_seq[r0 + j] = seq[j];
        p.slots[r0 + j] = slot[j];
      }
  }
}

template <bool EXTEND>
int launch_tables(const TableArgs& a, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(a.sequences) * (EXTEND ? 3 : 2) * 4;
  if (smem > 40 * 1024) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = allow_shared_memory(done, reinterpret_cast<const void*>(page_tables_kernel<EXTEND>), CACHEIR_B200_MAX_SEQUENCES * 12);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const bool few = a.sequences <= 128 && (!EXTEND || a.rows <= 512);
  const int blocks = a.sequences > 256 || (EXTEND && a.rows > 1024) ? kClusterBlocks : 1;
  cudaError_t e = launch_clusters(page_tables_kernel<EXTEND>, dim3(blocks), dim3(few ? 128 : kThreads), smem, stream, dim3(blocks), a);
  if (EXTEND && !a.fills && e == cudaSuccess)
    e = launch_chained(token_rows_kernel, dim3((a.rows + 8 * kRowsPerWarp - 1) / (8 * kRowsPerWarp)), dim3(256), 0, stream, a);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_extend_page_tables(const cacheir_b200_tables_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_tables_args& a = *args;
  if (a.sequences <= 0 || a.rows <= 0) return 0;
  if (!a.page_table || !a.seq_lens || !a.change || !a.free_pages || !a.free_count || !a.positions || !a.row_seq || !a.slots || !a.cu_rows || !a.status ||
      a.max_pages <= 0 || a.page_size <= 0 || a.capacity <= 0)
    return CACHEIR_B200_EINVAL;
  if (a.sequences > CACHEIR_B200_MAX_SEQUENCES || static_cast<long long>(a.max_pages) * a.page_size > 0x7fffffffLL) return CACHEIR_B200_ELIMIT;
  return launch_tables<true>(TableArgs{a, a.rows <= kOwnRows ? 1 : 0}, as_stream(stream));
}

extern "C" int cacheir_b200_shrink_page_tables(const cacheir_b200_tables_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_tables_args& a = *args;
  if (a.sequences <= 0) return 0;
  if (!a.page_table || !a.seq_lens || !a.change || !a.free_pages || !a.free_count || !a.status || a.max_pages <= 0 || a.page_size <= 0 || a.capacity <= 0)
    return CACHEIR_B200_EINVAL;
  if (a.sequences > CACHEIR_B200_MAX_SEQUENCES || static_cast<long long>(a.max_pages) * a.page_size > 0x7fffffffLL) return CACHEIR_B200_ELIMIT;
  return launch_tables<false>(TableArgs{a, 0}, as_stream(stream));
}
