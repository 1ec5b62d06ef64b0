// Attention of drafted tokens over their sequence's pages: general kernels (any element type, head size, page size, heads per key/value head)
// and the C entry point.
//
// A tile is 32 (row, head) pairs of one sequence that share a key/value head; its keys are cut into pieces, which leave their maximum, sum and
// unnormalised output, and the pieces of a row are joined in order; with one piece the output is written as it ends. Within a piece 64 keys at a time, 64 columns of them at a time in shared memory as 32-bit floats;
// a thread has 2 x 4 scores, and for every 64 columns 2 x 4 outputs in registers, reads four numbers at a time of either operand, and has the next 64 columns on their way
// meanwhile. 32 trees of 12 to 16 tokens behind 256 to 4096, 32 query and 8 key/value heads, take 1970 us in fp32 with heads of 128, 2440 in bf16 with heads of
// 96 and 4640 with heads of 256 (with tiles of eight rows and a number at a time 6652 and 5226 of the first two; the ordinary decode attention of as many single rows 2685, 3060 and 3350).
// Most of that is waiting: two barriers around every 64 columns. So as many blocks as the registers allow share an SM, though a few numbers are spilled: three took 1980 and
// 4630 us where two took 2541 and 7700, and four 2205 in fp32; heads of more than 256 two blocks (14.4 ms with heads of 512, 22.8 with one).
#include "tree_attention.cuh"

namespace cb200 {
namespace {

constexpr int kTileRows = 32;
constexpr int kTileKeys = 64;
constexpr int kColumns = 64;                   // of keys or values in shared memory
constexpr int kLine = kColumns + 4;            // floats of a row of them (lanes that read rows beside one another reach different banks)
constexpr int kGeneralThreads = 256;
constexpr int kGeneralDim = 512;
constexpr int chunks_of(int dim) { return (dim + kColumns - 1) / kColumns; }
// queries [kTileRows][columns + 4], keys or values [kTileKeys][kLine], weights [kTileRows][kTileKeys + 4]
constexpr size_t general_smem(int dim) {
  return (static_cast<size_t>(kTileRows) * (chunks_of(dim) * kColumns + 4) + kTileKeys * kLine + kTileRows * (kTileKeys + 4)) * 4;
}

struct TreeParts {
  float* ml;       // [pieces][rows][heads][2]
  float* acc;      // [pieces][rows][heads][dim]
  int pieces;      // 1: there is no scratch
};

// Heads of up to kChunks * kColumns.
template <typename T, int kChunks>
__global__ void __launch_bounds__(kGeneralThreads, kChunks > 4 ? 2 : 3)
tree_general_kernel(const cacheir_b200_tree_args a, const TreeParts parts) {
  chain_enter();
  extern __shared__ __align__(16) float smem[];
  __shared__ long long s_line[2][kTileKeys];           // where a key of this tile, or of the next, begins in the pools; -1: it is not there
  __shared__ float s_scale[kTileRows], s_sum[kTileRows];
  const int D = a.dim, group = a.heads / a.kv_heads, chunks = chunks_of(D), q_line = chunks * kColumns + 4;
  const int piece = blockIdx.x % parts.pieces, kvh = blockIdx.x / parts.pieces % a.kv_heads, place = blockIdx.x / parts.pieces / a.kv_heads;
  float* s_q = smem;                                   // [kTileRows][q_line]
  float* s_kv = s_q + kTileRows * q_line;              // [kTileKeys][kLine]
  float* s_p = s_kv + kTileKeys * kLine;               // [kTileRows][kTileKeys + 4]
  // Sequence b has the tiles from floor(first row group / kTileRows) + b on: at least as many up to those of the next one as its rows fill.
  auto first_tile = [&](int b) { return static_cast<int>(static_cast<long long>(min(max(a.cu_rows[b], 0), a.rows)) * group / kTileRows) + b; };
  int b = 0, above = a.sequences;
  while (above - b > 1) {
    const int mid = (b + above) >> 1;
    if (first_tile(mid) <= place) b = mid; else above = mid;
  }
  const TreeSequence s = tree_sequence(a, b);
  const int first = (place - first_tile(b)) * kTileRows, rows = min(kTileRows, s.rows * group - first);
  if (first < 0 || rows <= 0) return;
  const int32_t* pages = a.page_table + static_cast<size_t>(b) * a.max_pages;
  const int step = ((s.keys + parts.pieces - 1) / parts.pieces + kTileKeys - 1) / kTileKeys * kTileKeys;
  const long long begin = static_cast<long long>(piece) * step;
  const int lo = static_cast<int>(min(begin, static_cast<long long>(s.keys))), hi = static_cast<int>(min(begin + step, static_cast<long long>(s.keys)));

  constexpr int kEach = kTileRows * kColumns / kGeneralThreads;  // queries of a thread in 64 columns, asked for together
  for (int c = threadIdx.x & (kColumns - 1); c < chunks * kColumns; c += kColumns) {
    float v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int r = threadIdx.x / kColumns + i * (kTileRows / kEach), pair = first + r;
      v[i] = r < rows && c < D ? Elem<T>::ld(static_cast<const T*>(a.q) + static_cast<size_t>(s.row + pair / group) * a.q_stride + (kvh * group + pair % group) * D + c) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) s_q[(threadIdx.x / kColumns + i * (kTileRows / kEach)) * q_line + c] = v[i];
  }
  const float qscale = a.softmax_scale * 1.4426950408889634f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;        // rows 2 ty, 2 ty + 1; keys tx + 16 j, or columns 4 tx ..
  float acc[kChunks][2][4] = {};
  float m_run[4], l_run[4];                                      // rows 4 warp ..
#pragma unroll
  for (int e = 0; e < 4; ++e) { m_run[e] = -INFINITY; l_run[e] = 0.f; }
  constexpr int kOwn = kTileKeys * kColumns / kGeneralThreads;   // numbers of a thread in 64 columns: one of every fourth key
  const int column = threadIdx.x & (kColumns - 1), own = threadIdx.x / kColumns;
  float ahead[kOwn];
  auto locate = [&](int k0, int place) {                         // the keys of the tile from k0 on
    if (threadIdx.x < kTileKeys) {
      const int t = k0 + threadIdx.x, id = t < hi ? pages[t / a.page_size] : -1;
      s_line[place][threadIdx.x] = id >= 0 && id < a.num_slots ? ((static_cast<long long>(id) * a.kv_heads + kvh) * a.page_size + t % a.page_size) * D : -1;
    }
  };
  auto ask = [&](const void* pool, int chunk, int place) {       // 64 columns of a tile's keys or values
    const int c = chunk * kColumns + column;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const long long line = s_line[place][own + i * (kTileKeys / kOwn)];
      ahead[i] = line >= 0 && c < D ? Elem<T>::ld(static_cast<const T*>(pool) + line + c) : 0.f;
    }
  };
  auto put = [&] {                                               // .. into shared memory, when everybody is done with what is there
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) s_kv[(own + i * (kTileKeys / kOwn)) * kLine + column] = ahead[i];
    __syncthreads();
  };
  int line_place = 0;
  if (lo < hi) {
    locate(lo, 0);
    __syncthreads();
    ask(a.k_cache, 0, 0);
  }
  for (int k0 = lo; k0 < hi; k0 += kTileKeys, line_place ^= 1) {
    const int n = min(kTileKeys, hi - k0);
    locate(k0 + kTileKeys, line_place ^ 1);
    // ---- scores ----
    float sc[2][4] = {};
    for (int chunk = 0; chunk < chunks; ++chunk) {
      put();
      if (chunk + 1 < chunks) ask(a.k_cache, chunk + 1, line_place);
      else ask(a.v_cache, 0, line_place);
      const float* q0 = s_q + 2 * ty * q_line + chunk * kColumns;
#pragma unroll 4
      for (int c = 0; c < kColumns; c += 4) {
        const float4 x = *reinterpret_cast<const float4*>(q0 + c), y = *reinterpret_cast<const float4*>(q0 + q_line + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 k = *reinterpret_cast<const float4*>(s_kv + (tx + 16 * j) * kLine + c);
          sc[0][j] = fmaf(x.x, k.x, fmaf(x.y, k.y, fmaf(x.z, k.z, fmaf(x.w, k.w, sc[0][j]))));
          sc[1][j] = fmaf(y.x, k.x, fmaf(y.y, k.y, fmaf(y.z, k.z, fmaf(y.w, k.w, sc[1][j]))));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s_p[(2 * ty + i) * (kTileKeys + 4) + tx + 16 * j] = sc[i][j];
    __syncthreads();
    // ---- weights: a warp has four rows, a lane two keys ----
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 4 * warp + e;
      float x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = k0 + lane + 32 * h, j = t - s.front;
        const bool seen = r < rows && lane + 32 * h < n && (j < 0 || (tree_word(a, s, (first + r) / group, j >> 5) >> (j & 31) & 1));
        x[h] = seen ? s_p[r * (kTileKeys + 4) + lane + 32 * h] * qscale : -INFINITY;
      }
      const float m_new = fmaxf(m_run[e], warp_max(fmaxf(x[0], x[1])));
      const float less = m_new > -INFINITY ? m_new : 0.f;             // (nothing seen yet: weights 0, but what is no number stays none)
      const float corr = exp2f(m_run[e] - less), p0 = exp2f(x[0] - less), p1 = exp2f(x[1] - less);
      l_run[e] = l_run[e] * corr + warp_sum(p0 + p1);
      m_run[e] = m_new;
      s_p[r * (kTileKeys + 4) + lane] = p0;
      s_p[r * (kTileKeys + 4) + lane + 32] = p1;
      if (lane == 0) s_scale[r] = corr;
    }
    // ---- outputs ----
    const bool drafted = k0 + n > s.front;                       // keys that not every row sees, and which may hold anything
#pragma unroll
    for (int chunk = 0; chunk < kChunks; ++chunk) {
      if (chunk >= chunks) break;
      put();
      if (chunk + 1 < chunks) ask(a.v_cache, chunk + 1, line_place);
      else if (k0 + kTileKeys < hi) ask(a.k_cache, 0, line_place ^ 1);
      const float f0 = s_scale[2 * ty], f1 = s_scale[2 * ty + 1];
      float o[2][4] = {};
      const float* p0 = s_p + 2 * ty * (kTileKeys + 4);
#pragma unroll 2
      for (int t = 0; t < kTileKeys; t += 4) {
        const float4 x4 = *reinterpret_cast<const float4*>(p0 + t), y4 = *reinterpret_cast<const float4*>(p0 + kTileKeys + 4 + t);
        const float x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 v = *reinterpret_cast<const float4*>(s_kv + (t + j) * kLine + 4 * tx);
          const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (!drafted || x[j] != 0.f) o[0][c] = fmaf(x[j], vs[c], o[0][c]);
            if (!drafted || y[j] != 0.f) o[1][c] = fmaf(y[j], vs[c], o[1][c]);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc[chunk][0][c] = acc[chunk][0][c] * f0 + o[0][c];
        acc[chunk][1][c] = acc[chunk][1][c] * f1 + o[1][c];
      }
    }
  }
  if (parts.pieces == 1) {                                       // nobody else has keys of these rows
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane == 0) s_sum[4 * warp + e] = l_run[e];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (2 * ty + i >= rows) continue;
      const int pair = first + 2 * ty + i;
      const float l = s_sum[2 * ty + i];
      T* to = static_cast<T*>(a.out) + static_cast<size_t>(s.row + pair / group) * a.out_stride + static_cast<size_t>(kvh * group + pair % group) * D;
#pragma unroll
      for (int chunk = 0; chunk < kChunks; ++chunk) {
        if (chunk >= chunks) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int d = chunk * kColumns + 4 * tx + c;
          if (d < D) Elem<T>::st(to + d, l > 0.f || l != l ? acc[chunk][i][c] / l : 0.f);
        }
      }
    }
    return;
  }
  auto at_pair = [&](int r) {                                    // of the scratch
    const int pair = first + r;
    return (static_cast<size_t>(piece) * a.rows + s.row + pair / group) * a.heads + kvh * group + pair % group;
  };
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = 4 * warp + e;
    if (r < rows && lane == 0) {
      parts.ml[2 * at_pair(r)] = m_run[e];
      parts.ml[2 * at_pair(r) + 1] = l_run[e];
    }
  }
#pragma unroll
  for (int chunk = 0; chunk < kChunks; ++chunk) {
    if (chunk >= chunks) break;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (2 * ty + i >= rows) continue;
      float* to = parts.acc + at_pair(2 * ty + i) * D;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = chunk * kColumns + 4 * tx + c;
        if (d < D) to[d] = acc[chunk][i][c];
      }
    }
  }
}

// One block per row and head; rows outside every sequence are left alone.
template <typename T>
__global__ void __launch_bounds__(128)
tree_join_kernel(const cacheir_b200_tree_args a, const TreeParts parts) {
  chain_enter();
  const int head = blockIdx.x % a.heads, row = blockIdx.x / a.heads;
  const int begin = min(max(a.cu_rows[0], 0), a.rows), end = min(max(a.cu_rows[a.sequences], 0), a.rows);
  if (row < begin || row >= end) return;
  const size_t at = static_cast<size_t>(row) * a.heads + head, step = static_cast<size_t>(a.rows) * a.heads;
  float m = -INFINITY, l = 0.f;
#pragma unroll 8
  for (int s = 0; s < parts.pieces; ++s) m = fmaxf(m, parts.ml[(s * step + at) * 2]);
#pragma unroll 8
  for (int s = 0; s < parts.pieces; ++s) {
    const float ms = parts.ml[(s * step + at) * 2];
    l = fmaf(parts.ml[(s * step + at) * 2 + 1], ms > -INFINITY ? exp2f(ms - m) : 1.f, l);
  }
  for (int d = threadIdx.x; d < a.dim; d += 128) {
    float o = 0.f;
#pragma unroll 8
    for (int s = 0; s < parts.pieces; ++s) {
      const float ms = parts.ml[(s * step + at) * 2], v = parts.acc[(s * step + at) * a.dim + d];
      o = ms > -INFINITY ? fmaf(v, exp2f(ms - m), o) : o;
    }
    Elem<T>::st(static_cast<T*>(a.out) + static_cast<size_t>(row) * a.out_stride + static_cast<size_t>(head) * a.dim + d, l > 0.f || l != l ? o / l : 0.f);
  }
}

template <typename T, int kChunks>
cudaError_t launch_tiles(const cacheir_b200_tree_args& a, const TreeParts& parts, long long blocks, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  auto kern = tree_general_kernel<T, kChunks>;
  cudaError_t e = allow_shared_memory(done, reinterpret_cast<const void*>(kern), static_cast<int>(general_smem(kChunks * kColumns)));
  if (e == cudaSuccess) e = launch_chained(kern, dim3(static_cast<unsigned>(blocks)), dim3(kGeneralThreads), general_smem(a.dim), stream, a, parts);
  return e;
}

template <typename T>
int launch_general(const cacheir_b200_tree_args& a, cudaStream_t stream) {
  const int group = a.heads / a.kv_heads;
  const long long tiles = static_cast<long long>(a.rows) * group / kTileRows + a.sequences;
  TreeParts parts;
  const long long want = 4LL * kNumSMs / (tiles * a.kv_heads), most = tree_pieces(a.rows, a.heads, a.dim);
  parts.pieces = static_cast<int>(want < 1 ? 1 : want > most ? most : want);
  parts.ml = static_cast<float*>(a.workspace);
  parts.acc = parts.ml + static_cast<size_t>(parts.pieces) * a.rows * a.heads * 2;
  const long long blocks = tiles * a.kv_heads * parts.pieces, ends = static_cast<long long>(a.rows) * a.heads;
  if (blocks > 0x7fffffffLL || ends > 0x7fffffffLL) return CACHEIR_B200_ELIMIT;
  const int chunks = chunks_of(a.dim);
  cudaError_t e = chunks == 1 ? launch_tiles<T, 1>(a, parts, blocks, stream) : chunks == 2 ? launch_tiles<T, 2>(a, parts, blocks, stream)
                  : chunks <= 4 ? launch_tiles<T, 4>(a, parts, blocks, stream) : launch_tiles<T, kGeneralDim / kColumns>(a, parts, blocks, stream);
  if (e == cudaSuccess && parts.pieces > 1) e = launch_chained(tree_join_kernel<T>, dim3(static_cast<unsigned>(ends)), dim3(128), 0, stream, a, parts);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" size_t cacheir_b200_tree_attention_workspace_bytes(int rows, int heads, int dim) {
  if (rows <= 0 || heads <= 0 || dim <= 0) return 0;
  const int pieces = tree_pieces(rows, heads, dim);
  const size_t general = pieces > 1 ? static_cast<size_t>(pieces) * rows * heads * (dim + 2) * 4 : 0, fast = tree_fast_bytes(dim);
  return general > fast ? general : fast;
}

extern "C" int cacheir_b200_tree_attention(const cacheir_b200_tree_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  cacheir_b200_tree_args a = *args;
  if (a.rows <= 0 || a.sequences <= 0 || a.heads <= 0) return 0;
  if (!a.q || !a.k_cache || !a.v_cache || !a.out || !a.page_table || !a.seq_lens || !a.cu_rows || a.kv_heads <= 0 || a.heads % a.kv_heads != 0 || a.dim <= 0 ||
      a.page_size <= 0 || a.num_slots <= 0 || a.max_pages <= 0 || (a.visible && a.words <= 0) || dtype_size(a.dtype) == 0)
    return CACHEIR_B200_EINVAL;
  if (a.dim > kGeneralDim) return CACHEIR_B200_EUNSUPPORTED;
  if (a.sequences > 65535 || a.rows > 1 << 24 || a.kv_heads > 65535 || static_cast<long long>(a.max_pages) * a.page_size > 1LL << 30 ||
      (a.visible && a.words > CACHEIR_B200_MAX_DRAFT_WORDS))
    return CACHEIR_B200_ELIMIT;
  const size_t need = cacheir_b200_tree_attention_workspace_bytes(a.rows, a.heads, a.dim);
  if ((need > 0 && !a.workspace) || a.workspace_bytes < need) return CACHEIR_B200_EWORKSPACE;
  if (!aligned_to(a.workspace, 16)) return CACHEIR_B200_EALIGN;
  if (!(a.softmax_scale > 0.f)) a.softmax_scale = 1.0f / sqrtf(static_cast<float>(a.dim));
  if (a.rows == 1) a.q_stride = a.out_stride = static_cast<long long>(a.heads) * a.dim;
  if (tree_fast_supported(a)) return launch_tree_fast(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F32) return launch_general<float>(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16) return launch_general<__half>(a, as_stream(stream));
  return launch_general<__nv_bfloat16>(a, as_stream(stream));
}

extern "C" int cacheir_b200_drafts_device_status(int reset) { return tree_device_status(reset != 0); }
