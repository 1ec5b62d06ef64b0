// Attention of drafted tokens over their sequence's pages: general kernels (any element type, head size, page size, heads per key/value head)
// and the C entry point.
//
// A tile is eight (row, head) pairs of one sequence that share a key/value head; its keys are cut into pieces, which leave their maximum, sum and
// unnormalised output, and the pieces of a row are joined in order. Right for every case, not fast: each value is loaded by itself and a tile has only eight
// query rows for the keys that it reads.
#include "tree_attention.cuh"

namespace cb200 {
namespace {

constexpr int kTileRows = 8;
constexpr int kTileKeys = 32;
constexpr int kGeneralThreads = 128;
constexpr int kGeneralDim = 512;
// queries, keys (a float further a row, so that lanes reach different banks), values, weights, scales
constexpr size_t general_smem(int dim) { return (static_cast<size_t>(kTileRows) * dim + kTileKeys * (2 * dim + 1) + kTileRows * (kTileKeys + 2)) * 4; }

struct TreeParts {
  float* ml;       // [pieces][rows][heads][2]
  float* acc;      // [pieces][rows][heads][dim]
  int pieces;
};

template <typename T>
__global__ void __launch_bounds__(kGeneralThreads)
tree_general_kernel(const cacheir_b200_tree_args a, const TreeParts parts) {
  chain_enter();
  extern __shared__ float smem[];
  const int D = a.dim, group = a.heads / a.kv_heads;
  const int piece = blockIdx.x % parts.pieces, kvh = blockIdx.x / parts.pieces % a.kv_heads, place = blockIdx.x / parts.pieces / a.kv_heads;
  float* s_q = smem;                                   // [kTileRows][D]
  float* s_k = s_q + kTileRows * D;                    // [kTileKeys][D + 1]
  float* s_v = s_k + kTileKeys * (D + 1);              // [kTileKeys][D]
  float* s_p = s_v + kTileKeys * D;                    // [kTileRows][kTileKeys + 1]
  float* s_scale = s_p + kTileRows * (kTileKeys + 1);  // [kTileRows]
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

  for (int i = threadIdx.x; i < rows * D; i += kGeneralThreads) {
    const int r = first + i / D;
    s_q[i] = Elem<T>::ld(static_cast<const T*>(a.q) + static_cast<size_t>(s.row + r / group) * a.q_stride + (kvh * group + r % group) * D + i % D);
  }
  const float qscale = a.softmax_scale * 1.4426950408889634f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float acc[kTileRows][kGeneralDim / kGeneralThreads] = {};
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};    // rows 2 warp, 2 warp + 1
  for (int k0 = lo; k0 < hi; k0 += kTileKeys) {
    const int n = min(kTileKeys, hi - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < kTileKeys * D; i += kGeneralThreads) {
      const int t = i / D, d = i - t * D;
      float kv = 0.f, vv = 0.f;
      if (t < n) {
        const int id = pages[(k0 + t) / a.page_size];
        if (id >= 0 && id < a.num_slots) {
          const size_t at = ((static_cast<size_t>(id) * a.kv_heads + kvh) * a.page_size + (k0 + t) % a.page_size) * D + d;
          kv = Elem<T>::ld(static_cast<const T*>(a.k_cache) + at);
          vv = Elem<T>::ld(static_cast<const T*>(a.v_cache) + at);
        }
      }
      s_k[t * (D + 1) + d] = kv;
      s_v[i] = vv;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * warp + e;
      if (r >= rows) continue;
      float x = 0.f;
      for (int d = 0; d < D; ++d) x = fmaf(s_q[r * D + d], s_k[lane * (D + 1) + d], x);
      const int t = k0 + lane, j = t - s.front;
      const bool seen = lane < n && (j < 0 || (tree_word(a, s, (first + r) / group, j >> 5) >> (j & 31) & 1));
      x = seen ? x * qscale : -INFINITY;
      const float m_new = fmaxf(m_run[e], warp_max(x));
      const float less = m_new > -INFINITY ? m_new : 0.f;             // (nothing seen yet: weights 0, but what is no number stays none)
      const float corr = exp2f(m_run[e] - less), p = exp2f(x - less);
      l_run[e] = l_run[e] * corr + warp_sum(p);
      m_run[e] = m_new;
      s_p[r * (kTileKeys + 1) + lane] = p;
      if (lane == 0) s_scale[r] = corr;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kGeneralDim / kGeneralThreads; ++j) {
      const int d = threadIdx.x + j * kGeneralThreads;
      if (d >= D) break;
      for (int r = 0; r < rows; ++r) {
        float o = 0.f;
        for (int t = 0; t < n; ++t) {
          const float p = s_p[r * (kTileKeys + 1) + t];
          if (p != 0.f) o = fmaf(p, s_v[t * D + d], o);     // (keys that a row does not see may hold anything)
        }
        // constant indices keep the sums in registers
#pragma unroll
        for (int q = 0; q < kTileRows; ++q)
          if (q == r) acc[q][j] = acc[q][j] * s_scale[r] + o;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * warp + e;
    if (i < rows && lane == 0) {
      const int r = first + i;
      float* ml = parts.ml + ((static_cast<size_t>(piece) * a.rows + s.row + r / group) * a.heads + kvh * group + r % group) * 2;
      ml[0] = m_run[e];
      ml[1] = l_run[e];
    }
  }
#pragma unroll
  for (int j = 0; j < kGeneralDim / kGeneralThreads; ++j) {
    const int d = threadIdx.x + j * kGeneralThreads;
    if (d >= D) break;
#pragma unroll
    for (int i = 0; i < kTileRows; ++i)
      if (i < rows) {
        const int r = first + i;
        parts.acc[((static_cast<size_t>(piece) * a.rows + s.row + r / group) * a.heads + kvh * group + r % group) * D + d] = acc[i][j];
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
  for (int s = 0; s < parts.pieces; ++s) m = fmaxf(m, parts.ml[(s * step + at) * 2]);
  for (int s = 0; s < parts.pieces; ++s) {
    const float ms = parts.ml[(s * step + at) * 2];
    l = fmaf(parts.ml[(s * step + at) * 2 + 1], ms > -INFINITY ? exp2f(ms - m) : 1.f, l);
  }
  for (int d = threadIdx.x; d < a.dim; d += 128) {
    float o = 0.f;
    for (int s = 0; s < parts.pieces; ++s) {
      const float ms = parts.ml[(s * step + at) * 2];
      if (ms > -INFINITY) o = fmaf(parts.acc[(s * step + at) * a.dim + d], exp2f(ms - m), o);
    }
    Elem<T>::st(static_cast<T*>(a.out) + static_cast<size_t>(row) * a.out_stride + static_cast<size_t>(head) * a.dim + d, l > 0.f || l != l ? o / l : 0.f);
  }
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
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_shared_memory(done, reinterpret_cast<const void*>(tree_general_kernel<T>), static_cast<int>(general_smem(kGeneralDim)));
  if (e == cudaSuccess)
    e = launch_chained(tree_general_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kGeneralThreads), general_smem(a.dim), stream, a, parts);
  if (e == cudaSuccess) e = launch_chained(tree_join_kernel<T>, dim3(static_cast<unsigned>(ends)), dim3(128), 0, stream, a, parts);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" size_t cacheir_b200_tree_attention_workspace_bytes(int rows, int heads, int dim) {
  if (rows <= 0 || heads <= 0 || dim <= 0) return 0;
  const size_t general = static_cast<size_t>(tree_pieces(rows, heads, dim)) * rows * heads * (dim + 2) * 4, fast = tree_fast_bytes(dim);
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
  if (!a.workspace || a.workspace_bytes < cacheir_b200_tree_attention_workspace_bytes(a.rows, a.heads, a.dim)) return CACHEIR_B200_EWORKSPACE;
  if (!aligned_to(a.workspace, 16)) return CACHEIR_B200_EALIGN;
  if (!(a.softmax_scale > 0.f)) a.softmax_scale = 1.0f / sqrtf(static_cast<float>(a.dim));
  if (a.rows == 1) a.q_stride = a.out_stride = static_cast<long long>(a.heads) * a.dim;
  if (tree_fast_supported(a)) return launch_tree_fast(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F32) return launch_general<float>(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16) return launch_general<__half>(a, as_stream(stream));
  return launch_general<__nv_bfloat16>(a, as_stream(stream));
}

extern "C" int cacheir_b200_drafts_device_status(int reset) { return tree_device_status(reset != 0); }
