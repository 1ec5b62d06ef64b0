// Decode attention of groups of sequences with a common prefix: general kernels (any element type, head size, page size, heads per
// key/value head) and the C entry points.
//
// softmax over t < len of q K_t splits into the common keys, t < P, and the row's own ones. The common ones are read once for a tile of
// query rows, which are the (row, head) pairs of a group that share a key/value head; the own ones once for the heads of one row. Each
// part is cut into pieces; a piece leaves its maximum, sum and unnormalised output, and the pieces of a row are joined in order.
//
// These kernels are right for every case, not fast: bound by their own instructions, as each value is loaded by itself and a tile has only eight
// query rows for the keys it reads. They are slower than the ordinary decode attention, which reads every row's keys (32 query and 8 key/value
// heads, from a graph: 32 rows behind 2048 tokens 1485 us for 582 in float32 with heads of 128, 1027 for 343 in bf16 with heads of 96; 64 rows
// behind 32768 tokens 26120 for 4950 and 20193 for 5884).
#include "shared_prefix.cuh"

namespace cb200 {
namespace {

constexpr int kTileRows = 8;
constexpr int kTileKeys = 32;
constexpr int kGeneralThreads = 128;
constexpr int kGeneralDim = 512;
// queries, keys (a float further a row, so that lanes reach different banks), values, weights, scales
constexpr size_t general_smem(int dim) { return (static_cast<size_t>(kTileRows) * dim + kTileKeys * (2 * dim + 1) + kTileRows * (kTileKeys + 2)) * 4; }

template <typename T>
__global__ void __launch_bounds__(kGeneralThreads)
prefix_general_kernel(const cacheir_b200_prefix_args a, const PrefixParts parts, const int common_tiles) {
  chain_enter();
  extern __shared__ float smem[];
  // Blocks in the order of tiles, key/value heads, pieces: the common parts, which are long, come first.
  const int D = a.dim, group = a.heads / a.kv_heads, half = parts.pieces / 2;
  const int piece = blockIdx.x % half, kvh = blockIdx.x / half % a.kv_heads, place = blockIdx.x / half / a.kv_heads;
  float* s_q = smem;                                   // [kTileRows][D]
  float* s_k = s_q + kTileRows * D;                    // [kTileKeys][D + 1]
  float* s_v = s_k + kTileKeys * (D + 1);              // [kTileKeys][D]
  float* s_p = s_v + kTileKeys * D;                    // [kTileRows][kTileKeys + 1]
  float* s_scale = s_p + kTileRows * (kTileKeys + 1);  // [kTileRows]
  const bool common = place < common_tiles;
  // ---- which query rows (row = base + i / group, head i % group) and which keys ----
  int base, first, rows, key_lo, key_hi;
  const int32_t* pages;
  if (common) {
    // Group g has the tiles from floor(start heads / kTileRows) + g on: at least as many up to those of the next group as its rows fill.
    auto first_tile = [&](int g) { return static_cast<int>(static_cast<long long>(group_start(a, g)) * group / kTileRows) + g; };
    int g = 0, hi = a.groups;
    while (hi - g > 1) {
      const int mid = (g + hi) >> 1;
      if (first_tile(mid) <= place) g = mid; else hi = mid;
    }
    base = group_start(a, g);
    first = (place - first_tile(g)) * kTileRows;
    rows = min(kTileRows, (group_start(a, g + 1) - base) * group - first);
    if (first < 0) return;                             // (rows before the first group)
    key_lo = 0;
    key_hi = rows <= 0 ? 0 : prefix_of_group(a, g);    // (a tile of no rows looks at no keys)
    pages = a.prefix_table + static_cast<size_t>(g) * a.prefix_pages;
  } else {
    const int per_row = (group + kTileRows - 1) / kTileRows, tile = place - common_tiles;
    base = tile / per_row;
    first = tile % per_row * kTileRows;
    rows = min(kTileRows, group - first);
    group_of_row(a, base, &key_lo);
    key_hi = min(max(a.seq_lens[base], 0), a.max_pages * a.page_size);
    pages = a.page_table + static_cast<size_t>(base) * a.max_pages;
  }
  // neighbouring pieces of the same size, whole key tiles
  const int keys = max(key_hi - key_lo, 0), step = ((keys + half - 1) / half + kTileKeys - 1) / kTileKeys * kTileKeys;
  const long long begin = key_lo + static_cast<long long>(piece) * step;
  const int lo = static_cast<int>(min(begin, static_cast<long long>(key_hi))), hi = static_cast<int>(min(begin + step, static_cast<long long>(key_hi)));

  for (int i = threadIdx.x; i < rows * D; i += kGeneralThreads) {
    const int r = first + i / D;
    s_q[i] = Elem<T>::ld(static_cast<const T*>(a.q) + static_cast<size_t>(base + r / group) * a.q_stride + (kvh * group + r % group) * D + i % D);
  }
  const float qscale = a.softmax_scale * 1.4426950408889634f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float acc[kTileRows][kGeneralDim / kGeneralThreads] = {};
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};    // rows 2 warp, 2 warp + 1
  int row_len[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * warp + e;
    row_len[e] = i < rows ? a.seq_lens[base + (first + i) / group] : 0;
  }
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
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(s_q[r * D + d], s_k[lane * (D + 1) + d], s);
      s = lane < n && k0 + lane < row_len[e] ? s * qscale : -INFINITY;
      const float m_new = fmaxf(m_run[e], warp_max(s));
      const float less = m_new > -INFINITY ? m_new : 0.f;             // (nothing seen yet: weights 0, but what is no number stays none)
      const float corr = exp2f(m_run[e] - less), p = exp2f(s - less);
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
  const int slot = common ? piece : half + piece;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * warp + e;
    if (i < rows && lane == 0) {
      const int r = first + i;
      float* ml = parts.ml + ((static_cast<size_t>(slot) * a.batch + base + r / group) * a.heads + kvh * group + r % group) * 2;
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
        parts.acc[((static_cast<size_t>(slot) * a.batch + base + r / group) * a.heads + kvh * group + r % group) * D + d] = acc[i][j];
      }
  }
}

template <typename T>
__global__ void __launch_bounds__(128)
prefix_join_kernel(const cacheir_b200_prefix_args a, const PrefixParts parts) {
  chain_enter();
  const int head = blockIdx.x, row = blockIdx.y, half = parts.pieces / 2;
  int prefix;
  const int from = group_of_row(a, row, &prefix) < 0 ? half : 0;      // no group: no common pieces were written
  const size_t at = static_cast<size_t>(row) * a.heads + head, step = static_cast<size_t>(a.batch) * a.heads;
  float m = -INFINITY, l = 0.f;
  for (int s = from; s < parts.pieces; ++s) m = fmaxf(m, parts.ml[(s * step + at) * 2]);
  for (int s = from; s < parts.pieces; ++s) {
    const float ms = parts.ml[(s * step + at) * 2];
    l = fmaf(parts.ml[(s * step + at) * 2 + 1], ms > -INFINITY ? exp2f(ms - m) : 0.f, l);
  }
  for (int d = threadIdx.x; d < a.dim; d += 128) {
    float o = 0.f;
    for (int s = from; s < parts.pieces; ++s) {
      const float ms = parts.ml[(s * step + at) * 2];
      if (ms > -INFINITY) o = fmaf(parts.acc[(s * step + at) * a.dim + d], exp2f(ms - m), o);
    }
    Elem<T>::st(static_cast<T*>(a.out) + static_cast<size_t>(row) * a.out_stride + static_cast<size_t>(head) * a.dim + d, l > 0.f || l != l ? o / l : 0.f);
  }
}

template <typename T>
int launch_general(const cacheir_b200_prefix_args& a, PrefixParts parts, cudaStream_t stream) {
  const int group = a.heads / a.kv_heads;
  const long long common = static_cast<long long>(a.batch) * group / kTileRows + a.groups;
  const long long tiles = (a.groups > 0 ? common : 0) + static_cast<long long>(a.batch) * ((group + kTileRows - 1) / kTileRows);
  const long long want = 4LL * kNumSMs / (tiles * a.kv_heads);
  const int half = static_cast<int>(want < 1 ? 1 : want > parts.pieces / 2 ? parts.pieces / 2 : want);
  parts.pieces = 2 * half;
  const long long blocks = tiles * a.kv_heads * half;
  if (blocks > 0x7fffffffLL) return CACHEIR_B200_ELIMIT;
  const size_t smem = general_smem(a.dim);
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_shared_memory(done, reinterpret_cast<const void*>(prefix_general_kernel<T>), static_cast<int>(general_smem(kGeneralDim)));
  if (e == cudaSuccess)
    e = launch_chained(prefix_general_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kGeneralThreads), smem, stream, a, parts,
                       static_cast<int>(a.groups > 0 ? common : 0));
  if (e == cudaSuccess) e = launch_chained(prefix_join_kernel<T>, dim3(a.heads, a.batch), dim3(128), 0, stream, a, parts);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" size_t cacheir_b200_shared_prefix_workspace_bytes(int batch, int heads, int dim) {
  if (batch <= 0 || heads <= 0 || dim <= 0) return 0;
  const int pieces = prefix_pieces(batch, heads, dim) + own_parts(batch);
  return prefix_plan_bytes(batch) + prefix_ml_bytes(batch, heads, pieces) + static_cast<size_t>(pieces) * batch * heads * dim * 4;
}

extern "C" int cacheir_b200_shared_prefix_launches(int batch, int heads, int kv_heads, int dim, int page_size, int groups, int dtype) {
  if (batch <= 0 || heads <= 0) return 0;
  if (kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0 || page_size <= 0) return CACHEIR_B200_EINVAL;
  cacheir_b200_prefix_args a{};
  a.batch = batch;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.page_size = page_size;
  a.num_slots = a.max_pages = a.prefix_pages = 1;
  a.groups = groups;
  a.dtype = dtype;
  return prefix_fast_supported(a) ? prefix_fast_launches(groups) : 2;
}

extern "C" int cacheir_b200_shared_prefix_attention(const cacheir_b200_prefix_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  cacheir_b200_prefix_args a = *args;
  if (a.batch <= 0 || a.heads <= 0) return 0;
  if (!a.q || !a.k_cache || !a.v_cache || !a.out || !a.page_table || !a.seq_lens || a.kv_heads <= 0 || a.heads % a.kv_heads != 0 || a.dim <= 0 ||
      a.page_size <= 0 || a.num_slots <= 0 || a.max_pages <= 0 || a.groups < 0 || dtype_size(a.dtype) == 0)
    return CACHEIR_B200_EINVAL;
  if (a.groups > a.batch) return CACHEIR_B200_EINVAL;
  if (a.groups > 0 && (!a.group_rows || !a.prefix_table || !a.prefix_lens || a.prefix_pages <= 0)) return CACHEIR_B200_EINVAL;
  if (a.dim > kGeneralDim) return CACHEIR_B200_EUNSUPPORTED;
  if (a.batch > 65535 || a.kv_heads > 65535 || static_cast<long long>(a.max_pages) * a.page_size > 1LL << 30 ||
      static_cast<long long>(a.prefix_pages) * a.page_size > 1LL << 30)
    return CACHEIR_B200_ELIMIT;
  if (!a.workspace || a.workspace_bytes < cacheir_b200_shared_prefix_workspace_bytes(a.batch, a.heads, a.dim)) return CACHEIR_B200_EWORKSPACE;
  if (!aligned_to(a.workspace, 16)) return CACHEIR_B200_EALIGN;
  if (!(a.softmax_scale > 0.f)) a.softmax_scale = 1.0f / sqrtf(static_cast<float>(a.dim));
  PrefixParts parts;
  parts.pieces = prefix_pieces(a.batch, a.heads, a.dim);
  parts.own = own_parts(a.batch);
  char* scratch = static_cast<char*>(a.workspace);
  parts.plan = reinterpret_cast<PrefixPlan*>(scratch);
  parts.ml = reinterpret_cast<float*>(scratch += prefix_plan_bytes(a.batch));
  parts.acc = reinterpret_cast<float*>(scratch + prefix_ml_bytes(a.batch, a.heads, parts.pieces + parts.own));
  if (prefix_fast_supported(a)) return launch_prefix_fast(a, parts, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F32) return launch_general<float>(a, parts, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16) return launch_general<__half>(a, parts, as_stream(stream));
  return launch_general<__nv_bfloat16>(a, parts, as_stream(stream));
}

extern "C" int cacheir_b200_serving_device_status(int reset) {
  const int found[] = {prefix_device_status(reset != 0), logprobs_device_status(reset != 0)};
  for (int status : found)
    if (status != 0) return status;
  return 0;
}
