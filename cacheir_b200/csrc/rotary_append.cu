// Rotary positions of q and k rows, both pair layouts, whole heads or the first part of each, with the append of k and v to the page
// pool by slot.
//
//   (a, b) -> factor * (a cos - b sin, a sin + b cos), angle = position * frequency
//
// Bound by memory: every value is read and written once. One block per row; its cosines are worked out once for all heads. Where there are
// many rows, small blocks: 16384 rows of 64 + 8 heads of 128 in fp16 take 116 us (5.8 TB/s; from a graph, in bursts: 126 on end, under the power
// cap) with 64 threads a block, 119 with 128 and 134 with 192; few rows want more of a row under way (32 rows: 4.8, 3.5 and 3.1 us). Asking for the values before the cosines, cosines in
// registers, and rows streamed through shared memory by bulk copies (201 us) were all slower.
#include "cacheir_b200_serving.h"
#include "common.cuh"
#include "rotary_turn.cuh"

namespace cb200 {
namespace {

constexpr int kMaxThreads = 256;
constexpr int kMaxDim = 1024;

// A unit is VEC pairs (or 2 VEC values that are only copied): two vectors of VEC values.
template <typename T, int VEC>
__global__ void __launch_bounds__(kMaxThreads)
rotary_append_kernel(const cacheir_b200_rotary_args p) {
  chain_enter();
  __shared__ float2 s_turn[kMaxDim / 2];
  const int row = blockIdx.x, threads = blockDim.x;
  long long line = 0;                                       // of the pool, in rows of a kv head
  if (p.slots) {
    const int slot = p.slots[row];
    if (slot < 0 || slot / p.page_size >= p.num_slots) return;
    line = static_cast<long long>(slot / p.page_size) * p.kv_heads * p.page_size + slot % p.page_size;
  }
  const int half = p.rot / 2, position = p.positions[row];
  for (int i = threadIdx.x; i < half; i += threads) s_turn[i] = turn_cos_sin(p.turns[i], position, p.factor);
  __syncthreads();
  const int turning = half / VEC, units = turning + (p.dim - p.rot + 2 * VEC - 1) / (2 * VEC);       // per head
  const int heads = p.heads + (p.slots ? 2 : 1) * p.kv_heads;
  for (int u = threadIdx.x; u < heads * units; u += threads) {
    const int head = u / units, j = u - head * units;
    const bool is_q = head < p.heads, is_v = head >= p.heads + p.kv_heads;
    const int h = is_q ? head : (head - p.heads) % p.kv_heads;
    const T* src = is_q ? static_cast<const T*>(p.q) + row * p.q_stride
                        : is_v ? static_cast<const T*>(p.v) + row * p.v_stride : static_cast<const T*>(p.k) + row * p.k_stride;
    src += static_cast<size_t>(h) * p.dim;
    const bool turns = j < turning;
    const int at = !turns ? p.rot + (j - turning) * 2 * VEC : p.layout == CACHEIR_B200_ROTARY_HALF ? j * VEC : j * 2 * VEC;
    const int second = turns && p.layout == CACHEIR_B200_ROTARY_HALF ? at + half : at + VEC;
    const bool both = second < p.dim;                       // (an odd rest of single values)
    float a[VEC], b[VEC];
    VecIO<T, VEC>::ld(src + at, a);
    if (both) VecIO<T, VEC>::ld(src + second, b);
    if (turns && !is_v) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 t = s_turn[j * VEC + i];
        float x, y;
        if (VEC == 1 || p.layout == CACHEIR_B200_ROTARY_HALF) { x = a[i]; y = b[i]; }
        else { x = i < VEC / 2 ? a[2 * i % VEC] : b[2 * i % VEC]; y = i < VEC / 2 ? a[(2 * i + 1) % VEC] : b[(2 * i + 1) % VEC]; }
        const float rx = __fmaf_rn(x, t.x, -__fmul_rn(y, t.y)), ry = __fmaf_rn(x, t.y, __fmul_rn(y, t.x));
        if (VEC == 1 || p.layout == CACHEIR_B200_ROTARY_HALF) { a[i] = rx; b[i] = ry; }
        else if (i < VEC / 2) { a[2 * i % VEC] = rx; a[(2 * i + 1) % VEC] = ry; }
        else { b[2 * i % VEC] = rx; b[(2 * i + 1) % VEC] = ry; }
      }
    }
    auto put = [&](void* base, size_t from) {
      T* dst = static_cast<T*>(base) + from;
      VecIO<T, VEC>::st(dst + at, a);
      if (both) VecIO<T, VEC>::st(dst + second, b);
    };
    const size_t pooled = (static_cast<size_t>(line) + static_cast<size_t>(h) * p.page_size) * p.dim;
    if (is_q) {
      if (p.q_out) put(p.q_out, static_cast<size_t>(row) * p.q_out_stride + static_cast<size_t>(h) * p.dim);
    } else if (is_v) {
      put(p.v_cache, pooled);
    } else {
      if (p.k_out) put(p.k_out, static_cast<size_t>(row) * p.k_out_stride + static_cast<size_t>(h) * p.dim);
      if (p.slots) put(p.k_cache, pooled);
    }
  }
}

template <typename T>
int launch_rotary(const cacheir_b200_rotary_args& a, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  bool wide = a.dim % VEC == 0 && (a.dim - a.rot) % (2 * VEC) == 0 && a.rot % (2 * VEC) == 0;
  for (const void* ptr : {a.q, a.k, a.v, static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_out), static_cast<const void*>(a.k_cache),
                          static_cast<const void*>(a.v_cache)})
    wide = wide && aligned_to(ptr, 16);
  for (long long stride : {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride}) wide = wide && stride % VEC == 0;
  const int threads = a.rows > 4096 ? 64 : a.rows > 4 * kNumSMs ? 128 : kMaxThreads;
  const cudaError_t e = wide ? launch_chained(rotary_append_kernel<T, VEC>, dim3(a.rows), dim3(threads), 0, stream, a)
                             : launch_chained(rotary_append_kernel<T, 1>, dim3(a.rows), dim3(threads), 0, stream, a);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_rotary_append(const cacheir_b200_rotary_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  cacheir_b200_rotary_args a = *args;
  if (a.rows <= 0) return 0;
  if (!a.q || !a.k || !a.positions || !a.turns || a.heads <= 0 || a.kv_heads <= 0 || a.dim <= 0 || a.rot <= 0 || a.rot % 2 != 0 || a.rot > a.dim ||
      (a.layout != CACHEIR_B200_ROTARY_INTERLEAVED && a.layout != CACHEIR_B200_ROTARY_HALF) || dtype_size(a.dtype) == 0)
    return CACHEIR_B200_EINVAL;
  if (a.dim > kMaxDim) return CACHEIR_B200_ELIMIT;
  if (a.slots ? (!a.v || !a.k_cache || !a.v_cache || a.num_slots <= 0 || a.page_size <= 0) : (a.k_cache || a.v_cache || !a.k_out || !a.q_out))
    return CACHEIR_B200_EINVAL;
  if (static_cast<long long>(a.heads + 2 * a.kv_heads) * a.dim > 0x7fffffffLL) return CACHEIR_B200_ELIMIT;
  if (a.dtype == CACHEIR_B200_F32) return launch_rotary<float>(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16) return launch_rotary<__half>(a, as_stream(stream));
  return launch_rotary<__nv_bfloat16>(a, as_stream(stream));
}
