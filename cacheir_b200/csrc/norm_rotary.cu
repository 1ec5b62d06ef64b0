// Norms of query and key heads, rotary positions and the append to the page pool, in one pass over q, k and v.
//
//   y = x / sqrt(mean x^2 + eps) * (weight + offset), (a, b) -> factor * (a cos - b sin, a sin + b cos)
//
// Bound by memory: every value is read and written once, as without norms. A head lies in the registers of a few neighbouring lanes, each of
// which has both values of its pairs, so that the sum of squares is three exchanges of lanes (heads of 128 in 16 bits) and the turn none. Squares, sums, angles and
// products are in 32 bits; a value is rounded once, where it is stored.
#include "cacheir_b200_drafts.h"
#include "common.cuh"
#include "rotary_turn.cuh"

namespace cb200 {
namespace {

constexpr int kMaxThreads = 256;
constexpr int kMaxDim = 1024;

// Row `row`'s place in the pool, in rows of a key/value head; -1: outside it.
__device__ __forceinline__ long long pool_line(const cacheir_b200_rotary_args& p, int row) {
  if (!p.slots) return 0;
  const int slot = p.slots[row];
  if (slot < 0 || slot / p.page_size >= p.num_slots) return -1;
  return static_cast<long long>(slot / p.page_size) * p.kv_heads * p.page_size + slot % p.page_size;
}

// A unit is VEC pairs (or 2 VEC values that do not turn): two vectors of VEC values. `lanes` units (a power of two, up to 32) are a head.
template <typename T, int VEC>
__global__ void __launch_bounds__(kMaxThreads)
norm_rotary_kernel(const cacheir_b200_norm_rotary_args args, const int lanes) {
  chain_enter();
  __shared__ float2 s_turn[kMaxDim / 2];
  const cacheir_b200_rotary_args& p = args.rotary;
  const int row = blockIdx.x, threads = blockDim.x;
  const long long line = pool_line(p, row);
  if (line < 0) return;
  const int half = p.rot / 2, position = p.positions[row];
  for (int i = threadIdx.x; i < half; i += threads) s_turn[i] = turn_cos_sin(p.turns[i], position, p.factor);
  __syncthreads();
  const int turning = half / VEC, j = threadIdx.x & (lanes - 1);
  const bool turns = j < turning, wide_turn = p.layout == CACHEIR_B200_ROTARY_HALF;
  const int at = !turns ? p.rot + (j - turning) * 2 * VEC : wide_turn ? j * VEC : j * 2 * VEC;
  const int second = turns && wide_turn ? at + half : at + VEC;
  const int heads = p.heads + (p.slots ? 2 : 1) * p.kv_heads;
  for (int u0 = 0; u0 < heads * lanes; u0 += threads) {
    const int head = (u0 + static_cast<int>(threadIdx.x)) / lanes;
    const bool active = head < heads, is_q = head < p.heads, is_v = head >= p.heads + p.kv_heads;
    const int h = is_q ? head : (head - p.heads) % p.kv_heads;
    float a[VEC] = {}, b[VEC] = {};
    if (active) {
      const T* src = is_q ? static_cast<const T*>(p.q) + row * p.q_stride
                          : is_v ? static_cast<const T*>(p.v) + row * p.v_stride : static_cast<const T*>(p.k) + row * p.k_stride;
      src += static_cast<size_t>(h) * p.dim;
      VecIO<T, VEC>::ld(src + at, a);
      VecIO<T, VEC>::ld(src + second, b);
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
    for (int off = lanes >> 1; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (!active) continue;
    if (!is_v) {
      const float r = rsqrtf(sum / static_cast<float>(p.dim) + args.eps);
      const void* weight = is_q ? args.q_weight : args.k_weight;
      if (weight) {
        float wa[VEC], wb[VEC];
        if (sizeof(T) == 4 || args.weight_dtype != CACHEIR_B200_F32) {
          VecIO<T, VEC>::ld(static_cast<const T*>(weight) + at, wa);
          VecIO<T, VEC>::ld(static_cast<const T*>(weight) + second, wb);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            wa[i] = static_cast<const float*>(weight)[at + i];
            wb[i] = static_cast<const float*>(weight)[second + i];
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          a[i] = a[i] * r * (wa[i] + args.offset);
          b[i] = b[i] * r * (wb[i] + args.offset);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) { a[i] *= r; b[i] *= r; }
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 t = s_turn[j * VEC + i];
          float x, y;
          if (wide_turn) { x = a[i]; y = b[i]; }
          else { x = i < VEC / 2 ? a[2 * i % VEC] : b[2 * i % VEC]; y = i < VEC / 2 ? a[(2 * i + 1) % VEC] : b[(2 * i + 1) % VEC]; }
          const float rx = __fmaf_rn(x, t.x, -__fmul_rn(y, t.y)), ry = __fmaf_rn(x, t.y, __fmul_rn(y, t.x));
          if (wide_turn) { a[i] = rx; b[i] = ry; }
          else if (i < VEC / 2) { a[2 * i % VEC] = rx; a[(2 * i + 1) % VEC] = ry; }
          else { b[2 * i % VEC] = rx; b[(2 * i + 1) % VEC] = ry; }
        }
      }
    }
    auto put = [&](void* base, size_t from) {
      T* dst = static_cast<T*>(base) + from;
      VecIO<T, VEC>::st(dst + at, a);
      VecIO<T, VEC>::st(dst + second, b);
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

// Any head size, stride and alignment: a warp a head, which it reads twice.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads)
norm_rotary_any_kernel(const cacheir_b200_norm_rotary_args args) {
  chain_enter();
  __shared__ float2 s_turn[kMaxDim / 2];
  const cacheir_b200_rotary_args& p = args.rotary;
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const long long line = pool_line(p, row);
  if (line < 0) return;
  const int half = p.rot / 2, position = p.positions[row];
  for (int i = threadIdx.x; i < half; i += blockDim.x) s_turn[i] = turn_cos_sin(p.turns[i], position, p.factor);
  __syncthreads();
  const int heads = p.heads + (p.slots ? 2 : 1) * p.kv_heads;
  for (int head = threadIdx.x >> 5; head < heads; head += blockDim.x >> 5) {
    const bool is_q = head < p.heads, is_v = head >= p.heads + p.kv_heads;
    const int h = is_q ? head : (head - p.heads) % p.kv_heads;
    const T* src = (is_q ? static_cast<const T*>(p.q) + row * p.q_stride
                         : is_v ? static_cast<const T*>(p.v) + row * p.v_stride : static_cast<const T*>(p.k) + row * p.k_stride) +
                   static_cast<size_t>(h) * p.dim;
    const size_t pooled = (static_cast<size_t>(line) + static_cast<size_t>(h) * p.page_size) * p.dim;
    T* out = nullptr;
    T* pool = nullptr;
    if (is_q) out = p.q_out ? static_cast<T*>(p.q_out) + static_cast<size_t>(row) * p.q_out_stride + static_cast<size_t>(h) * p.dim : nullptr;
    else if (is_v) pool = static_cast<T*>(p.v_cache) + pooled;
    else {
      out = p.k_out ? static_cast<T*>(p.k_out) + static_cast<size_t>(row) * p.k_out_stride + static_cast<size_t>(h) * p.dim : nullptr;
      pool = p.slots ? static_cast<T*>(p.k_cache) + pooled : nullptr;
    }
    auto put = [&](int d, float v) {
      if (out) Elem<T>::st(out + d, v);
      if (pool) Elem<T>::st(pool + d, v);
    };
    if (is_v) {
      for (int d = lane; d < p.dim; d += 32) put(d, Elem<T>::ld(src + d));
      continue;
    }
    float sum = 0.f;
    for (int d = lane; d < p.dim; d += 32) {
      const float x = Elem<T>::ld(src + d);
      sum = fmaf(x, x, sum);
    }
    const float r = rsqrtf(warp_sum(sum) / static_cast<float>(p.dim) + args.eps);
    const void* weight = is_q ? args.q_weight : args.k_weight;
    auto normed = [&](int d) {
      const float x = Elem<T>::ld(src + d) * r;
      if (!weight) return x;
      const float w = sizeof(T) == 4 || args.weight_dtype != CACHEIR_B200_F32 ? Elem<T>::ld(static_cast<const T*>(weight) + d) : static_cast<const float*>(weight)[d];
      return x * (w + args.offset);
    };
    // (a lane writes what it has read itself, so that outputs may be their inputs)
    for (int i = lane; i < half; i += 32) {
      const int d0 = p.layout == CACHEIR_B200_ROTARY_HALF ? i : 2 * i, d1 = p.layout == CACHEIR_B200_ROTARY_HALF ? i + half : 2 * i + 1;
      const float x = normed(d0), y = normed(d1);
      const float2 t = s_turn[i];
      put(d0, __fmaf_rn(x, t.x, -__fmul_rn(y, t.y)));
      put(d1, __fmaf_rn(x, t.y, __fmul_rn(y, t.x)));
    }
    for (int d = p.rot + lane; d < p.dim; d += 32) put(d, normed(d));
  }
}

template <typename T>
int launch_norm_rotary(const cacheir_b200_norm_rotary_args& args, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const cacheir_b200_rotary_args& a = args.rotary;
  const int lanes = a.dim / (2 * VEC);
  bool wide = a.dim % (2 * VEC) == 0 && a.rot % (2 * VEC) == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0;
  for (const void* ptr : {a.q, a.k, a.v, static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_out), static_cast<const void*>(a.k_cache),
                          static_cast<const void*>(a.v_cache), args.q_weight, args.k_weight})
    wide = wide && aligned_to(ptr, 16);
  for (long long stride : {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride}) wide = wide && stride % VEC == 0;
  const int threads = a.rows > 4096 ? 64 : a.rows > 4 * kNumSMs ? 128 : kMaxThreads;
  const cudaError_t e = wide ? launch_chained(norm_rotary_kernel<T, VEC>, dim3(a.rows), dim3(threads), 0, stream, args, lanes)
                             : launch_chained(norm_rotary_any_kernel<T>, dim3(a.rows), dim3(threads), 0, stream, args);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_norm_rotary_append(const cacheir_b200_norm_rotary_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_norm_rotary_args n = *args;
  const cacheir_b200_rotary_args& a = n.rotary;
  if (a.rows <= 0) return 0;
  if (!a.q || !a.k || !a.positions || !a.turns || a.heads <= 0 || a.kv_heads <= 0 || a.dim <= 0 || a.rot <= 0 || a.rot % 2 != 0 || a.rot > a.dim ||
      (a.layout != CACHEIR_B200_ROTARY_INTERLEAVED && a.layout != CACHEIR_B200_ROTARY_HALF) || dtype_size(a.dtype) == 0 || !(n.eps >= 0.f))
    return CACHEIR_B200_EINVAL;
  if ((n.q_weight || n.k_weight) && n.weight_dtype != a.dtype && n.weight_dtype != CACHEIR_B200_F32) return CACHEIR_B200_EINVAL;
  if (a.dim > kMaxDim) return CACHEIR_B200_ELIMIT;
  if (a.slots ? (!a.v || !a.k_cache || !a.v_cache || a.num_slots <= 0 || a.page_size <= 0) : (a.k_cache || a.v_cache || !a.k_out || !a.q_out))
    return CACHEIR_B200_EINVAL;
  if (static_cast<long long>(a.heads + 2 * a.kv_heads) * a.dim > 0x7fffffffLL) return CACHEIR_B200_ELIMIT;
  if (a.dtype == CACHEIR_B200_F32) return launch_norm_rotary<float>(n, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16) return launch_norm_rotary<__half>(n, as_stream(stream));
  return launch_norm_rotary<__nv_bfloat16>(n, as_stream(stream));
}
