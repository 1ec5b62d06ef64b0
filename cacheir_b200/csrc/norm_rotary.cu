// Norms of query and key heads, rotary positions and the append to the page pool, in one pass over q, k and v.
//
//   y = x / sqrt(mean x^2 + eps) * (weight + offset), (a, b) -> factor * (a cos - b sin, a sin + b cos)
//
// Bound by memory, and nearly as much by instructions: every value is read and written once, as without norms (16384 rows of 64 + 8 + 8 heads of 128 in fp16: 130 us, of
// which 103 us are the bytes, and 116 without norms; 2001 rows of 32 + 8 + 8 in bf16 15.8 us; 32 rows 3.5 us). A head lies in the registers of a few neighbouring lanes, each of
// which has both values of its pairs, so that the sum of squares is three exchanges of lanes (heads of 128 in 16 bits) and the turn none. Squares, sums, angles and
// products are in 32 bits; a value is rounded once, where it is stored. What moved it: two heads of a lane under way (155 us with one, 137 with three, 176 with four), pairs of
// floats in one instruction and lanes of a head known to the compiler (146 to 130).
#include "cacheir_b200_drafts.h"
#include "common.cuh"
#include "float_pairs.cuh"
#include "rotary_turn.cuh"

namespace cb200 {
namespace {

constexpr int kMaxThreads = 256;
constexpr int kMaxDim = 1024;
constexpr int kTogether = 2;                // heads that a lane has under way

using ptx::f32x2;

// Row `row`'s place in the pool, in rows of a key/value head; -1: outside it.
__device__ __forceinline__ long long pool_line(const cacheir_b200_rotary_args& p, int row) {
  if (!p.slots) return 0;
  const int slot = p.slots[row];
  if (slot < 0 || slot / p.page_size >= p.num_slots) return -1;
  return static_cast<long long>(slot / p.page_size) * p.kv_heads * p.page_size + slot % p.page_size;
}

// A lane has VEC pairs (or 2 VEC values that do not turn) of a head, as two vectors of VEC values; LANES lanes are a head. pair_x(i), pair_y(i): which of
// the 2 VEC values are the two of pair i.
template <int VEC, bool HALF>
__device__ __forceinline__ constexpr int pair_x(int i) { return HALF ? i : 2 * i; }
template <int VEC, bool HALF>
__device__ __forceinline__ constexpr int pair_y(int i) { return HALF ? VEC + i : 2 * i + 1; }

template <typename T, int VEC, int LANES, bool HALF>
__global__ void __launch_bounds__(kMaxThreads)
norm_rotary_kernel(const cacheir_b200_norm_rotary_args args) {
  chain_enter();
  __shared__ __align__(16) float2 s_turn[LANES * VEC];
  const cacheir_b200_rotary_args& p = args.rotary;
  const int row = blockIdx.x, threads = blockDim.x, groups = threads / LANES;
  const long long line = pool_line(p, row);
  if (line < 0) return;
  const int half = p.rot / 2, position = p.positions[row];
  for (int i = threadIdx.x; i < half; i += threads) s_turn[i] = turn_cos_sin(p.turns[i], position, p.factor);
  __syncthreads();
  const int turning = half / VEC, j = threadIdx.x & (LANES - 1);
  const bool turns = j < turning;
  const int at = !turns ? p.rot + (j - turning) * 2 * VEC : HALF ? j * VEC : j * 2 * VEC;
  const int second = turns && HALF ? at + half : at + VEC;
  const int behind_q = p.heads, behind_k = p.heads + p.kv_heads, heads = behind_k + (p.slots ? p.kv_heads : 0);
  // the weights of this lane's values, of queries or keys, as pairs of pairs
  f32x2 wx[VEC / 2], wy[VEC / 2];
  const void* loaded = nullptr;
  auto load_weights = [&](const void* weight) {
    float w[2 * VEC];
    if (!weight) {
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) w[i] = 1.f;
    } else if (sizeof(T) == 4 || args.weight_dtype != CACHEIR_B200_F32) {
      float a[VEC], b[VEC];
      VecIO<T, VEC>::ld(static_cast<const T*>(weight) + at, a);
      VecIO<T, VEC>::ld(static_cast<const T*>(weight) + second, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) { w[i] = a[i] + args.offset; w[VEC + i] = b[i] + args.offset; }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        w[i] = static_cast<const float*>(weight)[at + i] + args.offset;
        w[VEC + i] = static_cast<const float*>(weight)[second + i] + args.offset;
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      wx[i / 2] = ptx::pair(w[pair_x<VEC, HALF>(i)], w[pair_x<VEC, HALF>(i + 1)]);
      wy[i / 2] = ptx::pair(w[pair_y<VEC, HALF>(i)], w[pair_y<VEC, HALF>(i + 1)]);
    }
    loaded = weight;
  };
  load_weights(args.q_weight);
  const float inverse = 1.f / static_cast<float>(p.dim);
  // (values of several heads are asked for together: a store might be to what a later load reads, so that loads wait for the stores before them)
  for (int head0 = threadIdx.x / LANES; head0 - static_cast<int>(threadIdx.x & 31) / LANES < heads; head0 += kTogether * groups) {         // (whole warps)
    uint4 raw[kTogether][2];
#pragma unroll
    for (int e = 0; e < kTogether; ++e) {
      const int head = head0 + e * groups;
      if (head >= heads) continue;
      const T* src = head < behind_q ? static_cast<const T*>(p.q) + row * p.q_stride + head * p.dim
                                     : head < behind_k ? static_cast<const T*>(p.k) + row * p.k_stride + (head - behind_q) * p.dim
                                                       : static_cast<const T*>(p.v) + row * p.v_stride + (head - behind_k) * p.dim;
      raw[e][0] = *reinterpret_cast<const uint4*>(src + at);
      raw[e][1] = *reinterpret_cast<const uint4*>(src + second);
    }
#pragma unroll
    for (int e = 0; e < kTogether; ++e) {
      const int head = head0 + e * groups;
      float v[2 * VEC];
      f32x2 x[VEC / 2], y[VEC / 2], squares = 0ull;
      {
        float a[VEC], b[VEC];
        VecIO<T, VEC>::ld(reinterpret_cast<const T*>(&raw[e][0]), a);
        VecIO<T, VEC>::ld(reinterpret_cast<const T*>(&raw[e][1]), b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) { v[i] = a[i]; v[VEC + i] = b[i]; }
      }
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        x[i / 2] = ptx::pair(v[pair_x<VEC, HALF>(i)], v[pair_x<VEC, HALF>(i + 1)]);
        y[i / 2] = ptx::pair(v[pair_y<VEC, HALF>(i)], v[pair_y<VEC, HALF>(i + 1)]);
        squares = ptx::fma2(x[i / 2], x[i / 2], ptx::fma2(y[i / 2], y[i / 2], squares));
      }
      float sum, more;
      ptx::unpair(squares, sum, more);
      sum += more;
#pragma unroll
      for (int off = LANES / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (head >= heads) continue;
      if (head >= behind_k) {                              // values are copied
        T* dst = static_cast<T*>(p.v_cache) + (static_cast<size_t>(line) + static_cast<size_t>(head - behind_k) * p.page_size) * p.dim;
        *reinterpret_cast<uint4*>(dst + at) = raw[e][0];
        *reinterpret_cast<uint4*>(dst + second) = raw[e][1];
        continue;
      }
      const void* weight = head < behind_q ? args.q_weight : args.k_weight;
      if (weight != loaded) load_weights(weight);
      const float r = rsqrtf(fmaf(sum, inverse, args.eps));
      const f32x2 r2 = ptx::pair(r, r);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        x[i] = ptx::mul2(ptx::mul2(x[i], r2), wx[i]);
        y[i] = ptx::mul2(ptx::mul2(y[i], r2), wy[i]);
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float4 t = *reinterpret_cast<const float4*>(&s_turn[j * VEC + 2 * i]);       // two cosines and sines
          const f32x2 c = ptx::pair(t.x, t.z), s = ptx::pair(t.y, t.w), less = ptx::pair(-t.y, -t.w);
          const f32x2 turned = ptx::fma2(x[i], c, ptx::mul2(y[i], less));
          y[i] = ptx::fma2(x[i], s, ptx::mul2(y[i], c));
          x[i] = turned;
        }
      }
      float a[VEC], b[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        ptx::unpair(x[i / 2], v[pair_x<VEC, HALF>(i)], v[pair_x<VEC, HALF>(i + 1)]);
        ptx::unpair(y[i / 2], v[pair_y<VEC, HALF>(i)], v[pair_y<VEC, HALF>(i + 1)]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) { a[i] = v[i]; b[i] = v[VEC + i]; }
      auto put = [&](void* base, size_t from) {
        T* dst = static_cast<T*>(base) + from;
        VecIO<T, VEC>::st(dst + at, a);
        VecIO<T, VEC>::st(dst + second, b);
      };
      if (head < behind_q) {
        if (p.q_out) put(p.q_out, static_cast<size_t>(row) * p.q_out_stride + static_cast<size_t>(head) * p.dim);
      } else {
        const int h = head - behind_q;
        if (p.k_out) put(p.k_out, static_cast<size_t>(row) * p.k_out_stride + static_cast<size_t>(h) * p.dim);
        if (p.slots) put(p.k_cache, (static_cast<size_t>(line) + static_cast<size_t>(h) * p.page_size) * p.dim);
      }
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

template <typename T, int VEC, int LANES>
cudaError_t launch_lanes(const cacheir_b200_norm_rotary_args& args, int threads, cudaStream_t stream) {
  return args.rotary.layout == CACHEIR_B200_ROTARY_HALF ? launch_chained(norm_rotary_kernel<T, VEC, LANES, true>, dim3(args.rotary.rows), dim3(threads), 0, stream, args)
                                                        : launch_chained(norm_rotary_kernel<T, VEC, LANES, false>, dim3(args.rotary.rows), dim3(threads), 0, stream, args);
}

template <typename T>
int launch_norm_rotary(const cacheir_b200_norm_rotary_args& args, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const cacheir_b200_rotary_args& a = args.rotary;
  bool wide = a.dim % (2 * VEC) == 0 && a.rot % (2 * VEC) == 0;
  for (const void* ptr : {a.q, a.k, a.v, static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_out), static_cast<const void*>(a.k_cache),
                          static_cast<const void*>(a.v_cache), args.q_weight, args.k_weight})
    wide = wide && aligned_to(ptr, 16);
  for (long long stride : {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride}) wide = wide && stride % VEC == 0;
  // Few rows want as much of a row under way as there is; many want small blocks. Of 64 and 96 threads the larger where its blocks are through in as many rounds of the SMs as
  // the smaller's, 12 or 8 on an SM by their registers (fp32 16 or 10): 1000 rows of 32 + 8 + 8 heads of 128 in bf16 7.6 us with 96 threads, 9.5 with 64; 1500 rows 14.0 and
  // 11.7; 2001 16.0 and 17.2; 2600 20.4 and 19.5; 16384 94 and 87; in fp32 2001 rows 22.1 and 19.6, 2600 25.1 and 29.2. Heads that the general kernel serves are a warp's work each, with
  // more to wait for: 2001 rows of 32 + 8 + 8 of 96 in bf16 50.9 us with 256 threads, 60.5 with 128, 83 with 64; 5000 rows 110.5, 111 and 126; 16384 341, 329 and 337.
  const int lanes = wide ? a.dim / (2 * VEC) : 0;
  const bool general = lanes != 4 && lanes != 8 && lanes != 16 && lanes != 32;
  auto rounds = [&](int blocks) { return (a.rows + blocks * kNumSMs - 1) / (blocks * kNumSMs); };
  int threads = kMaxThreads;
  if (general) threads = a.rows > 4096 ? 128 : kMaxThreads;
  else if (a.rows > 4 * kNumSMs) threads = rounds(sizeof(T) == 4 ? 10 : 8) == rounds(sizeof(T) == 4 ? 16 : 12) ? 96 : 64;
  cudaError_t e;
  switch (lanes) {
    case 4: e = launch_lanes<T, VEC, 4>(args, threads, stream); break;
    case 8: e = launch_lanes<T, VEC, 8>(args, threads, stream); break;
    case 16: e = launch_lanes<T, VEC, 16>(args, threads, stream); break;
    case 32: e = launch_lanes<T, VEC, 32>(args, threads, stream); break;
    default: e = launch_chained(norm_rotary_any_kernel<T>, dim3(a.rows), dim3(threads), 0, stream, args);
  }
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
