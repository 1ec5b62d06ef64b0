// Log probabilities of given tokens, entropies and the likeliest alternatives of rows of logits.
//
// In units of log 2, y = x log2(e) / T:  Z = sum 2^(y - m),  log p(t) = ln 2 (y_t - m) - ln Z,  H = ln Z - ln 2 sum 2^(y - m) (y - m) / Z
// with m the row's largest y: both terms of H are non-negative, nothing cancels. Sums are 32-bit floats, one per thread with a running
// maximum, joined by a tree.
#include "cacheir_b200_serving.h"
#include "common.cuh"

namespace cb200 {
namespace {

constexpr int kThreads = 512;
constexpr float kLowest = -1e30f;          // stands for masked values: 2^(kLowest - m) is 0 and its product with (y - m) too

struct Sums { float m, z, s; };             // largest value (unscaled), sum of e = 2^(c (x - m)), sum of e c (x - m)

// log2-domain change of reference
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b, float c) {
  if (!(b.m > -INFINITY) && b.m == b.m) return a;           // nothing in b
  if (!(a.m > -INFINITY) && a.m == a.m) return b;
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = fmaxf((a.m - r.m) * c, kLowest), db = fmaxf((b.m - r.m) * c, kLowest);
  const float wa = exp2f(da), wb = exp2f(db);
  r.z = a.z * wa + b.z * wb;
  r.s = (a.s + da * a.z) * wa + (b.s + db * b.z) * wb;
  return r;
}

// Values as integers of the same order, NaN above all; -0 is 0.
__device__ __forceinline__ uint32_t ordered_bits(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t b) {
  return b == 0xffffffffu ? NAN : __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const T* __restrict__ logits, long long stride, const int64_t* __restrict__ tokens, float* __restrict__ logprobs,
                      float* __restrict__ entropy, int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs, int vocab, int top, double inv_t) {
  chain_enter();
  __shared__ Sums s_sums[kThreads / 32];
  __shared__ unsigned long long s_key[kThreads / 32];
  __shared__ int s_nan[1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* row = logits + static_cast<size_t>(blockIdx.x) * stride;
  const float c = static_cast<float>(inv_t * 1.4426950408889634);
  Sums a{-INFINITY, 0.f, 0.f};
  bool bad = false;
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const float x = Elem<T>::ld(row + i);
    if (!(x < INFINITY)) bad = true;
    else if (x > -INFINITY) a = joined(a, Sums{x, 1.f, 0.f}, c);
  }
  if (threadIdx.x == 0) s_nan[0] = 0;
  const bool nan = __syncthreads_or(bad ? 1 : 0) != 0;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    Sums o{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.z, off), __shfl_xor_sync(0xffffffffu, a.s, off)};
    a = lane & off ? joined(o, a, c) : joined(a, o, c);
  }
  if (lane == 0) s_sums[warp] = a;
  __syncthreads();
  a = s_sums[0];
  for (int w = 1; w < kThreads / 32; ++w) a = joined(a, s_sums[w], c);
  const bool empty = !(a.m > -INFINITY);
  const float log_z = logf(a.z);
  auto log_p = [&](float x) {
    if (nan) return static_cast<float>(NAN);
    if (empty) return -INFINITY;
    return static_cast<float>(static_cast<double>(x - a.m) * inv_t - static_cast<double>(log_z));
  };
  if (threadIdx.x == 0) {
    if (logprobs) {
      const int64_t t = tokens[blockIdx.x];
      logprobs[blockIdx.x] = t < 0 ? 0.f : t >= vocab ? static_cast<float>(NAN) : log_p(Elem<T>::ld(row + t));
    }
    if (entropy) entropy[blockIdx.x] = nan ? static_cast<float>(NAN) : empty ? 0.f : log_z - 0.6931471805599453f * a.s / a.z;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const unsigned long long key = (static_cast<unsigned long long>(ordered_bits(Elem<T>::ld(row + i))) << 32) | static_cast<uint32_t>(~i);
      if (key > best && key < last) best = key;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, off);
      if (o > best) best = o;
    }
    __syncthreads();
    if (lane == 0) s_key[warp] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) if (s_key[w] > best) best = s_key[w];
    last = best;
    if (threadIdx.x == 0) {
      const size_t at = static_cast<size_t>(blockIdx.x) * top + k;
      top_ids[at] = static_cast<int64_t>(~static_cast<uint32_t>(best));
      top_logprobs[at] = log_p(from_ordered(static_cast<uint32_t>(best >> 32)));
    }
  }
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_token_logprobs(const void* logits, long long row_stride, const int64_t* tokens, float* logprobs, float* entropy,
                                           int64_t* top_ids, float* top_logprobs, int rows, int vocab, int top, double temperature, int dtype,
                                           void* stream) {
  if (rows <= 0 || vocab <= 0) return 0;
  if (!logits || (logprobs && !tokens) || top < 0 || (top > 0 && (!top_ids || !top_logprobs)) || !(temperature > 0.0) || temperature > 1e30 ||
      temperature < 1e-30 || dtype_size(dtype) == 0 || (row_stride != 0 && row_stride < vocab && rows > 1))
    return CACHEIR_B200_EINVAL;
  if (top > CACHEIR_B200_MAX_TOP || top > vocab) return CACHEIR_B200_ELIMIT;
  if (row_stride == 0) row_stride = vocab;
#define CB200_LOGPROBS(T)                                                                                                                    \
  launch_chained(token_logprobs_kernel<T>, dim3(rows), dim3(kThreads), 0, as_stream(stream), static_cast<const T*>(logits), row_stride, tokens, \
                 logprobs, entropy, top_ids, top_logprobs, vocab, top, 1.0 / temperature)
  cudaError_t e;
  if (dtype == CACHEIR_B200_F32) e = CB200_LOGPROBS(float);
  else if (dtype == CACHEIR_B200_F16) e = CB200_LOGPROBS(__half);
  else e = CB200_LOGPROBS(__nv_bfloat16);
#undef CB200_LOGPROBS
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}
