// Log probabilities of given tokens, entropies and the likeliest alternatives of rows of logits, in one pass over the row.
//
// With m the row's largest value and y = (x - m) log2(e) / T:  Z = sum 2^y,  S = sum 2^y y,
//   log p(t) = (x_t - m) / T - ln Z,   H = ln Z - ln 2 S / Z   (both terms are non-negative: nothing cancels).
// Every lane keeps 32-bit sums of its own relative to the largest value that it has met; they are joined by trees.
//
// The likeliest `top` come out of the same pass. A lane looks at 64 bytes at a time (a group: neighbouring values) and leaves the group's
// largest value in shared memory. Of the groups only the `top` first by (largest value, lower index) can hold one of the `top` first values
// by (value, lower index): each group before a given one has a value before all of that one's. So a few hundred values are read again, and
// that holds for any data, ties and masks included.
//
// Bound by memory for many rows (2048 x 128256 in bf16: 90 us, 5.8 TB/s), by latency for few (1 x 128256 in fp16 with 5 alternatives: 7.9 us,
// 64 x 50001 in fp32 with 20: 13.8 us; from a graph, in bursts: a second of the first on end runs into the power cap, 106 us). A row is read by one block, or by a thread-block cluster where
// there are few; every warp copies 4 KB pieces (bulk copies, a ring of its own: no barrier between warps) and has two of them on
// their way. Per value that is half an instruction for the maximum, one to widen it, one for the exponent's argument, one
// exponential (16 a cycle and SM: 73 % of the memory's rate), half each for the two sums.
#include "cacheir_b200_serving.h"
#include "hybrid_common.cuh"
#include "serving_status.h"
#include "tc_ptx.cuh"

namespace cb200 {
namespace {

using namespace ptx;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTileBytes = 4096;           // of a warp's copy: two groups a lane
constexpr int kStages = 2;
constexpr int kMaxTiles = 128;             // of a block, where its groups' largest values are kept
constexpr int kMaxCluster = 8;
constexpr int kList = 256;                 // candidates that are ranked against one another
constexpr float kMasked = -1e30f;          // what is at or below it weighs nothing beside anything above it
constexpr float kHuge = 1e30f;
constexpr float kFar = -1e6f;              // 2^kFar is 0, and kFar times a sum is a number

__device__ int g_logprobs_status = 0;

struct Args {
  const void* logits;
  long long stride;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  int vocab, top, cluster;
  double inv_t;
};

struct Sums {
  float m, z, s;                           // the largest x (-inf: nothing yet), Z, S
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The lanes' sums as one, in every lane.
__device__ __forceinline__ Sums joined(const Sums& a, float c) {
  Sums r;
  r.m = warp_max(a.m);
  const float d = a.m > -INFINITY ? fmaxf((a.m - r.m) * c, kFar) : kFar, w = ex2(d);
  r.z = warp_sum(a.z * w);
  r.s = warp_sum((a.s + d * a.z) * w);
  return r;
}

// Values as integers of the same order, NaN above all; -0 is 0. 0 is no value.
__device__ __forceinline__ uint32_t ordered_bits(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t b) {
  return b == 0xffffffffu ? NAN : __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ unsigned long long key_of(uint32_t value, uint32_t index) { return static_cast<unsigned long long>(value) << 32 | (~index & 0xffffffffu); }

// two floats of a register pair at a time
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 x, f32x2 y, f32x2 z) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 x, f32x2 y) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 x, f32x2 y) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  return d;
}

// 64 bytes of a row: largest value (NaN if there is one), and its values two by two
template <typename T>
struct Group;
template <>
struct Group<float> {
  static constexpr int kPairs = 8;
  static __device__ __forceinline__ float largest(const uint32_t (&w)[16]) {
    float mx = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 1; i < 15; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(mx) : "f"(__uint_as_float(w[i])), "f"(__uint_as_float(w[i + 1])));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx) : "f"(__uint_as_float(w[15])));
    return mx;
  }
  static __device__ __forceinline__ void two(const uint32_t (&w)[16], int i, float& lo, float& hi) { lo = __uint_as_float(w[2 * i]); hi = __uint_as_float(w[2 * i + 1]); }
  static constexpr uint32_t kNothing = 0xff800000u;       // -inf
};
template <>
struct Group<__half> {
  static constexpr int kPairs = 16;
  static __device__ __forceinline__ float largest(const uint32_t (&w)[16]) {
    __half2 mx = *reinterpret_cast<const __half2*>(&w[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = __hmax2_nan(mx, *reinterpret_cast<const __half2*>(&w[i]));
    return __half2float(__hmax_nan(__low2half(mx), __high2half(mx)));
  }
  static __device__ __forceinline__ void two(const uint32_t (&w)[16], int i, float& lo, float& hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    lo = f.x;
    hi = f.y;
  }
  static constexpr uint32_t kNothing = 0xfc00fc00u;
};
template <>
struct Group<__nv_bfloat16> {
  static constexpr int kPairs = 16;
  static __device__ __forceinline__ float largest(const uint32_t (&w)[16]) {
    __nv_bfloat162 mx = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = __hmax2_nan(mx, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    return __bfloat162float(__hmax_nan(__low2bfloat16(mx), __high2bfloat16(mx)));
  }
  static __device__ __forceinline__ void two(const uint32_t (&w)[16], int i, float& lo, float& hi) {
    lo = __uint_as_float(w[i] << 16);
    hi = __uint_as_float(w[i] & 0xffff0000u);
  }
  static constexpr uint32_t kNothing = 0xff80ff80u;
};

__device__ __forceinline__ uint32_t ld_rank_u32(const void* local, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_rank(smem_u32(local), rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long ld_rank_u64(const void* local, uint32_t rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_rank(smem_u32(local), rank)) : "memory");
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3)
token_logprobs_kernel(const __grid_constant__ Args p) {
  chain_enter();
  using G = Group<T>;
  constexpr int kGroup = 64 / sizeof(T), kTile = kTileBytes / sizeof(T), kVec = 16 / sizeof(T);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[kWarps * kStages];
  __shared__ Sums s_sums[kWarps];
  __shared__ int s_flags[kWarps];
  __shared__ Sums s_block;
  __shared__ int s_block_flags;
  __shared__ unsigned long long s_top[CACHEIR_B200_MAX_TOP];
  __shared__ uint32_t s_warp_bound[kWarps];
  __shared__ uint32_t s_bound;
  __shared__ int s_count;
  __shared__ int s_selected[CACHEIR_B200_MAX_TOP];
  __shared__ unsigned long long s_round[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = p.cluster > 1 ? blockIdx.x % p.cluster : 0, row = blockIdx.x / p.cluster;
  const T* x = static_cast<const T*>(p.logits) + static_cast<size_t>(row) * p.stride;
  // The row as single values up to the first 16-byte boundary, tiles, and single values behind the last whole 16 bytes.
  const int head = min(p.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int body = (p.vocab - head) / kVec * kVec, tail = p.vocab - head - body, all_tiles = (body + kTile - 1) / kTile;
  const int per_block = (all_tiles + p.cluster - 1) / p.cluster, tile0 = min(all_tiles, rank * per_block), tiles = min(all_tiles, tile0 + per_block) - tile0;
  uint8_t* ring = smem + warp * kStages * kTileBytes;
  uint32_t* s_max = reinterpret_cast<uint32_t*>(smem + kWarps * kStages * kTileBytes);      // [tiles * 64 groups] ordered, with `top` only
  const uint32_t bar = smem_u32(&s_bar[warp * kStages]);
  const float c = static_cast<float>(p.inv_t * 1.4426950408889634);

  const int mine = warp < tiles ? (tiles - warp + kWarps - 1) / kWarps : 0;            // this warp's tiles: warp + i * kWarps
  auto bytes_of = [&](int i) { return min(kTile, body - (tile0 + warp + i * kWarps) * kTile) * static_cast<int>(sizeof(T)); };
  auto copy = [&](int i, int s) {                          // (one lane)
    const uint32_t n = bytes_of(i);
    mbar_expect_tx(bar + s * 8, n);
    bulk_load(smem_u32(ring + s * kTileBytes), x + head + static_cast<size_t>(tile0 + warp + i * kWarps) * kTile, n, bar + s * 8);
  };
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bar + s * 8, 1);
    mbar_fence_init();
    for (int s = 0; s < kStages && s < mine; ++s) copy(s, s);
  }
  __syncwarp();

  const bool asks = warp == 0 && rank == 0 && p.logprobs;
  const int64_t token = asks ? p.tokens[row] : -1;         // (on its way beside the row's first pieces, its value beside the sums)
  float m = -INFINITY;
  f32x2 z2 = 0ull, s2 = 0ull;                              // (both halves)
  int flags = 0;                                           // 1: NaN or +inf, 2: values beyond kHuge, 4: some at or below kMasked that are not -inf
  auto rescale = [&](float mx) {                           // the lane's sums become relative to mx
    if (m > -INFINITY) {
      const float d = fmaxf((m - mx) * c, kFar), w = ex2(d);
      const f32x2 w2 = pair(w, w), d2 = pair(d, d);
      s2 = mul2(fma2(d2, z2, s2), w2);
      z2 = mul2(z2, w2);
    }
    m = mx;
  };
  // A few values at a time are added as they are; what is masked weighs nothing.
  auto add_one = [&](float v) {
    if (!(v < kHuge)) { flags |= v < INFINITY ? 2 : 1; return; }
    if (v <= kMasked) { if (v > -INFINITY) flags |= 4; return; }
    if (v > m) rescale(v);
    const float y = (v - m) * c, e = ex2(y);
    z2 = add2(z2, pair(e, 0.f));
    s2 = fma2(pair(e, 0.f), pair(y, 0.f), s2);
  };
  int stage = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    if (!__all_sync(0xffffffffu, mbar_wait(bar + stage * 8, phase, &g_logprobs_status, (16 << 8) | 1))) {
      for (int k = i; k < min(mine, i + kStages); ++k) {   // the copies that are still under way
        mbar_wait(bar + stage * 8, phase, &g_logprobs_status, (16 << 8) | 2);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      flags |= 1;                                          // (the row's results are no numbers)
      break;
    }
    const int n16 = bytes_of(i) / 16;
    const uint8_t* tile = ring + stage * kTileBytes;
#pragma unroll
    for (int half = 0; half < 2; ++half) {                 // a lane has 128 bytes: two groups
      const int which = half ^ (lane >> 2 & 1);
      uint32_t w[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = lane * 8 + which * 4 + ((j + lane) & 3);        // (in an order in which eight lanes reach all banks)
        const uint4 v = *reinterpret_cast<const uint4*>(tile + at * 16);
        w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
        if (at >= n16) w[4 * j] = w[4 * j + 1] = w[4 * j + 2] = w[4 * j + 3] = G::kNothing;
      }
      if (half == 1) {
        __syncwarp();
        if (lane == 0 && i + kStages < mine) copy(i + kStages, stage);
      }
      const float mx = G::largest(w);
      if (p.top > 0) s_max[((warp + i * kWarps) * 32 + lane) * 2 + which] = lane * 8 + which * 4 < n16 ? ordered_bits(mx) : 0u;
      if (!(mx < kHuge)) {
        flags |= mx < INFINITY ? 2 : 1;
      } else if (mx <= kMasked) {
        if (mx > -INFINITY) flags |= 4;
      } else {
        if (mx > m) rescale(mx);
        const f32x2 c2 = pair(c, c), less = pair(-m, -m);
        f32x2 gz[2] = {0ull, 0ull}, gs[2] = {0ull, 0ull};
#pragma unroll
        for (int k = 0; k < G::kPairs; ++k) {
          float lo, hi, y0, y1;
          G::two(w, k, lo, hi);
          const f32x2 y = mul2(add2(pair(lo, hi), less), c2);
          unpair(y, y0, y1);
          const f32x2 e = pair(ex2(y0), ex2(y1));
          gz[k & 1] = add2(gz[k & 1], e);
          gs[k & 1] = fma2(e, y, gs[k & 1]);
        }
        gs[0] = add2(gs[0], gs[1]);
        float s0, s1;
        unpair(gs[0], s0, s1);
        if (!(s0 + s1 == s0 + s1)) {                       // a masked value: its weight of 0 times -inf is no number
          gs[0] = 0ull;
#pragma unroll
          for (int k = 0; k < G::kPairs; ++k) {
            float lo, hi, y0, y1;
            G::two(w, k, lo, hi);
            const f32x2 y = mul2(add2(pair(fmaxf(lo, kMasked), fmaxf(hi, kMasked)), less), c2);
            unpair(y, y0, y1);
            gs[0] = fma2(pair(ex2(y0), ex2(y1)), y, gs[0]);
          }
        }
        z2 = add2(z2, add2(gz[0], gz[1]));
        s2 = add2(s2, gs[0]);
      }
    }
    if (++stage == kStages) { stage = 0; phase ^= 1; }
  }
  const float asked = token >= 0 && token < p.vocab ? Elem<T>::ld(x + token) : 0.f;
  // the single values of both ends: lanes of the first block's first warp, of the last block's
  if (warp == 0 && rank == 0 && lane < head) add_one(Elem<T>::ld(x + lane));
  if (warp == 0 && rank == p.cluster - 1 && lane < tail) add_one(Elem<T>::ld(x + head + body + lane));

  // ---- sums ----
  Sums a;
  {
    float z0, z1, s0, s1;
    unpair(z2, z0, z1);
    unpair(s2, s0, s1);
    a = Sums{m, z0 + z1, s0 + s1};
  }
  a = joined(a, c);
  flags = __reduce_or_sync(0xffffffffu, flags);
  if (lane == 0) { s_sums[warp] = a; s_flags[warp] = flags; }
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();                                         // (the rings are drained)
  if (warp == 0) {
    a = joined(lane < kWarps ? s_sums[lane] : Sums{-INFINITY, 0.f, 0.f}, c);
    flags = __reduce_or_sync(0xffffffffu, lane < kWarps ? s_flags[lane] : 0);
    if (lane == 0) { s_block = a; s_block_flags = flags; }
  }

  // ---- the block's likeliest `top` ----
  if (p.top > 0) {
    const int top = p.top, ends = (rank == 0 && head > 0 ? 1 : 0) + (rank == p.cluster - 1 && tail > 0 ? 1 : 0);
    const int first = rank == 0 && head > 0 ? 1 : 0, groups = tiles * 64 + ends;       // in order: the head, those of the tiles, the tail
    unsigned long long* s_list = reinterpret_cast<unsigned long long*>(smem);          // [kList], over the rings
    auto value_of = [&](int g) -> uint32_t {
      if (g >= first && g - first < tiles * 64) return s_max[g - first];
      const bool front = g < first;
      uint32_t best = 0;
      for (int i = 0; i < (front ? head : tail); ++i) best = max(best, ordered_bits(Elem<T>::ld(x + (front ? 0 : head + body) + i)));
      return best;
    };
    auto range_of = [&](int g, int* from) {                // its values
      if (g >= first && g - first < tiles * 64) {
        const int at = tile0 * kTile + (g - first) * kGroup;
        *from = head + at;
        return min(kGroup, body - at);
      }
      *from = g < first ? 0 : head + body;
      return g < first ? head : tail;
    };
    auto list = [&](bool wanted, unsigned long long key) { // (a whole warp; any order: they are ranked)
      const uint32_t who = __ballot_sync(0xffffffffu, wanted);
      if (who == 0) return;
      int at = 0;
      if (lane == __ffs(who) - 1) at = atomicAdd(&s_count, __popc(who));
      at = __shfl_sync(0xffffffffu, at, __ffs(who) - 1) + __popc(who & ((1u << lane) - 1));
      if (wanted && at < kList) s_list[at] = key;
    };
    // the largest key below `last` that anybody offers (the slow way, for lists that do not fit)
    auto next_best = [&](unsigned long long best) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, off);
        if (o > best) best = o;
      }
      __syncthreads();
      if (lane == 0) s_round[warp] = best;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w)
        if (s_round[w] > best) best = s_round[w];
      return best;
    };
    // A bound from below that `top` groups reach: every warp's share of them among its lanes' best ones, and the least of that.
    uint32_t best = 0;
    for (int g = threadIdx.x; g < groups; g += kThreads) best = max(best, value_of(g));
    uint32_t nth = 0;
    for (int k = 0; k < (top + kWarps - 1) / kWarps; ++k) {
      nth = __reduce_max_sync(0xffffffffu, best);
      if (lane == __ffs(__ballot_sync(0xffffffffu, best == nth)) - 1) best = 0;
    }
    if (lane == 0) s_warp_bound[warp] = nth;
    if (threadIdx.x < CACHEIR_B200_MAX_TOP) { s_selected[threadIdx.x] = -1; s_top[threadIdx.x] = 0; }
    __syncthreads();
    uint32_t bound = s_warp_bound[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bound = min(bound, s_warp_bound[w]);
    for (int g = threadIdx.x; g - lane < groups; g += kThreads) {
      const uint32_t v = g < groups ? value_of(g) : 0u;
      list(v >= bound && v > 0, key_of(v, g));
    }
    __syncthreads();
    const int found = s_count;
    if (found <= kList) {
      if (static_cast<int>(threadIdx.x) < found) {
        const unsigned long long key = s_list[threadIdx.x];
        int before = 0;
        for (int i = 0; i < found; ++i) before += s_list[i] > key ? 1 : 0;
        if (before < top) {
          s_selected[before] = static_cast<int>(~static_cast<uint32_t>(key));
          if (before == top - 1) s_bound = static_cast<uint32_t>(key >> 32);
        }
      }
      if (found < top && threadIdx.x == 0) s_bound = 0;
    } else {
      unsigned long long last = ~0ull;
      for (int k = 0; k < top; ++k) {
        unsigned long long mine_best = 0;
        for (int g = threadIdx.x; g < groups; g += kThreads) {
          const unsigned long long key = key_of(value_of(g), g);
          if (key < last && key > mine_best && (key >> 32) > 0) mine_best = key;
        }
        last = next_best(mine_best);
        if (threadIdx.x == 0) {
          s_selected[k] = static_cast<int>(~static_cast<uint32_t>(last));
          s_bound = static_cast<uint32_t>(last >> 32);
        }
      }
    }
    __syncthreads();
    // Their values: every one that can be among the first has at least the last selected group's largest value.
    constexpr int kPer = CACHEIR_B200_MAX_TOP * kGroup / kThreads;
    unsigned long long keys[kPer];
    const uint32_t least = s_bound;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int at = threadIdx.x + j * kThreads, k = at / kGroup, e = at % kGroup;
      int from;
      keys[j] = 0;
      if (k < top && s_selected[k] >= 0 && e < range_of(s_selected[k], &from)) {
        const uint32_t v = ordered_bits(Elem<T>::ld(x + from + e));
        if (v >= least) keys[j] = key_of(v, from + e);
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) list(keys[j] > 0, keys[j]);
    __syncthreads();
    const int values = s_count;
    if (values <= kList) {
      if (static_cast<int>(threadIdx.x) < values) {
        const unsigned long long key = s_list[threadIdx.x];
        int before = 0;
        for (int i = 0; i < values; ++i) before += s_list[i] > key ? 1 : 0;
        if (before < top) s_top[before] = key;
      }
    } else {
      unsigned long long last = ~0ull;
      for (int k = 0; k < top; ++k) {
        unsigned long long mine_best = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (keys[j] < last && keys[j] > mine_best) mine_best = keys[j];
        last = next_best(mine_best);
        if (threadIdx.x == 0) s_top[k] = last;
      }
    }
  }

  // ---- the row ----
  __syncthreads();
  if (p.cluster > 1) cluster_sync_release();
  if (rank == 0) {
    if (p.cluster > 1) {
      const Sums o{__uint_as_float(ld_rank_u32(&s_block.m, lane % p.cluster)), __uint_as_float(ld_rank_u32(&s_block.z, lane % p.cluster)),
                   __uint_as_float(ld_rank_u32(&s_block.s, lane % p.cluster))};
      a = joined(lane < p.cluster ? o : Sums{-INFINITY, 0.f, 0.f}, c);
      flags = __reduce_or_sync(0xffffffffu, static_cast<int>(ld_rank_u32(&s_block_flags, lane % p.cluster)));
    } else {
      a = s_block;
      flags = s_block_flags;
    }
    double log_z = 0.0, entropy = 0.0;
    const bool nan = (flags & 1) != 0;
    bool empty = false;
    if (!nan && ((flags & 2) || (a.m == -INFINITY && (flags & 4)))) {
      // Values of 1e30 and more, or none above -1e30: the same in 64 bits, relative to the largest one.
      double mx = -INFINITY, z = 0.0, s = 0.0;
      for (int i = threadIdx.x; i < p.vocab; i += kThreads) mx = fmax(mx, static_cast<double>(Elem<T>::ld(x + i)));
      __shared__ double s_wide[3][kThreads];
      s_wide[0][threadIdx.x] = mx;
      __syncthreads();
      for (int i = 0; i < kThreads; ++i) mx = fmax(mx, s_wide[0][i]);
      for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
        const double y = (static_cast<double>(Elem<T>::ld(x + i)) - mx) * p.inv_t;
        if (y > -1e4) {
          const double e = exp(y);
          z += e;
          s += e * y;
        }
      }
      s_wide[1][threadIdx.x] = z;
      s_wide[2][threadIdx.x] = s;
      __syncthreads();
      z = s = 0.0;
      for (int i = 0; i < kThreads; ++i) { z += s_wide[1][i]; s += s_wide[2][i]; }
      a.m = static_cast<float>(mx);
      log_z = log(z);
      entropy = log_z - s / z;
    } else if (!nan && a.m == -INFINITY) {
      empty = true;
    } else if (!nan) {
      const float lz = logf(a.z);
      log_z = lz;
      entropy = lz - 0.6931471805599453f * (a.s / a.z);
    }
    auto log_p = [&](float v) {
      if (nan) return static_cast<float>(NAN);
      if (empty || v == -INFINITY) return -INFINITY;
      return static_cast<float>((static_cast<double>(v) - static_cast<double>(a.m)) * p.inv_t - log_z);
    };
    if (threadIdx.x == 0) {
      if (p.logprobs) {
        p.logprobs[row] = token < 0 ? 0.f : token >= p.vocab ? static_cast<float>(NAN) : log_p(asked);
      }
      if (p.entropy) p.entropy[row] = nan ? static_cast<float>(NAN) : empty ? 0.f : static_cast<float>(entropy);
    }
    if (p.top > 0) {
      unsigned long long key = 0;
      int before = -1;
      if (p.cluster == 1) {
        if (static_cast<int>(threadIdx.x) < p.top) { key = s_top[threadIdx.x]; before = threadIdx.x; }
      } else {                                             // the blocks' lists ranked against one another
        unsigned long long* s_list = reinterpret_cast<unsigned long long*>(smem);
        const int n = p.cluster * p.top;
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const int r = i / p.top, k = i % p.top;
          s_list[i] = ld_rank_u64(&s_top[k], r);
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < n) {
          key = s_list[threadIdx.x];
          before = 0;
          for (int i = 0; i < n; ++i) before += s_list[i] > key ? 1 : 0;
        }
      }
      if (before >= 0 && before < p.top && key > 0) {
        const size_t at = static_cast<size_t>(row) * p.top + before;
        p.top_ids[at] = static_cast<int64_t>(~static_cast<uint32_t>(key));
        p.top_logprobs[at] = log_p(from_ordered(static_cast<uint32_t>(key >> 32)));
      }
    }
  }
  if (p.cluster > 1) {
    __syncwarp();
    cluster_sync_release();                                // nobody leaves while its results are being read
  }
}

// Blocks for a row: as many waves of them as there are places (three on an SM), each as long as its tiles and what begins and ends it, about
// 12 tiles' time.
int cluster_of(int rows, int tiles, int least) {
  int best = least;
  long long shortest = -1;
  for (int n = least; n <= kMaxCluster; n *= 2) {
    const long long waves = (static_cast<long long>(rows) * n + 3 * kNumSMs - 1) / (3 * kNumSMs);
    const long long time = waves * ((tiles + n - 1) / n + 12);
    if (shortest < 0 || time < shortest) { shortest = time; best = n; }
  }
  return best;
}

template <typename T>
int launch_logprobs(Args a, int rows, cudaStream_t stream) {
  const long long tiles = (static_cast<long long>(a.vocab) * sizeof(T) + kTileBytes - 1) / kTileBytes;
  int least = 1;
  if (a.top > 0)
    while (least < kMaxCluster && tiles > static_cast<long long>(least) * kMaxTiles) least *= 2;
  if (a.top > 0 && tiles > static_cast<long long>(least) * kMaxTiles) return CACHEIR_B200_ELIMIT;
  a.cluster = cluster_of(rows, static_cast<int>(tiles), least);

  const int per_block = static_cast<int>((tiles + a.cluster - 1) / a.cluster);
  const size_t smem = static_cast<size_t>(kWarps) * kStages * kTileBytes + (a.top > 0 ? static_cast<size_t>(per_block) * 64 * 4 : 0);
  auto kern = token_logprobs_kernel<T>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_shared_memory(done, reinterpret_cast<const void*>(kern), kWarps * kStages * kTileBytes + kMaxTiles * 64 * 4);
  if (e == cudaSuccess) e = launch_clusters(kern, dim3(static_cast<unsigned>(rows) * a.cluster), dim3(kThreads), smem, stream, dim3(a.cluster), a);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace

int logprobs_device_status(bool reset) { return device_status_word(g_logprobs_status, reset); }

}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_token_logprobs(const cacheir_b200_logprobs_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  const cacheir_b200_logprobs_args& g = *args;
  if (g.rows <= 0 || g.vocab <= 0) return 0;
  if (!g.logits || (g.logprobs && !g.tokens) || g.top < 0 || (g.top > 0 && (!g.top_ids || !g.top_logprobs)) || !(g.temperature >= 1e-6) ||
      g.temperature > 1e6 || dtype_size(g.dtype) == 0 || (g.row_stride != 0 && g.row_stride < g.vocab && g.rows > 1))
    return CACHEIR_B200_EINVAL;
  if (g.top > CACHEIR_B200_MAX_TOP || g.top > g.vocab || g.rows > 0x7fffffff / kMaxCluster) return CACHEIR_B200_ELIMIT;
  if (!aligned_to(g.logits, dtype_size(g.dtype))) return CACHEIR_B200_EALIGN;
  const Args a{g.logits, g.row_stride == 0 ? g.vocab : g.row_stride, g.tokens, g.logprobs, g.entropy, g.top_ids, g.top_logprobs, g.vocab, g.top, 1,
               1.0 / g.temperature};
  if (g.dtype == CACHEIR_B200_F32) return launch_logprobs<float>(a, g.rows, as_stream(stream));
  if (g.dtype == CACHEIR_B200_F16) return launch_logprobs<__half>(a, g.rows, as_stream(stream));
  return launch_logprobs<__nv_bfloat16>(a, g.rows, as_stream(stream));
}
