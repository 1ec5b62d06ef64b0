// Penalties for repeated tokens, biases and grammar masks, in one pass over the logits.
//
//   c(t) = times that token t was said, known = c > 0 or t in the prompt
//   x = known ? (x > 0 ? x / repetition : x * repetition) : x;  x -= frequency c;  x -= presence [c > 0];  x += bias(t);  -inf where not allowed
//
// Bound by memory: logits are read and written once, in a pass that knows nothing but the grammar's bits. A block has a slice of the vocabulary and a run of rows.
// The tokens that fall into its slice are counted in shared memory, once for all neighbouring rows of one sequence, and listed; behind the pass the threads
// share out (row, listed token) pairs, whose logits are asked for once more, mostly from L2. Looking at counts while the vectors are in registers was slower by far: eight
// copies of the penalties' code a vector, of which instruction fetches alone took half the time (512 rows of 128256, 4096 tokens said: 325 us).
// Drafted tokens are a short list beside the counts, of which every row takes those that it sees. Counts are integers: the order of the
// additions does not matter.
//
// 512 rows of 128256 in bf16 (32 sequences of up to 4096 tokens, 16 drafted rows each, a grammar): 81 us, of which 41 us are the bytes at the copy's rate; with the grammar
// alone 50 us. The rest is latency: a block counts before its pass (5 us, 3000 tokens in four rounds of loads and three barriers) and changes listed
// tokens behind it (3 us, 13 where the frequent tokens are), and only the other blocks of its SM are at work meanwhile. 64 rows of 50001 in fp32 9.1 us, one row 3.8 us.
#include "cacheir_b200_drafts.h"
#include "common.cuh"
#include "serving_status.h"

namespace cb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;                           // tokens of a block, at most
constexpr int kPairs = 2;                             // logits of listed tokens that a thread has under way
constexpr int kRun = 8;                                // rows of a block, at most (16 took 111 us where 8 took 95, as there are fewer blocks to even the work out)
constexpr int kSaid = 4;                               // tokens of the history that a thread has under way
constexpr uint32_t kInPrompt = 0x80000000u;
constexpr uint32_t kDrafted = 0x40000000u;             // the list of drafted tokens has the token
constexpr uint32_t kBiased = 0x20000000u;
constexpr uint32_t kTimes = 0x1fffffffu;

struct LogitsParams {
  cacheir_b200_logits_args a;
  int slice;                  // tokens of a block, a multiple of 32
  int run;                    // rows of a block
};

__device__ __forceinline__ bool aligned_to_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Shared memory: marks [slice / 32], then, where tokens can be marked, counts [slice], (with a bias) entries of it [slice], (with drafts) the drafted
// tokens and what the rows see of them, and the list of marked tokens [slice].
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 3 : 4)
adjust_logits_kernel(const LogitsParams p) {
  constexpr int NV = kSlice / VEC / kThreads;          // vectors of a thread in a row
  constexpr bool kWide = VEC > 1;
  chain_enter();
  extern __shared__ uint32_t smem[];
  __shared__ int s_marked, s_drafted, s_seq[kRun];
  const cacheir_b200_logits_args& a = p.a;
  const int lo = blockIdx.x * p.slice, size = min(p.slice, a.vocab - lo), words = p.slice / 32;
  const bool biased = a.biases > 0, counting = a.history || a.draft_ids || biased;
  uint32_t* marks = smem;
  uint32_t* counts = marks + words;
  int* entry = reinterpret_cast<int*>(counts + (counting ? p.slice : 0));
  uint32_t* drafted = reinterpret_cast<uint32_t*>(entry + (biased ? p.slice : 0));   // token of the slice << 16 | row of the sequence
  uint32_t* sees = drafted + (a.draft_ids ? 32 * a.words : 0);                       // [rows of the block][words]
  uint16_t* marked = reinterpret_cast<uint16_t*>(sees + (a.draft_ids ? p.run * a.words : 0));
  const int begin = blockIdx.y * p.run, last = min(a.rows, begin + p.run), allowed_words = (a.vocab + 31) / 32;
  if (static_cast<int>(threadIdx.x) < last - begin) {
    const int seq = a.row_seq ? a.row_seq[begin + threadIdx.x] : begin + threadIdx.x;
    s_seq[threadIdx.x] = seq < a.sequences ? seq : -1;
  }
  if (a.draft_ids)
    for (int i = threadIdx.x; i < (last - begin) * a.words; i += kThreads) sees[i] = static_cast<uint32_t>(a.visible[static_cast<size_t>(begin) * a.words + i]);
  __syncthreads();
  auto input = [&](int row) { return static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.row_stride + lo; };
  auto output = [&](int row) { return static_cast<O*>(a.out) + static_cast<size_t>(row) * a.out_stride + lo; };
  auto grammar = [&](int row) { return reinterpret_cast<const uint32_t*>(a.allowed) + static_cast<size_t>(row) * allowed_words + lo / 32; };
  // vectors begin where addresses allow it: `skew` tokens before the slice
  auto skew_of = [&](const T* in) { return kWide ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % VEC) : 0; };
  const bool same = a.logits == a.out;

  for (int row0 = begin; row0 < last;) {
    const int seq = s_seq[row0 - begin];
    int end = row0 + 1;
    if (seq < 0) { row0 = end; continue; }
    while (end < last && s_seq[end - begin] == seq) ++end;
    // ---- the pass over the rows: values and bits of one are asked for while the one before is worked on (or tokens are counted) ----
    const bool pass = !same || a.allowed;
    uint4 ahead[kWide ? NV : 1];
    uint2 bits[kWide ? NV : 1];
    auto ask = [&](int row) {
      const T* in = input(row);
      const int skew = skew_of(in);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int t0 = (k * kThreads + static_cast<int>(threadIdx.x)) * VEC - skew;
        if (t0 < 0 || t0 + VEC > size) continue;
        ahead[k] = *reinterpret_cast<const uint4*>(in + t0);
        if (a.allowed) {
          const uint32_t* may = grammar(row) + (t0 >> 5);
          bits[k].x = may[0];
          if ((t0 & 31) + VEC > 32) bits[k].y = may[1];        // (the vector ends in the next word, which so there is)
        }
      }
    };
    if (kWide && pass) ask(row0);
    // ---- what the sequence has said (loads that do not depend on one another go out together) ----
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (counting) {
      const int n = a.history ? min(a.history_lens[seq], a.history_width) : 0, prompt = a.history && a.prompt_lens ? a.prompt_lens[seq] : 0;
      const int first = a.draft_ids ? min(max(a.cu_rows[seq], 0), a.rows) : 0;
      const int drafts = a.draft_ids ? min(min(max(a.cu_rows[seq + 1], 0), a.rows) - first, 32 * a.words) : 0;
      if (a.repetition) rep = a.repetition[seq];
      if (a.frequency) freq = a.frequency[seq];
      if (a.presence) pres = a.presence[seq];
      const int32_t* said = a.history + static_cast<size_t>(seq) * a.history_width;
      const size_t of_bias = static_cast<size_t>(seq) * a.biases;
      int id[kSaid];
#pragma unroll
      for (int e = 0; e < kSaid; ++e) {
        const int i = threadIdx.x + e * kThreads;
        id[e] = a.history && i < a.history_width ? said[i] : -1;
      }
      const int bias_id = static_cast<int>(threadIdx.x) < a.biases ? a.bias_ids[of_bias + threadIdx.x] : -1;
      __syncthreads();
      for (int i = threadIdx.x; i < words; i += kThreads) marks[i] = 0;
      for (int i = threadIdx.x; i < p.slice; i += kThreads) counts[i] = 0;
      if (biased) for (int i = threadIdx.x; i < p.slice; i += kThreads) entry[i] = 0;
      if (threadIdx.x == 0) s_marked = s_drafted = 0;
      __syncthreads();
      auto mark = [&](uint32_t t) {
        const uint32_t bit = 1u << (t & 31);
        if (!(atomicOr(&marks[t >> 5], bit) & bit)) marked[atomicAdd(&s_marked, 1)] = static_cast<uint16_t>(t);
      };
      for (int i0 = threadIdx.x; i0 < n; i0 += kSaid * kThreads) {
        int next[kSaid];
#pragma unroll
        for (int e = 0; e < kSaid; ++e) {
          const int i = i0 + (kSaid + e) * kThreads;
          next[e] = i < n ? said[i] : -1;
        }
#pragma unroll
        for (int e = 0; e < kSaid; ++e) {
          const int i = i0 + e * kThreads;
          if (i < n && id[e] >= lo && id[e] - lo < size) {
            const uint32_t t = static_cast<uint32_t>(id[e] - lo);
            if (i < prompt) atomicOr(&counts[t], kInPrompt);
            else atomicAdd(&counts[t], 1u);
            mark(t);
          }
        }
#pragma unroll
        for (int e = 0; e < kSaid; ++e) id[e] = next[e];
      }
      for (int j = threadIdx.x; j < drafts; j += kThreads) {
        const int64_t token = a.draft_ids[first + j];
        if (token >= lo && token - lo < size) {
          const uint32_t t = static_cast<uint32_t>(token - lo);
          drafted[atomicAdd(&s_drafted, 1)] = t << 16 | static_cast<uint32_t>(j);
          atomicOr(&counts[t], kDrafted);
          mark(t);
        }
      }
      for (int i = threadIdx.x; i < a.biases; i += kThreads) {
        const int token = i < kThreads ? bias_id : a.bias_ids[of_bias + i];
        if (token >= lo && token - lo < size) {
          atomicMax(&entry[token - lo], i + 1);
          atomicOr(&counts[token - lo], kBiased);
          mark(token - lo);
        }
      }
    }
    if (pass) {
      for (int row = row0; row < end; ++row) {
        const T* in = input(row);
        O* out = output(row);
        auto one = [&](int t) {
          if (a.allowed && !(grammar(row)[t >> 5] >> (t & 31) & 1)) Elem<O>::st(out + t, -INFINITY);
          else if (!same) Elem<O>::st(out + t, Elem<T>::ld(in + t));
        };
        if constexpr (kWide) {
          uint4 raw[NV];
          uint2 may[NV];
#pragma unroll
          for (int k = 0; k < NV; ++k) { raw[k] = ahead[k]; may[k] = bits[k]; }
          if (row + 1 < end) ask(row + 1);
          const int skew = skew_of(in);
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            const int t0 = (k * kThreads + static_cast<int>(threadIdx.x)) * VEC - skew;
            if (t0 < 0 || t0 + VEC > size) continue;
            const uint32_t yes = a.allowed ? __funnelshift_r(may[k].x, may[k].y, t0 & 31) | ~((1u << VEC) - 1) : 0xffffffffu;
            if (same && yes == 0xffffffffu) continue;
            float x[VEC];
            VecIO<T, VEC>::ld(reinterpret_cast<const T*>(&raw[k]), x);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              if (!(yes >> i & 1)) x[i] = -INFINITY;
            if constexpr (sizeof(O) == sizeof(T)) {
              VecIO<O, VEC>::st(out + t0, x);
            } else if (aligned_to_16(out + t0)) {
#pragma unroll
              for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(out + t0 + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
            } else {
#pragma unroll
              for (int i = 0; i < VEC; ++i) Elem<O>::st(out + t0 + i, x[i]);
            }
          }
          // tokens of vectors that the slice has only a part of: fewer than VEC at either end
          const int head = min((VEC - skew) % VEC, size), tail = head + (size - head) / VEC * VEC, i = threadIdx.x;
          if (i < head) one(i);
          else if (i >= 32 && tail + i - 32 < size) one(tail + i - 32);
        } else {
#pragma unroll 4
          for (int t = threadIdx.x; t < size; t += kThreads) one(t);
        }
      }
    }
    // ---- tokens that were said, are drafted or have a bias ----
    if (counting) {
      __syncthreads();
      const int many = s_drafted, rows = end - row0, pairs = s_marked * rows;
      for (int i0 = threadIdx.x; i0 < pairs; i0 += kPairs * kThreads) {
        T value[kPairs];
        uint32_t may[kPairs];
        float bias[kPairs];
        int token[kPairs], at[kPairs];
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {                     // (asked for together)
          const int i = min(i0 + e * kThreads, pairs - 1), k = i / rows;
          token[e] = marked[k];
          at[e] = row0 + i - k * rows;
          value[e] = input(at[e])[token[e]];
          may[e] = a.allowed ? grammar(at[e])[token[e] >> 5] : 0xffffffffu;
          bias[e] = counts[token[e]] & kBiased ? a.bias_values[static_cast<size_t>(seq) * a.biases + entry[token[e]] - 1] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          const int t = token[e], row = at[e];
          if (i0 + e * kThreads >= pairs || !(may[e] >> (t & 31) & 1)) continue;
          float x = Elem<T>::ld(&value[e]);
          const uint32_t c = counts[t];
          uint32_t times = c & kTimes;
          if (c & kDrafted)
            for (int d = 0; d < many; ++d) {
              const uint32_t v = drafted[d], j = v & 0xffffu;
              if (v >> 16 == static_cast<uint32_t>(t)) times += sees[(row - begin) * a.words + (j >> 5)] >> (j & 31) & 1;
            }
          if (times || (c & kInPrompt)) x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
          if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(times))), pres);
          if (c & kBiased) x = __fadd_rn(x, bias[e]);
          Elem<O>::st(output(row) + t, x);
        }
      }
    }
    row0 = end;
  }
}

template <typename T, typename O>
int launch_adjust(const cacheir_b200_logits_args& a, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  // Slices and runs: enough blocks for all SMs before rows share a count.
  LogitsParams p{a, kSlice, 1};
  while (p.slice > 1024 && static_cast<long long>(a.rows) * ((a.vocab + p.slice - 1) / p.slice) < 4 * kNumSMs) p.slice /= 2;
  const int slices = (a.vocab + p.slice - 1) / p.slice;
  while (p.run < kRun && static_cast<long long>(a.rows) * slices >= 6LL * p.run * kNumSMs) p.run *= 2;
  if (a.rows > kRun * 65535LL) return CACHEIR_B200_ELIMIT;
  if (a.rows > 65535) p.run = kRun;
  const bool counting = a.history || a.draft_ids || a.biases > 0;
  const size_t smem = (p.slice / 32 + (counting ? p.slice : 0) + (a.biases > 0 ? p.slice : 0) + (a.draft_ids ? (32 + p.run) * a.words : 0)) * sizeof(uint32_t) +
                      p.slice * sizeof(uint16_t);
  // vectors where a row's input and output begin at the same place of 16 bytes (with outputs of the same size)
  const bool wide = reinterpret_cast<uintptr_t>(a.logits) % sizeof(T) == 0 &&
                    (sizeof(T) != sizeof(O) || ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                                                (a.row_stride - a.out_stride) % VEC == 0));
  auto kern = wide ? adjust_logits_kernel<T, O, VEC> : adjust_logits_kernel<T, O, 1>;
  const dim3 grid(slices, (a.rows + p.run - 1) / p.run);
  static std::atomic<unsigned long long> done_wide{0}, done_any{0};
  constexpr int most = (kSlice / 32 + 2 * kSlice + (32 + kRun) * CACHEIR_B200_MAX_DRAFT_WORDS) * 4 + kSlice * 2;
  cudaError_t e = allow_shared_memory(wide ? done_wide : done_any, reinterpret_cast<const void*>(kern), most);
  if (e == cudaSuccess) e = launch_chained(kern, grid, dim3(kThreads), smem, stream, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

// Whether a row of out lies over a row of logits (rows may lie between one another).
bool rows_overlap(const cacheir_b200_logits_args& a) {
  const uintptr_t in = reinterpret_cast<uintptr_t>(a.logits), out = reinterpret_cast<uintptr_t>(a.out);
  const uint64_t in_row = static_cast<uint64_t>(a.vocab) * dtype_size(a.dtype), out_row = static_cast<uint64_t>(a.vocab) * dtype_size(a.out_dtype);
  auto in_at = [&](int r) { return in + static_cast<uint64_t>(r) * static_cast<uint64_t>(a.row_stride) * dtype_size(a.dtype); };
  auto out_at = [&](int r) { return out + static_cast<uint64_t>(r) * static_cast<uint64_t>(a.out_stride) * dtype_size(a.out_dtype); };
  if (in_at(a.rows - 1) + in_row <= out || out_at(a.rows - 1) + out_row <= in) return false;
  for (int i = 0, j = 0; i < a.rows && j < a.rows;) {          // in the order of their addresses
    const uint64_t x = in_at(i), y = out_at(j);
    if (x < y + out_row && y < x + in_row) return true;
    if (x < y) ++i; else ++j;
  }
  return false;
}

}  // namespace
}  // namespace cb200

using namespace cb200;

extern "C" int cacheir_b200_adjust_logits(const cacheir_b200_logits_args* args, void* stream) {
  if (!args) return CACHEIR_B200_EINVAL;
  cacheir_b200_logits_args a = *args;
  if (a.rows <= 0 || a.vocab <= 0) return 0;
  if (!a.logits || !a.out || a.sequences <= 0 || dtype_size(a.dtype) == 0 || (a.out_dtype != a.dtype && a.out_dtype != CACHEIR_B200_F32)) return CACHEIR_B200_EINVAL;
  if (a.row_stride == 0) a.row_stride = a.vocab;
  if (a.out_stride == 0) a.out_stride = a.vocab;
  if ((a.rows > 1 && (a.row_stride < a.vocab || a.out_stride < a.vocab)) || a.biases < 0 || (a.history && (!a.history_lens || a.history_width <= 0)) ||
      (a.draft_ids && (!a.cu_rows || !a.visible || a.words <= 0)) || (a.biases > 0 && (!a.bias_ids || !a.bias_values)))
    return CACHEIR_B200_EINVAL;
  const bool same = a.logits == a.out;
  if (same ? a.dtype != a.out_dtype || (a.rows > 1 && a.row_stride != a.out_stride) : rows_overlap(a)) return CACHEIR_B200_EINVAL;
  if (a.vocab > 1 << 28 || a.history_width >= 1 << 29 || (a.draft_ids && a.words > CACHEIR_B200_MAX_DRAFT_WORDS)) return CACHEIR_B200_ELIMIT;
  if (a.biases == 0) a.bias_ids = nullptr;
  if (a.dtype == CACHEIR_B200_F32) return launch_adjust<float, float>(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16)
    return a.out_dtype == CACHEIR_B200_F32 ? launch_adjust<__half, float>(a, as_stream(stream)) : launch_adjust<__half, __half>(a, as_stream(stream));
  return a.out_dtype == CACHEIR_B200_F32 ? launch_adjust<__nv_bfloat16, float>(a, as_stream(stream))
                                         : launch_adjust<__nv_bfloat16, __nv_bfloat16>(a, as_stream(stream));
}
