// Penalties for repeated tokens, biases and grammar masks, in one pass over the logits.
//
//   c(t) = times that token t was said, known = c > 0 or t in the prompt
//   x = known ? (x > 0 ? x / repetition : x * repetition) : x;  x -= frequency c;  x -= presence [c > 0];  x += bias(t);  -inf where not allowed
//
// Bound by memory: logits are read and written once. A block has a slice of the vocabulary and a run of rows. The tokens that fall into its slice
// are counted in shared memory, once for all neighbouring rows of one sequence, and marked as bits; while the slice streams through registers only marked
// tokens look at their counts. Counts are integers: the order of the additions does not matter.
#include "cacheir_b200_drafts.h"
#include "common.cuh"
#include "serving_status.h"

namespace cb200 {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;

struct LogitsParams {
  cacheir_b200_logits_args a;
  int slice;                  // tokens of a block, a multiple of 32
  int run;                    // rows of a block
};

// Shared memory: marks [slice / 32 + 1], then counts [slice] (with a history or drafts), then entries of the bias [slice] (with one).
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kThreads)
adjust_logits_kernel(const LogitsParams p) {
  chain_enter();
  extern __shared__ uint32_t smem[];
  const cacheir_b200_logits_args& a = p.a;
  const int lo = blockIdx.x * p.slice, size = min(p.slice, a.vocab - lo), words = p.slice / 32;
  const bool counting = a.history || a.draft_ids, biased = a.biases > 0;
  uint32_t* marks = smem;                              // (one word more, which stays 0)
  uint32_t* counts = smem + words + 1;
  int* entry = reinterpret_cast<int*>(counts + (counting ? p.slice : 0));
  const int last = min(a.rows, static_cast<int>(blockIdx.y + 1) * p.run);
  int current = -1;
  for (int row = blockIdx.y * p.run; row < last; ++row) {
    const int seq = a.row_seq ? a.row_seq[row] : row;
    if (seq < 0 || seq >= a.sequences) continue;
    if (seq != current) {                              // count what its history says
      __syncthreads();
      for (int i = threadIdx.x; i <= words; i += kThreads) marks[i] = 0;
      if (counting) for (int i = threadIdx.x; i < p.slice; i += kThreads) counts[i] = 0;
      if (biased) for (int i = threadIdx.x; i < p.slice; i += kThreads) entry[i] = 0;
      __syncthreads();
      if (a.history) {
        const int32_t* said = a.history + static_cast<size_t>(seq) * a.history_width;
        const int n = min(a.history_lens[seq], a.history_width), prompt = a.prompt_lens ? a.prompt_lens[seq] : 0;
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const uint32_t t = static_cast<uint32_t>(said[i] - lo);
          if (said[i] >= 0 && t < static_cast<uint32_t>(size)) {
            if (i < prompt) atomicOr(&counts[t], kInPrompt);
            else atomicAdd(&counts[t], 1u);
            atomicOr(&marks[t >> 5], 1u << (t & 31));
          }
        }
      }
      for (int i = threadIdx.x; i < a.biases; i += kThreads) {
        const int id = a.bias_ids[static_cast<size_t>(seq) * a.biases + i];
        const uint32_t t = static_cast<uint32_t>(id - lo);
        if (id >= 0 && t < static_cast<uint32_t>(size)) {
          atomicMax(&entry[t], i + 1);
          atomicOr(&marks[t >> 5], 1u << (t & 31));
        }
      }
      current = seq;
      __syncthreads();
    }
    // the drafted tokens that this row sees (taken off again behind it)
    auto drafted = [&](int sign) {
      const int first = min(max(a.cu_rows[seq], 0), a.rows), end = min(max(a.cu_rows[seq + 1], 0), a.rows);
      for (int j = threadIdx.x; j < min(end - first, 32 * a.words); j += kThreads)
        if (a.visible[static_cast<size_t>(row) * a.words + (j >> 5)] >> (j & 31) & 1) {
          const int64_t id = a.draft_ids[first + j];
          if (id >= lo && id < lo + size) {
            const uint32_t t = static_cast<uint32_t>(id - lo);
            atomicAdd(&counts[t], static_cast<uint32_t>(sign));
            atomicOr(&marks[t >> 5], 1u << (t & 31));
          }
        }
      __syncthreads();
    };
    if (a.draft_ids) drafted(1);
    const float rep = a.repetition ? a.repetition[seq] : 1.f, freq = a.frequency ? a.frequency[seq] : 0.f, pres = a.presence ? a.presence[seq] : 0.f;
    const float* values = a.bias_values + static_cast<size_t>(seq) * a.biases;
    auto marked = [&](float x, int t) {                // token t of the slice
      if (counting) {
        const uint32_t c = counts[t], times = c & ~kInPrompt;
        if (c) x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
        if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(times))), pres);
      }
      if (biased && entry[t]) x = __fadd_rn(x, values[entry[t] - 1]);
      return x;
    };
    const T* in = static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.row_stride + lo;
    O* out = static_cast<O*>(a.out) + static_cast<size_t>(row) * a.out_stride + lo;
    const uint32_t* allowed = a.allowed ? reinterpret_cast<const uint32_t*>(a.allowed) + static_cast<size_t>(row) * ((a.vocab + 31) / 32) + lo / 32 : nullptr;
    const int allowed_words = (a.vocab + 31) / 32 - lo / 32;
    // vectors begin where addresses allow it: `skew` tokens before the slice
    const int skew = VEC > 1 ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % VEC) : 0;
    const bool same = static_cast<const void*>(in) == static_cast<const void*>(out) && sizeof(T) == sizeof(O);
    for (int v = threadIdx.x; v * VEC < size + skew; v += kThreads) {
      const int t0 = v * VEC - skew, w = max(t0, 0) >> 5, sh = t0 & 31;
      uint32_t mark, may = 0xffffffffu;                // bits of the vector's tokens
      if (t0 < 0) {
        mark = marks[0] << -t0;
        if (allowed) may = allowed[0] << -t0;
      } else {
        mark = __funnelshift_r(marks[w], marks[w + 1], sh);
        if (allowed) may = __funnelshift_r(allowed[w], w + 1 < allowed_words && sh + VEC > 32 ? allowed[w + 1] : 0u, sh);
      }
      if (VEC < 32) { mark &= (1u << VEC) - 1; may &= (1u << VEC) - 1; }
      const bool whole = t0 >= 0 && t0 + VEC <= size;
      if (same && mark == 0 && (!allowed || may == (1u << VEC) - 1)) continue;
      if (whole) {
        float x[VEC];
        VecIO<T, VEC>::ld(in + t0, x);
        if (mark)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (mark >> i & 1) x[i] = marked(x[i], t0 + i);
        if (allowed)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (!(may >> i & 1)) x[i] = -INFINITY;
        if constexpr (sizeof(O) == sizeof(T)) {
          VecIO<O, VEC>::st(out + t0, x);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) Elem<O>::st(out + t0 + i, x[i]);
        }
      } else {
        for (int i = max(-t0, 0); i < VEC && t0 + i < size; ++i) {
          float x = Elem<T>::ld(in + t0 + i);
          if (mark >> i & 1) x = marked(x, t0 + i);
          if (allowed && !(may >> i & 1)) x = -INFINITY;
          Elem<O>::st(out + t0 + i, x);
        }
      }
    }
    if (a.draft_ids) {
      __syncthreads();
      drafted(-1);
    }
  }
}

template <typename T, typename O>
int launch_adjust(const cacheir_b200_logits_args& a, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  // Slices and runs: enough blocks for all SMs before rows share a count.
  LogitsParams p{a, 8192, 1};
  while (p.slice > 1024 && static_cast<long long>(a.rows) * ((a.vocab + p.slice - 1) / p.slice) < 4 * kNumSMs) p.slice /= 2;
  const int slices = (a.vocab + p.slice - 1) / p.slice;
  while (p.run < 8 && static_cast<long long>(a.rows) * slices >= 16LL * p.run * kNumSMs) p.run *= 2;
  const int runs = (a.rows + p.run - 1) / p.run;
  if (runs > 65535) p.run = (a.rows + 65534) / 65535;
  const bool counting = a.history || a.draft_ids;
  const size_t smem = (p.slice / 32 + 1 + (counting ? p.slice : 0) + (a.biases > 0 ? p.slice : 0)) * sizeof(uint32_t);
  // vectors where a row's input and output begin at the same place of 16 bytes (with outputs of the same size)
  const bool wide = reinterpret_cast<uintptr_t>(a.logits) % sizeof(T) == 0 &&
                    (sizeof(T) != sizeof(O) || ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                                                (a.row_stride - a.out_stride) % VEC == 0));
  auto kern = wide ? adjust_logits_kernel<T, O, VEC> : adjust_logits_kernel<T, O, 1>;
  const dim3 grid(slices, (a.rows + p.run - 1) / p.run);
  static std::atomic<unsigned long long> done_wide{0}, done_any{0};
  constexpr int most = (8192 / 32 + 1 + 2 * 8192) * 4;
  cudaError_t e = allow_shared_memory(wide ? done_wide : done_any, reinterpret_cast<const void*>(kern), most);
  if (e == cudaSuccess) e = launch_chained(kern, grid, dim3(kThreads), smem, stream, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
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
  if (a.logits == a.out && a.dtype != a.out_dtype) return CACHEIR_B200_EINVAL;
  if (a.vocab > 1 << 28 || (a.draft_ids && a.words > CACHEIR_B200_MAX_DRAFT_WORDS)) return CACHEIR_B200_ELIMIT;
  if (a.biases == 0) a.bias_ids = nullptr;
  if (a.dtype == CACHEIR_B200_F32) return launch_adjust<float, float>(a, as_stream(stream));
  if (a.dtype == CACHEIR_B200_F16)
    return a.out_dtype == CACHEIR_B200_F32 ? launch_adjust<__half, float>(a, as_stream(stream)) : launch_adjust<__half, __half>(a, as_stream(stream));
  return a.out_dtype == CACHEIR_B200_F32 ? launch_adjust<__nv_bfloat16, float>(a, as_stream(stream))
                                         : launch_adjust<__nv_bfloat16, __nv_bfloat16>(a, as_stream(stream));
}
