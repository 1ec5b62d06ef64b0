// Decode attention of groups of sequences with a common prefix on the tensor cores: 16-bit types, head sizes 64 and 128, pages of a multiple
// of 16 tokens, up to 64 query heads per key/value head.
//
// Three kernels. The first one multiplies the common keys of a group, once, with the queries of all of its rows that share a key/value
// head: S = Q K^T and O = P V as tcgen05 MMAs of 128 query rows, scores, probabilities and outputs in tensor memory. The second one takes
// every row's own keys with warp MMAs, like the ordinary decode attention, beside the first one on the SMs that are left to it. The third
// one joins the pieces.
//
// Common part. An item is (group, key/value head, tile of up to 256 query rows); its keys come in tiles of 128. The key tiles of all items,
// in a row, are cut evenly over the blocks, so that lengths and sizes of groups do not matter; an item that is cut leaves one piece per
// block. One warp brings keys and one values (TMA, 16 tokens at a time, into a ring of 32 KB slots; by one warp the copies' issue, 66 cycles
// each, was what the tensor cores waited for), one issues the MMAs, and two groups of four warps do the softmax, a thread per query row.
// Above 128 rows each group of warps has its own 128 of them and the two take turns on the tensor cores with the same keys; else the first
// one has them all and scores run one tile ahead. A row's maximum is a reference that moves only when it is exceeded by 2^14, so that the
// outputs, which stay in tensor memory, are hardly ever rescaled; probabilities are rounded to the element type as the second MMA's operand,
// their sums are not.
//
// Measured (32 query and 8 key/value heads of 128, fp16; all three kernels, replayed from a graph in bursts at 1965 MHz; a second of calls on end,
// under the power cap, is slower: 60 us for the first): 64 rows behind 32768 common tokens 52.2 us, of which 25.6 us are the bytes and 20.8 us
// the products; 32 rows behind 2048 tokens 20.3 us (bytes 7.1 us). 128 rows in 16 groups of ragged prefixes with 64 and 8 heads, bf16: 66.6 us
// (bytes 46.5 us). A call spends about 5.5 us before the first scores (launch, plan, page ids, copies), and about 3 us on joining. In between a
// tile of 256 query rows takes 3300 cycles, of which the tensor cores work 2048: probabilities lie over the scores they come from, so that a
// group of warps' next scores are issued behind its second product, and its step is scores (512), softmax (2300, 1500 of them exponentials) and
// second product (512) one after the other, beside which only the other group's run. Neither a share of the exponentials by polynomials nor
// reading scores once into 128 registers changed that (56.0 us became 55.7 and 56.3).
#include "shared_prefix.cuh"

#include "attention_ptx.cuh"
#include "hybrid_common.cuh"

namespace cb200 {
namespace {

using namespace ptx;

constexpr int kKeys = 128;                     // keys of a tile
constexpr int kFirst = 96;                     // .. whose probabilities go to the second MMA first: less of it is left when the others come
constexpr int kRows = 128;                     // query rows of a group of warps
constexpr int kCommonThreads = 352;
constexpr int kPlanGroups = 64;                // groups that every block lays out by itself
constexpr int kMaxHeadsPerKv = 64;
constexpr float kAhead = 6.f;                  // a new reference is the maximum less this: probabilities start at 2^6 ..
constexpr float kStale = 14.f;                 // .. and may grow to 2^14 (in fp16: 2^-24 of that is still a number)

__device__ int g_prefix_status = 0;

struct CommonParams {
  cacheir_b200_prefix_args a;
  PrefixParts parts;
  int plan_ready;                              // the plan is in the scratch already
  int tile_rows;                               // batch rows of an item
  int own_heads;                               // blocks that a row has for its own keys
  float scale_log2;
};

// A warp's wait; false in all lanes where it gave up in one.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, &g_prefix_status, code));
}
// n / d for a d that mostly is a power of two (pages).
struct Division {
  int d, shift;
  __device__ __forceinline__ explicit Division(int n) {
    d = n;
    shift = (n & (n - 1)) == 0 ? 31 - __clz(n) : -1;
  }
  __device__ __forceinline__ int of(int n) const { return shift >= 0 ? n >> shift : n / d; }
};

// ---- how the common parts are cut ----
// An item of n key tiles is kItemUnits + n units: what it costs to begin with (queries, the first tile's latency, the output) is about
// that of so many tiles. The units are dealt out as evenly as whole numbers can be.
constexpr int kItemUnits = 2;

struct Deal {
  int share, more;             // every block has `share` units, the first `more` one more
  __device__ __forceinline__ Deal(int units, int ctas) : share(units / ctas), more(units % ctas) {}
  __device__ __forceinline__ int begin(int block) const { return block * share + min(block, more); }
  __device__ __forceinline__ int owner(int unit) const {
    const int big = more * (share + 1);
    return unit < big ? unit / (share + 1) : more + (unit - big) / share;
  }
};

__device__ __forceinline__ int key_tiles(int keys) { return (keys + kKeys - 1) / kKeys; }
// Group g, and its units (the launcher has seen that all of them fit an int).
__device__ __forceinline__ int group_units(const cacheir_b200_prefix_args& a, int tile_rows, int g, PlanGroup* out) {
  out->row = group_start(a, g);
  out->rows = max(group_start(a, g + 1) - out->row, 0);
  out->prefix = prefix_of_group(a, g);
  return out->rows > 0 && out->prefix > 0 ? a.kv_heads * ((out->rows + tile_rows - 1) / tile_rows) * (kItemUnits + key_tiles(out->prefix)) : 0;
}
// What decides how many blocks take part, besides the units.
struct Weights {
  int longest;                 // key tiles of the longest item
  long long common;            // tokens times rows of the common parts
  long long cost;              // units, those of items for two groups of warps half as much again
};
__device__ __forceinline__ Weights group_weights(const PlanGroup& g, int units, int half_rows) {
  return Weights{units > 0 ? key_tiles(g.prefix) : 0, static_cast<long long>(g.rows) * g.prefix, g.rows > half_rows ? units + units / 2 : units};
}
// Blocks that take part. No item may be in more pieces than there is scratch for: n tiles touch ceil((n - 1) / share) + 1 blocks at most. And
// the common parts get as many SMs as is their share of the work, so that the other kernel can have the rest of them meanwhile: 16 own
// tokens of a key/value head (8 KB) take an SM about a twentieth of a unit's time (64 KB), and a row's own part costs as much as eleven of
// those before it has any. `lens`: tokens of all rows. (Device times: 64 rows with 144 own tokens on average behind 32768, 128 rows with 350 behind up to 4095:
// 51.2 and 66.6 us; an eighteenth 51.3 and 68.5, a twenty-second 52.8 and 66.5, fourteen and a twentieth 51.4 and 68.2.)
__device__ __forceinline__ int plan_ctas(const cacheir_b200_prefix_args& a, int pieces, int own_heads, int units, const Weights& w, long long lens, int grid) {
  if (units <= 0) return 0;
  const int least = max(1, (w.longest - 1 + pieces - 2) / (pieces - 1));
  const float cost = static_cast<float>(w.cost), own = __fmul_rn(static_cast<float>(max(lens - w.common, 0LL) / kChunk + 11LL * a.batch), own_heads / 20.f);
  const float sms = __fdiv_rn(__fmul_rn(kNumSMs, cost), __fadd_rn(cost, own));       // (two kernels work this out and have to agree)
  return max(1, min(min(grid, units / least), static_cast<int>(sms) + 1));
}
// Tokens of all rows, a thread's part of them.
__device__ __forceinline__ long long lens_part(const cacheir_b200_prefix_args& a, int thread, int threads) {
  const int room = a.max_pages * a.page_size;
  long long sum = 0;
  for (int b = thread; b < a.batch; b += threads) sum += min(max(a.seq_lens[b], 0), room);
  return sum;
}
__device__ __forceinline__ long long warp_sum64(long long v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The plan of more groups than a block lays out by itself.
__global__ void __launch_bounds__(1024)
prefix_plan_kernel(const CommonParams p, const int grid) {
  chain_enter();
  __shared__ int s_sum[32], s_longest[32];
  __shared__ long long s_wide[3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  Weights all{0, 0, 0};
  for (int g0 = 0; g0 < p.a.groups; g0 += 1024) {
    const int g = g0 + threadIdx.x;
    PlanGroup group{};
    const int own = g < p.a.groups ? group_units(p.a, p.tile_rows, g, &group) : 0;
    int sum = own;
    const Weights w = group_weights(group, own, p.tile_rows / 2);
    all = Weights{max(all.longest, w.longest), all.common + w.common, all.cost + w.cost};
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += up;
    }
    if (lane == 31) s_sum[warp] = sum;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w];
    }
    group.start = base + before + sum - own;
    if (g < p.a.groups) p.parts.plan->group[g] = group;
    base += total;
    __syncthreads();
  }
  const int longest = __reduce_max_sync(0xffffffffu, all.longest);
  const long long lens = warp_sum64(lens_part(p.a, threadIdx.x, 1024)), common = warp_sum64(all.common), cost = warp_sum64(all.cost);
  if (lane == 0) { s_longest[warp] = longest; s_wide[0][warp] = lens; s_wide[1][warp] = common; s_wide[2][warp] = cost; }
  __syncthreads();
  if (threadIdx.x == 0) {
    Weights w{0, 0, 0};
    long long tokens = 0;
    for (int i = 0; i < 32; ++i) {
      w = Weights{max(w.longest, s_longest[i]), w.common + s_wide[1][i], w.cost + s_wide[2][i]};
      tokens += s_wide[0][i];
    }
    p.parts.plan->group[p.a.groups].start = base;
    p.parts.plan->units = base;
    p.parts.plan->ctas = plan_ctas(p.a, p.parts.pieces, p.own_heads, base, w, tokens, grid);
  }
}

// A block's share of the units, item by item.
struct Walk {
  const PlanGroup* groups;
  Deal deal;
  int at, end;
  // the item
  int group, kvh, row0, rows, tile, tiles, prefix, piece;      // key tiles tile .. tile + tiles - 1 of it are this block's

  __device__ __forceinline__ Walk(const PlanGroup* g, int units, int ctas) : groups(g), deal(units, ctas) {
    at = deal.begin(blockIdx.x);
    end = deal.begin(blockIdx.x + 1);
  }
  __device__ __forceinline__ bool next(const CommonParams& p) {
    while (at < end) {
      int lo = 0, hi = p.a.groups;                             // last group that starts at or before `at` (empty ones start where the next does)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (groups[mid].start <= at) lo = mid; else hi = mid;
      }
      const PlanGroup of = groups[lo];
      const int all = kItemUnits + key_tiles(of.prefix), row_tiles = (of.rows + p.tile_rows - 1) / p.tile_rows;
      const int rel = at - of.start, item = rel / all, item0 = of.start + item * all, tile0 = item0 + kItemUnits;
      const int stop = min(end, item0 + all);
      tile = max(at - tile0, 0);
      tiles = stop - tile0 - tile;
      at = stop;
      if (tiles <= 0) continue;                                // (no more than an item's beginning: the next block has its tiles)
      group = lo;
      prefix = of.prefix;
      kvh = item / row_tiles;
      row0 = of.row + (item - kvh * row_tiles) * p.tile_rows;
      rows = min(p.tile_rows, of.row + of.rows - row0);
      piece = blockIdx.x - deal.owner(tile0);
      return true;
    }
    return false;
  }
};

template <int D>
struct CommonSmem {
  static constexpr int kSlotBytes = kKeys * D * 2;
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kTiles = 2 * kQBytes + kSlots * kSlotBytes;
  // then: barriers full, empty [slots], q[2], place of q[2], s[2], p[2][2], o[2]; tensor memory address; groups
  static constexpr int kBarriers = 2 * kSlots + 12;
  static constexpr int kBytes = 1024 + kTiles + kBarriers * 8 + 16 + (kPlanGroups + 1) * static_cast<int>(sizeof(PlanGroup));
};

template <typename T, int D>
__global__ void __launch_bounds__(kCommonThreads, 1)
prefix_common_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_q,
                     const __grid_constant__ CommonParams p) {
  using L = CommonSmem<D>;
  constexpr int kSlots = L::kSlots;
  chain_enter();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;                                         // [2][D / 64][128 rows][128 B]
  uint8_t* s_kv = smem + 2 * L::kQBytes;                       // [slots][D / 64][128 keys][128 B]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kTiles);
  uint64_t* empty = full + kSlots;
  uint64_t* bar_q = empty + kSlots;                            // queries of a group of warps are there
  uint64_t* bar_free = bar_q + 2;                              // .. and their place is free again
  uint64_t* bar_s = bar_free + 2;                              // scores are in tensor memory
  uint64_t* bar_p = bar_s + 2;                                 // probabilities are, [buffer][first keys, the others]
  uint64_t* bar_o = bar_p + 4;                                 // .. and have been added to the output
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_o + 2);
  PlanGroup* s_group = reinterpret_cast<PlanGroup*>(tmem_slot + 4);
  __shared__ int s_plan[2], s_scan[kPlanGroups / 32], s_longest[kPlanGroups / 32];
  __shared__ long long s_lens[kCommonThreads / 32], s_common[kPlanGroups / 32], s_cost[kPlanGroups / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const cacheir_b200_prefix_args& a = p.a;

  if (warp == 8) tc_alloc(smem_u32(tmem_slot), 512);           // (beside the loads of the plan)
  if (threadIdx.x == 288) {
    prefetch_map(&tmap_q);
    prefetch_map(&tmap_k);
    prefetch_map(&tmap_v);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_q[b]), 1);
      mbar_init(smem_u32(&bar_free[b]), 4);
      mbar_init(smem_u32(&bar_s[b]), 1);
      mbar_init(smem_u32(&bar_p[2 * b]), kRows);
      mbar_init(smem_u32(&bar_p[2 * b + 1]), kRows);
      mbar_init(smem_u32(&bar_o[b]), 1);
    }
    mbar_fence_init();
  }
  // ---- the plan ----
  if (!p.plan_ready) {
    PlanGroup mine{};
    int own = 0, sum = 0;
    const long long lens = lens_part(a, threadIdx.x, kCommonThreads);
    if (warp < kPlanGroups / 32) {
      own = static_cast<int>(threadIdx.x) < a.groups ? group_units(a, p.tile_rows, threadIdx.x, &mine) : 0;
      const Weights w = group_weights(mine, own, p.tile_rows / 2);
      const int longest = __reduce_max_sync(0xffffffffu, w.longest);
      const long long common = warp_sum64(w.common), cost = warp_sum64(w.cost);
      sum = own;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += up;
      }
      if (lane == 31) { s_scan[warp] = sum; s_longest[warp] = longest; s_common[warp] = common; s_cost[warp] = cost; }
    }
    const long long warp_lens = warp_sum64(lens);
    if (lane == 0) s_lens[warp] = warp_lens;
    __syncthreads();
    if (warp < kPlanGroups / 32) {
      int before = 0, all = 0;
      Weights w{0, 0, 0};
#pragma unroll
      for (int i = 0; i < kPlanGroups / 32; ++i) {
        if (i < warp) before += s_scan[i];
        all += s_scan[i];
        w = Weights{max(w.longest, s_longest[i]), w.common + s_common[i], w.cost + s_cost[i]};
      }
      mine.start = before + sum - own;
      if (static_cast<int>(threadIdx.x) < a.groups) s_group[threadIdx.x] = mine;
      if (threadIdx.x == 0) {
        long long tokens = 0;
#pragma unroll
        for (int i = 0; i < kCommonThreads / 32; ++i) tokens += s_lens[i];
        s_group[a.groups].start = all;
        s_plan[0] = all;
        s_plan[1] = plan_ctas(a, p.parts.pieces, p.own_heads, all, w, tokens, gridDim.x);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const PlanGroup* groups = p.plan_ready ? p.parts.plan->group : s_group;
  const int units = p.plan_ready ? p.parts.plan->units : s_plan[0], ctas = p.plan_ready ? p.parts.plan->ctas : s_plan[1];
  if (!p.plan_ready && blockIdx.x == 0) {                      // for the kernel that joins
    for (int g = threadIdx.x; g < a.groups; g += kCommonThreads) p.parts.plan->group[g] = s_group[g];
    if (threadIdx.x == 0) {
      p.parts.plan->units = units;
      p.parts.plan->ctas = ctas;
    }
  }
  const uint32_t tmem = *tmem_slot;                            // scores [2][128 columns] (probabilities over them), outputs [2][D]
  const uint32_t tmem_o = tmem + 2 * kKeys;
  const int group = a.heads / a.kv_heads, half_rows = p.tile_rows / 2;        // batch rows of a group of warps
  const bool takes_part = static_cast<int>(blockIdx.x) < ctas;
  Walk walk(groups, max(units, 1), max(ctas, 1));
  if (!takes_part) walk.end = walk.at;
  bool ok = true;

  if (warp >= 9) {
    // ------- copies: warp 9 keys, a lane per 16 of them and 64 columns; warp 10 values, a lane per 16 of them -------
    const bool keys = warp == 9;
    const int boxes = keys ? D / 64 : 1, chunk = lane / boxes, box = lane % boxes;
    const bool copies = chunk < kKeys / kChunk;
    const int outside = a.num_slots * a.kv_heads * a.page_size;         // rows behind the pool read as zeros
    const uint32_t dst = smem_u32(s_kv) + (keys ? box * kKeys * 128 + chunk * kChunk * 128 : chunk * kChunk * D * 2);
    const Division by_page(a.page_size);
    int slot = keys ? 0 : 1, q_place = 0;
    uint32_t phase = 1, sent = 0, q_phase = 3;                 // (slots of a tile: its keys', its values'; q_phase: a bit for either place)
    while (ok && walk.next(p)) {
      const int32_t* pages = a.prefix_table + static_cast<size_t>(walk.group) * a.prefix_pages;
      auto line_of = [&](int tile) {                           // first row of this lane's 16 in the pool
        const int key = tile * kKeys + chunk * kChunk;
        if (!copies || key >= walk.prefix) return outside;
        const int page = by_page.of(key), id = pages[page];
        return id >= 0 && id < a.num_slots ? (id * a.kv_heads + walk.kvh) * a.page_size + key - page * a.page_size : outside;
      };
      int line = line_of(walk.tile);
      if (!keys) {                                             // the item's queries: rows, heads, 64 columns at a time
        const bool two = walk.rows > half_rows;
        for (int w = 0; w < (two ? 2 : 1) && ok; ++w) {
          const int place = two ? w : q_place;
          ok = warp_wait(smem_u32(&bar_free[place]), q_phase >> place & 1, (15 << 8) | 7);
          if (!ok) break;
          q_phase ^= 1u << place;
          if (lane == 0) {
            mbar_expect_tx(smem_u32(&bar_q[place]), (D / 64) * half_rows * group * 128);
            for (int z = 0; z < D / 64; ++z)
              tma_load_4d(smem_u32(s_q + place * L::kQBytes + z * kRows * 128), &tmap_q, smem_u32(&bar_q[place]), 0, walk.kvh * group,
                          walk.row0 + w * half_rows, z);
          }
          __syncwarp();
        }
        if (!two) q_place ^= 1;
      }
      for (int t = walk.tile; t < walk.tile + walk.tiles && ok; ++t) {
        const int next = t + 1 < walk.tile + walk.tiles ? line_of(t + 1) : 0;
        ok = warp_wait(smem_u32(&empty[slot]), phase, (15 << 8) | 1);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(smem_u32(&full[slot]), L::kSlotBytes);
        __syncwarp();
        if (copies) {
          if (keys) tma_load_3d(dst + slot * L::kSlotBytes, &tmap_k, smem_u32(&full[slot]), 0, line, box);
          else tma_load_3d(dst + slot * L::kSlotBytes, &tmap_v, smem_u32(&full[slot]), 0, line, 0);
        }
        ++sent;
        slot += 2;
        if (slot >= kSlots) { slot -= kSlots; phase ^= 1; }
        line = next;
      }
    }
    // nothing may still be on its way when the block ends, also after a wait that gave up
    for (uint32_t i = sent > kSlots ? sent - kSlots : 0; i < sent; ++i) {
      const uint32_t n = 2 * i + (keys ? 0 : 1);
      if (ok && n + kSlots < 2 * sent) continue;               // its slot has been filled again since: it came, and that phase is long over
      mbar_wait(smem_u32(&full[n % kSlots]), (n / kSlots) & 1, &g_prefix_status, (15 << 8) | 2);
    }
    // (queries are waited for by the products; after a wait that gave up: both phases of both places)
    if (!keys && !ok)
      for (int w = 0; w < 4; ++w) mbar_wait(smem_u32(&bar_q[w >> 1]), w & 1, &g_prefix_status, (15 << 8) | 2);
  } else if (warp == 8) {
    // ---------------- MMA issue ----------------
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
    const uint32_t id_s = (1u << 4) | (kType << 7) | (kType << 10) | (static_cast<uint32_t>(kKeys >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
    const uint32_t id_o = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) |
                          (static_cast<uint32_t>(kRows >> 4) << 24);
    const uint64_t dq = smem_desc_sw128(smem_u32(s_q)), dk = smem_desc_sw128(smem_u32(s_kv)), dv = smem_desc_columns(smem_u32(s_kv));
    // An item's steps: a tile each, or a tile for either group of warps. Scores are two steps ahead of outputs, and are issued right behind the
    // output that frees their buffer. This is one warp's chain of dependent instructions, which the tensor cores wait for where it is not
    // done in time: whatever can be carried along is, and keys are waited for between the two halves of an output.
    const bool leader = elect_one();
    int b_s = 0, b_o = 0, k_slot = 0, v_slot = 1, q_place = 0; // buffers of scores and probabilities; slots
    uint32_t k_phase = 0, v_phase = 0, q_phase = 0, p_phase = 0;        // (of the two buffers of queries and probabilities: a bit each)
    while (ok && walk.next(p)) {
      const bool two = walk.rows > half_rows;
      const int steps = two ? 2 * walk.tiles : walk.tiles;
      auto wait_scores = [&](int j) {                          // the operands of step j's scores
        if (j < (two ? 2 : 1)) {                               // the item's first tile: its queries are new
          const int w = two ? b_s : q_place;
          if (!warp_wait(smem_u32(&bar_q[w]), q_phase >> w & 1, (15 << 8) | 3)) return false;
          q_phase ^= 1u << w;
        }
        return (two && (j & 1)) || warp_wait(smem_u32(&full[k_slot]), k_phase, (15 << 8) | 4);
      };
      auto score = [&](int j) {                                // (one lane)
        const uint64_t q_at = dq + ((two ? b_s : q_place) * L::kQBytes >> 4), k_at = dk + (k_slot * L::kSlotBytes >> 4);
        const uint32_t to = tmem + b_s * kKeys;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          constexpr int kHalf = kRows * 128 >> 4;              // 64 columns further
          mma_ss(to, q_at + (k >> 2) * kHalf + (k & 3) * 2, k_at + (k >> 2) * kHalf + (k & 3) * 2, id_s, k > 0 ? 1u : 0u);
        }
        tc_commit(smem_u32(&bar_s[b_s]));
        if (!two || (j & 1)) tc_commit(smem_u32(&empty[k_slot]));
      };
      auto scored = [&](int j) {                               // (the whole warp)
        b_s ^= 1;
        if (!two || (j & 1)) {
          k_slot += 2;
          if (k_slot >= kSlots) { k_slot -= kSlots; k_phase ^= 1; }
        }
      };
      for (int j = 0; j < 2 && j < steps && ok; ++j) {
        ok = wait_scores(j);
        if (!ok) break;
        tc_fence_after();
        if (leader) score(j);
        __syncwarp();
        scored(j);
      }
      for (int j = 0; j < steps && ok; ++j) {
        if (!(two && (j & 1))) ok = warp_wait(smem_u32(&full[v_slot]), v_phase, (15 << 8) | 5);
        ok = ok && warp_wait(smem_u32(&bar_p[2 * b_o]), p_phase >> b_o & 1, (15 << 8) | 6);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v_at = dv + (v_slot * L::kSlotBytes >> 4);
        const uint32_t to = tmem_o + (two ? b_o * D : 0), from = tmem + b_o * kKeys, add = j < (two ? 2 : 1) ? 0u : 1u;
        const bool frees = !two || (j & 1), more = j + 2 < steps;
        if (leader) {                                          // (the first keys while the others' probabilities are worked out)
#pragma unroll
          for (int k = 0; k < kFirst / 16; ++k) mma_ts(to, from + k * 8, v_at + k * (kChunk * D * 2 >> 4), id_o, k == 0 ? add : 1u);
        }
        __syncwarp();
        if (more) ok = wait_scores(j + 2);
        ok = ok && warp_wait(smem_u32(&bar_p[2 * b_o + 1]), p_phase >> b_o & 1, (15 << 8) | 6);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = kFirst / 16; k < kKeys / 16; ++k) mma_ts(to, from + k * 8, v_at + k * (kChunk * D * 2 >> 4), id_o, 1u);
          tc_commit(smem_u32(&bar_o[b_o]));
          if (frees) tc_commit(smem_u32(&empty[v_slot]));
          if (more) score(j + 2);
        }
        __syncwarp();
        p_phase ^= 1u << b_o;
        b_o ^= 1;
        if (frees) {
          v_slot += 2;
          if (v_slot >= kSlots) { v_slot -= kSlots; v_phase ^= 1; }
        }
        if (more) scored(j + 2);
      }
      if (!two) q_place ^= 1;
    }
  } else {
    // ---------------- softmax: a thread per query row ----------------
    const int w = warp >> 2, r = threadIdx.x & (kRows - 1);
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int by_group = (65536 + group - 1) / group;          // n / group = n * by_group >> 16 for n < 256, group <= 64
    int step = 0, tile = 0, q_place = 0;                       // of the block so far; where the queries of an item of one group of warps are
    while (ok && walk.next(p)) {
      const int two = walk.rows > half_rows ? 1 : 0, steps = walk.tiles * (two ? 2 : 1);
      if (!two && w == 1) {                                    // (its barrier's phases pass all the same)
        for (int s = step | 1; s < step + steps && ok; s += 2) ok = warp_wait(smem_u32(&bar_s[1]), (s >> 1) & 1, (15 << 8) | 14);
        step += steps;
        tile += walk.tiles;
        q_place ^= 1;
        continue;
      }
      const int place = two ? w : q_place;
      if (!two) q_place ^= 1;
      const int in_tile = w * half_rows + (r * by_group >> 16);          // this thread's row of the item
      const bool real = r < half_rows * group && in_tile < walk.rows;
      const int b_row = walk.row0 + (real ? in_tile : 0), head = walk.kvh * group + (real ? r - (r * by_group >> 16) * group : 0);
      // Keys that the row sees: all, or none where it ends inside the prefix. What stands behind its end may hold anything, also values that are
      // no numbers, and 0 * value would not be 0: such a row's keys are its own, and the outputs that it gets here have no weight.
      const int limit = real && a.seq_lens[b_row] < walk.prefix ? 0 : walk.prefix;
      float m_ref = -INFINITY, l_run = 0.f;
      int last = 0;
      for (int t = 0, s = two ? step + ((step ^ w) & 1) : step; t < walk.tiles && ok; ++t, s += two ? 2 : 1) {
        const int b = s & 1, base = (walk.tile + t) * kKeys;
        ok = warp_wait(smem_u32(&bar_s[b]), (s >> 1) & 1, (15 << 8) | 8);
        if (!ok) break;
        tc_fence_after();
        const uint32_t scores = tmem + b * kKeys + lane_addr;
        const bool whole = __all_sync(0xffffffffu, base + kKeys <= limit);
        // The row's 128 scores are looked at twice. For the maximum the second half comes first: the first half then stays in registers,
        // and its probabilities may be written over scores 0 .. 31 while the second half is still where it was.
        uint32_t x[32], y[32];
        auto masked = [&](uint32_t (&v)[32], int first) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (base + first + i >= limit) v[i] = 0xff800000u;           // -inf
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto largest = [&](const uint32_t (&v)[32]) {
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            asm("max.f32 %0, %1, %2, %0;" : "+f"(mx[(i >> 1) & 3]) : "f"(__uint_as_float(v[i])), "f"(__uint_as_float(v[i + 1])));
        };
        tmem_ld_x32(scores + 64, x);
        tmem_ld_x32(scores + 96, y);
        tmem_wait_ld(x);
        tmem_wait_ld(y);
        if (!whole) { masked(x, 64); masked(y, 96); }
        largest(x);
        largest(y);
        tmem_ld_x32(scores, x);
        tmem_ld_x32(scores + 32, y);
        tmem_wait_ld(x);
        tmem_wait_ld(y);
        if (!whole) { masked(x, 0); masked(y, 32); }
        largest(x);
        largest(y);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
        const bool grown = top > m_ref + kStale;
        if (__any_sync(0xffffffffu, grown)) {
          const float fresh = grown ? top - kAhead : m_ref, alpha = grown ? ex2(m_ref - fresh) : 1.f;
          m_ref = fresh;
          l_run *= alpha;
          if (t > 0) {                                         // bring the output to the new reference
            // (with two groups of warps this buffer's last output came before these scores)
            if (!two) ok = warp_wait(smem_u32(&bar_o[(s - 1) & 1]), ((s - 1) >> 1) & 1, (15 << 8) | 9);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tc_ld_x16(tmem_o + w * D + lane_addr + c, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_x16(tmem_o + w * D + lane_addr + c, o);
            }
          }
        }
        // keys behind the prefix in its last page may hold anything: zero their values, so that 0 * value stays 0
        auto clear_values = [&] {
          const int rest = walk.prefix - base;
          if (rest >= kKeys || rest % kChunk == 0) return;
          const int at = 2 * (tile + t) + 1, slot = at % kSlots;
          ok = warp_wait(smem_u32(&full[slot]), (at / kSlots) & 1, (15 << 8) | 10) && ok;
          const int rows = kChunk - rest % kChunk;
          for (int i = r; i < rows * (D / 8); i += kRows) {
            const int key = rest + i / (D / 8), c = i % (D / 8);
            *reinterpret_cast<uint4*>(s_kv + slot * L::kSlotBytes + (key / kChunk) * kChunk * D * 2 + (c >> 3) * kChunk * 128 + key % kChunk * 128 + ((c & 7) << 4)) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_smem();
        };
        const float less = m_ref > -INFINITY ? -m_ref : 0.f;
        f32x2 sum[2] = {0ull, 0ull};
        const f32x2 scale2 = pair(p.scale_log2, p.scale_log2), less2 = pair(less, less);
        auto weigh = [&](const uint32_t (&v)[32], uint32_t* out) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float a0, a1;
            unpair(fma2(pair(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), scale2, less2), a0, a1);
            a0 = ex2(a0);
            a1 = ex2(a1);
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pair(a0, a1));
            out[i >> 1] = pack_pair<T>(a0, a1);
          }
        };
        {
          uint32_t out[32];
          weigh(x, out);
          tmem_ld_x32(scores + 64, x);                         // (on its way meanwhile)
          weigh(y, out + 16);
          tmem_wait_ld(x);
          tmem_ld_x32(scores + 96, y);
          tmem_st_x32(scores, out);
          if (!whole) masked(x, 64);
          uint32_t rest[16];
          weigh(x, rest);
          tmem_wait_ld(y);
          tmem_st_x16(scores + 32, rest);
          tmem_wait_st();
          clear_values();
          tc_fence_before();
          mbar_arrive(smem_u32(&bar_p[2 * b]));
          if (!whole) masked(y, 96);
          weigh(y, rest);
          tmem_st_x16(scores + 48, rest);
        }
        float s0, s1, s2, s3;
        unpair(sum[0], s0, s1);
        unpair(sum[1], s2, s3);
        l_run += (s0 + s1) + (s2 + s3);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&bar_p[2 * b + 1]));
        last = s;
      }
      step += steps;
      tile += walk.tiles;
      if (!ok) break;
      ok = warp_wait(smem_u32(&bar_o[last & 1]), (last >> 1) & 1, (15 << 8) | 11);
      if (!ok) break;
      tc_fence_after();
      const int at = real ? b_row * a.heads + head : -1;
      const size_t piece0 = static_cast<size_t>(walk.piece) * a.batch * a.heads;
      if (real) *reinterpret_cast<float2*>(p.parts.ml + 2 * (piece0 + at)) = make_float2(m_ref, l_run);
      // By way of shared memory (the queries' place), so that a store writes whole lines: a lane has a row, a store 128 bytes of four rows.
      float* s_row = reinterpret_cast<float*>(s_q + place * L::kQBytes + (warp & 3) * (L::kQBytes / 4));
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld_x32(tmem_o + w * D + lane_addr + c, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(s_row + lane * 32 + ((i ^ (lane & 7)) << 2)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 4 * i + (lane >> 3), to = __shfl_sync(0xffffffffu, at, row);
          const uint4 v = *reinterpret_cast<const uint4*>(s_row + row * 32 + (((lane & 7) ^ (row & 7)) << 2));
          if (to >= 0) *reinterpret_cast<uint4*>(p.parts.acc + (piece0 + to) * D + c + (lane & 7) * 4) = v;
        }
        __syncwarp();
      }
      tc_fence_before();
      fence_async_smem();                                      // (the next queries come by copies)
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_free[place]));
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tc_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Every row's own keys. One block per (part of the row's own keys, key/value head and up to 16 of its query heads, row). Keys and values come
// 16 tokens at a time (TMA): every warp takes every WARPS-th chunk of the part through a ring of its own, with warp MMAs that have the query
// heads as their 16 rows. Bound by the memory's rate where there are many rows: then blocks of two warps, six of them on an SM, so that
// while some begin or end others keep the memory busy; where there are few, blocks of four or eight, and the longest row counts: a chunk takes
// a warp about 1 us, half its copy's latency and half its own chain of instructions (masks and cleared values only in chunks that are not
// whole, two chains of products a score, and the scale inside the exponent's argument made 20.0 us of 21.7 for 32 rows of up to 512 own
// tokens; a reference that moves as seldom as that of the common keys made nothing of it). None of that needs the common part's
// kernel: this one starts as soon as that one's blocks have their places, on the SMs that they leave.
struct OwnParams {
  cacheir_b200_prefix_args a;
  PrefixParts parts;
  int common;                                  // a kernel of common parts runs before
  int tile_rows, head_chunks, splits;
  int grid;                                    // .. its blocks
  float scale_log2;
};

template <int D, int WARPS>
struct OwnSmem {
  static constexpr int kStages = WARPS <= 4 ? 2 : 3;
  static constexpr int kTileBytes = kChunk * D * 2;
  static constexpr int kRing = WARPS * kStages * 2 * kTileBytes;
  static constexpr int kJoin = WARPS * 16 * (D + 2) * 4;       // over the ring afterwards: the warps' states
  static constexpr int kBytes = 1024 + (kRing > kJoin ? kRing : kJoin) + WARPS * kStages * 8;
};

__device__ __forceinline__ void ldsm_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma_pair(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
  else
    mma_bf16(c, x, b0, b1);
}
// A row's group (rows and prefix 0 outside every group). Up to 32 groups, a lane each, the warp lays the plan out beside that, as nothing of it
// has to wait for the common part's kernel.
struct RowGroup {
  PlanGroup in;
  int group, planned, units;                   // planned: its first unit, the number of units and what decides about blocks are known already
  Weights weights;
};
__device__ __forceinline__ RowGroup row_group(const cacheir_b200_prefix_args& a, int tile_rows, int row) {
  RowGroup r{};
  r.group = -1;
  if (a.groups <= 0) return r;
  if (a.groups > 32) {
    r.group = group_of_row(a, row, &r.in.prefix);
    if (r.group >= 0) {
      r.in.row = group_start(a, r.group);
      r.in.rows = group_start(a, r.group + 1) - r.in.row;
    }
    return r;
  }
  const int lane = threadIdx.x & 31;
  PlanGroup mine{};
  const int own = lane < a.groups ? group_units(a, tile_rows, lane, &mine) : 0;
  int sum = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += up;
  }
  r.planned = 1;
  r.units = __shfl_sync(0xffffffffu, sum, 31);
  const Weights w = group_weights(mine, own, tile_rows / 2);
  r.weights = Weights{__reduce_max_sync(0xffffffffu, w.longest), warp_sum64(w.common), warp_sum64(w.cost)};
  const uint32_t found = __ballot_sync(0xffffffffu, mine.rows > 0 && mine.row <= row && row < mine.row + mine.rows);
  if (found == 0) return r;
  r.group = 31 - __clz(found);
  r.in.start = __shfl_sync(0xffffffffu, sum - own, r.group);
  r.in.row = __shfl_sync(0xffffffffu, mine.row, r.group);
  r.in.rows = __shfl_sync(0xffffffffu, mine.rows, r.group);
  r.in.prefix = __shfl_sync(0xffffffffu, mine.prefix, r.group);
  return r;
}

template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
prefix_own_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ OwnParams p) {
  using L = OwnSmem<D, WARPS>;
  constexpr int kThreads = WARPS * 32, kStages = L::kStages;
  // This kernel reads what was there before the common part's kernel began, whose blocks let this one in only after they had waited for all
  // earlier ones. (One block waits for that kernel in the end, so that the end of this one implies the end of both.)
  if (!p.common) chain_wait();
  chain_next();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const cacheir_b200_prefix_args& a = p.a;
  const int split = blockIdx.x, kvh = blockIdx.y / p.head_chunks, row = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.kv_heads, head0 = kvh * group + blockIdx.y % p.head_chunks * 16, heads = min(16, (kvh + 1) * group - head0);
  const uint32_t bars = smem_u32(smem_raw + L::kBytes - WARPS * kStages * 8) + warp * kStages * 8;
  const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * L::kTileBytes;
  const int g = lane >> 2, t4 = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bars + s * 8, 1);
    mbar_fence_init();
    if (warp == 0) {
      prefetch_map(&tmap_k);
      prefetch_map(&tmap_v);
    }
  }
  // Lengths, group, first page ids and queries are asked for together as far as they can be.
  const int tokens = max(a.seq_lens[row], 0);
  int prefix;
  const int in_group = group_of_row(a, row, &prefix);
  const bool inside = tokens < prefix;                           // (no key of it is common)
  const int len = inside ? tokens : min(tokens, a.max_pages * a.page_size), from = inside ? 0 : min(prefix, len);
  const int chunk0 = from / kChunk, chunks = len > from ? (len + kChunk - 1) / kChunk - chunk0 : 0, per = (chunks + p.splits - 1) / p.splits;
  const int begin = chunk0 + min(chunks, split * per), end = chunk0 + min(chunks, (split + 1) * per);
  uint32_t qa[D / 16][4];                                        // queries as the A operand: rows = heads
  {
    const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(row) * a.q_stride + static_cast<size_t>(head0) * D;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = g + (i & 1) * 8, col = k * 16 + 2 * t4 + (i >> 1) * 8;
        qa[k][i] = h < heads ? *reinterpret_cast<const uint32_t*>(q + static_cast<size_t>(h) * D + col) : 0u;
      }
  }
  const int32_t* pages = inside ? a.prefix_table + static_cast<size_t>(in_group) * a.prefix_pages : a.page_table + static_cast<size_t>(row) * a.max_pages;
  const int outside = a.num_slots * a.kv_heads * a.page_size;   // rows behind the pool read as zeros
  const int mine = begin + warp < end ? (end - begin - warp + WARPS - 1) / WARPS : 0;          // chunks begin + warp + i * WARPS
  const Division by_page(a.page_size);
  auto line_of = [&](int i) {                                    // first row of this warp's i-th chunk in the pool
    if (i >= mine) return outside;
    const int key = (begin + warp + i * WARPS) * kChunk, page = by_page.of(key), id = pages[page];
    return id >= 0 && id < a.num_slots ? (id * a.kv_heads + kvh) * a.page_size + key - page * a.page_size : outside;
  };
  int lines = line_of(lane), lines_next = mine > 32 ? line_of(32 + lane) : outside;            // of chunks 32 k + lane, k rising
  __syncwarp();
  auto copy = [&](int i, int s) {                                // chunk i into stage s: a lane for the keys, one for the values
    const int line = __shfl_sync(0xffffffffu, lines, i & 31);
    if (lane == 0) mbar_expect_tx(bars + s * 8, 2 * L::kTileBytes);
    __syncwarp();
    if (lane < 2) tma_load_3d(ring + (2 * s + lane) * L::kTileBytes, lane == 0 ? &tmap_k : &tmap_v, bars + s * 8, 0, line, 0);
  };
  for (int s = 0; s < kStages; ++s)
    if (s < mine) copy(s, s);

  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const uint32_t lrow = lane & 7, lmat = lane >> 3;
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
#pragma unroll 1
  for (int it = 0; it < mine; ++it) {
    ok = warp_wait(bars + stage * 8, phase, (15 << 8) | 12);
    if (!ok) {                                                   // the copies that are still under way are waited for
      for (int i = it; i < min(mine, it + kStages); ++i) {
        mbar_wait(bars + stage * 8, phase, &g_prefix_status, (15 << 8) | 13);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      break;
    }
    const uint32_t kbase = ring + stage * 2 * L::kTileBytes, vbase = kbase + L::kTileBytes;
    float sc[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float odd[4] = {0.f, 0.f, 0.f, 0.f};                       // (two chains of products a score: this warp waits for its own results only)
      sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
      const uint32_t token = n * 8 + lrow;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const uint32_t c = 4 * k + lmat;
        uint32_t kb[4];
        ldsm_x4(kbase + (c >> 3) * (kChunk * 128) + token * 128 + (((c & 7) ^ (token & 7)) << 4), kb);
        mma_pair<T>(sc[n], qa[2 * k], kb[0], kb[1]);
        mma_pair<T>(odd, qa[2 * k + 1], kb[2], kb[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][e] += odd[e];
    }
    const int key0 = (begin + warp + it * WARPS) * kChunk;
    const bool whole = key0 >= from && key0 + kChunk <= len;
    if (!whole) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + 2 * t4 + (e & 1);
          if (key < from || key >= len) sc[n][e] = -INFINITY;
        }
    }
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) top[r] = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
    float corr[2], less[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float m_new = fmaxf(m_run[r], top[r] * p.scale_log2);                  // (-inf where all scores so far are)
      less[r] = m_new > -INFINITY ? m_new : 0.f;
      corr[r] = ex2(m_run[r] - less[r]);
      m_run[r] = m_new;
    }
    float pr[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[n][e] = ex2(fmaf(sc[n][e], p.scale_log2, -less[e >> 1]));
#pragma unroll
    for (int r = 0; r < 2; ++r) l_run[r] = l_run[r] * corr[r] + (pr[0][2 * r] + pr[0][2 * r + 1] + pr[1][2 * r] + pr[1][2 * r + 1]);
    const uint32_t pa[4] = {pack_pair<T>(pr[0][0], pr[0][1]), pack_pair<T>(pr[0][2], pr[0][3]), pack_pair<T>(pr[1][0], pr[1][1]),
                            pack_pair<T>(pr[1][2], pr[1][3])};
    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) { o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1]; }
    }
    auto add_values = [&](auto clear, const uint32_t keep0, const uint32_t keep1) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const uint32_t token = (lmat & 1) * 8 + lrow, c = 2 * j + (lmat >> 1);
        uint32_t vb[4];
        ldsm_trans(vbase + (c >> 3) * (kChunk * 128) + token * 128 + (((c & 7) ^ (token & 7)) << 4), vb);
        if constexpr (decltype(clear)::value) {
          vb[0] &= keep0; vb[1] &= keep1; vb[2] &= keep0; vb[3] &= keep1;
        }
        mma_pair<T>(o[2 * j], pa, vb[0], vb[1]);
        mma_pair<T>(o[2 * j + 1], pa, vb[2], vb[3]);
      }
    };
    if (whole) {
      add_values(std::false_type{}, 0u, 0u);
    } else {                                                     // values of keys that do not count may hold anything: cleared, so that 0 * value stays 0
      uint32_t keep[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = key0 + i * 8 + 2 * t4;
        keep[i] = (key >= from && key < len ? 0x0000ffffu : 0u) | (key + 1 >= from && key + 1 < len ? 0xffff0000u : 0u);
      }
      add_values(std::true_type{}, keep[0], keep[1]);
    }
    __syncwarp();                                                // the stage has been read
    const int ahead = it + kStages;
    if (ahead < mine) {
      if ((ahead & 31) == 0) {                                   // (its line and those behind it are the next round's)
        lines = lines_next;
        lines_next = line_of(ahead + 32 + lane);
      }
      copy(ahead, stage);
    }
    if (++stage == kStages) { stage = 0; phase ^= 1; }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
  }

  // ---------------- the warps' states in warp order ----------------
  __syncthreads();                                               // the rings are drained
  float* s_wm = reinterpret_cast<float*>(smem);                  // [warps][16] maxima, denominators
  float* s_wl = s_wm + WARPS * 16;
  float* s_wo = s_wl + WARPS * 16;                               // [warps][16][D]
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int h = g + r * 8;
    if (t4 == 0) { s_wm[warp * 16 + h] = m_run[r]; s_wl[warp * 16 + h] = l_run[r]; }
    if (h < heads) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(s_wo + (warp * 16 + h) * D + i * 8 + 2 * t4) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    }
  }
  __syncthreads();
  const size_t to = (static_cast<size_t>(p.parts.pieces + split) * a.batch + row) * a.heads + head0;
  for (int i = threadIdx.x; i < heads * (D / 4); i += kThreads) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < WARPS; ++k) m = fmaxf(m, s_wm[k * 16 + h]);
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float mk = s_wm[k * 16 + h], wgt = mk > -INFINITY ? ex2(mk - m) : 0.f;
      l = fmaf(s_wl[k * 16 + h], wgt, l);
      const float4 x = *reinterpret_cast<const float4*>(s_wo + (k * 16 + h) * D + d);
      v[0] = fmaf(x.x, wgt, v[0]); v[1] = fmaf(x.y, wgt, v[1]); v[2] = fmaf(x.z, wgt, v[2]); v[3] = fmaf(x.w, wgt, v[3]);
    }
    *reinterpret_cast<float4*>(p.parts.acc + (to + h) * D + d) = make_float4(v[0], v[1], v[2], v[3]);
    if (d == 0) *reinterpret_cast<float2*>(p.parts.ml + 2 * (to + h)) = make_float2(m, l);
  }
  if (p.common && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) chain_wait();
}

// ---------------------------------------------------------------------------------------------------------------------------------
// The pieces of a row, in order: its own keys' parts, then the common ones. A block per key/value head (and up to 16 of its query heads) and
// row; bound by latency: which pieces there are is known before the kernels that write them have ended (up to 32 groups), and the first
// outputs are asked for together with the maxima. (32 rows behind 2048 tokens: 2.1 us from the end of the kernel before to that of this one, 3.8
// with the plan read back, then the maxima, then the outputs.)
constexpr int kJoinThreads = 128;
constexpr int kSources = kMaxPieces + kMaxOwnParts;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
prefix_join_pieces_kernel(const __grid_constant__ OwnParams p) {
  __shared__ float s_w[16][kSources];
  __shared__ long long s_lens[kJoinThreads / 32];
  const cacheir_b200_prefix_args& a = p.a;
  const int kvh = blockIdx.x / p.head_chunks, row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.kv_heads, head0 = kvh * group + blockIdx.x % p.head_chunks * 16, heads = min(16, (kvh + 1) * group - head0);
  int pieces = 0;
  if (p.common) {
    // (the kernel before this one was let in after all earlier ones had ended, and so was this one: groups and lengths may be read ahead)
    RowGroup of = row_group(a, p.tile_rows, row);
    int ctas = 0;
    if (of.planned) {
      const long long mine = warp_sum64(lens_part(a, threadIdx.x, kJoinThreads));
      if (lane == 0) s_lens[warp] = mine;
      __syncthreads();
      long long lens = 0;
#pragma unroll
      for (int i = 0; i < kJoinThreads / 32; ++i) lens += s_lens[i];
      ctas = plan_ctas(a, p.parts.pieces, a.kv_heads * p.head_chunks, of.units, of.weights, lens, p.grid);
    }
    const int row_tiles = (of.in.rows + p.tile_rows - 1) / p.tile_rows, all = kItemUnits + key_tiles(of.in.prefix);
    const int rel = (kvh * row_tiles + (row - of.in.row) / p.tile_rows) * all;
    if (!of.planned) {
      chain_wait();
      if (of.group >= 0) {
        of.in.start = p.parts.plan->group[of.group].start;
        of.units = p.parts.plan->units;
        ctas = p.parts.plan->ctas;
      }
    }
    if (of.in.prefix > 0 && ctas > 0) {                          // (then the row is in a group that has items)
      const Deal deal(of.units, ctas);
      const int item0 = of.in.start + rel;
      pieces = min(max(deal.owner(item0 + all - 1) - deal.owner(item0 + kItemUnits) + 1, 0), p.parts.pieces);      // (as it is where groups ascend)
    }
  }
  chain_wait();
  chain_next();
  const size_t at0 = static_cast<size_t>(row) * a.heads + head0, step = static_cast<size_t>(a.batch) * a.heads;
  const int sources = p.splits + pieces;
  auto slot_of = [&](int k) { return k < p.splits ? p.parts.pieces + k : k - p.splits; };
  // A warp per head: the weight of every source.
  auto weigh = [&] {
    for (int h = warp; h < heads; h += kJoinThreads / 32) {
      float m = -INFINITY, l = 0.f, ms[3], ls[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {                              // (at most 72)
        const int k = i * 32 + lane;
        float2 x = make_float2(-INFINITY, 0.f);
        if (k < sources) x = *reinterpret_cast<const float2*>(p.parts.ml + 2 * (slot_of(k) * step + at0 + h));
        ms[i] = x.x;
        ls[i] = x.y;
        m = fmaxf(m, ms[i]);
      }
      m = warp_max(m);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        ms[i] = ms[i] > -INFINITY ? ex2(ms[i] - m) : 0.f;
        l += ls[i] * ms[i];
      }
      l = warp_sum(l);
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i * 32 + lane < sources) s_w[h][i * 32 + lane] = ms[i] * inv;
    }
    __syncthreads();
  };
  // Four neighbouring outputs are a place; ITEMS places of a thread and DEEP pieces of each are on their way at once. A piece without weight
  // does not count: a row that ends before it has zeros there, times values that may be no numbers.
  const int places = heads * (D / 4);
  const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 7) == 0 && a.out_stride % 4 == 0;
  auto finish = [&](auto items, auto deep) {
    constexpr int ITEMS = decltype(items)::value, DEEP = decltype(deep)::value;
    for (int first = 0; first < places; first += ITEMS * kJoinThreads) {
      float v[ITEMS][4];
      const float* acc[ITEMS];
      const float* wgt[ITEMS];
      bool live[ITEMS];
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) {
        const int at = first + threadIdx.x + j * kJoinThreads;
        live[j] = at < places;
        const int i = live[j] ? at : 0, h = i / (D / 4), d = i % (D / 4) * 4;
        acc[j] = p.parts.acc + (at0 + h) * D + d;
        wgt[j] = s_w[h];
        v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.f;
      }
      float4 x[DEEP][ITEMS];
      auto load = [&](int k) {
#pragma unroll
        for (int e = 0; e < DEEP; ++e)
#pragma unroll
          for (int j = 0; j < ITEMS; ++j)
            x[e][j] = live[j] && k + e < sources ? *reinterpret_cast<const float4*>(acc[j] + slot_of(k + e) * step * D) : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      load(0);
      if (first == 0) weigh();
#pragma unroll 1
      for (int k = 0; k < sources; k += DEEP) {
        if (k > 0) load(k);
#pragma unroll
        for (int e = 0; e < DEEP; ++e)
#pragma unroll
          for (int j = 0; j < ITEMS; ++j) {
            const float f = k + e < sources ? wgt[j][k + e] : 0.f;
            if (f != 0.f) {
              v[j][0] = fmaf(x[e][j].x, f, v[j][0]); v[j][1] = fmaf(x[e][j].y, f, v[j][1]);
              v[j][2] = fmaf(x[e][j].z, f, v[j][2]); v[j][3] = fmaf(x[e][j].w, f, v[j][3]);
            }
          }
      }
#pragma unroll
      for (int j = 0; j < ITEMS; ++j)
        if (live[j]) {
          const int i = first + threadIdx.x + j * kJoinThreads, h = i / (D / 4), d = i % (D / 4) * 4;
          T* out = static_cast<T*>(a.out) + static_cast<size_t>(row) * a.out_stride + static_cast<size_t>(head0 + h) * D + d;
          if (wide) *reinterpret_cast<uint2*>(out) = make_uint2(pack_pair<T>(v[j][0], v[j][1]), pack_pair<T>(v[j][2], v[j][3]));
          else
#pragma unroll
            for (int e = 0; e < 4; ++e) Elem<T>::st(out + e, v[j][e]);
        }
    }
  };
  if (places <= kJoinThreads) finish(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  else finish(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
}

template <typename T, int D, int WARPS>
int launch_own(const OwnParams& o, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t stream) {
  auto kern = prefix_own_kernel<T, D, WARPS>;
  constexpr int bytes = OwnSmem<D, WARPS>::kBytes;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_shared_memory(done, reinterpret_cast<const void*>(kern), bytes);
  if (e == cudaSuccess)
    e = launch_chained(kern, dim3(o.splits, o.a.kv_heads * o.head_chunks, o.a.batch), dim3(WARPS * 32), bytes, stream, tk, tv, o);
  if (e == cudaSuccess)
    e = launch_chained(prefix_join_pieces_kernel<T, D>, dim3(o.a.kv_heads * o.head_chunks, o.a.batch), dim3(kJoinThreads), 0, stream, o);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

// Units of all items, at most.
long long most_units(const cacheir_b200_prefix_args& a, int tile_rows) {
  const long long tiles = (static_cast<long long>(a.prefix_pages) * a.page_size + kKeys - 1) / kKeys;
  return (kItemUnits + tiles) * a.kv_heads * (a.batch / tile_rows + a.groups);
}
// Batch rows of an item: as many as two groups of warps have rows for.
int rows_of_tile(const cacheir_b200_prefix_args& a) { return 2 * (kRows / (a.heads / a.kv_heads)); }

template <typename T, int D>
int launch_fast(const cacheir_b200_prefix_args& a, const PrefixParts& parts, cudaStream_t stream) {
  CUtensorMap tk, tv, tk_half, tq;
  const uint64_t rows = static_cast<uint64_t>(a.num_slots) * a.kv_heads * a.page_size;
  if (!encode_pool<T>(&tk, a.k_cache, rows, D, true) || !encode_pool<T>(&tv, a.v_cache, rows, D, true) ||
      (a.groups > 0 && (!encode_pool<T>(&tk_half, a.k_cache, rows, D, false) || !encode_queries<T>(&tq, a.q, a.batch, a.heads, a.kv_heads, D, a.q_stride, rows_of_tile(a) / 2))))
    return CACHEIR_B200_EUNSUPPORTED;
  const int group = a.heads / a.kv_heads, tile_rows = rows_of_tile(a);
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const long long most = most_units(a, tile_rows);
  const int grid = static_cast<int>(most < kNumSMs ? most : kNumSMs);
  if (a.groups > 0) {
    const CommonParams c{a, parts, a.groups > kPlanGroups ? 1 : 0, tile_rows, a.kv_heads * ((group + 15) / 16), scale_log2};
    cudaError_t e = cudaSuccess;
    if (c.plan_ready) e = launch_chained(prefix_plan_kernel, dim3(1), dim3(1024), 0, stream, c, grid);
    auto kern = prefix_common_kernel<T, D>;
    static std::atomic<unsigned long long> done{0};
    if (e == cudaSuccess) e = allow_shared_memory(done, reinterpret_cast<const void*>(kern), CommonSmem<D>::kBytes);
    if (e == cudaSuccess) e = launch_chained(kern, dim3(grid), dim3(kCommonThreads), CommonSmem<D>::kBytes, stream, tk_half, tv, tq, c);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  OwnParams o{a, parts, a.groups > 0 ? 1 : 0, tile_rows, (group + 15) / 16, 1, grid, scale_log2};
  const long long blocks = static_cast<long long>(a.batch) * a.kv_heads * o.head_chunks;
  // (Device times: 64 rows behind a document, 512 blocks: 51.2 us with two warps, 52.5 with four; 32 rows behind instructions, 256 blocks: 20.1
  // with four, 23.5 with two, 23.1 with eight, which have rings of three stages and so an SM for themselves; 2 rows of 16000 own tokens, 16 blocks
  // in eight parts: 26.9 with eight, 28.2 with four)
  if (blocks > 3 * kNumSMs) return launch_own<T, D, 2>(o, tk, tv, stream);
  if (blocks > kNumSMs) return launch_own<T, D, 4>(o, tk, tv, stream);
  // Parts of a row's own keys while there are SMs for them, but no more than there are chunks to share.
  const long long chunks = static_cast<long long>(a.max_pages) * a.page_size / kChunk;
  while (2 * o.splits <= parts.own && 2 * o.splits * blocks <= kNumSMs && 2 * o.splits * 8 <= chunks) o.splits *= 2;
  return launch_own<T, D, 8>(o, tk, tv, stream);
}

}  // namespace

bool prefix_fast_supported(const cacheir_b200_prefix_args& a) {
  const int group = a.heads / a.kv_heads;
  return (a.dtype == CACHEIR_B200_F16 || a.dtype == CACHEIR_B200_BF16) && (a.dim == 64 || a.dim == 128) && a.page_size % kChunk == 0 &&
         group <= kMaxHeadsPerKv && aligned_to(a.q, 16) && a.q_stride % 8 == 0 && aligned_to(a.k_cache, 16) && aligned_to(a.v_cache, 16) &&
         static_cast<long long>(a.num_slots) * a.kv_heads * a.page_size <= 0x7fffffffLL - kChunk &&
         static_cast<long long>(a.kv_heads) * ((group + 15) / 16) <= 65535 && most_units(a, rows_of_tile(a)) <= 0x7fffffffLL;
}

int prefix_fast_launches(int groups) { return groups > kPlanGroups ? 4 : groups > 0 ? 3 : 2; }

int launch_prefix_fast(const cacheir_b200_prefix_args& a, const PrefixParts& parts, cudaStream_t stream) {
  if (a.dtype == CACHEIR_B200_F16) return a.dim == 128 ? launch_fast<__half, 128>(a, parts, stream) : launch_fast<__half, 64>(a, parts, stream);
  return a.dim == 128 ? launch_fast<__nv_bfloat16, 128>(a, parts, stream) : launch_fast<__nv_bfloat16, 64>(a, parts, stream);
}

int prefix_device_status(bool reset) { return device_status_word(g_prefix_status, reset); }

}  // namespace cb200
