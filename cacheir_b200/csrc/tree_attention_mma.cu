// Attention of drafted tokens over their sequence's pages on the tensor cores: 16-bit types, head sizes 64 and 128, pages of a multiple of 16
// tokens, up to 64 query heads per key/value head.
//
// S = Q K^T and O = P V as tcgen05 MMAs of 128 query rows, which are the (token, head) pairs of a sequence that share a key/value head; scores,
// probabilities and outputs in tensor memory. An item is (sequence, up to 256 query rows, key/value head); its keys come in tiles of 128, from
// the sequence's first token to the last that one of its rows can see, so that a sequence's keys are read once for all rows of an item. The key tiles of all items, in a row, are cut
// evenly over the blocks, whatever the lengths. An item that one block has alone is written as it ends; of others every block leaves a piece, and a second kernel joins them.
//
// One warp brings keys and one values (TMA, 16 tokens at a time, into a ring of slots), one issues the MMAs, and two groups of four warps do the
// softmax, a thread per query row, each with scores, probabilities and an output of its own in tensor memory. Above 128 query rows each group
// has its own 128 of them and both use the same keys. With fewer, which is what decoding with drafts has mostly, both have the same
// rows and take turns with the key tiles: what bounds such an item is the memory's rate, and one group alone would not keep up with it. The two halves are added up
// from tensor memory at the item's end, by the group that had its first tile, while the other one is at work on the next item.
//
// Masks are looked at only in tiles that hold drafted tokens: 128 bits a row, shifted to the tile. Whatever stands in a key that a row does not
// see, its weight is 0; but 0 times a value that is no number is none. So one more warp looks through the drafted tokens' values before the second product has them, puts
// zeros for infinities and NaN, and says that it did; rows that see such a value get it added at the end, by their warp.
//
// A row's maximum is a reference that moves only when it is exceeded by 2^14, so that outputs are hardly ever rescaled; probabilities are rounded to
// the element type as the second MMA's operand, their sums are not (errors against 64 bits 1.2 to 1.45 times those of probabilities in 32 bits).
//
// Measured (both kernels, replayed from a graph; 32 query and 8 key/value heads of 128 in fp16 where nothing else is said): 32 trees of 12 to 16 tokens behind 256 to
// 4096 75 us, of which 47 us are the bytes; 4 chains of up to 5 tokens behind 90000 to 131072 315 to 330 us (bytes 263); 16 trees of 40 to 64 tokens behind 1000 to
// 8192, 64 heads, bf16, 195 to 200 us called on end, 182 in short bursts (products 80, at the rate of those); two trees of 8 tokens behind 300 10.9 us. In the main loop an item of one group's
// rows takes 1.5 us a tile, which is the memory's rate; one of two groups' rows 1.8 us, 3300 cycles, of which the tensor cores work 2048: probabilities lie over the scores that they come from,
// so that a group's scores, softmax (1024 cycles of exponentials alone) and second product follow one another, and only the other group's fill the gaps. First scores come
// 4 to 7 us after the launch, an item's end takes 1.5 to 3 us, the pieces 5. Scores of 64 keys at a time, in two places a group, would close the gaps,
// but the tensor cores take as long for 64 keys as for 128 (the queries are read again): 84, 372 and 216 us for the first three.
#include "attention_ptx.cuh"
#include "hybrid_common.cuh"
#include "tree_attention.cuh"

namespace cb200 {
namespace {

using namespace ptx;

constexpr int kKeys = 128;                     // keys of a tile
constexpr int kFirst = 96;                     // .. whose probabilities go to the second MMA first: less of it is left when the others come
constexpr int kRows = 128;                     // query rows of a group of warps
constexpr int kThreads = 384;
constexpr int kMaxHeadsPerKv = 64;
// Tokens that tables have room for, in tiles, up to which items are not cut: joining their pieces takes longer than a block takes for all of them (67 sequences of up to 502
// tokens 52 us, cut 57; 3 of up to 897 with one key/value head 13.2, cut 15.7).
constexpr int kWholeTiles = 8;
constexpr int kPlanThreads = 128;              // that lay the plan out, some sequences each
constexpr float kAhead = 6.f;                  // a new reference is the maximum less this: probabilities start at 2^6 ..
constexpr float kStale = 14.f;                 // .. and may grow to 2^14 (in fp16: 2^-24 of that is still a number)

__device__ int g_tree_status = 0;

// What a block that ends an item which others began leaves for the kernel that joins (rows 0: nothing).
struct TreeJoin {
  int row, rows, kvh, first;                   // first row and number of rows; the blocks from `first` to this one have a piece each
};
struct FastParams {
  cacheir_b200_tree_args a;
  TreeJoin* joins;                             // [blocks]
  float* ml;                                   // [blocks][2 pieces][2 groups][128][2]: maxima (log2 domain) and denominators
  float* acc;                                  // [blocks][2 pieces][2 groups][dim / 4][128][4]: unnormalised outputs, rows side by side as the lanes are that have them
  int half_rows;                               // tokens of a group of warps
  int whole;                                   // items are not cut
  int out_wide;                                // rows of out begin at 32 bytes
  float scale_log2;
};

// A warp's wait; false in all lanes where it gave up in one.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, &g_tree_status, code));
}
__device__ __forceinline__ void store_32_bytes(void* to, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
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

// ---- how the work is cut ----
// An item of n key tiles is kItemUnits + n kTileUnits units (kTwoUnits where two groups of warps have rows of their own, whose tiles take the longer the less
// the memory is waited for): what it costs to begin with (queries, the first tile's latency, the output) is about that of three tiles. The units are dealt out
// as evenly as whole numbers can be; a block has the tiles whose first unit is its own. Where items are not cut, each is a unit. (32 trees and 16 wide ones: 6, 2, 3 units
// 75.9 and 186 us; 4, 2, 3 75.0 and 193; 2, 2, 3 75.0 and 200; 4, 2, 4 75.0 and 221; 3, 2, 2 74.6 and 190.)
constexpr int kItemUnits = 6;
constexpr int kTileUnits = 2;
constexpr int kTwoUnits = 3;

struct Deal {
  int share, more;             // every block has `share` units, the first `more` one more
  __device__ __forceinline__ Deal(int units, int ctas) : share(units / ctas), more(units % ctas) {}
  __device__ __forceinline__ int begin(int block) const { return block * share + min(block, more); }
  __device__ __forceinline__ int owner(int unit) const {
    const int big = more * (share + 1);
    return unit < big ? unit / (share + 1) : more + (unit - big) / share;
  }
};
// Keys that rows below `end` of a sequence can see (with a mask any of its tokens), and the units of such an item.
__device__ __forceinline__ int item_keys(const cacheir_b200_tree_args& a, const TreeSequence& s, int end) {
  return a.visible ? s.keys : max(min(s.keys, s.front + min(end, s.rows)), 0);
}
__device__ __forceinline__ int item_tiles(int keys) { return max((keys + kKeys - 1) / kKeys, 1); }
struct Cost {
  int tile_rows, whole;
  // the units of a tile, and of an item, of so many rows
  __device__ __forceinline__ int tile(int rows) const { return 2 * rows > tile_rows ? kTwoUnits : kTileUnits; }
  __device__ __forceinline__ int item(int rows, int keys) const { return whole ? 1 : kItemUnits + item_tiles(keys) * tile(rows); }
};
// Of a sequence, for one key/value head after the other in every tile of rows.
__device__ __forceinline__ int sequence_units(const cacheir_b200_tree_args& a, const TreeSequence& s, const Cost& cost) {
  const int tiles = (s.rows + cost.tile_rows - 1) / cost.tile_rows;
  if (tiles == 0) return 0;
  int units = 0;
  if (a.visible) units = (tiles - 1) * cost.item(cost.tile_rows, s.keys);
  else for (int j = 1; j < tiles; ++j) units += cost.item(cost.tile_rows, item_keys(a, s, j * cost.tile_rows));
  return a.kv_heads * (units + cost.item(s.rows - (tiles - 1) * cost.tile_rows, s.keys));
}

// A block's share of the units, item by item.
struct Walk {
  const cacheir_b200_tree_args& a;
  Cost cost;
  Deal deal;
  int at, end;
  int b, start;                // the sequence, and the first unit of its row tile
  TreeSequence s;
  int row0, rows, keys, units; // .. the row tile: rows from row0 of the sequence on, what they see, and the units of an item in it
  // the item
  int kvh, tile, tiles, first; // key tiles tile .. tile + tiles - 1 of it are this block's; block `first` has its first one
  bool begins, ends;

  __device__ __forceinline__ void row_tile(int from) {
    row0 = from;
    rows = min(cost.tile_rows, s.rows - row0);
    keys = item_keys(a, s, row0 + rows);
    units = cost.item(rows, keys);
  }
  // starts: the first units of runs of `run` sequences
  __device__ __forceinline__ Walk(const cacheir_b200_tree_args& args, const Cost& c, const int* starts, int run, int total, int ctas) : a(args), cost(c), deal(total, ctas) {
    at = deal.begin(blockIdx.x);
    end = deal.begin(blockIdx.x + 1);
    int lo = 0, hi = kPlanThreads;                             // last run that starts at or before `at` (empty ones start where the next does)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= at) lo = mid; else hi = mid;
    }
    b = min(lo * run, a.sequences - 1);
    start = starts[lo];
    s = tree_sequence(a, b);
    row_tile(0);
  }
  __device__ __forceinline__ bool next() {
    while (at < end) {
      while (rows <= 0 || start + a.kv_heads * units <= at) {  // to the row tile that `at` is in
        if (rows > 0) start += a.kv_heads * units;
        if (rows > 0 && row0 + rows < s.rows) {
          row_tile(row0 + rows);
        } else {
          if (++b >= a.sequences) return false;
          s = tree_sequence(a, b);
          row_tile(0);
        }
      }
      kvh = (at - start) / units;
      const int item0 = start + kvh * units, stop = min(end, item0 + units), all = item_tiles(keys);
      const int each = cost.tile(rows), tile0 = item0 + kItemUnits;
      auto behind = [&](int unit) { return cost.whole ? (unit > item0 ? all : 0) : min((max(unit - tile0, 0) + each - 1) / each, all); };      // tiles that begin before a unit
      tile = behind(at);
      tiles = behind(stop) - tile;
      begins = tile == 0;
      ends = tile + tiles == all;
      at = stop;
      if (tiles <= 0) continue;                                // (no tile begins here)
      first = begins ? static_cast<int>(blockIdx.x) : deal.owner(tile0);
      return true;
    }
    return false;
  }
};

// What the warps other than the keys' need to know of an item.
struct Item {
  TreeSequence s;
  int b, row0, rows, kvh;
  int tile, tiles, keys;       // (tiles 0: there are no more items)
  int flags;                   // 1: begins here, 2: ends here
};

template <int D>
struct Smem {
  static constexpr int kSlotBytes = kKeys * D * 2;
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int kQBytes = kRows * D * 2;
  // Items in shared memory. The keys' warp, which goes through them, is no more tiles ahead of the outputs than there are slots (where their number is even, of the
  // scores, which are two steps ahead of the outputs), but a group of warps may be any number of items behind these: those of one tile that follow may all be the other group's. So
  // both groups say when they are done with a place; whoever else reads it has done so by then, as no group ends an item before its outputs are there.
  static constexpr int kItems = D == 128 ? 8 : 16;
  static constexpr int kTiles = 2 * kQBytes + kSlots * kSlotBytes;
  // then: barriers of keys, of values, empty, clean [slots], q[2], place of q[2], s[2], p[2][2], o[2], given[2], taken[2], items, places of items;
  // tensor memory address; items; starts of runs, and later
  // maxima and denominators that one group of warps hands to the other
  static constexpr int kBarriers = 4 * kSlots + 16 + 2 * kItems;
  static constexpr int kBytes = 1024 + kTiles + kBarriers * 8 + 16 + kItems * static_cast<int>(sizeof(Item)) + kRows * 8;
};

// What the rows of a warp's lanes get of values that are no numbers, of the tokens that they see in the tiles from `tile` on, added to the places
// `to`, which the lanes have written: rows of out, or with floats of the scratch, whose columns lie in fours, 128 of them apart. The whole warp calls it; lanes whose row
// is not there, or is NaN already, do not take part. The lanes look through 32 tokens at a time, then have some columns each of every token found, and a bit per row of
// what comes to a column: infinity, its negative, or both, which is NaN (a chain of 6000 rows with one infinite value, two key/value heads of 128: 0.51 ms, 0.24 without it, 26
// with lanes that each go through all tokens).
template <typename T, int D, typename O>
__device__ __noinline__ void add_spoilt(const cacheir_b200_tree_args& a, const TreeSequence s, const int32_t* pages, int row, int head, bool takes, int tile, int tiles,
                                        int keys, O* to) {
  constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr int kOwn = D / 32;                                 // columns of a lane
  const int lane = threadIdx.x & 31, kvh = head / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(s.row + row) * a.q_stride + static_cast<size_t>(head) * D;
  const T* k_pool = static_cast<const T*>(a.k_cache);
  const T* v_pool = static_cast<const T*>(a.v_cache);
  float largest = 0.f;
  for (int d = 0; d < D; ++d) largest = fmaxf(largest, fabsf(Elem<T>::ld(q + d)));
  uint32_t plus[kOwn] = {}, minus[kOwn] = {};
  const int end = min((tile + tiles) * kKeys, keys);
  for (int t0 = max(tile * kKeys, max(s.front, 0)); t0 < end; t0 += 32) {
    const int t = t0 + lane, id = t < end ? pages[t / a.page_size] : -1;
    long long at = 0;
    uint32_t bad = 0;
    if (id >= 0 && id < a.num_slots) {
      at = ((static_cast<long long>(id) * a.kv_heads + kvh) * a.page_size + t % a.page_size) * D;
#pragma unroll
      for (int i = 0; i < D; i += 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(v_pool + at + i);
        bad |= __vcmpeq2(v.x & kExponent, kExponent) | __vcmpeq2(v.y & kExponent, kExponent) | __vcmpeq2(v.z & kExponent, kExponent) | __vcmpeq2(v.w & kExponent, kExponent);
      }
    }
    for (uint32_t found = __ballot_sync(0xffffffffu, bad != 0); found; found &= found - 1) {
      const int from = __ffs(found) - 1, j = t0 + from - s.front;
      const long long line = __shfl_sync(0xffffffffu, at, from);
      const T* k = k_pool + line;
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) most = fmaxf(most, fabsf(Elem<T>::ld(k + lane * kOwn + i)));
      most = warp_max(most);
      bool counts = takes && (tree_word(a, s, row, j >> 5) >> (j & 31) & 1);
      if (counts && !(most * largest < 1e38f / D)) {           // a score of -inf has no weight
        float score = 0.f;
        for (int d = 0; d < D; ++d) score = fmaf(Elem<T>::ld(q + d), Elem<T>::ld(k + d), score);
        counts = score != -INFINITY;
      }
      const uint32_t rows = __ballot_sync(0xffffffffu, counts);
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const float x = Elem<T>::ld(v_pool + line + lane * kOwn + i);
        if (isfinite(x)) continue;
        if (!(x < 0.f)) plus[i] |= rows;
        if (!(x > 0.f)) minus[i] |= rows;
      }
    }
  }
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) any |= plus[i] | minus[i];
  __syncwarp();                                                // (other lanes' rows are there)
  for (any = __reduce_or_sync(0xffffffffu, any); any; any &= any - 1) {
    const int r = __ffs(any) - 1;
    O* const line = reinterpret_cast<O*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), r));
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int c = lane * kOwn + i;
      const bool up = plus[i] >> r & 1, down = minus[i] >> r & 1;
      O* const x = line + (std::is_same<O, float>::value ? (c >> 2) * (kRows * 4) + (c & 3) : c);
      if (up || down) Elem<O>::st(x, Elem<O>::ld(x) + (up ? down ? NAN : INFINITY : -INFINITY));
    }
  }
}

template <typename T, int D, bool RUN_ON>
__global__ void __launch_bounds__(kThreads, 1)
tree_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_q,
            const __grid_constant__ FastParams p) {
  using L = Smem<D>;
  constexpr int kSlots = L::kSlots, kItems = L::kItems;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;                                         // [2][D / 64][128 rows][128 B]
  uint8_t* s_kv = smem + 2 * L::kQBytes;                       // [slots][D / 64][128 keys][128 B]
  // Keys and values take the slots in turn: those of the block's tile u are in slots 2 u and 2 u + 1 modulo their number. Their barriers go by u, so that
  // whoever looks at one kind only never meets a phase of the other.
  uint64_t* key_full = reinterpret_cast<uint64_t*>(smem + L::kTiles);
  uint64_t* value_full = key_full + kSlots;
  uint64_t* empty = value_full + kSlots;                       // (by slot)
  uint64_t* bar_clean = empty + kSlots;                        // values have been looked through
  uint64_t* bar_q = bar_clean + kSlots;                        // queries of a group of warps are there
  uint64_t* bar_free = bar_q + 2;                              // .. and their place is free again
  uint64_t* bar_s = bar_free + 2;                              // scores are in tensor memory
  uint64_t* bar_p = bar_s + 2;                                 // probabilities are, [group of warps][first keys, the others]
  uint64_t* bar_o = bar_p + 4;                                 // .. and have been added to the output
  uint64_t* bar_given = bar_o + 2;                             // a group's part of an item is done
  uint64_t* bar_taken = bar_given + 2;                         // .. and has been added to the other one's
  uint64_t* bar_item = bar_taken + 2;                            // the item is known
  uint64_t* bar_done = bar_item + kItems;                      // .. and both groups of warps are done with it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + kItems);
  Item* s_item = reinterpret_cast<Item*>(tmem_slot + 4);
  int* s_start = reinterpret_cast<int*>(s_item + kItems);
  float2* s_ml = reinterpret_cast<float2*>(s_start);           // (when the first item ends the keys' warp has long found its share)
  static_assert(kPlanThreads * 4 <= kRows * 8, "starts and maxima share their place");
  __shared__ int s_scan[kPlanThreads / 32];
  __shared__ volatile int s_spoilt[kItems];                    // the last item of this place some of whose values are no numbers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const cacheir_b200_tree_args& a = p.a;

  if (threadIdx.x == 288) {
    prefetch_map(&tmap_q);
    prefetch_map(&tmap_k);
    prefetch_map(&tmap_v);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(smem_u32(&key_full[s]), 1);
      mbar_init(smem_u32(&value_full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
      mbar_init(smem_u32(&bar_clean[s]), 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&bar_q[w]), 1);
      mbar_init(smem_u32(&bar_free[w]), 1);
      mbar_init(smem_u32(&bar_s[w]), 1);
      mbar_init(smem_u32(&bar_p[2 * w]), kRows);
      mbar_init(smem_u32(&bar_p[2 * w + 1]), kRows);
      mbar_init(smem_u32(&bar_o[w]), 1);
      mbar_init(smem_u32(&bar_given[w]), 4);
      mbar_init(smem_u32(&bar_taken[w]), 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(smem_u32(&bar_item[i]), 1);
      mbar_init(smem_u32(&bar_done[i]), 2 * kRows / 32);
    }
    mbar_fence_init();
  }
  if (threadIdx.x >= 256 && threadIdx.x < 256 + kItems) s_spoilt[threadIdx.x - 256] = 0;
  chain_enter();
  if (warp == 8) tc_alloc(smem_u32(tmem_slot), 512);           // (beside the loads of the plan)
  // ---- the plan: units of runs of sequences, a thread each ----
  const Cost cost{2 * p.half_rows, p.whole};
  const int run = (a.sequences + kPlanThreads - 1) / kPlanThreads;
  int sum = 0, own = 0;
  if (threadIdx.x < kPlanThreads) {
    for (int b = threadIdx.x * run; b < min(static_cast<int>(threadIdx.x + 1) * run, a.sequences); ++b) own += sequence_units(a, tree_sequence(a, b), cost);
    sum = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += up;
    }
    if (lane == 31) s_scan[warp] = sum;
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 32; ++i) {
    if (i < warp) sum += s_scan[i];
    total += s_scan[i];
  }
  if (threadIdx.x < kPlanThreads) s_start[threadIdx.x] = sum - own;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;                            // scores [2][128 columns] (probabilities over them), outputs [2][D]
  const uint32_t tmem_o = tmem + 2 * kKeys;
  const int group = a.heads / a.kv_heads, half_rows = p.half_rows;
  // (no block between those of an item's first and last tile is without one)
  const int ctas = max(1, min(p.whole ? total : total / kTwoUnits, static_cast<int>(gridDim.x)));
  bool ok = true;
  Item it;
  int item = 0;                                                // of the block, counted from 1
  auto next_item = [&] {
    const int place = item % kItems;
    ok = ok && warp_wait(smem_u32(&bar_item[place]), (item / kItems) & 1, (17 << 8) | 14);
    if (!ok) return false;
    it = s_item[place];
    ++item;
    return it.tiles > 0;
  };

  if (warp == 11) {
    // ------- values: those of drafted tokens are looked through, those behind the last key cleared -------
    constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr int kLanes = D / 8;                              // of a key's values
    int slot = 1, turn = 0;
    uint32_t phase = 0;
    while (next_item()) {
      for (int t = it.tile; t < it.tile + it.tiles && ok; ++t) {
        ok = warp_wait(smem_u32(&value_full[turn]), phase, (17 << 8) | 12);
        if (!ok) break;
        // (behind the 16 keys in which the last one lies there are zeros already)
        const int base = t * kKeys, from = max(min(it.s.front, it.keys) - base, 0), until = min((it.keys - base + kChunk - 1) / kChunk * kChunk, kKeys);
        if (from < until) {
          bool spoilt = false;
          constexpr int kAtOnce = 2;                           // 16-byte words of a lane under way
          for (int first = from + lane / kLanes; first < until; first += kAtOnce * (32 / kLanes)) {
            const int c = lane % kLanes;
            auto word = [&](int key) {
              return reinterpret_cast<uint4*>(s_kv + slot * L::kSlotBytes + (key / kChunk) * kChunk * D * 2 + (c >> 3) * kChunk * 128 + key % kChunk * 128 + ((c & 7) << 4));
            };
            uint4 v[kAtOnce];
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) v[e] = *word(min(first + e * (32 / kLanes), until - 1));
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
              const int key = first + e * (32 / kLanes);
              const uint32_t bad[4] = {__vcmpeq2(v[e].x & kExponent, kExponent), __vcmpeq2(v[e].y & kExponent, kExponent), __vcmpeq2(v[e].z & kExponent, kExponent),
                                       __vcmpeq2(v[e].w & kExponent, kExponent)};
              const bool behind = base + key >= it.keys;       // (nobody sees it)
              if (key < until && (behind || (bad[0] | bad[1] | bad[2] | bad[3]))) {
                spoilt = spoilt || !behind;
                *word(key) = behind ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(v[e].x & ~bad[0], v[e].y & ~bad[1], v[e].z & ~bad[2], v[e].w & ~bad[3]);
              }
            }
          }
          if (__any_sync(0xffffffffu, spoilt) && lane == 0) s_spoilt[(item - 1) % kItems] = item;
          fence_async_smem();
          __threadfence_block();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_clean[turn]));
        slot += 2;
        if (slot >= kSlots) slot -= kSlots;
        if (++turn == kSlots) { turn = 0; phase ^= 1; }
      }
    }
  } else if (warp >= 9) {
    // ------- copies: warp 9 keys, a lane per 16 of them and 64 columns; warp 10 values, a lane per 16 of them -------
    const bool keys = warp == 9;
    const int boxes = keys ? D / 64 : 1, chunk = lane / boxes, box = lane % boxes;
    const bool copies = chunk < kKeys / kChunk;
    const int outside = a.num_slots * a.kv_heads * a.page_size;         // rows behind the pool read as zeros
    const uint32_t dst = smem_u32(s_kv) + (keys ? box * kKeys * 128 + chunk * kChunk * 128 : chunk * kChunk * D * 2);
    const Division by_page(a.page_size);
    uint64_t* full = keys ? key_full : value_full;
    int slot = keys ? 0 : 1, turn = 0, q_place = 0;
    uint32_t phase = 1, sent = 0, q_phase = 3;                 // (slots of a tile: its keys', its values'; q_phase: a bit for either place)
    auto line_of = [&](int tile) {                             // first row of this lane's 16 in the pool
      const int key = tile * kKeys + chunk * kChunk;
      if (!copies || key >= it.keys) return outside;
      const int page = by_page.of(key), id = a.page_table[static_cast<size_t>(it.b) * a.max_pages + page];
      return id >= 0 && id < a.num_slots ? (id * a.kv_heads + it.kvh) * a.page_size + key - page * a.page_size : outside;
    };
    auto copy_tiles = [&](int line) {
      for (int t = it.tile; t < it.tile + it.tiles && ok; ++t) {
        const int next = t + 1 < it.tile + it.tiles ? line_of(t + 1) : 0;
        ok = warp_wait(smem_u32(&empty[slot]), phase, (17 << 8) | 1);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(smem_u32(&full[turn]), L::kSlotBytes);
        __syncwarp();
        if (copies) {
          if (keys) tma_load_3d(dst + slot * L::kSlotBytes, &tmap_k, smem_u32(&full[turn]), 0, line, box);
          else tma_load_3d(dst + slot * L::kSlotBytes, &tmap_v, smem_u32(&full[turn]), 0, line, 0);
        }
        ++sent;
        slot += 2;
        if (slot >= kSlots) { slot -= kSlots; phase ^= 1; }
        turn = turn + 1 == kSlots ? 0 : turn + 1;
        line = next;
      }
    };
    if (keys) {                                                // this warp goes through the block's share and says what the items are
      Walk walk(a, cost, s_start, run, max(total, 1), ctas);
      if (static_cast<int>(blockIdx.x) >= min(ctas, total)) walk.end = walk.at;
      TreeJoin join{};
      bool more = true;
      while (ok && more) {
        more = walk.next();
        ok = warp_wait(smem_u32(&bar_done[item % kItems]), ((item / kItems) & 1) ^ 1, (17 << 8) | 15);
        if (!ok) break;
        it = Item{walk.s, walk.b, walk.row0, walk.rows, walk.kvh, walk.tile, more ? walk.tiles : 0, walk.keys, (walk.begins ? 1 : 0) | (walk.ends ? 2 : 0)};
        if (lane == 0) {
          s_item[item % kItems] = it;
          mbar_arrive(smem_u32(&bar_item[item % kItems]));
        }
        ++item;
        if (!more) break;
        if (walk.ends && !walk.begins) join = TreeJoin{walk.s.row + walk.row0, walk.rows, walk.kvh, walk.first};
        copy_tiles(line_of(it.tile));
      }
      if (lane == 0) p.joins[blockIdx.x] = join;
    } else {
      while (next_item()) {
        const int line = line_of(it.tile);
        const bool two = it.rows > half_rows;                  // the item's queries: rows, heads, 64 columns at a time
        for (int w = 0; w < (two ? 2 : 1) && ok; ++w) {
          const int place = two ? w : q_place;
          ok = warp_wait(smem_u32(&bar_free[place]), q_phase >> place & 1, (17 << 8) | 7);
          if (!ok) break;
          q_phase ^= 1u << place;
          if (lane == 0) {
            mbar_expect_tx(smem_u32(&bar_q[place]), (D / 64) * half_rows * group * 128);
            for (int z = 0; z < D / 64; ++z)
              tma_load_4d(smem_u32(s_q + place * L::kQBytes + z * kRows * 128), &tmap_q, smem_u32(&bar_q[place]), 0, it.kvh * group,
                          it.s.row + it.row0 + w * half_rows, z);
          }
          __syncwarp();
        }
        if (!two) q_place ^= 1;
        copy_tiles(line);
      }
    }
    // nothing may still be on its way when the block ends, also after a wait that gave up
    for (uint32_t i = sent > kSlots ? sent - kSlots : 0; i < sent; ++i)
      mbar_wait(smem_u32(&full[i % kSlots]), (i / kSlots) & 1, &g_tree_status, (17 << 8) | 2);
    // (queries are waited for by the products; after a wait that gave up: both phases of both places)
    if (!keys && !ok)
      for (int w = 0; w < 4; ++w) mbar_wait(smem_u32(&bar_q[w >> 1]), w & 1, &g_tree_status, (17 << 8) | 2);
  } else if (warp == 8) {
    // ---------------- MMA issue ----------------
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
    const uint32_t id_s = (1u << 4) | (kType << 7) | (kType << 10) | (static_cast<uint32_t>(kKeys >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
    const uint32_t id_o = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) |
                          (static_cast<uint32_t>(kRows >> 4) << 24);
    const uint64_t dq = smem_desc_sw128(smem_u32(s_q)), dk = smem_desc_sw128(smem_u32(s_kv)), dv = smem_desc_columns(smem_u32(s_kv));
    // An item's steps: a tile each, or a tile for either half of the rows. They go to the two groups of warps in turn; scores are two steps ahead of outputs, and are
    // issued right behind the output that frees their place. RUN_ON: both also across the end of an item, so that items of one tile keep both groups at work.
    const bool leader = elect_one();
    auto load_item = [&](int& n, Item& into) {
      const int place = n % kItems;
      ok = ok && warp_wait(smem_u32(&bar_item[place]), (n / kItems) & 1, (17 << 8) | 14);
      if (!ok) return false;
      into = s_item[place];
      ++n;
      return into.tiles > 0;
    };
    // the scores' side
    int s_items = 0, s_step = 0, s_steps = 0, s_place = 0, s_group = 0, k_slot = 0, k_turn = 0;         // (s_place: of the next shared queries)
    uint32_t k_phase = 0, q_phase = 0;                         // (q_phase: a bit for either place)
    bool s_two = false, s_more = true;
    uint64_t s_queries = dq;                                   // descriptor of the item's queries (of its first half)
    // Waits for what the next step's scores need; false where there is no further step, or a wait gave up.
    auto prepare = [&] {
      if (!s_more) return false;
      if (s_step == s_steps) {
        Item next;
        s_more = load_item(s_items, next);
        if (!s_more) return false;
        s_two = next.rows > half_rows;
        s_steps = s_two ? 2 * next.tiles : next.tiles;
        s_step = 0;
        s_queries = dq + (s_two ? 0 : s_place * L::kQBytes >> 4);
      }
      if (s_step < (s_two ? 2 : 1)) {                          // the item's queries are new
        const int place = s_two ? s_step : s_place;
        ok = warp_wait(smem_u32(&bar_q[place]), q_phase >> place & 1, (17 << 8) | 3);
        q_phase ^= 1u << place;
      }
      if (!(s_two && (s_step & 1))) ok = ok && warp_wait(smem_u32(&key_full[k_turn]), k_phase, (17 << 8) | 4);
      return ok;
    };
    auto score = [&] {                                         // (one lane)
      const bool second = s_two && (s_step & 1);
      const uint64_t q_at = s_queries + (second ? L::kQBytes >> 4 : 0), k_at = dk + (k_slot * L::kSlotBytes >> 4);
      const uint32_t to = tmem + s_group * kKeys;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        constexpr int kHalf = kRows * 128 >> 4;                // 64 columns further
        mma_ss(to, q_at + (k >> 2) * kHalf + (k & 3) * 2, k_at + (k >> 2) * kHalf + (k & 3) * 2, id_s, k > 0 ? 1u : 0u);
      }
      tc_commit(smem_u32(&bar_s[s_group]));
      if (!s_two || second) tc_commit(smem_u32(&empty[k_slot]));
      if (s_step >= s_steps - (s_two ? 2 : 1)) tc_commit(smem_u32(&bar_free[s_two ? s_step & 1 : s_place]));        // (the last that look at these queries)
    };
    auto scored = [&] {                                        // (the whole warp)
      if (!s_two || (s_step & 1)) {
        k_slot += 2;
        if (k_slot >= kSlots) k_slot -= kSlots;
        if (++k_turn == kSlots) { k_turn = 0; k_phase ^= 1; }
      }
      ++s_step;
      s_group ^= 1;
      if (s_step == s_steps && !s_two) s_place ^= 1;
    };
    auto first_scores = [&] {
      for (int j = 0; j < 2; ++j) {
        if (!prepare()) break;
        tc_fence_after();
        if (leader) score();
        __syncwarp();
        scored();
        if (!RUN_ON && s_step == s_steps) break;
      }
    };
    if (RUN_ON) first_scores();
    // the outputs' side
    int a_items = 0, group_of = 0, v_slot = 1, v_turn = 0;
    uint32_t v_phase = 0, p_phase = 0;                         // (p_phase: a bit for either group)
    Item add_item;
    while (ok && load_item(a_items, add_item)) {
      const bool two = add_item.rows > half_rows;
      const int steps = two ? 2 * add_item.tiles : add_item.tiles;
      if (!RUN_ON) {
        s_group = group_of = 0;
        first_scores();
      }
      for (int j = 0; j < steps && ok; ++j) {
        const int w = group_of;
        const bool frees = !two || (j & 1);
        if (!(two && (j & 1))) ok = warp_wait(smem_u32(&bar_clean[v_turn]), v_phase, (17 << 8) | 5);
        ok = ok && warp_wait(smem_u32(&bar_p[2 * w]), p_phase >> w & 1, (17 << 8) | 6);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v_at = dv + (v_slot * L::kSlotBytes >> 4);
        const uint32_t to = tmem_o + w * D, from = tmem + w * kKeys, add = j < 2 ? 0u : 1u;
        if (leader) {                                          // (the first keys while the others' probabilities are worked out)
#pragma unroll
          for (int k = 0; k < kFirst / 16; ++k) mma_ts(to, from + k * 8, v_at + k * (kChunk * D * 2 >> 4), id_o, k == 0 ? add : 1u);
        }
        __syncwarp();
        // (mostly the item goes on, and its next keys are all there is to wait for: this warp's chain of instructions is what the tensor cores wait for)
        bool more;
        if (s_step >= 2 && s_step < s_steps) more = ok = (s_two && (s_step & 1)) || warp_wait(smem_u32(&key_full[k_turn]), k_phase, (17 << 8) | 4);
        else more = RUN_ON && prepare();
        ok = ok && warp_wait(smem_u32(&bar_p[2 * w + 1]), p_phase >> w & 1, (17 << 8) | 6);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = kFirst / 16; k < kKeys / 16; ++k) mma_ts(to, from + k * 8, v_at + k * (kChunk * D * 2 >> 4), id_o, 1u);
          tc_commit(smem_u32(&bar_o[w]));
          if (frees) tc_commit(smem_u32(&empty[v_slot]));
          if (more) score();
        }
        __syncwarp();
        p_phase ^= 1u << w;
        group_of ^= 1;
        if (frees) {
          v_slot += 2;
          if (v_slot >= kSlots) v_slot -= kSlots;
          if (++v_turn == kSlots) { v_turn = 0; v_phase ^= 1; }
        }
        if (more) scored();
      }
    }
  } else {
    // ---------------- softmax: a thread per query row ----------------
    const int w = warp >> 2, r = threadIdx.x & (kRows - 1);
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int by_group = (65536 + group - 1) / group;          // n / group = n * by_group >> 16 for n < 256, group <= 64
    const int token = r * by_group >> 16, head_of = r - token * group;
    uint32_t s_phase = 0, o_phase = 0, given_phase = 0, taken_phase = 0;
    bool lent = false;                                         // this group's output has not been added to the other one's yet
    int before = 0;                                            // steps of the items before, modulo 2: they go to the groups in turn
    // (an item's numbers stay in shared memory: in registers they were spilled)
    for (;; ) {
      const int ring = item % kItems;
      ok = ok && warp_wait(smem_u32(&bar_item[ring]), (item / kItems) & 1, (17 << 8) | 14);
      if (!ok) break;
      ++item;
      const Item& now = s_item[ring];
      if (now.tiles <= 0) break;
      auto done = [&] {                                        // (`now` is not looked at any more)
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_done[ring]));
      };
      const bool two = now.rows > half_rows;
      // which half of the rows is this group's, or its first tile (the group that has the item's first tile also stores what comes of it)
      const int place_of = w ^ before;
      if (!two) {
        if (RUN_ON) before ^= now.tiles & 1;
        if (place_of >= now.tiles) {                            // (an item of one tile, which is the other group's)
          done();
          continue;
        }
      }
      const int in_item = (two ? place_of * half_rows : 0) + token;      // this thread's token of the item
      const bool real = r < half_rows * group && in_item < now.rows;
      const bool idle = !__any_sync(0xffffffffu, real);        // (a warp without rows: whatever it leaves as probabilities goes to outputs of nobody)
      const int row = now.row0 + (real ? in_item : 0), head = now.kvh * group + head_of;
      const int masked_from = min(now.s.front, now.keys);    // keys behind this need a look at the row's mask
      float m_ref = -INFINITY, l_run = 0.f;
      int steps = 0;
      for (int t = two ? 0 : place_of; t < now.tiles && ok; t += two ? 1 : 2, ++steps) {
        const int base = (now.tile + t) * kKeys;
        const bool whole = base + kKeys <= masked_from;
        uint32_t see[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (!whole) {                                          // 128 bits of the row, from the tile's first key on
          const int from = base - now.s.front, sh = from & 31;
          uint32_t low = tree_word(a, now.s, row, from >> 5);
          if (from >> 5 < 0) low = 0xffffffffu;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int q = (from >> 5) + i + 1;
            const uint32_t high = q < 0 ? 0xffffffffu : tree_word(a, now.s, row, q);
            const int left = now.keys - base - 32 * i;        // keys there are from this word on
            see[i] = __funnelshift_r(low, high, sh) & (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
            low = high;
          }
        }
        ok = warp_wait(smem_u32(&bar_s[w]), s_phase, (17 << 8) | 8);
        if (!ok) break;
        s_phase ^= 1;
        auto returned = [&] {                                  // the output may be written over
          if (!lent) return;
          lent = false;
          ok = warp_wait(smem_u32(&bar_taken[w]), taken_phase, (17 << 8) | 13) && ok;
          taken_phase ^= 1;
        };
        if (idle) {
          returned();
          mbar_arrive(smem_u32(&bar_p[2 * w]));
          mbar_arrive(smem_u32(&bar_p[2 * w + 1]));
          continue;
        }
        tc_fence_after();
        const uint32_t scores = tmem + w * kKeys + lane_addr;
        // The row's 128 scores are looked at twice. For the maximum the second half comes first: the first half then stays in registers,
        // and its probabilities may be written over scores 0 .. 31 while the second half is still where it was.
        uint32_t x[32], y[32];
        auto masked = [&](uint32_t (&v)[32], uint32_t bits) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(bits >> i & 1)) v[i] = 0xff800000u;          // -inf
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
        if (!whole) { masked(x, see[2]); masked(y, see[3]); }
        largest(x);
        largest(y);
        tmem_ld_x32(scores, x);
        tmem_ld_x32(scores + 32, y);
        tmem_wait_ld(x);
        tmem_wait_ld(y);
        if (!whole) { masked(x, see[0]); masked(y, see[1]); }
        largest(x);
        largest(y);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
        const bool grown = real && top > m_ref + kStale;
        if (__any_sync(0xffffffffu, grown)) {
          const float fresh = grown ? top - kAhead : m_ref, alpha = grown ? ex2(m_ref - fresh) : 1.f;
          m_ref = fresh;
          l_run *= alpha;
          if (steps > 0) {                                     // bring the output to the new reference (its last part came before these scores)
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
        const float less = m_ref > -INFINITY ? -m_ref : 0.f;
        f32x2 sum2[2] = {0ull, 0ull};
        const f32x2 scale2 = pair(p.scale_log2, p.scale_log2), less2 = pair(less, less);
        auto weigh = [&](const uint32_t (&v)[32], uint32_t* out) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float a0, a1;
            unpair(fma2(pair(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), scale2, less2), a0, a1);
            a0 = ex2(a0);
            a1 = ex2(a1);
            sum2[(i >> 1) & 1] = add2(sum2[(i >> 1) & 1], pair(a0, a1));
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
          if (!whole) masked(x, see[2]);
          uint32_t rest[16];
          weigh(x, rest);
          tmem_wait_ld(y);
          tmem_st_x16(scores + 32, rest);
          tmem_wait_st();
          returned();
          tc_fence_before();
          mbar_arrive(smem_u32(&bar_p[2 * w]));
          if (!whole) masked(y, see[3]);
          weigh(y, rest);
          tmem_st_x16(scores + 48, rest);
        }
        float s0, s1, s2, s3;
        unpair(sum2[0], s0, s1);
        unpair(sum2[1], s2, s3);
        l_run += (s0 + s1) + (s2 + s3);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&bar_p[2 * w + 1]));
      }
      if (!ok) break;
      // ---- the item's end ----
      o_phase ^= (steps - 1) & 1;                              // (the phase of this group's last output; those before it have not been waited for)
      ok = warp_wait(smem_u32(&bar_o[w]), o_phase, (17 << 8) | 11);
      if (!ok) break;
      o_phase ^= 1;
      tc_fence_after();
      // An item that both groups have had: one leaves its maxima and denominators and goes on, the one that had the first tile adds its output to its own. (Each of
      // them storing half of the columns, and waiting for the other one three times, took 2 us an item longer.)
      float f_own = 1.f, f_other = 0.f;
      if (!two && place_of == 1) {
        s_ml[r] = make_float2(m_ref, l_run);
        lent = true;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_given[w]));
        done();
        continue;
      }
      const bool joins = !two && now.tiles > 1;
      if (joins) {
        ok = warp_wait(smem_u32(&bar_given[w ^ 1]), given_phase, (17 << 8) | 13);
        if (!ok) break;
        given_phase ^= 1;
        tc_fence_after();
        const float2 other = s_ml[r];
        const float m = fmaxf(m_ref, other.x);
        f_own = m_ref > -INFINITY ? ex2(m_ref - m) : 0.f;
        f_other = other.x > -INFINITY ? ex2(other.x - m) : 0.f;
        // (a group whose keys all scored -inf has a sum of 0, or of NaN, which stays)
        l_run = l_run * (m_ref > -INFINITY ? f_own : 1.f) + other.y * (other.x > -INFINITY ? f_other : 1.f);
        m_ref = m;
      }
      const bool direct = now.flags == 3;
      if (!idle) {
        const float scale = direct ? (l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f) : 1.f;
        f_own *= scale;
        f_other *= scale;
        const size_t place = (static_cast<size_t>(2 * blockIdx.x + (now.flags & 1)) * 2 + (two ? place_of : 0));          // of the piece in the scratch
        T* const to = static_cast<T*>(a.out) + static_cast<size_t>(now.s.row + row) * a.out_stride + static_cast<size_t>(head) * D;
        float* const acc = p.acc + place * (kRows * D) + r * 4;
        if (!direct && real) *reinterpret_cast<float2*>(p.ml + (place * kRows + r) * 2) = make_float2(m_ref, l_run);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t x[32];
          float o[32];
          if (__any_sync(0xffffffffu, f_own != 0.f)) {
            tmem_ld_x32(tmem_o + w * D + lane_addr + c, x);
            tmem_wait_ld(x);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = f_own != 0.f ? __uint_as_float(x[i]) * f_own : 0.f;
          if (joins && __any_sync(0xffffffffu, f_other != 0.f)) {
            tmem_ld_x32(tmem_o + (w ^ 1) * D + lane_addr + c, x);
            tmem_wait_ld(x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = f_other != 0.f ? fmaf(__uint_as_float(x[i]), f_other, o[i]) : o[i];
          }
          if (l_run != l_run)                                  // (NaN among the scores of a group whose reference never moved)
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = l_run;
          if (!real) continue;
          if (direct) {
            uint32_t v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = pack_pair<T>(o[2 * i], o[2 * i + 1]);
            if (p.out_wide) {
              store_32_bytes(to + c, v);
              store_32_bytes(to + c + 16, v + 8);
            } else {
#pragma unroll
              for (int i = 0; i < 16; i += 2) *reinterpret_cast<uint2*>(to + c + 2 * i) = make_uint2(v[i], v[i + 1]);
            }
          } else {                                             // (a lane's neighbours have the rows beside its own)
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(acc + (c + i) * kRows) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (s_spoilt[ring] == item) {
          const int32_t* pages = a.page_table + static_cast<size_t>(now.b) * a.max_pages;
          const bool takes = real && l_run == l_run;
          if (direct) add_spoilt<T, D, T>(a, now.s, pages, row, head, takes, now.tile, now.tiles, now.keys, to);
          else add_spoilt<T, D, float>(a, now.s, pages, row, head, takes, now.tile, now.tiles, now.keys, acc);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (joins && lane == 0) mbar_arrive(smem_u32(&bar_taken[w ^ 1]));
      done();
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

// ---- the pieces of items that were cut ----
// A block per (block of the first kernel, group of warps of its item), a lane a query row, pieces in their order. Up to 32 rows a warp has them all and a sixteenth of the
// columns, and with fewer rows its lanes share the pieces out as well (one row of 32 heads behind 100000 tokens, 19 pieces of four query rows each: 33 us with a row's lane for itself).
// Output rows are put together in shared memory, so that a store writes whole lines.
constexpr int kJoinThreads = 512;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
tree_pieces_kernel(const FastParams p) {
  chain_enter();
  constexpr int kLine = D * 2 + 16;                            // bytes of a row in shared memory (so that lanes beside one another reach different banks)
  __shared__ __align__(16) uint8_t s_out[kRows * kLine];
  const TreeJoin j = p.joins[blockIdx.x];
  const int group_of = blockIdx.y;
  if (j.rows <= group_of * p.half_rows) return;
  const cacheir_b200_tree_args& a = p.a;
  const int group = a.heads / a.kv_heads, n = static_cast<int>(blockIdx.x) - j.first + 1;
  const int rows = min(p.half_rows, j.rows - group_of * p.half_rows) * group;        // query rows that there are
  auto place_of = [&](int i) { return static_cast<size_t>(2 * (j.first + i) + (i == 0 ? 1 : 0)) * 2 + group_of; };
  // Row r, every `parts`th four columns from `part` on, every `shares`th piece from `share` on (by the lanes of a warp).
  auto join = [&](auto fours, auto deep, int r, int part, int parts, int share, int shares) {
    constexpr int kFours = decltype(fours)::value, kDeep = decltype(deep)::value;    // fours of a thread; pieces under way
    const bool real = r < rows;
    float m = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int i = share; i < n; i += shares) m = fmaxf(m, real ? p.ml[(place_of(i) * kRows + r) * 2] : -INFINITY);
    for (int off = 16; off >= 32 / shares && off > 0 && shares > 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    float4 o[kFours] = {};
    for (int i0 = share; i0 < n; i0 += kDeep * shares) {
      float2 ml[kDeep];
      float4 v[kDeep][kFours];
#pragma unroll
      for (int e = 0; e < kDeep; ++e) {
        const int i = i0 + e * shares;
        ml[e] = make_float2(-INFINITY, 0.f);
        if (real && i < n) {
          ml[e] = *reinterpret_cast<const float2*>(p.ml + (place_of(i) * kRows + r) * 2);
          const float* acc = p.acc + place_of(i) * (kRows * D) + r * 4;
#pragma unroll
          for (int k = 0; k < kFours; ++k) v[e][k] = *reinterpret_cast<const float4*>(acc + (part + k * parts) * (kRows * 4));
        }
      }
#pragma unroll
      for (int e = 0; e < kDeep; ++e) {
        const float f = ml[e].x > -INFINITY ? exp2f(ml[e].x - m) : 0.f;
        l += ml[e].y * (ml[e].x > -INFINITY ? f : 1.f);        // (a piece whose keys all scored -inf has a sum of 0, or of NaN, which stays)
        if (f != 0.f)
#pragma unroll
          for (int k = 0; k < kFours; ++k) {
            o[k].x = fmaf(v[e][k].x, f, o[k].x);
            o[k].y = fmaf(v[e][k].y, f, o[k].y);
            o[k].z = fmaf(v[e][k].z, f, o[k].z);
            o[k].w = fmaf(v[e][k].w, f, o[k].w);
          }
      }
    }
    for (int off = 16; off >= 32 / shares && off > 0 && shares > 1; off >>= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
      for (int k = 0; k < kFours; ++k) {
        o[k].x += __shfl_xor_sync(0xffffffffu, o[k].x, off);
        o[k].y += __shfl_xor_sync(0xffffffffu, o[k].y, off);
        o[k].z += __shfl_xor_sync(0xffffffffu, o[k].z, off);
        o[k].w += __shfl_xor_sync(0xffffffffu, o[k].w, off);
      }
    }
    if (!real || share != 0) return;
    const float scale = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int k = 0; k < kFours; ++k) {
      if (scale != scale) o[k] = make_float4(scale, scale, scale, scale);
      *reinterpret_cast<uint2*>(s_out + r * kLine + (part + k * parts) * 8) =
          make_uint2(pack_pair<T>(o[k].x * scale, o[k].y * scale), pack_pair<T>(o[k].z * scale, o[k].w * scale));
    }
  };
  constexpr int kWarps = kJoinThreads / 32, kParts = kJoinThreads / kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (rows <= 32) {
    const int wide = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;           // lanes that have rows of their own
    join(std::integral_constant<int, D / 4 / kWarps>{}, std::integral_constant<int, 4>{}, lane & (wide - 1), warp, kWarps, lane / wide, 32 / wide);
  } else {
    join(std::integral_constant<int, D / 4 / kParts>{}, std::integral_constant<int, 2>{}, threadIdx.x & (kRows - 1), threadIdx.x / kRows, kParts, 0, 1);
  }
  __syncthreads();
  constexpr int kLanes = D / 4;                                // of a row, 8 bytes each
  const int first_token = j.row + group_of * p.half_rows;
  for (int i = threadIdx.x; i < rows * kLanes; i += kJoinThreads) {
    const int row = i / kLanes, c = i % kLanes * 4;
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + static_cast<size_t>(first_token + row / group) * a.out_stride + static_cast<size_t>(j.kvh * group + row % group) * D + c) =
        *reinterpret_cast<const uint2*>(s_out + row * kLine + c * 2);
  }
}

int half_rows_of(const cacheir_b200_tree_args& a) { return kRows / (a.heads / a.kv_heads); }
// Units of all items, at most.
long long most_units(const cacheir_b200_tree_args& a) {
  const long long tiles = (static_cast<long long>(a.max_pages) * a.page_size + kKeys - 1) / kKeys;
  return (kItemUnits + kTwoUnits * tiles) * a.kv_heads * (a.rows / (2 * half_rows_of(a)) + a.sequences);
}

template <typename T, int D>
int launch_fast(const cacheir_b200_tree_args& a, cudaStream_t stream) {
  CUtensorMap tk, tv, tq;
  const uint64_t rows = static_cast<uint64_t>(a.num_slots) * a.kv_heads * a.page_size;
  FastParams p;
  p.a = a;
  p.half_rows = half_rows_of(a);
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  if (!encode_pool<T>(&tk, a.k_cache, rows, D, false) || !encode_pool<T>(&tv, a.v_cache, rows, D, true) ||
      !encode_queries<T>(&tq, a.q, a.rows, a.heads, a.kv_heads, D, a.q_stride, p.half_rows))
    return CACHEIR_B200_EUNSUPPORTED;
  const long long most = most_units(a);
  const int grid = static_cast<int>(most < kNumSMs ? most : kNumSMs);
  p.whole = static_cast<long long>(a.max_pages) * a.page_size <= kWholeTiles * kKeys;
  p.out_wide = aligned_to(a.out, 32) && a.out_stride % 16 == 0;
  p.joins = static_cast<TreeJoin*>(a.workspace);
  p.ml = reinterpret_cast<float*>(p.joins + kNumSMs);
  p.acc = p.ml + static_cast<size_t>(kNumSMs) * 2 * 2 * kRows * 2;
  // Blocks with several short items each go on from one to the next (150 sequences of up to 66 tokens, 32 query and 8 key/value heads of 64: 43.8 us without, 35.5 with;
  // 16 trees on long sequences: 183.6 without, 192.9 with, as the warp that issues the products has more to look after).
  const bool run_on = p.whole && (a.rows / (2 * p.half_rows) + static_cast<long long>(a.sequences)) * a.kv_heads > 2 * kNumSMs;
  auto kern = run_on ? tree_kernel<T, D, true> : tree_kernel<T, D, false>;
  static std::atomic<unsigned long long> done[2]{{0}, {0}};
  cudaError_t e = allow_shared_memory(done[run_on], reinterpret_cast<const void*>(kern), Smem<D>::kBytes);
  if (e == cudaSuccess) e = launch_chained(kern, dim3(grid), dim3(kThreads), Smem<D>::kBytes, stream, tk, tv, tq, p);
  if (e == cudaSuccess && !p.whole) e = launch_chained(tree_pieces_kernel<T, D>, dim3(grid, a.rows > p.half_rows ? 2 : 1), dim3(kJoinThreads), 0, stream, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

}  // namespace

size_t tree_fast_bytes(int dim) {
  if (dim != 64 && dim != 128) return 0;
  return kNumSMs * sizeof(TreeJoin) + static_cast<size_t>(kNumSMs) * 2 * 2 * kRows * (2 + dim) * 4;
}

bool tree_fast_supported(const cacheir_b200_tree_args& a) {
  return (a.dtype == CACHEIR_B200_F16 || a.dtype == CACHEIR_B200_BF16) && (a.dim == 64 || a.dim == 128) && a.page_size % kChunk == 0 &&
         a.heads / a.kv_heads <= kMaxHeadsPerKv && aligned_to(a.q, 16) && a.q_stride % 8 == 0 && aligned_to(a.k_cache, 16) && aligned_to(a.v_cache, 16) &&
         aligned_to(a.out, 8) && a.out_stride % 4 == 0 && static_cast<long long>(a.num_slots) * a.kv_heads * a.page_size <= 0x7fffffffLL - kChunk &&
         most_units(a) <= 0x7fffffffLL;
}

int launch_tree_fast(const cacheir_b200_tree_args& a, cudaStream_t stream) {
  if (a.dtype == CACHEIR_B200_F16) return a.dim == 128 ? launch_fast<__half, 128>(a, stream) : launch_fast<__half, 64>(a, stream);
  return a.dim == 128 ? launch_fast<__nv_bfloat16, 128>(a, stream) : launch_fast<__nv_bfloat16, 64>(a, stream);
}

int tree_device_status(bool reset) { return device_status_word(g_tree_status, reset); }

}  // namespace cb200
