// Attention of a few new rows per sequence over the paged 8-bit cache (decode, drafted tokens).
//
// Every cached byte is needed once and meets at most 32 query rows (new tokens x query heads of
// its key head), so HBM bounds the kernel; the work is to keep the byte stream going and
// everything else underneath it.
//
//  * Tokens are the M side of both products: S^T = K Q^T (128 tokens x rows) and
//    O^T = V^T P^T (head_dim x rows).  K and V^T are read by tcgen05.mma straight from the TMA
//    tiles (V as an MN-major operand), with the block scales of the cache as the hardware's block
//    scales: no cached value passes through a register.  A token row is a lane of tensor memory.
//  * Queries and weights are E4M3 terms (kv_attention.cuh).  The terms lie side by side along N,
//    so that one pass of the K or V tile serves all of them, and are added in 32 bits afterwards.
//    With at most 96 columns an MMA costs what its 128-row operand costs (about 33 ns).
//  * Warps: 0-3 and 4-7 softmax (one lane per token; the two groups take alternate tiles, each
//    with its own running maximum and output accumulator, because one group needs about as long
//    for a tile as HBM does), 8 and 9 TMA of K and of V (one warp for both held heads of 128 back:
//    131072 tokens x 8 heads, 8 rows each: 65 us, with two 55), 10 MMAs of the scores (two tiles
//    ahead), 11 MMAs of the outputs, 12 and 13 quantise queries and describe the segments.
//  * The list of (sequence, key head, tile of 128 tokens) is cut into equal shares, one per CTA
//    (one per SM), whatever the lengths are: the cut follows the lengths on the device.  A CTA
//    whose share covers all tiles of a (sequence, head) writes its rows; otherwise it leaves
//    unnormalised rows with their maximum and sum, and a second kernel (launched as a
//    programmatic dependent) joins them in the order of the tiles, so the result does not depend
//    on timing.
//  * Online softmax without touching the output.  The weights of a row are taken relative to the
//    largest score among the warp's own 32 tokens, rounded to a power of two, and that power
//    (relative to a reference fixed by the first tile) is the hardware block scale of the
//    weights: 32 tokens is one scale block of the second product.  So no maximum crosses warps
//    and no accumulator is rescaled from tile to tile.  Only where a tile exceeds the reference
//    by more than 2^16 the four warps move it and shrink the accumulator.  It is also the more
//    exact way: each block's largest weight is in (181, 363), so E4M3's smallest step never
//    reaches a weight that counts.  The sums of the weights, as they were rounded, are a product
//    with ones.
//
// Measured inside a CUDA graph (copy rate 6.57 TB/s): 131072 tokens of one sequence, 4 key heads of
// 256, 6 rows each: 52 us, 5.2 TB/s; 32 sequences of up to 8192: 53 us, 4.9 TB/s; 32 sequences of
// 8001: 91 us, 5.8 TB/s.  With more rows the softmax of a tile takes longer than its bytes: 131072
// tokens, 8 key heads of 128: 55 us with 8 rows, 59 with 16, 79 with 24; 48 sequences of 4 drafted
// tokens (16 rows, up to 4096 tokens): 68 us, 2.9 TB/s, of which about 3 us for every segment's start
// and end, where the groups meet.  Tried and left: a third softmax group (78 us for the last case).
#include "kv_attention.cuh"

#include <cfloat>
#include <climits>
#include <cstdlib>

namespace mx {

int* device_status_word(int device);

namespace {

constexpr int kThreads = 448;
constexpr int kGroupWarps = 4;  // warps of a softmax group, one per 32 lanes of tensor memory
constexpr int kKeyWarp = 8, kValueWarp = 9, kScoreWarp = 10, kOutputWarp = 11, kQueryWarp = 12, kQueryWarps = 2;
// Query buffers.  Scores run two tiles ahead of the outputs, so a tile of one segment may be
// waiting for its output while the scores of the second segment behind it are due.
constexpr int kQueries = 3;
constexpr float kWeightLog2 = 8.0f;     // weights are scaled by 256 before they become E4M3 terms
constexpr float kMostLog2 = 16.0f;      // a tile may exceed the reference by 2^16
constexpr int kSms = 148;
constexpr int kJoinThreads = 256;
// Items of at most this many tiles are not cut, and not joined: 32 sequences of 1000 tokens, 8 key
// heads of 128: 22 us, cut 27 us; one sequence 10.3 us, cut 11.2 us.  At 16 tiles 32 sequences still
// gain (35.2 -> 32.7 us), but one sequence loses (11.3 -> 15.3 us).  The rule goes by the longest sequence
// that the block table can name, which the host knows: the same 32 sequences under a table of 2048
// columns of 64 tokens are cut, 23 against 19 us in a graph (one of 200 tokens: 9.5 against 8.3 us).
constexpr int kWholeTiles = 8;
constexpr int kMinUnits = 3;      // units that a CTA takes at least

template <int D, int RP, int TERMS>
struct DecodeCfg {
  static constexpr int kN = RP * TERMS;              // columns of both products
  static constexpr int kRowBytes = D < 128 ? D : 128;  // bytes of a token row in one sub-tile
  static constexpr int kSubs = D / kRowBytes;
  static constexpr int kSubBytes = kKvTile * kRowBytes;
  static constexpr int kSlotBytes = kKvTile * D;     // a K or V tile
  static constexpr int kQBytes = (kN * D + 1023) / 1024 * 1024;
  static constexpr int kPBytes = kN * kKvTile;
  // Weights are buffered twice per softmax group, so that it need not wait for the output of its
  // last tile (about 0.6 us) before it writes the next; a head of 256 spends the room on its ring.
  static constexpr int kPBuffers = D < 256 ? 2 : 1;
  static constexpr int kFixedBytes = 8192 + 2 * D * 4;
  static constexpr int kBudget = 227 * 1024 - 1024;
  static constexpr int kFit =
      (kBudget - kFixedBytes - kQueries * kQBytes - 2 * kPBuffers * kPBytes) / (kSlotBytes + 512);
  static constexpr int kSlots = kFit > 16 ? 16 : kFit;
  // Two rings: the scores run ahead of the outputs, so K has the odd slot.
  static constexpr int kKeySlots = (kSlots + 1) / 2, kValueSlots = kSlots / 2;
  static_assert(kValueSlots >= 2 * kPBuffers, "the softmax groups wait for V by the output that far back");
  static constexpr int kSmemBytes =
      1024 + kSlots * (kSlotBytes + 512) + kQueries * kQBytes + 2 * kPBuffers * kPBytes + kFixedBytes;
  // Tensor memory columns: two score tiles; per softmax group an output of one or two halves
  // and the sums of the weights; scales.
  static constexpr int kHalves = D > 128 ? 2 : 1;
  static constexpr int kOCol = 2 * kN;
  static constexpr int kLCol = kOCol + 2 * kHalves * kN;  // sums of the weights, per group
  static constexpr int kSfCol = kLCol + 2 * kN;
  static constexpr int kOnesCol = kSfCol + 2 * kPBuffers * 12;  // a set per group and buffer of weights
  static constexpr int kColsUsed = kOnesCol + 4;
  static constexpr int kChunk = RP % 16 == 0 ? 16 : 8;  // rows of a score tile held at a time
  static constexpr int kTmemCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  static_assert(kColsUsed <= 512, "tensor memory");
  static constexpr uint64_t kSwizzle = kRowBytes == 128 ? ptx::kSwizzle128 : ptx::kSwizzle64;
  static constexpr int kGroup = 8 * kRowBytes;  // bytes of eight token rows
  // Partial rows of one CTA end: RP rows of D values, then RP pairs (maximum, sum).
  static constexpr int kPartialFloats = RP * D + 2 * RP;
};

// Rows (new tokens x query heads) of the widest variant: tensor memory holds, for two groups,
// scores, sums and one or two output halves of rows x terms columns.
constexpr int most_rows(int d, int terms) {
  return d == 256 ? (terms == 3 ? 16 : 24) : (terms == 3 ? 24 : 32);
}

// Rows of the variant that `rows` take: the softmax works through all of a variant's (65536 tokens, 8
// key heads of 128, 24 rows: 44 us, as 32 rows 49 us).
constexpr int variant_rows(int rows, int d, int terms) {
  return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 24 && most_rows(d, terms) > 24 ? 24 : most_rows(d, terms);
}

// The work list and its cut, the same arithmetic in both kernels.  An item is a (sequence, key
// head); it counts its tiles and item_units more for the rows' start and end (a CTA that takes
// seven short items was 60 % later than one that takes 27 tiles of one).  A CTA gets the tiles
// whose units lie in its share.
struct Share {
  int64_t total;  // units in all
  int ctas;
};
__host__ __device__ __forceinline__ int64_t share_begin(const Share& s, int cta) {
  return s.total * cta / s.ctas;
}
__device__ __forceinline__ Share share_of(int64_t total, int grid) {
  Share s;
  s.total = total;
  // Fewer, larger shares while the list is short: joining costs more than a second tile.
  const int64_t want = (total + kMinUnits - 1) / kMinUnits;
  s.ctas = (int)(want < grid ? (want < 1 ? 1 : want) : grid);
  return s;
}
__device__ __forceinline__ int units_of(const AttentionArgs& a, int tiles) {
  return tiles == 0 ? 0 : tiles + a.item_units;
}

// Units of all sequences (one key head), by a full warp.
__device__ __forceinline__ int64_t warp_total_units(const AttentionArgs& a, int lane) {
  int64_t mine = 0;
  for (int b = lane; b < a.batch.batch; b += 32) mine += units_of(a, kv_sequence(a, b).tiles);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  return mine;
}

// A place in the work list and the sequence it belongs to.
struct Cursor {
  int b, head, tile;
  KvSequence seq;
  __device__ __forceinline__ void load(const AttentionArgs& a) { seq = kv_sequence(a, b); }
  // Next tile; the caller knows that there is one.
  __device__ __forceinline__ void next(const AttentionArgs& a) {
    if (++tile < seq.tiles) return;
    tile = 0;
    if (++head < a.cache.kv_heads) return;
    head = 0;
    do {
      if (++b >= a.batch.batch) {
        b = a.batch.batch - 1;  // behind the end: only reached by look-ahead
        seq.tiles = 1;
        return;
      }
      seq = kv_sequence(a, b);
    } while (seq.tiles == 0);
  }
};

// The first tile at or behind unit `at`, by a full warp: returns its number in the list of all
// tiles and, in all lanes, the place and the first unit of its item.  `whole`: items are not cut, the place is the first item that
// begins at or behind `at`.
__device__ __forceinline__ int64_t warp_locate(const AttentionArgs& a, int64_t at, bool whole,
                                               int lane, Cursor* place, int64_t* item_begin) {
  const int heads = a.cache.kv_heads;
  int64_t units = 0, tiles = 0;  // of all heads of the sequences before this group of 32
  place->b = a.batch.batch - 1;
  place->head = place->tile = 0;
  for (int b0 = 0; b0 < a.batch.batch; b0 += 32) {
    const int b = b0 + lane;
    const int mine = b < a.batch.batch ? kv_sequence(a, b).tiles : 0;
    int64_t upto = (int64_t)units_of(a, mine) * heads, tiles_upto = (int64_t)mine * heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
      const int64_t t = __shfl_up_sync(0xffffffffu, tiles_upto, o);
      if (lane >= o) {
        upto += u;
        tiles_upto += t;
      }
    }
    // The sequence whose last item's last tile is not before `at`.
    const int64_t reach = units + upto - (whole ? units_of(a, mine) - 1 : 0);
    const unsigned reached = __ballot_sync(0xffffffffu, mine > 0 && reach > at);
    if (reached != 0) {
      const int l = __ffs(reached) - 1;
      const int count = __shfl_sync(0xffffffffu, mine, l);
      const int64_t per_item = units_of(a, count);
      const int64_t first = units + __shfl_sync(0xffffffffu, upto, l) - per_item * heads;
      const int64_t into = at > first ? at - first : 0;
      place->b = b0 + l;
      *item_begin = first + into / per_item * per_item;
      if (whole) {
        place->head = (int)((into + per_item - 1) / per_item);
      } else {
        place->head = (int)(into / per_item);
        const int64_t in_item = into % per_item - a.item_units;
        place->tile = in_item > 0 ? (int)in_item : 0;
      }
      return tiles + __shfl_sync(0xffffffffu, tiles_upto, l) - (int64_t)count * heads +
             (int64_t)place->head * count + place->tile;
    }
    units += __shfl_sync(0xffffffffu, upto, 31);
    tiles += __shfl_sync(0xffffffffu, tiles_upto, 31);
  }
  return tiles;
}

// What the joining kernel needs to know about the border behind a CTA's share: the item in which the
// next share begins.
struct Border {
  int64_t row;  // first token row of the item
  int rows;     // query rows
  int head;
  int parts;    // CTAs over which the item goes, 1: nothing to join here
  int pad[3];
};
// With many rows it is told, in the workspace before the partial rows: its CTAs do not fit the GPU at
// once, and most have nothing to do.  With few it finds out while the main kernel ends.  131072 tokens,
// 6 rows: told 52.4 us, finding out 51.7; 48 sequences of 16 rows: told 68.0, finding out 71.2.
template <int RP>
constexpr bool kToldBorders = RP > 8;
__device__ __forceinline__ Border* borders_of(const AttentionArgs& a) {
  return reinterpret_cast<Border*>(a.partials) - kSms;
}
__device__ __forceinline__ Border border_of(const AttentionArgs& a, const Share& s, int cta, int64_t begin,
                                            int b, int head) {
  Border border{0, 0, head, 1, {}};
  if (cta + 1 >= s.ctas) return border;
  const KvSequence seq = kv_sequence(a, b);
  border.row = seq.row;
  border.rows = seq.rows * a.group;
  const int64_t u0 = begin + a.item_units, u1 = u0 + seq.tiles - 1;
  // CTA of a unit: the last one whose share begins at or before it.
  if (u1 >= u0 && (int)(((u0 + 1) * s.ctas - 1) / s.total) == cta)
    border.parts = (int)(((u1 + 1) * s.ctas - 1) / s.total) - cta + 1;
  return border;
}

// A segment: the tiles of one item that a CTA takes, and where its rows go.  Filled by the query
// warps, one segment ahead.
template <int RP>
struct Segment {
  int64_t out[RP];  // offset of each output row
  float scale[RP];  // of the quantised query rows, times the softmax scale and log2(e)
  int64_t first_position;  // of the first row; rows see cached tokens up to their own
  int length;       // cached tokens
  int rows;         // query rows: new tokens x group
  int tile;         // first tile
  int tiles;
  int whole;        // all tiles of the item are here
};

template <int D, int RP, int TERMS>
__global__ void __launch_bounds__(kThreads, 1)
kv_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const AttentionArgs a) {
  using C = DecodeCfg<D, RP, TERMS>;
  using T = typename std::conditional<TERMS == 2, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* slots = smem;
  uint8_t* q_tiles = slots + C::kSlots * C::kSlotBytes;        // [buffer][sub][column][row bytes]
  uint8_t* p_tiles = q_tiles + kQueries * C::kQBytes;                 // [group][buffer][column][128 tokens]
  uint8_t* sf_tiles = p_tiles + 2 * C::kPBuffers * C::kPBytes;                // scale atom of every slot
  uint8_t* fixed = sf_tiles + C::kSlots * 512;
  uint64_t* bars = reinterpret_cast<uint64_t*>(fixed);
  uint8_t* ones = fixed + 512;                                 // scale atom of factors of one
  uint8_t* p_sf = fixed + 1024;                                // scale atoms of the weights, as p_tiles
  uint8_t* one_values = fixed + 1024 + 2048;                   // E4M3 ones, see the sums
  Segment<RP>* segments = reinterpret_cast<Segment<RP>*>(fixed + 5120);  // [buffer]
  float* red_max = reinterpret_cast<float*>(segments + kQueries);     // [group][warp][RP]
  float* red_top = red_max + 8 * RP;                           // [group][RP]
  int* nan_table = reinterpret_cast<int*>(red_top + 2 * RP);   // [segment parity][head_dim], see clear_nan
  Cursor* start = reinterpret_cast<Cursor*>(nan_table + 2 * D);  // of this share, of the next
  int64_t* share_smem = reinterpret_cast<int64_t*>(start + 2);  // begin, end, all units, begin of the item at the end
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(share_smem + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ask_flag = abort_flag + 1;                     // [group][2]
  volatile int* nan_flag = ask_flag + 4;                       // [segment parity]
  volatile uint32_t* slot_named = reinterpret_cast<volatile uint32_t*>(nan_flag + 2);  // [slot]
  static_assert(5120 + kQueries * sizeof(Segment<RP>) + 10 * RP * 4 + 2 * D * 4 + 2 * sizeof(Cursor) + 32 + 8 + 16 + 72 <=
                    C::kFixedBytes,
                "fixed area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = ptx::smem_u32(bars);
  const uint32_t empty0 = full0 + 8 * C::kSlots;
  const uint32_t sfull0 = empty0 + 8 * C::kSlots;  // one per group; of the weights', one per buffer
  const uint32_t pfull0 = sfull0 + 16;
  const uint32_t pvdone0 = pfull0 + 16 * C::kPBuffers;
  const uint32_t qfull0 = pvdone0 + 16 * C::kPBuffers;
  const uint32_t qempty0 = qfull0 + 8 * kQueries;
  const uint32_t vsync0 = qempty0 + 8 * kQueries;
  const uint32_t sread0 = vsync0 + 16;
  static_assert(8 * (2 * 16 + 6 + 4 * C::kPBuffers + 2 * kQueries) <= 512, "barriers");

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 4; ++i) ask_flag[i] = 0;
    nan_flag[0] = nan_flag[1] = 0;
    for (int s = 0; s < C::kSlots; ++s) {
      ptx::mbar_init(full0 + 8 * s, 2);  // the copies' bytes, and the scales
      ptx::mbar_init(empty0 + 8 * s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(sfull0 + 8 * i, 1);
      for (int b = 0; b < C::kPBuffers; ++b) {
        ptx::mbar_init(pfull0 + 8 * (i * C::kPBuffers + b), kGroupWarps);
        ptx::mbar_init(pvdone0 + 8 * (i * C::kPBuffers + b), 1);
      }
      ptx::mbar_init(vsync0 + 8 * i, kGroupWarps);
      ptx::mbar_init(sread0 + 8 * i, kGroupWarps);
    }
    for (int i = 0; i < kQueries; ++i) {
      ptx::mbar_init(qfull0 + 8 * i, kQueryWarps);
      ptx::mbar_init(qempty0 + 8 * i, 1 + 2 * kGroupWarps);
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
  }
  if (threadIdx.x < 128) reinterpret_cast<uint32_t*>(ones)[threadIdx.x] = 0x7f7f7f7fu;
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) nan_table[i] = INT_MAX;
  for (int i = threadIdx.x; i < 512; i += kThreads)
    reinterpret_cast<uint32_t*>(one_values)[i] = 0x38383838u;
  ptx::fence_proxy_async();
  if (warp == kScoreWarp) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), C::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  // From here on everything before this kernel has completed, also for the joining kernel, which may
  // read the same lengths before it waits for this one.
  ptx::grid_launch_dependents();
  if (warp < 2) {
    // Warp 0 finds the first tile of this CTA, warp 1 the first of the next.
    const Share s = share_of(warp_total_units(a, lane) * a.cache.kv_heads, (int)gridDim.x);
    const int cta = (int)blockIdx.x + warp;
    Cursor c{};
    int64_t tile = 0;
    int64_t begin = 0;
    if ((int)blockIdx.x < s.ctas)
      tile = warp_locate(a, share_begin(s, cta), a.whole_items != 0, lane, &c, &begin);
    if (lane == 0) {
      share_smem[warp] = tile;
      start[warp] = c;
      if (warp == 1) {
        share_smem[2] = s.total;
        share_smem[3] = begin;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int count = (int)(share_smem[1] - share_smem[0]);  // tiles of this CTA
  const int per_page = a.cache.page_size / kKvBlock;
  // E4M3 x E4M3, UE8M0 scales, M = 128, N = kN; K-major unless bit 15 says otherwise for A.
  constexpr uint32_t kIdesc = ((uint32_t)(C::kN >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24);

  if (count > 0 && (warp == kKeyWarp || warp == kValueWarp)) {
    // ---------------- TMA producers, one for K and one for V ----------------
    // Lane l looks up block l % 4 of tile l / 4 of a group of eight tiles and later issues that
    // block's copies itself; the next group's lookups are in flight while this group is copied.
    const bool is_v = warp == kValueWarp;
    const int first_slot = is_v ? C::kKeySlots : 0;
    const int end_slot = is_v ? C::kSlots : C::kKeySlots;
    const CUtensorMap* map = is_v ? &tm_v : &tm_k;
    const uint8_t* scales = is_v ? a.cache.v_scales : a.cache.k_scales;
    Cursor mine = *start;
    mine.load(a);
    for (int i = 0; i < (lane >> 2); ++i) mine.next(a);
    int64_t page = -1, next_page = -1;  // scale block of this lane's block of tokens, or -1
    uint32_t scale = 127, next_scale = 127;
    auto lookup_page = [&]() -> int64_t {
      const int block = mine.tile * kKvTileBlocks + (lane & 3);
      if (block * kKvBlock >= mine.seq.length) return -1;
      const int64_t p = kv_page(a.batch, a.cache, mine.b, block);
      return p < 0 ? -1 : (p * a.cache.kv_heads + mine.head) * per_page + block % per_page;
    };
    page = lookup_page();
    if (page >= 0) scale = scales[page];
    int slot = first_slot;
    uint32_t phase = 0;
    bool ok = true;
    const bool leads = (lane & 3) % per_page == 0;  // first block of a page in its tile
    const uint32_t page_bytes = (uint32_t)(a.cache.page_size * D);
    const uint32_t slots_s = ptx::smem_u32(slots) + (lane & 3) * kKvBlock * C::kRowBytes;
    for (int i0 = 0; ok && i0 < count; i0 += 8) {
      const bool more = i0 + 8 < count;
      if (more) {
        for (int i = 0; i < 8; ++i) mine.next(a);
        next_page = lookup_page();
      }
      // One copy per page and 128 columns; blocks of no page are left as they are.
      const bool issue = leads && page >= 0;
      const uint32_t issued = __ballot_sync(0xffffffffu, issue);
      const uint32_t named = __ballot_sync(0xffffffffu, page >= 0);
      for (int j = 0; j < 8 && i0 + j < count; ++j) {
        const int src = 4 * j;  // lanes src .. src + 3 know the tile's blocks
        ok = ok && __all_sync(0xffffffffu, bounded_wait(empty0 + 8 * slot, phase ^ 1u, abort_flag,
                                                        a.status, 401));
        if (!ok) break;
        const uint32_t bar = full0 + 8 * slot;
        if (lane == src) ptx::mbar_arrive_expect_tx(bar, __popc(issued >> src & 15u) * page_bytes);
        __syncwarp();
        if (issue && (lane & ~3) == src) {
#pragma unroll
          for (int s = 0; s < C::kSubs; ++s)
            ptx::tma_load_2d(slots_s + slot * C::kSlotBytes + s * C::kSubBytes, map, s * 128,
                             (int)(page * kKvBlock), bar);
        }
        // Scale atom: lane = row % 32.  Keys: row block c of 32 tokens has one factor for all of
        // head_dim; values: every row has the factors of the four 32-token steps along K.
        uint32_t sf[kKvTileBlocks];
#pragma unroll
        for (int i = 0; i < kKvTileBlocks; ++i) sf[i] = __shfl_sync(0xffffffffu, scale, src + i);
        const uint32_t all = sf[0] | sf[1] << 8 | sf[2] << 16 | sf[3] << 24;
        reinterpret_cast<uint4*>(sf_tiles + slot * 512)[lane] =
            is_v ? make_uint4(all, all, all, all)
                 : make_uint4(sf[0] * 0x01010101u, sf[1] * 0x01010101u, sf[2] * 0x01010101u,
                              sf[3] * 0x01010101u);
        if (lane == 0) slot_named[slot] = named >> src & 15u;
        ptx::fence_proxy_async();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar);
        if (++slot == end_slot) {
          slot = first_slot;
          phase ^= 1u;
        }
        if (j == 3 && more) next_scale = next_page >= 0 ? scales[next_page] : 127u;
      }
      page = next_page;
      scale = next_scale;
    }
  } else if (count > 0 && warp == kScoreWarp) {
    // ---------------- scores ----------------
    // Two warps issue MMAs: with one, the scores of a tile waited behind the outputs of the tile
    // before it, whose weights are not there yet.
    const uint32_t sf0 = tmem + C::kSfCol, ones_t = tmem + C::kOnesCol;  // sets of keys, values, weights
    if (ptx::elect_one()) ptx::tc_cp_32x128b_warpx4(ones_t, ptx::smem_desc_scale_atom(ptx::smem_u32(ones)));
    __syncwarp();
    bool ok = true;
    int left = 0;  // tiles of the segment that are still to come
    for (int i = 0, segment = -1; ok && i < count; ++i) {
      if (left == 0) {
        ++segment;
        ok = __all_sync(0xffffffffu, bounded_wait(qfull0 + 8 * (segment % kQueries),
                                                  (uint32_t)(segment / kQueries) & 1u, abort_flag,
                                                  a.status, 402));
        left = segments[segment % kQueries].tiles;
      }
      --left;
      const int slot = i % C::kKeySlots;
      // The score tile of two tiles ago has been read.
      if (i >= 2)
        ok = ok && __all_sync(0xffffffffu, bounded_wait(sread0 + 8 * (i & 1), (uint32_t)((i - 2) >> 1) & 1u,
                                                        abort_flag, a.status, 415));
      ok = ok && __all_sync(0xffffffffu,
                            bounded_wait(full0 + 8 * slot, (uint32_t)(i / C::kKeySlots) & 1u,
                                         abort_flag, a.status, 403));
      if (!ok) break;
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        const uint32_t sf_t = sf0 + 12 * (i & 1);
        ptx::tc_cp_32x128b_warpx4(sf_t, ptx::smem_desc_scale_atom(ptx::smem_u32(sf_tiles + slot * 512)));
        const uint32_t k_s = ptx::smem_u32(slots + slot * C::kSlotBytes);
        const uint32_t q_s = ptx::smem_u32(q_tiles + (segment % kQueries) * C::kQBytes);
#pragma unroll
        for (int s = 0; s < C::kSubs; ++s) {
          const uint64_t ad = ptx::smem_desc(k_s + s * C::kSubBytes, 0, C::kGroup, C::kSwizzle);
          const uint64_t bd = ptx::smem_desc(q_s + s * C::kN * C::kRowBytes, 0, C::kGroup, C::kSwizzle);
#pragma unroll
          for (int ks = 0; ks < C::kRowBytes / 32; ++ks)
            ptx::tc_mma_mxf8f6f4(tmem + (i & 1) * C::kN, ad + 2 * ks, bd + 2 * ks, kIdesc, sf_t,
                                 ones_t, (s > 0 || ks > 0) ? 1u : 0u);
        }
        ptx::tc_commit(sfull0 + 8 * (i & 1));
        ptx::tc_commit(empty0 + 8 * slot);
        if (left == 0) ptx::tc_commit(qempty0 + 8 * (segment % kQueries));
      }
      __syncwarp();
    }
  } else if (count > 0 && warp == kOutputWarp) {
    // ---------------- outputs and sums ----------------
    const uint32_t sf0 = tmem + C::kSfCol;
    const uint32_t ones_t = tmem + C::kOnesCol;  // written before the first scores, which the weights follow
    bool ok = true;
    int left = 0, number = 0;  // tiles of the segment that are still to come, that were
    for (int i = 0, segment = -1; i < count; ++i) {
      const int slot = C::kKeySlots + i % C::kValueSlots;
      const int weights = (i & 1) * C::kPBuffers + (i >> 1) % C::kPBuffers;
      ok = ok && __all_sync(0xffffffffu,
                            bounded_wait(pfull0 + 8 * weights, (uint32_t)((i >> 1) / C::kPBuffers) & 1u,
                                         abort_flag, a.status, 404));
      ok = ok && __all_sync(0xffffffffu,
                            bounded_wait(full0 + 8 * slot, (uint32_t)(i / C::kValueSlots) & 1u,
                                         abort_flag, a.status, 405));
      if (!ok) break;
      if (left == 0) {
        ++segment;
        left = segments[segment % kQueries].tiles;
        number = 0;
      }
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        const uint32_t sf_t = sf0 + 12 * (i % (2 * C::kPBuffers)) + 4, weight_t = sf_t + 4;
        ptx::tc_cp_32x128b_warpx4(sf_t, ptx::smem_desc_scale_atom(ptx::smem_u32(sf_tiles + slot * 512)));
        ptx::tc_cp_32x128b_warpx4(weight_t, ptx::smem_desc_scale_atom(ptx::smem_u32(p_sf + weights * 512)));
        const uint32_t v_s = ptx::smem_u32(slots + slot * C::kSlotBytes);
        const uint64_t bd =
            ptx::smem_desc(ptx::smem_u32(p_tiles + weights * C::kPBytes), 0, 1024, ptx::kSwizzle128);
        const bool first = number < 2;  // of its group in the segment
#pragma unroll
        for (int h = 0; h < C::kHalves; ++h) {
          // V^T: 128 values of head_dim along M (MN-major), 32 tokens per step.  With a head of
          // 64 the upper 64 rows of M are the next eight tokens' bytes: lanes nobody reads.
          const uint64_t ad = ptx::smem_desc(v_s + h * C::kSubBytes, C::kGroup, C::kGroup, C::kSwizzle);
#pragma unroll
          for (int ks = 0; ks < kKvTileBlocks; ++ks) {
            const uint32_t idesc = kIdesc | (1u << 15) | ((uint32_t)ks << 29) | ((uint32_t)ks << 4);
            ptx::tc_mma_mxf8f6f4(tmem + C::kOCol + ((i & 1) * C::kHalves + h) * C::kN,
                                 ad + ks * (kKvBlock * C::kRowBytes / 16), bd + 2 * ks, idesc, sf_t,
                                 weight_t, (!first || ks > 0) ? 1u : 0u);
          }
        }
        // Sums of the weights as they were rounded and scaled, so that they add up to one: a
        // product with ones (eight rows of shared memory serve all 128).
        const uint64_t ones_d = ptx::smem_desc(ptx::smem_u32(one_values), 0, 0, ptx::kSwizzle128);
#pragma unroll
        for (int ks = 0; ks < kKvTileBlocks; ++ks)
          ptx::tc_mma_mxf8f6f4(tmem + C::kLCol + (i & 1) * C::kN, ones_d, bd + 2 * ks,
                               kIdesc | ((uint32_t)ks << 4), ones_t, weight_t,
                               (!first || ks > 0) ? 1u : 0u);
        ptx::tc_commit(pvdone0 + 8 * weights);
        ptx::tc_commit(empty0 + 8 * slot);
      }
      __syncwarp();
      --left;
      ++number;
    }
  } else if (count > 0 && warp >= kQueryWarp) {
    // ---------------- query terms ----------------
    Cursor c = *start;
    c.load(a);
    int left = count;
    bool ok = true;
    for (int segment = 0; ok && left > 0; ++segment) {
      const int buffer = segment % kQueries;
      ok = __all_sync(0xffffffffu, bounded_wait(qempty0 + 8 * buffer, ((uint32_t)(segment / kQueries) & 1u) ^ 1u,
                                                abort_flag, a.status, 406));
      if (!ok) break;
      Segment<RP>& seg = segments[buffer];
      uint8_t* q_s = q_tiles + buffer * C::kQBytes;
      const int rows = c.seq.rows * a.group;
      const int tiles = min(left, c.seq.tiles - c.tile);
      // Lane r: where row r is read (padding rows: row 0, unused) and where it goes.
      const int own = lane < rows ? lane : 0;
      const int64_t own_token = c.seq.row + own / a.group;
      const int64_t own_head = c.head * a.group + own % a.group;
      const int64_t own_q = own_token * a.q_token_stride + own_head * a.q_head_stride;
      if (warp == kQueryWarp) {
        if (lane < RP) seg.out[lane] = own_token * a.out_token_stride + own_head * a.out_head_stride;
        if (lane == 0) {
          seg.first_position = c.seq.last - c.seq.rows + 1;
          seg.length = c.seq.length;
          seg.rows = rows;
          seg.tile = c.tile;
          seg.tiles = tiles;
          seg.whole = c.tile == 0 && tiles == c.seq.tiles;
        }
      }
      constexpr int kPer = D / 32;   // values per lane
      constexpr int kBatch = 4;      // rows in flight
#pragma unroll 1
      for (int r0 = warp - kQueryWarp; r0 < RP; r0 += kBatch * kQueryWarps) {
        // Row r0 + n * kQueryWarps is batch entry n.
        uint32_t raw[kBatch][kPer / 2];
        const int64_t offset = __shfl_sync(0xffffffffu, own_q, (r0 + lane * kQueryWarps) % 32);
        load_query_rows<kBatch, kPer>(static_cast<const uint16_t*>(a.q) + lane * kPer, offset, 0, a.vector, raw);
        // All maxima first: the rows' conversions then overlap.
        float scale[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n)
          scale[n] = query_scale<T, kPer>(raw[n], r0 + n * kQueryWarps < rows);
        float mine = scale[0];
#pragma unroll
        for (int n = 1; n < kBatch; ++n) mine = lane == n ? scale[n] : mine;
        if (lane < kBatch) seg.scale[r0 + lane * kQueryWarps] = mine * a.scale_log2;
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const int r = r0 + n * kQueryWarps;
          uint32_t codes[TERMS][kPer / 2];
          query_terms<T, TERMS, kPer>(raw[n], r < rows, scale[n], 1.0f, codes);
          const int d0 = lane * kPer;
#pragma unroll
          for (int k = 0; k < TERMS; ++k) {
            const int col = k * RP + r;
            const int in_row = d0 % C::kRowBytes;
            const int swizzle = C::kRowBytes == 128 ? (col & 7) : ((col >> 1) & 3);
            uint8_t* dst = q_s + (d0 / C::kRowBytes) * C::kN * C::kRowBytes + col * C::kRowBytes +
                           (((in_row >> 4) ^ swizzle) << 4) + (in_row & 15);
            if constexpr (kPer == 8) {
              *reinterpret_cast<uint2*>(dst) = make_uint2(codes[k][0] | codes[k][1] << 16,
                                                          codes[k][2] | codes[k][3] << 16);
            } else if constexpr (kPer == 4) {
              *reinterpret_cast<uint32_t*>(dst) = codes[k][0] | codes[k][1] << 16;
            } else {
              *reinterpret_cast<uint16_t*>(dst) = (uint16_t)codes[k][0];
            }
          }
        }
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(qfull0 + 8 * buffer);
      // On to the first tile of the next item of this share.
      left -= tiles;
      c.tile = c.seq.tiles - 1;
      if (left > 0) c.next(a);
    }
  } else if (count > 0 && warp < 2 * kGroupWarps) {
    // ---------------- softmax: lane = token of the tile ----------------
    // Two groups of four warps take alternate tiles, each with its own reference, sum and output
    // accumulator; they meet at the end of a segment.  A wait that runs out ends the warp's tiles,
    // and the vote at the end of the segment ends both groups together.
    const int group = warp / kGroupWarps, quarter = warp % kGroupWarps;
    const int token = quarter * 32 + lane;  // within the tile; quarter = its scale block
    const uint32_t lane_t = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_t = lane_t + group * C::kN;
    const uint32_t sfull = sfull0 + 8 * group, vsync = vsync0 + 8 * group, sread = sread0 + 8 * group;
    // Weights are stored four tokens at a time: the lane's are tokens lane & ~3 .. | 3 of row
    // lane % 4 of every four.
    uint8_t* p_s0 = p_tiles + group * C::kPBuffers * C::kPBytes + (lane & 3) * 128 + (token & 12);
    const uint32_t p_chunk = (token & 0x70) ^ ((lane & 3) << 4);
    const uint32_t turn1 = lane & 1 ? 0x3715 : 0x6240, turn2 = lane & 2 ? 0x3276 : 0x5410;
    float* my_max = red_max + group * 4 * RP;
    bool failed = false;
    uint32_t done = 0;     // tiles this group has taken
    uint32_t syncs = 0;    // times the four warps of the group have met
    uint32_t votes = 0;    // of them, to ask for another reference
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
      if (!failed) failed = !__all_sync(0xffffffffu, bounded_wait(bar, parity, abort_flag, a.status, code));
    };
    // The output of the group's tile `number`, one of its last kPBuffers.
    auto wait_output = [&](uint32_t number, int code) {
      wait(pvdone0 + 8 * (group * C::kPBuffers + number % C::kPBuffers), number / C::kPBuffers & 1u, code);
    };
    for (int segment = 0, i0 = 0; i0 < count; ++segment) {
      wait(qfull0 + 8 * (segment % kQueries), (uint32_t)(segment / kQueries) & 1u, 407);
      const Segment<RP>& seg = segments[segment % kQueries];
      const int tiles = failed ? 0 : seg.tiles, length = seg.length;
      const int64_t first_position = seg.first_position;
      float ref = -INFINITY;  // of row lane % RP, the same in the four warps
      const int j0 = (group ^ i0) & 1;
#pragma unroll 1
      for (int j = j0; j < tiles; j += 2, ++done) {
        const int i = i0 + j;
        const int t0 = (seg.tile + j) * kKvTile;
        const int held = min(kKvTile, length - t0);  // tokens of this tile that exist
        wait(sfull, done & 1u, 409);
        // PV of this group's tile kPBuffers before, i - 2 * kPBuffers, has read the weights that this
        // tile's replace.  It also shows that V of tile i - kValueSlots, which had this tile's slot,
        // has landed: copies land in any order, and one phase further back the parity would be the
        // same.
        if (done >= C::kPBuffers) wait_output(done - C::kPBuffers, 410);
        const uint32_t weights = group * C::kPBuffers + done % C::kPBuffers;
        uint8_t* p_s = p_s0 + done % C::kPBuffers * C::kPBytes;
        const int slot = C::kKeySlots + i % C::kValueSlots;
        wait(full0 + 8 * slot, (uint32_t)(i / C::kValueSlots) & 1u, 408);
        if (failed) break;
        ptx::tc_fence_after();
        const bool named = (slot_named[slot] >> quarter & 1u) != 0;
        const bool here = named && token < held, full = named && (quarter + 1) * 32 <= held;
        if (!full) {
          // Rows of V without a token may hold anything, NaN among them, and 0 * NaN is NaN.
          uint8_t* v_s = slots + slot * C::kSlotBytes;
          const int from = named ? max(0, held - quarter * 32) : 0;
          for (int at16 = from * (D / 16) + lane; at16 < 32 * (D / 16); at16 += 32) {
            const int t = at16 / (D / 16), piece = at16 % (D / 16);
            const int sub = piece / (C::kRowBytes / 16), in_row = piece % (C::kRowBytes / 16);
            *reinterpret_cast<uint4*>(v_s + sub * C::kSubBytes + (quarter * 32 + t) * C::kRowBytes +
                                      in_row * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        const bool bounded = a.causal && t0 + held - 1 > first_position;  // some row does not see all
        if (bounded) {
          __syncwarp();
          clear_nan<D>(slots + slot * C::kSlotBytes, quarter * 32, 32, t0, nan_table + (segment & 1) * D,
                       nan_flag + (segment & 1), lane);
        }
        float my_top = -INFINITY;  // of row lane % RP in this warp's 32 tokens
#pragma unroll
        for (int c0 = 0; c0 < RP; c0 += C::kChunk) {
          float s[C::kChunk];
#pragma unroll
          for (int r0 = 0; r0 < C::kChunk; r0 += 8) {
            uint32_t raw[TERMS][8];
#pragma unroll
            for (int k = 0; k < TERMS; ++k) ptx::tmem_ld_x8(s_t + k * RP + c0 + r0, raw[k]);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              float v = __uint_as_float(raw[TERMS - 1][n]);
#pragma unroll
              for (int k = TERMS - 2; k >= 0; --k) v = v * 0.0625f + __uint_as_float(raw[k][n]);
              s[r0 + n] = v * seg.scale[c0 + r0 + n];
            }
          }
          if (c0 + C::kChunk == RP) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(sread);
          }
          if (!full) {
#pragma unroll
            for (int r = 0; r < C::kChunk; ++r)
              if (!here) s[r] = -INFINITY;
          }
          if (bounded) {
#pragma unroll
            for (int r = 0; r < C::kChunk; ++r)
              if (t0 + token > first_position + (c0 + r) / a.group) s[r] = -INFINITY;
          }
#pragma unroll
          for (int r = 0; r < C::kChunk; r += 4) {
            float p[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              // To the nearest power of two: the largest weight is in (181, 363).  Where nothing is
              // seen (-inf) the lowest finite base keeps the weights zero.
              const float top = rintf(ptx::warp_max(s[r + n]));
              if (lane % RP == c0 + r + n) my_top = top;
              p[n] = ptx::exp2_approx(s[r + n] - (fmaxf(top, -FLT_MAX) - kWeightLog2));
            }
            uint32_t lo[TERMS], hi[TERMS];
            e4m3_terms_half<TERMS>(__floats2half2_rn(p[0], p[1]), lo);
            e4m3_terms_half<TERMS>(__floats2half2_rn(p[2], p[3]), hi);
#pragma unroll
            for (int k = 0; k < TERMS; ++k) {
              // This token's bytes of four rows become four tokens' bytes of row lane % 4.
              uint32_t w = __byte_perm(lo[k], hi[k], 0x5410);
              w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 1), turn1);
              w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 2), turn2);
              const int col = k * RP + c0 + r;  // a multiple of four; the lane's is col + lane % 4
              *reinterpret_cast<uint32_t*>(p_s + col * 128 + (p_chunk ^ ((col & 7) << 4))) = w;
            }
          }
        }
        // Does any row of the four warps need another reference?
        volatile int* asked = ask_flag + group * 2 + (votes++ & 1u);
        const bool ask = __any_sync(0xffffffffu, my_top > ref + kMostLog2);
        if (lane == 0) {
          if (ask) *asked = 1;
          ptx::mbar_arrive(vsync);
        }
        wait(vsync, syncs & 1u, 413);
        ++syncs;
        if (!failed && *asked != 0) {
          // The first tokens that a row sees, or a maximum far above its reference: the four
          // warps agree on a new one.
          if (lane < RP) my_max[quarter * RP + lane] = my_top;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(vsync);
          wait(vsync, syncs & 1u, 414);
          ++syncs;
          if (quarter == 0 && lane == 0) *asked = 0;  // not used by the next vote, but the one after
          const int r = lane % RP;
          const float m = fmaxf(fmaxf(my_max[r], my_max[RP + r]),
                                fmaxf(my_max[2 * RP + r], my_max[3 * RP + r]));
          const bool up = m > ref + kMostLog2;
          const float f = up ? pow2_whole(ref - m) : 1.0f;
          if (up) ref = m;
          if (j != j0 && !failed) {
            // What has been added up so far shrinks.
            wait_output(done - 1, 412);
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < C::kN; c0 += 8) {
              float g[8];
#pragma unroll
              for (int n = 0; n < 8; ++n) g[n] = __shfl_sync(0xffffffffu, f, (c0 + n) % RP);
#pragma unroll
              for (int h = 0; h <= C::kHalves; ++h) {
                uint32_t o[8];
                const uint32_t at_o = lane_t + c0 + (h < C::kHalves
                                                         ? C::kOCol + (group * C::kHalves + h) * C::kN
                                                         : C::kLCol + group * C::kN);
                ptx::tmem_ld_x8(at_o, o);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int n = 0; n < 8; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * g[n]);
                ptx::tmem_st_x8(at_o, o);
              }
            }
            ptx::tmem_st_wait();
          }
        }
        // 2^(top - ref), between 2^-126 and 2^16: its exponent field is the UE8M0 code.
        const uint32_t my_code =
            my_top == -INFINITY ? 127u : __float_as_uint(pow2_whole(my_top - ref)) >> 23;
        if (failed) break;
        // Scale atom of the weights: column col is row col % 32 of the atom, word col / 32, and
        // this warp's tokens are byte `quarter` of the word.
#pragma unroll
        for (int col0 = 0; col0 < C::kN; col0 += 32) {
          const int col = col0 + lane;
          uint32_t code = my_code;
          if constexpr (RP == 24) code = __shfl_sync(0xffffffffu, my_code, col % RP);
          if (col < C::kN) p_sf[weights * 512 + lane * 16 + (col0 / 32) * 4 + quarter] = (uint8_t)code;
        }
        ptx::fence_proxy_async();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(pfull0 + 8 * weights);
      }
      // ---- the output of this CTA's tiles of the item ----
      if (quarter == 0 && lane < RP) red_top[group * RP + lane] = ref;
      if (j0 < tiles) wait_output(done - 1, 411);
      failed = ptx::barrier_any(3, 2 * kGroupWarps * 32, failed);
      if (failed) break;
      ptx::tc_fence_after();
      // The table of the segment before this one is of the next.
      const int* nan_from = nan_table + (segment & 1) * D;
      const bool nans = nan_flag[segment & 1] != 0;
      if (threadIdx.x < D) nan_table[(segment + 1 & 1) * D + threadIdx.x] = INT_MAX;
      if (threadIdx.x == 0) nan_flag[segment + 1 & 1] = 0;
      // Lane r: what row r's two accumulators are multiplied by (RP <= 32).
      float factor_a = 0.0f, factor_b = 0.0f;
      if (lane < RP) {
        const float ta = red_top[lane], tb = red_top[RP + lane], most = fmaxf(ta, tb);
        // A reference is -inf where the row saw nothing (NaN scores leave it there too).
        factor_a = ta == most ? 1.0f : pow2_whole(ta - most);
        factor_b = tb == most ? 1.0f : pow2_whole(tb - most);
      }
      // A share that begins inside an item uses the CTA's first partial slot for it, one that ends
      // inside the second.
      float* part = a.partials +
                    (int64_t)(2 * blockIdx.x + (seg.tile != 0 ? 0 : 1)) * C::kPartialFloats;
      const int rows = seg.rows;
      const bool whole = seg.whole != 0;
      // The groups share the output by halves of head_dim, or by eight rows.
#pragma unroll 1
      for (int unit = group; unit < C::kHalves * (RP / 8); unit += 2) {
        const int h = unit % C::kHalves, r0 = unit / C::kHalves * 8;
        if (r0 >= rows) continue;
        float v[8], l[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) v[n] = l[n] = 0.0f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g == 1 && tiles < 2) break;  // only one group had a tile
          const int owner = (g ^ i0) & 1;  // group of the segment's tile g
          uint32_t raw[TERMS][8], sums[TERMS][8];
#pragma unroll
          for (int k = 0; k < TERMS; ++k) {
            ptx::tmem_ld_x8(lane_t + C::kOCol + (owner * C::kHalves + h) * C::kN + k * RP + r0, raw[k]);
            ptx::tmem_ld_x8(lane_t + C::kLCol + owner * C::kN + k * RP + r0, sums[k]);
          }
          ptx::tmem_ld_wait();
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            float x = __uint_as_float(raw[TERMS - 1][n]), y = __uint_as_float(sums[TERMS - 1][n]);
#pragma unroll
            for (int k = TERMS - 2; k >= 0; --k) {
              x = x * 0.0625f + __uint_as_float(raw[k][n]);
              y = y * 0.0625f + __uint_as_float(sums[k][n]);
            }
            const float f = __shfl_sync(0xffffffffu, owner ? factor_b : factor_a, r0 + n);
            v[n] += x * f;
            l[n] += y * f;
          }
        }
        if (!whole && h == 0 && quarter == 0) {
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            if (lane != n) continue;
            const int r = r0 + n;
            part[RP * D + 2 * r] = fmaxf(red_top[r], red_top[RP + r]);
            part[RP * D + 2 * r + 1] = l[n];
          }
        }
        const int d = h * 128 + token;
        if (nans && d < D) {
#pragma unroll
          for (int n = 0; n < 8; ++n)
            if (nan_from[d] <= first_position + (r0 + n) / a.group) v[n] = NAN;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int r = r0 + n;
          if (r < rows && d < D) {
            if (whole) {
              T* out = static_cast<T*>(a.out) + seg.out[r] + d;
              const float o = l[n] == 0.0f ? 0.0f : __fdividef(v[n], l[n]);
              if constexpr (TERMS == 2) *out = __float2bfloat16_rn(o);
              else *out = __float2half_rn(o);
            } else {
              part[r * D + d] = v[n];
            }
          }
        }
      }
      ptx::tc_fence_before();
      i0 += tiles;
      // The accumulators, sums and the segment's description have been read.
      if (i0 < count && ptx::barrier_any(3, 2 * kGroupWarps * 32, false)) break;
      if (lane == 0) ptx::mbar_arrive(qempty0 + 8 * (segment % kQueries));
    }
  }

  if constexpr (kToldBorders<RP>) {
    // Now that nothing waits for it.
    if (warp == kValueWarp && lane == 0 && a.whole_items == 0 && blockIdx.x + 1 < gridDim.x)
      borders_of(a)[blockIdx.x] = border_of(a, share_of(share_smem[2], (int)gridDim.x), (int)blockIdx.x,
                                            share_smem[3], start[1].b, start[1].head);
  }

  // ---------------- teardown ----------------
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // Give copies and MMAs still in flight time to land before the CTA's shared
    // and tensor memory are handed back.
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  if (warp == kScoreWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the partial rows of every item whose tiles went to more than one CTA, in the order of the
// tiles.  One CTA per row and border between two shares; the first border inside an item has it.
template <int D, int RP, int TERMS>
__global__ void __launch_bounds__(kJoinThreads)
kv_decode_join_kernel(const AttentionArgs a, int grid) {
  using C = DecodeCfg<D, RP, TERMS>;
  using T = typename std::conditional<TERMS == 2, __nv_bfloat16, __half>::type;
  constexpr int kColumns = D / 4;                     // four values a thread
  constexpr int kShares = kJoinThreads / kColumns;    // threads that share a column's parts
  __shared__ float factor[kSms];
  __shared__ float4 acc[kJoinThreads];
  const int c0 = (int)blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  Border item;
  if constexpr (kToldBorders<RP>) {
    ptx::grid_dependency_wait();
    item = borders_of(a)[c0];
  } else {
    // The lengths are final before the main kernel starts.
    __shared__ Border found;
    if (tid < 32) {
      const Share s = share_of(warp_total_units(a, lane) * a.cache.kv_heads, grid);
      Cursor c{};
      int64_t begin = 0;
      if (c0 + 1 < s.ctas) warp_locate(a, share_begin(s, c0 + 1), false, lane, &c, &begin);
      if (lane == 0) found = border_of(a, s, c0, begin, c.b, c.head);
    }
    __syncthreads();
    item = found;
    ptx::grid_dependency_wait();
  }
  const int parts = item.parts, head = item.head;
  if (parts == 1 || r >= item.rows) return;
  // The first CTA began before this item or with it, the others inside it.
  const int64_t first = 2 * c0 + 1, later = 2 * c0;  // slot of part p: p == 0 ? first : later + 2 p
  auto part_of = [&](int p) {
    return a.partials + (p == 0 ? first : later + 2 * p) * C::kPartialFloats;
  };
  // Every warp the same factors and the same sum in the same order.
  float top = -INFINITY, l = 0.0f;
  float2 mine[(kSms + 31) / 32];
#pragma unroll
  for (int i = 0; i < (kSms + 31) / 32; ++i) {
    const int p = i * 32 + lane;
    mine[i] = p < parts ? *reinterpret_cast<const float2*>(part_of(p) + RP * D + 2 * r)
                        : make_float2(-INFINITY, 0.0f);
    top = fmaxf(top, mine[i].x);
  }
  top = ptx::warp_max(top);
#pragma unroll
  for (int i = 0; i < (kSms + 31) / 32; ++i) {
    const int p = i * 32 + lane;
    const float f = mine[i].x == top ? 1.0f : pow2_whole(mine[i].x - top);
    l += p < parts ? f * mine[i].y : 0.0f;
    if (tid < 32 && p < parts) factor[p] = f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  __syncthreads();
  const int column = tid % kColumns, share = tid / kColumns;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int p = share; p < parts; p += kShares) {
    const float4 v = *reinterpret_cast<const float4*>(part_of(p) + r * D + column * 4);
    const float f = factor[p];
    o.x += f * v.x;
    o.y += f * v.y;
    o.z += f * v.z;
    o.w += f * v.w;
  }
  acc[tid] = o;
  __syncthreads();
  if (share != 0) return;
#pragma unroll
  for (int g = 1; g < kShares; ++g) {
    const float4 v = acc[g * kColumns + column];
    o.x += v.x;
    o.y += v.y;
    o.z += v.z;
    o.w += v.w;
  }
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.out) + (item.row + r / a.group) * a.out_token_stride +
           (int64_t)(head * a.group + r % a.group) * a.out_head_stride + column * 4;
  const float v[4] = {o.x * scale, o.y * scale, o.z * scale, o.w * scale};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TERMS == 2) out[i] = __float2bfloat16_rn(v[i]);
    else out[i] = __float2half_rn(v[i]);
  }
}

bool use_pdl() {
  static const bool enabled = []() {
    const char* env = std::getenv("MXFP6_B200_PDL");
    return env == nullptr || env[0] != '0';
  }();
  return enabled;
}

template <int D, int RP, int TERMS>
int launch(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttentionArgs& a, int grid,
           cudaStream_t stream) {
  using C = DecodeCfg<D, RP, TERMS>;
  static bool configured[64] = {};
  int device = 0;
  MX_CUDA(cudaGetDevice(&device));
  if (device >= 64 || !configured[device]) {
    MX_CUDA(cudaFuncSetAttribute(kv_decode_kernel<D, RP, TERMS>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    if (device < 64) configured[device] = true;
  }
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)grid);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = C::kSmemBytes;
  config.stream = stream;
  config.attrs = attribute;
  config.numAttrs = use_pdl() ? 1 : 0;
  MX_CUDA(cudaLaunchKernelEx(&config, kv_decode_kernel<D, RP, TERMS>, tm_k, tm_v, a));
  if (a.whole_items != 0 || grid == 1) return kOk;  // nothing was cut
  config.gridDim = dim3((unsigned)(grid - 1), (unsigned)a.max_rows);
  config.blockDim = dim3(kJoinThreads);
  config.dynamicSmemBytes = 0;
  MX_CUDA(cudaLaunchKernelEx(&config, kv_decode_join_kernel<D, RP, TERMS>, a, grid));
  return kOk;
}

template <int D, int TERMS>
int launch_rows(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttentionArgs& a, int grid,
                cudaStream_t stream) {
  if (a.max_rows <= 8) return launch<D, 8, TERMS>(tm_k, tm_v, a, grid, stream);
  if (a.max_rows <= 16) return launch<D, 16, TERMS>(tm_k, tm_v, a, grid, stream);
  if constexpr (most_rows(D, TERMS) > 24)
    if (a.max_rows <= 24) return launch<D, 24, TERMS>(tm_k, tm_v, a, grid, stream);
  return launch<D, most_rows(D, TERMS), TERMS>(tm_k, tm_v, a, grid, stream);
}

}  // namespace

// CTAs of a decode launch: at most one per SM and no more than there can be work for.
int kv_decode_grid(int64_t batch, int kv_heads, int64_t max_context) {
  const int64_t tiles = ceil_div64(max_context < 1 ? 1 : max_context, kKvTile);
  const int64_t items = batch * kv_heads;
  const int64_t want =
      tiles <= kWholeTiles ? items : ceil_div64(items * (tiles + 1), kMinUnits);
  return (int)(want < kSms ? want : kSms);
}

int kv_decode_rows(int head_dim, int dtype) { return most_rows(head_dim, dtype == kBF16 ? 2 : 3); }

int64_t kv_decode_workspace(int64_t batch, int kv_heads, int head_dim, int dtype, int rows,
                            int64_t max_context) {
  const int grid = kv_decode_grid(batch, kv_heads, max_context);
  if (grid == 1 || max_context <= kWholeTiles * kKvTile) return 0;
  const int rp = variant_rows(rows, head_dim, dtype == kBF16 ? 2 : 3);
  return kSms * (int64_t)sizeof(Border) + (int64_t)grid * 2 * (rp * head_dim + 2 * rp) * 4;
}

// Sequences with at most a.max_rows <= kv_decode_rows() rows (tokens x group); others are left
// alone.
int launch_kv_decode(const AttentionArgs& args, int dtype, cudaStream_t stream) {
  AttentionArgs a = args;
  // Measured: about 2.6 us beside 1.5 us a tile of 256, 3.1 us beside 1.1 us a tile of 128.
  a.item_units = a.cache.head_dim == 256 ? 2 : 3;
  a.whole_items = (int64_t)a.batch.table_width * a.cache.page_size <= kWholeTiles * kKvTile;
  static_assert(sizeof(Border) % 16 == 0, "partial rows stay aligned");
  a.partials = reinterpret_cast<float*>(reinterpret_cast<Border*>(args.partials) + kSms);
  CUtensorMap tm_k, tm_v;
  if (int rc = make_kv_map(&tm_k, a.cache.k_values, a.cache)) return rc;
  if (int rc = make_kv_map(&tm_v, a.cache.v_values, a.cache)) return rc;
  const int grid = kv_decode_grid(a.batch.batch, a.cache.kv_heads,
                                  (int64_t)a.batch.table_width * a.cache.page_size);
  const int d = a.cache.head_dim;
  if (dtype == kBF16) {
    if (d == 64) return launch_rows<64, 2>(tm_k, tm_v, a, grid, stream);
    if (d == 128) return launch_rows<128, 2>(tm_k, tm_v, a, grid, stream);
    return launch_rows<256, 2>(tm_k, tm_v, a, grid, stream);
  }
  if (d == 64) return launch_rows<64, 3>(tm_k, tm_v, a, grid, stream);
  if (d == 128) return launch_rows<128, 3>(tm_k, tm_v, a, grid, stream);
  return launch_rows<256, 3>(tm_k, tm_v, a, grid, stream);
}

}  // namespace mx
