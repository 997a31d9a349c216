// Attention of many new rows per sequence over the paged 8-bit cache (prompts, prompt chunks).
//
// S = Q K^T and O = P V on 128 rows (new tokens x query heads of a key head, flattened) by 128
// cached tokens.  K and V are read by tcgen05.mma as they lie in the pages (TMA tiles, block
// scales in hardware, V as an MN-major operand); Q and P are E4M3 terms (kv_attention.cuh): a
// BF16 product is two passes at the 8-bit rate, so the tensor cores bound it at what they give 16-bit
// operands, with half the bytes per cached token and no conversion of a cached value anywhere.  An
// FP16 product is three passes, half as much again.
//
//  * The terms of a product accumulate into the same tensor memory: their factors 1, 1/16, 1/256
//    are block scales of the A operand.
//  * Online softmax as in the decode kernel: a row's weights are taken relative to the largest
//    score of each block of 32 tokens, rounded to a power of two, and that power relative to the
//    row's reference is the block scale of P.  No maximum crosses threads and the output is not
//    rescaled, except where a block exceeds the reference by more than 2^16.
//  * Warps: 0-15 softmax (a thread holds the 32 scores of one row and scale block; with eight warps
//    of 64 scores the waits and loads of a tile did not overlap its exponentials), 16 TMA, 17 MMA,
//    18 copies the next item's rows to where its terms will be, as soon as the last scores of the
//    item before are out (bulk copies: loads into the registers of a few warps, at the latency that
//    memory has under this kernel, took 10 us an item); the softmax warps turn them into terms.
//    Scores of tile j + 1 are issued before the output of tile j.
//  * Work: the list of (sequence, row tile, key head) with its tiles of cached tokens is cut into
//    equal shares, one per SM; an item that is cut leaves partial rows, which a second kernel
//    joins in the order of the tiles.
//
// Measured inside a CUDA graph: a prompt of 8192 tokens, 24 query and 4 key heads of 256: 710 to 770 us,
// back to back 830 (boxes and clocks differ), 0.99 to 1.16 PFLOP/s of 16-bit products, tensor pipes 57 %
// active at 1.64 GHz; in FP16 1040 to 1100 us.  The scores' product reads both operands from shared
// memory, 128 bytes a clock, which is all it gives, beside the copies into the ring: without any
// exponential the time is the same, with half the products 690 us.
// Five chunks of 1500 tokens over 12000, 8 rows per key head of 128: 306 to 325 us, 0.58 to 0.62 PFLOP/s
// (FP16 390 to 400 us).  Here no unit is at its limit: issue slots 64 %, ALU 56 %, special functions 32 %,
// tensor pipes 31 %, shared memory 17 % of their peaks; four softmax warps a scheduler do not cover the
// chain of a tile (scores, maximum, exponentials, conversions, weights through shared memory, product).
// Without exponentials and E4M3 terms 252 us.
// Tried and left: the next rows' terms before the last rows' output (790 against 746 us, heads of 256).
#include "kv_attention.cuh"

#include <cfloat>
#include <climits>
#include <cstdlib>

namespace mx {
namespace {

constexpr int kThreads = 608;
constexpr int kSoftmaxWarps = 16;
constexpr int kTmaWarp = 16, kMmaWarp = 17, kQueryWarp = 18;
constexpr int kRows = 128;            // rows of an item
constexpr float kWeightLog2 = 8.0f;   // weights are scaled by 256 before they become E4M3 terms
constexpr float kMostLog2 = 16.0f;    // a block may exceed the reference by 2^16
constexpr int kSms = 148;
// What an item costs beside its tiles: about 8 us, a tile 1.7 us.  8192-token prompt, heads of 256: with
// 3 units 940 us, 4 810, 5 740, 6 750; five chunks, heads of 128: 329, 322, 327, 329 us.  Other lengths
// were not tried; part of the first row may be how 8192 tokens divide.
constexpr int kItemUnits = 5;
constexpr int kMinUnits = 4;          // units a CTA takes at least

template <int D, int TERMS>
struct PrefillCfg {
  static constexpr int kRowBytes = D < 128 ? D : 128;
  static constexpr int kSubs = D / kRowBytes;
  static constexpr int kSubBytes = kKvTile * kRowBytes;  // also of a Q sub-tile: 128 rows
  static constexpr int kSlotBytes = kKvTile * D;
  static constexpr int kQBytes = TERMS * kRows * D;
  // A head of 256 leaves room for one score tile in tensor memory and one P.  Two terms of P fit
  // tensor memory beside it, which frees shared memory for a fourth tile of keys and values: with
  // three, a tile came 0.4 us after the tensor cores wanted it.
  static constexpr int kBuffers = D == 256 ? 1 : 2;
  static constexpr bool kTmemP = D == 256 && TERMS == 2;
  static constexpr int kPBytes = kTmemP ? 0 : TERMS * kRows * kKvTile;
  static constexpr int kStageWarp = kTmemP ? 1024 : 2048;  // bytes a warp stages outputs in
  static constexpr int kStageBytes = kTmemP ? kSoftmaxWarps * kStageWarp : 0;  // else in P
  static constexpr int kFixedBytes = 12288;
  static constexpr int kBudget = 227 * 1024 - 1024;
  static constexpr int kFit = (kBudget - kFixedBytes - kStageBytes - kQBytes - kBuffers * kPBytes) / (kSlotBytes + 512);
  static constexpr int kSlots = kFit > 8 ? 8 : kFit;
  static_assert(kSlots >= 3 || (kSlots == 2 && kBuffers == 1), "see kEarlyClear");
  // The softmax warps wait for a V tile too, where rows of it have to be cleared.  Copies land in
  // any order, and while the tile that had the slot before is still missing, the slot's barrier
  // stands one phase further back, where the parity is the same; so they have to know that it has
  // landed.  Tile i's V has place 2 i + 2 (K0, K1, V0, K2, V1, ...).  Before its scores they know it
  // of the places up to K of tile i - 1, five places back, and of V of tile i - 2, four places back,
  // where one buffer made them wait for that output; with its scores, up to its K, three places
  // back; with the last tile's output, two places back.
  static constexpr bool kEarlyClear = kSlots >= (kBuffers == 1 ? 4 : 5);
  static constexpr int kSmemBytes =
      1024 + kSlots * (kSlotBytes + 512) + kQBytes + kBuffers * kPBytes + kStageBytes + kFixedBytes;
  static constexpr int kOCol = kBuffers * kKvTile;
  static constexpr int kSfCol = kOCol + D;
  // Scales: constants per term; per buffer (what an MMA may still read is not overwritten) keys,
  // values (8 for 256 rows of B), weights per term.
  static constexpr int kSfTerm = kSfCol, kSfSets = kSfTerm + 4 * TERMS;
  static constexpr int kSfV = 4, kSfP = 12, kSfSet = 12 + 4 * TERMS;
  static constexpr int kPCol = (kSfSets + kBuffers * kSfSet + 15) / 16 * 16;  // [term][32 columns]
  static_assert(kPCol + (kTmemP ? TERMS * 32 : 0) <= 512, "tensor memory");
  static constexpr uint64_t kSwizzle = kRowBytes == 128 ? ptx::kSwizzle128 : ptx::kSwizzle64;
  static constexpr int kGroup = 8 * kRowBytes;
  static constexpr int kPartialFloats = kRows * D + 2 * kRows;
};

struct Share {
  int64_t total;
  int ctas;
};
__device__ __forceinline__ int64_t share_begin(const Share& s, int cta) {
  return s.total * cta / s.ctas;
}
__device__ __forceinline__ Share share_of(int64_t total, int grid) {
  Share s;
  s.total = total;
  const int64_t want = (total + kMinUnits - 1) / kMinUnits;
  s.ctas = (int)(want < grid ? (want < 1 ? 1 : want) : grid);
  return s;
}

// A sequence: rows of q are new tokens x group, in tiles of 128.
struct Sequence {
  int64_t row;             // first token row
  int64_t first_position;  // of its first new token
  int rows;                // new tokens x group
  int length;              // cached tokens
};
__device__ __forceinline__ Sequence load_sequence(const AttentionArgs& a, int b) {
  const KvSpan s = kv_span(a.batch, a.cache.page_size, b);
  Sequence q;
  q.row = s.row;
  q.first_position = (int64_t)a.batch.seq_lens[b] - s.rows;
  const int64_t rows = (int64_t)s.rows * a.group;
  q.rows = rows > a.min_rows ? (int)rows : 0;  // shorter ones are the decode kernel's
  q.length = s.length;
  return q;
}
// Tiles of cached tokens that row tile t sees (one even if it sees none: it writes zeros).
__device__ __forceinline__ int tiles_of(const AttentionArgs& a, const Sequence& q, int t) {
  int64_t see = q.length;
  if (a.causal) {
    const int last = min(q.rows - 1, kRows * t + kRows - 1) / a.group;
    const int64_t upto = q.first_position + last + 1;
    see = upto < see ? upto : see;
  }
  return see <= 0 ? 1 : (int)((see + kKvTile - 1) / kKvTile);
}

// An item and a tile of it.
struct Place {
  int b, t, head, tile;
};

// Units of all items, by a full warp.
__device__ __forceinline__ int64_t warp_total_units(const AttentionArgs& a, int lane) {
  int64_t units = 0;  // of this lane's row tiles, one key head
  for (int b0 = 0; b0 < a.batch.batch; b0 += 32) {
    Sequence mine{};
    if (b0 + lane < a.batch.batch) mine = load_sequence(a, b0 + lane);
    unsigned todo = __ballot_sync(0xffffffffu, mine.rows > 0);
    while (todo != 0) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      Sequence q;
      q.first_position = __shfl_sync(0xffffffffu, mine.first_position, l);
      q.rows = __shfl_sync(0xffffffffu, mine.rows, l);
      q.length = __shfl_sync(0xffffffffu, mine.length, l);
      const int row_tiles = (q.rows + kRows - 1) / kRows;
      for (int t = lane; t < row_tiles; t += 32) units += tiles_of(a, q, t) + kItemUnits;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
  return units * a.cache.kv_heads;
}

// The first tile at or behind unit `at`, in the order sequence, row tile, head, by a full warp:
// returns its number in the list of all tiles and, in all lanes, its place and the first unit of
// its item.
__device__ __forceinline__ int64_t warp_locate(const AttentionArgs& a, int64_t at, int lane,
                                               Place* place, int64_t* item_begin) {
  int64_t units = 0, tiles = 0;  // of all heads before this group of 32 row tiles
  const int heads = a.cache.kv_heads;
  for (int b0 = 0; b0 < a.batch.batch; b0 += 32) {
    Sequence mine{};
    if (b0 + lane < a.batch.batch) mine = load_sequence(a, b0 + lane);
    unsigned todo = __ballot_sync(0xffffffffu, mine.rows > 0);
    while (todo != 0) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      Sequence q;
      q.first_position = __shfl_sync(0xffffffffu, mine.first_position, l);
      q.rows = __shfl_sync(0xffffffffu, mine.rows, l);
      q.length = __shfl_sync(0xffffffffu, mine.length, l);
      const int row_tiles = (q.rows + kRows - 1) / kRows;
      for (int t0 = 0; t0 < row_tiles; t0 += 32) {
        const int t = t0 + lane;
        const int n = t < row_tiles ? tiles_of(a, q, t) : 0;
        // A tile count is below 2^23 (2^30 tokens), so 32 of them fit 32 bits.
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += other;
        }
        const int items = min(lane + 1, row_tiles - t0);
        const int64_t units_upto = ((int64_t)upto + (int64_t)items * kItemUnits) * heads;
        const unsigned reached = __ballot_sync(0xffffffffu, n > 0 && units + units_upto > at);
        if (reached != 0) {
          const int k = __ffs(reached) - 1;
          const int count = __shfl_sync(0xffffffffu, n, k);
          const int64_t per_item = count + kItemUnits;
          const int64_t first = units + __shfl_sync(0xffffffffu, units_upto, k) - per_item * heads;
          const int64_t into = at > first ? at - first : 0;
          place->b = b0 + l;
          place->t = t0 + k;
          place->head = (int)(into / per_item);
          const int64_t in_item = into % per_item - kItemUnits;
          place->tile = in_item > 0 ? (int)in_item : 0;
          *item_begin = first + into / per_item * per_item;
          return tiles + (int64_t)(__shfl_sync(0xffffffffu, upto, k) - count) * heads +
                 (int64_t)place->head * count + place->tile;
        }
        units += __shfl_sync(0xffffffffu, units_upto, 31);
        tiles += (int64_t)__shfl_sync(0xffffffffu, upto, 31) * heads;
      }
    }
  }
  return tiles;
}

// What the joining kernel is told about the border behind each CTA's share; in the workspace,
// before the partial rows.
struct Border {
  int b, t, head;
  int parts;  // CTAs over which the item goes, 1: nothing to join here
};
__device__ __forceinline__ Border* borders_of(const AttentionArgs& a) {
  return reinterpret_cast<Border*>(a.partials) - kSms;
}

// A place with its sequence, stepped from item to item.
struct Cursor {
  Place at;
  Sequence seq;
  int tiles;  // of the item
  __device__ __forceinline__ void load(const AttentionArgs& a) {
    seq = load_sequence(a, at.b);
    tiles = tiles_of(a, seq, at.t);
  }
  __device__ __forceinline__ void next_item(const AttentionArgs& a) {
    at.tile = 0;
    if (++at.head < a.cache.kv_heads) return;
    at.head = 0;
    if (kRows * ++at.t < seq.rows) {
      tiles = tiles_of(a, seq, at.t);
      return;
    }
    at.t = 0;
    do {
      if (++at.b >= a.batch.batch) {
        at.b = a.batch.batch - 1;
        break;
      }
      seq = load_sequence(a, at.b);
    } while (seq.rows == 0);
    tiles = tiles_of(a, seq, 0);
  }
};

// The tiles of one item that a CTA takes.
struct Segment {
  float scale[kRows];      // of the quantised rows, times the softmax scale and log2(e)
  int64_t row;             // first token row of the sequence
  int64_t first_position;  // of the sequence's first new token
  int rows;                // rows of the sequence
  int row0;                // first row of the item
  int length;
  int head;
  int tile;
  int tiles;
  int whole;
  int b;
  int all_named;           // every page of its tiles is in the block table
};

template <int D, int TERMS>
__global__ void __launch_bounds__(kThreads, 1)
kv_prefill_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const AttentionArgs a) {
  using C = PrefillCfg<D, TERMS>;
  using T = typename std::conditional<TERMS == 2, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* slots = smem;
  uint8_t* q_tiles = slots + C::kSlots * C::kSlotBytes;  // [term][sub][row][row bytes]
  uint8_t* p_tiles = q_tiles + C::kQBytes;               // [buffer][term][row][128 tokens]
  uint8_t* stages = p_tiles + C::kBuffers * C::kPBytes;  // where P is in tensor memory
  uint8_t* sf_tiles = stages + C::kStageBytes;
  uint8_t* fixed = sf_tiles + C::kSlots * 512;
  uint64_t* bars = reinterpret_cast<uint64_t*>(fixed);
  uint8_t* term_sf = fixed + 512;                        // [term] atoms of 1, 1/16, 1/256
  uint8_t* p_sf = term_sf + 3 * 512;                     // [buffer][term]
  Segment* segments = reinterpret_cast<Segment*>(p_sf + 6 * 512);  // two
  float* row_sum = reinterpret_cast<float*>(segments + 2);         // [block][row]
  float* row_top = row_sum + 4 * kRows;                            // [block][row]
  int* nan_from = reinterpret_cast<int*>(row_top + 4 * kRows);     // [head_dim], see clear_nan
  Cursor* start = reinterpret_cast<Cursor*>(nan_from + 256);
  int64_t* share_smem = reinterpret_cast<int64_t*>(start + 1);  // begin, end, all units, begin of the item at the end
  Place* next = reinterpret_cast<Place*>(share_smem + 4);  // where the next share begins
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(next + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ask_flag = abort_flag + 1;               // [quarter][2]
  volatile int* nan_seen = ask_flag + 8;
  static_assert(512 + 9 * 512 + 2 * sizeof(Segment) + 8 * kRows * 4 + 1024 + sizeof(Cursor) + 32 + sizeof(Place) + 8 + 36 <=
                    C::kFixedBytes,
                "fixed area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = ptx::smem_u32(bars);
  const uint32_t empty0 = full0 + 8 * C::kSlots;
  const uint32_t sfull0 = empty0 + 8 * C::kSlots;
  const uint32_t sread0 = sfull0 + 16;
  const uint32_t pfull0 = sread0 + 16;
  const uint32_t pvdone0 = pfull0 + 16;
  const uint32_t sdone0 = pvdone0 + 16;  // softmax has left a segment (by its parity)
  const uint32_t qraw = sdone0 + 16;     // an item's rows have been copied
  const uint32_t qfull = qraw + 8, qfree = qfull + 8;
  const uint32_t vsync0 = qfree + 8;     // four: the four warps of a lane quarter
  static_assert(8 * (2 * 8 + 10 + 3 + 4) <= 512, "barriers");

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) ask_flag[i] = 0;
    for (int s = 0; s < C::kSlots; ++s) {
      ptx::mbar_init(full0 + 8 * s, 2);  // the copies' bytes, and the scales
      ptx::mbar_init(empty0 + 8 * s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(sfull0 + 8 * i, 1);
      ptx::mbar_init(sread0 + 8 * i, kSoftmaxWarps);
      ptx::mbar_init(pfull0 + 8 * i, kSoftmaxWarps);
      ptx::mbar_init(pvdone0 + 8 * i, 1);
      ptx::mbar_init(sdone0 + 8 * i, kSoftmaxWarps);
    }
    ptx::mbar_init(qraw, 2);  // the copies' bytes, and the description
    ptx::mbar_init(qfull, kSoftmaxWarps);
    ptx::mbar_init(qfree, 1);
    for (int i = 0; i < 4; ++i) ptx::mbar_init(vsync0 + 8 * i, 4);
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
  }
  if (threadIdx.x < 3 * 128)
    reinterpret_cast<uint32_t*>(term_sf)[threadIdx.x] =
        threadIdx.x < 128 ? 0x7f7f7f7fu : threadIdx.x < 256 ? 0x7b7b7b7bu : 0x77777777u;
  ptx::fence_proxy_async();
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (warp < 2) {
    // Warp 0 finds the first tile of this CTA, warp 1 the first of the next.
    Place p{};
    int64_t begin = 0, tile = 0;
    const Share s = share_of(warp_total_units(a, lane), (int)gridDim.x);
    const int cta = (int)blockIdx.x + warp;
    if ((int)blockIdx.x < s.ctas && s.total > 0) tile = warp_locate(a, share_begin(s, cta), lane, &p, &begin);
    if (lane == 0) {
      share_smem[warp] = tile;
      if (warp == 0) {
        start->at = p;
      } else {
        share_smem[2] = s.total;
        share_smem[3] = begin;
        *next = p;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int count = (int)(share_smem[1] - share_smem[0]);  // tiles of this CTA
  const int per_page = a.cache.page_size / kKvBlock;

  if (count > 0 && warp == kTmaWarp) {
    // ---------------- TMA producer: K0, K1, V0, K2, V1, ... per segment ----------------
    Cursor c = *start;
    c.load(a);
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    const bool leads = (lane & 3) % per_page == 0;  // first block of a page in its tile
    const uint32_t page_bytes = (uint32_t)(a.cache.page_size * D);
    const uint32_t slots_s = ptx::smem_u32(slots) + (lane & 3) * kKvBlock * C::kRowBytes;
    auto copy = [&](bool is_v, int64_t lane_page, uint32_t lane_sf, int src) {
      ok = ok && __all_sync(0xffffffffu, bounded_wait(empty0 + 8 * slot, phase ^ 1u, abort_flag,
                                                      a.status, 501));
      if (!ok) return;
      const uint32_t bar = full0 + 8 * slot;
      const bool issue = (lane & ~3) == src && leads && lane_page >= 0;
      const uint32_t pages = __popc(__ballot_sync(0xffffffffu, issue));
      if (lane == src) ptx::mbar_arrive_expect_tx(bar, pages * page_bytes);
      __syncwarp();
      if (issue) {
#pragma unroll
        for (int s = 0; s < C::kSubs; ++s)
          ptx::tma_load_2d(slots_s + slot * C::kSlotBytes + s * C::kSubBytes, is_v ? &tm_v : &tm_k,
                           s * 128, (int)(lane_page * kKvBlock), bar);
      }
      // Scale atom: lane = row % 32.  Keys: 32 tokens are a word of rows; values: every row has
      // the factors of the four 32-token steps along K.
      uint32_t sf[kKvTileBlocks];
#pragma unroll
      for (int i = 0; i < kKvTileBlocks; ++i) sf[i] = __shfl_sync(0xffffffffu, lane_sf, src + i);
      const uint32_t all = sf[0] | sf[1] << 8 | sf[2] << 16 | sf[3] << 24;
      reinterpret_cast<uint4*>(sf_tiles + slot * 512)[lane] =
          is_v ? make_uint4(all, all, all, all)
               : make_uint4(sf[0] * 0x01010101u, sf[1] * 0x01010101u, sf[2] * 0x01010101u,
                            sf[3] * 0x01010101u);
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar);
      if (++slot == C::kSlots) {
        slot = 0;
        phase ^= 1u;
      }
    };
    for (int left = count; ok && left > 0;) {
      const int tiles = min(left, c.tiles - c.at.tile);
      // Lane l looks up block l % 4 of tile l / 4 of a group of eight tiles.
      auto lookup_page = [&](int j) -> int64_t {
        const int block = (c.at.tile + j + (lane >> 2)) * kKvTileBlocks + (lane & 3);
        if (j + (lane >> 2) >= tiles || block * kKvBlock >= c.seq.length) return -1;
        const int64_t p = kv_page(a.batch, a.cache, c.at.b, block);
        return p < 0 ? -1 : (p * a.cache.kv_heads + c.at.head) * per_page + block % per_page;
      };
      int64_t page = lookup_page(0), next_page = -1, last_page = -1;
      uint32_t k_sf = 127, v_sf = 127, next_k = 127, next_v = 127, last_v = 127;
      if (page >= 0) {
        k_sf = a.cache.k_scales[page];
        v_sf = a.cache.v_scales[page];
      }
      for (int j0 = 0; ok && j0 < tiles; j0 += 8) {
        if (j0 + 8 < tiles) next_page = lookup_page(j0 + 8);
        for (int j = 0; ok && j < 8 && j0 + j < tiles; ++j) {
          copy(false, page, k_sf, 4 * j);
          if (j > 0) copy(true, page, v_sf, 4 * (j - 1));
          else if (j0 > 0) copy(true, last_page, last_v, 28);
          if (j == 3 && j0 + 8 < tiles) {
            next_k = next_page >= 0 ? a.cache.k_scales[next_page] : 127u;
            next_v = next_page >= 0 ? a.cache.v_scales[next_page] : 127u;
          }
        }
        last_page = page;
        last_v = v_sf;
        page = next_page;
        k_sf = next_k;
        v_sf = next_v;
      }
      copy(true, last_page, last_v, 4 * ((tiles - 1) & 7));
      left -= tiles;
      if (left > 0) c.next_item(a);
    }
  } else if (count > 0 && warp == kMmaWarp) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t kIdescS = ((uint32_t)(kKvTile >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24);
    constexpr uint32_t kIdescO =
        (1u << 16) | ((uint32_t)(D >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24);
    if (ptx::elect_one()) {
#pragma unroll
      for (int k = 0; k < TERMS; ++k)
        ptx::tc_cp_32x128b_warpx4(tmem + C::kSfTerm + 4 * k,
                                  ptx::smem_desc_scale_atom(ptx::smem_u32(term_sf + k * 512)));
    }
    __syncwarp();
    bool ok = true;
    int at = 0;  // place in the order of the copies
    auto scores = [&](int i, bool last) {
      const int slot = at % C::kSlots, buffer = i % C::kBuffers;
      // The tile that these scores replace has been read.
      if (i >= C::kBuffers)
        ok = ok && __all_sync(0xffffffffu, bounded_wait(sread0 + 8 * buffer,
                                                        (uint32_t)(i / C::kBuffers - 1) & 1u, abort_flag,
                                                        a.status, 502));
      ok = ok && __all_sync(0xffffffffu,
                            bounded_wait(full0 + 8 * slot, (uint32_t)(at / C::kSlots) & 1u,
                                         abort_flag, a.status, 503));
      if (!ok) return;
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        const uint32_t sf_t = tmem + C::kSfSets + buffer * C::kSfSet;
        ptx::tc_cp_32x128b_warpx4(sf_t, ptx::smem_desc_scale_atom(ptx::smem_u32(sf_tiles + slot * 512)));
        const uint32_t k_s = ptx::smem_u32(slots + slot * C::kSlotBytes);
        const uint32_t q_s = ptx::smem_u32(q_tiles);
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
#pragma unroll
          for (int s = 0; s < C::kSubs; ++s) {
            const uint64_t ad = ptx::smem_desc(q_s + (k * C::kSubs + s) * C::kSubBytes, 0, C::kGroup, C::kSwizzle);
            const uint64_t bd = ptx::smem_desc(k_s + s * C::kSubBytes, 0, C::kGroup, C::kSwizzle);
#pragma unroll
            for (int ks = 0; ks < C::kRowBytes / 32; ++ks)
              ptx::tc_mma_mxf8f6f4(tmem + buffer * kKvTile, ad + 2 * ks, bd + 2 * ks, kIdescS,
                                   tmem + C::kSfTerm + 4 * k, sf_t,
                                   (k > 0 || s > 0 || ks > 0) ? 1u : 0u);
          }
        }
        ptx::tc_commit(sfull0 + 8 * buffer);
        ptx::tc_commit(empty0 + 8 * slot);
        if (last) ptx::tc_commit(qfree);
      }
      __syncwarp();
      ++at;
    };
    for (int i0 = 0, segment = 0; ok && i0 < count; ++segment) {
      ok = __all_sync(0xffffffffu, bounded_wait(qfull, (uint32_t)segment & 1u, abort_flag, a.status, 504));
      if (!ok) break;
      const int tiles = segments[segment & 1].tiles;
      scores(i0, tiles == 1);
      for (int j = 0; ok && j < tiles; ++j) {
        const int i = i0 + j, buffer = i % C::kBuffers;
        if (j + 1 < tiles) scores(i + 1, j + 2 == tiles);
        const int slot = at % C::kSlots;
        ok = ok && __all_sync(0xffffffffu, bounded_wait(pfull0 + 8 * buffer, (uint32_t)(i / C::kBuffers) & 1u,
                                                        abort_flag, a.status, 505));
        ok = ok && __all_sync(0xffffffffu,
                              bounded_wait(full0 + 8 * slot, (uint32_t)(at / C::kSlots) & 1u,
                                           abort_flag, a.status, 506));
        if (!ok) break;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          const uint64_t v_atom = ptx::smem_desc_scale_atom(ptx::smem_u32(sf_tiles + slot * 512));
          const uint32_t sf_t = tmem + C::kSfSets + buffer * C::kSfSet;
          ptx::tc_cp_32x128b_warpx4(sf_t + C::kSfV, v_atom);
          if (D > 128) ptx::tc_cp_32x128b_warpx4(sf_t + C::kSfV + 4, v_atom);
#pragma unroll
          for (int k = 0; k < TERMS; ++k)
            ptx::tc_cp_32x128b_warpx4(sf_t + C::kSfP + 4 * k,
                                      ptx::smem_desc_scale_atom(ptx::smem_u32(p_sf + (buffer * TERMS + k) * 512)));
          // V: head_dim along N (MN-major), 32 tokens per step.
          const uint64_t bd = ptx::smem_desc(ptx::smem_u32(slots + slot * C::kSlotBytes), C::kSubBytes,
                                             C::kGroup, C::kSwizzle);
          const uint32_t p_s = ptx::smem_u32(p_tiles + buffer * C::kPBytes);
#pragma unroll
          for (int k = 0; k < TERMS; ++k) {
            const uint64_t ad = ptx::smem_desc(p_s + k * kRows * kKvTile, 0, 1024, ptx::kSwizzle128);
#pragma unroll
            for (int ks = 0; ks < kKvTileBlocks; ++ks) {
              const uint32_t idesc = kIdescO | ((uint32_t)ks << 29) | ((uint32_t)ks << 4);
              const uint64_t b_ks = bd + ks * (kKvBlock * C::kRowBytes / 16);
              const uint32_t add = (j > 0 || k > 0 || ks > 0) ? 1u : 0u;
              if constexpr (C::kTmemP)
                ptx::tc_mma_mxf8f6f4_ts(tmem + C::kOCol, tmem + C::kPCol + 32 * k + 8 * ks, b_ks, idesc,
                                        sf_t + C::kSfP + 4 * k, sf_t + C::kSfV, add);
              else
                ptx::tc_mma_mxf8f6f4(tmem + C::kOCol, ad + 2 * ks, b_ks, idesc, sf_t + C::kSfP + 4 * k,
                                     sf_t + C::kSfV, add);
            }
          }
          ptx::tc_commit(pvdone0 + 8 * buffer);
          ptx::tc_commit(empty0 + 8 * slot);
        }
        __syncwarp();
        ++at;
      }
      i0 += tiles;
    }
  } else if (count > 0 && warp == kQueryWarp) {
    // ---------------- rows and descriptions of the segments ----------------
    Cursor c = *start;
    c.load(a);
    bool ok = true;
    // Rows that lie together, as f(where, first row of the item, rows): the query heads of a token
    // where heads follow one another, else single rows.  A copy costs about 65 clocks to issue: 128
    // single rows kept an item waiting 4 us.
    const int together = a.q_head_stride == D ? a.group : 1;
    auto runs = [&](const Cursor& at, auto f) {
      const int begin = at.at.t * kRows, end = min(begin + kRows, at.seq.rows);
      for (int run = begin / together + lane; run * together < end; run += 32) {
        const int first = max(run * together, begin), behind = min((run + 1) * together, end);
        f(static_cast<const uint16_t*>(a.q) + (at.seq.row + first / a.group) * a.q_token_stride +
              (int64_t)(at.at.head * a.group + first % a.group) * a.q_head_stride,
          first - begin, behind - first);
      }
    };
    for (int left = count, segment = 0; ok && left > 0; ++segment) {
      // The rows' buffer is free with the last scores of the segment before, the description with
      // the end of the one before that.
      if (segment > 0)
        ok = __all_sync(0xffffffffu, bounded_wait(qfree, (uint32_t)(segment - 1) & 1u, abort_flag, a.status, 507));
      if (segment > 1)
        ok = ok && __all_sync(0xffffffffu, bounded_wait(sdone0 + 8 * (segment & 1),
                                                        (uint32_t)(segment / 2 - 1) & 1u, abort_flag,
                                                        a.status, 508));
      if (!ok) break;
      Segment& seg = segments[segment & 1];
      const int tiles = min(left, c.tiles - c.at.tile);
      const int row0 = c.at.t * kRows, rows = min(kRows, c.seq.rows - row0);
      if (lane == 0) ptx::mbar_arrive_expect_tx(qraw, a.vector ? (uint32_t)(rows * 2 * D) : 0u);
      __syncwarp();
      if (a.vector) {
        runs(c, [&](const uint16_t* src, int n, int count) {
          ptx::bulk_load(ptx::smem_u32(q_tiles + n * 2 * D), src, count * 2 * D, qraw);
        });
      } else {
        for (int n = lane; n < rows; n += 32) {
          const int r = row0 + n;
          const uint16_t* src = static_cast<const uint16_t*>(a.q) + (c.seq.row + r / a.group) * a.q_token_stride +
                                (int64_t)(c.at.head * a.group + r % a.group) * a.q_head_stride;
          for (int d = 0; d < D; ++d) reinterpret_cast<uint16_t*>(q_tiles)[n * D + d] = src[d];
        }
      }
      // Are all pages named?  Eight lookups in flight.
      bool named = true;
      const int end = (int)min((int64_t)c.seq.length, (int64_t)(c.at.tile + tiles) * kKvTile);
      const int pages = (end + a.cache.page_size - 1) / a.cache.page_size;
      const int32_t* table = a.batch.block_table + (int64_t)c.at.b * a.batch.table_stride;
      for (int p0 = c.at.tile * kKvTile / a.cache.page_size + lane; p0 < pages; p0 += 8 * 32) {
        int32_t id[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) id[n] = p0 + 32 * n < pages ? table[p0 + 32 * n] : 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) named = named && id[n] >= 0 && id[n] < a.cache.pages;
      }
      named = __all_sync(0xffffffffu, named);
      if (lane == 0) {
        seg.row = c.seq.row;
        seg.first_position = c.seq.first_position;
        seg.rows = c.seq.rows;
        seg.row0 = row0;
        seg.length = c.seq.length;
        seg.head = c.at.head;
        seg.tile = c.at.tile;
        seg.tiles = tiles;
        seg.whole = c.at.tile == 0 && tiles == c.tiles;
        seg.b = c.at.b;
        seg.all_named = named;
      }
      __syncwarp();  // the rows and the description are complete
      if (lane == 0) ptx::mbar_arrive(qraw);
      left -= tiles;
      if (left > 0) {
        c.next_item(a);
        if (a.vector) {
          // The next rows will come from the L2.
          runs(c, [&](const uint16_t* src, int, int count) { ptx::bulk_prefetch_l2(src, count * 2 * D); });
        }
      }
    }
  } else if (count > 0 && warp < kSoftmaxWarps) {
    // ---------------- softmax: a thread has 32 tokens of one row ----------------
    // A wait that runs out ends the warp's tiles, and the vote at the end of the segment ends all.
    const int quarter = warp & 3, block = warp >> 2;  // rows, and scale block of the tile
    const int row = quarter * 32 + lane;              // of the item
    const uint32_t lane_t = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t vsync = vsync0 + 8 * quarter;
    uint8_t* p_row = p_tiles + row * kKvTile;
    uint8_t* p_sf_row = p_sf + lane * 16 + quarter * 4 + block;
    bool failed = false;
    uint32_t syncs = 0, votes = 0;
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
      if (!failed) failed = !__all_sync(0xffffffffu, bounded_wait(bar, parity, abort_flag, a.status, code));
    };
    // The four warps of a quarter meet.
    auto meet = [&](int code) {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(vsync);
      wait(vsync, syncs & 1u, code);
      ++syncs;
    };
    // Turns a segment's rows into terms, in place.
    auto turn_rows = [&](int segment) {
      wait(qraw, (uint32_t)segment & 1u, 510);
      Segment& seg = segments[segment & 1];
      // Eight rows a warp: their words leave shared memory before any terms replace them.
      constexpr int kPer = D / 32, kBatch = kRows / kSoftmaxWarps;
      const int first_row = warp * kBatch, real = failed ? 0 : seg.rows - seg.row0;
      uint32_t words[kBatch][kPer / 2];
      float scale[kBatch];
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(q_tiles + (first_row + n) * 2 * D) + lane * (kPer / 2);
#pragma unroll
        for (int w = 0; w < kPer / 2; ++w) words[n][w] = src[w];
      }
#pragma unroll
      for (int n = 0; n < kBatch; ++n) scale[n] = query_scale<T, kPer>(words[n], first_row + n < real);
      failed = ptx::barrier_any(1, kSoftmaxWarps * 32, failed);
      if (failed) return;
      if (threadIdx.x < D) nan_from[threadIdx.x] = INT_MAX;
      if (threadIdx.x == 0) *nan_seen = 0;
      float mine = scale[0];
#pragma unroll
      for (int n = 1; n < kBatch; ++n) mine = lane == n ? scale[n] : mine;
      if (lane < kBatch) seg.scale[first_row + lane] = mine * fabsf(a.scale_log2);
      const float sign = a.scale_log2 < 0.0f ? -1.0f : 1.0f;  // the softmax takes a factor >= 0
      const int d0 = lane * kPer, in_row = d0 % C::kRowBytes;
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int r = first_row + n;
        uint32_t codes[TERMS][kPer / 2];
        query_terms<T, TERMS, kPer>(words[n], r < real, scale[n], sign, codes);
        const int swizzle = C::kRowBytes == 128 ? (r & 7) : ((r >> 1) & 3);
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
          uint8_t* dst = q_tiles + (k * C::kSubs + d0 / C::kRowBytes) * C::kSubBytes + r * C::kRowBytes +
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
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(qfull);
    };
    turn_rows(0);
    int at0 = 0;  // place of the segment in the order of the copies
    for (int i0 = 0, segment = 0; i0 < count; ++segment) {
      const Segment& seg = segments[segment & 1];
      wait(qfull, (uint32_t)segment & 1u, 520);  // the other warps' scales
      const int tiles = failed ? 0 : seg.tiles, length = seg.length, tile0 = seg.tile;
      const bool all_named = seg.all_named != 0;
      // Above zero, so that a masked score (-inf) stays one where the scale is zero; the smallest
      // normal number is far below any factor of a score that counts.
      const float row_factor = seg.scale[row] < FLT_MIN ? FLT_MIN : seg.scale[row];
      // Cached tokens that this row sees.
      int64_t sees = length;
      if (a.causal) sees = min(sees, seg.first_position + (seg.row0 + row) / a.group + 1);
      const int visible = sees < 0 ? 0 : (int)sees;
      // All rows of the item see the tokens below this.
      const int64_t all_see = a.causal ? seg.first_position + seg.row0 / a.group + 1 : length;
      float ref = -INFINITY, sum = 0.0f;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int i = i0 + j, buffer = i % C::kBuffers;
        const int t0 = (tile0 + j) * kKvTile + block * kKvBlock;  // this thread's first token
        const bool named = all_named || (t0 < length && kv_page(a.batch, a.cache, seg.b, t0 / kKvBlock) >= 0);
        if constexpr (!C::kEarlyClear) wait(sfull0 + 8 * buffer, (uint32_t)(i / C::kBuffers) & 1u, 512);
        const bool partly = (int64_t)(tile0 + j + 1) * kKvTile > all_see;  // the same in all warps
        if (partly || !named || t0 + kKvBlock > length) {
          // Rows of V without a token may hold anything, NaN among them, and 0 * NaN is NaN: clear
          // them once the tile has landed.  The four warps of a block clear eight rows each.
          if constexpr (C::kSlots == 2)
            if (i > 0) wait(pvdone0, (uint32_t)(i - 1) & 1u, 521);
          const int at = at0 + (j + 1 < tiles ? 2 * j + 2 : 2 * j + 1);
          const int slot = at % C::kSlots;
          wait(full0 + 8 * slot, (uint32_t)(at / C::kSlots) & 1u, 511);
          uint8_t* v_s = slots + slot * C::kSlotBytes;
          for (int t = quarter * 8; t < quarter * 8 + 8; ++t) {
            if (named && t0 + t < length) continue;
            for (int piece = lane; piece < D / 16; piece += 32) {
              const int sub = piece / (C::kRowBytes / 16), in_row = piece % (C::kRowBytes / 16);
              *reinterpret_cast<uint4*>(v_s + sub * C::kSubBytes + (block * kKvBlock + t) * C::kRowBytes +
                                        in_row * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          __syncwarp();
          if (partly && !failed)
            clear_nan<D>(v_s, block * kKvBlock + quarter * 8, 8, (tile0 + j) * kKvTile, nan_from, nan_seen, lane);
          ptx::fence_proxy_async();
        }
        if constexpr (C::kEarlyClear) wait(sfull0 + 8 * buffer, (uint32_t)(i / C::kBuffers) & 1u, 512);
        if (failed) break;
        ptx::tc_fence_after();
        uint32_t raw[32];
        ptx::tmem_ld_x32(lane_t + buffer * kKvTile + block * kKvBlock, raw);
        ptx::tmem_ld_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(sread0 + 8 * buffer);
        float factor = row_factor;
        if (!named || !__all_sync(0xffffffffu, t0 + kKvBlock <= visible)) {
          const int n = named ? visible - t0 : 0;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e >= n) raw[e] = 0xff800000u;  // -inf
          // A row whose query has an infinity or NaN has a factor of NaN: not where it sees nothing.
          if (n <= 0) factor = 1.0f;
        }
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int n = 0; n < 4; ++n)
            m[n] = fmaxf(m[n], fmaxf(__uint_as_float(raw[e + n]), __uint_as_float(raw[e + 4 + n])));
        // To the nearest power of two: the largest weight is in (181, 363).
        const float top = rintf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * factor);
        // The reference moves only where a block exceeds it by much, or was not set: the four
        // warps that share the rows agree.  The answer is not needed before the weights are done.
        volatile int* asked = ask_flag + quarter * 2 + (votes++ & 1u);
        const bool ask = __any_sync(0xffffffffu, top > ref + kMostLog2);
        if (lane == 0) {
          if (ask) *asked = 1;
          ptx::mbar_arrive(vsync);
        }
        // Where nothing is seen (-inf) the lowest finite base keeps the weights zero.
        const float base = fmaxf(top, -FLT_MAX) - kWeightLog2;
        uint32_t codes[TERMS][8];
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float p[4];
#pragma unroll
          for (int n = 0; n < 4; ++n)
            p[n] = ptx::exp2_approx(__uint_as_float(raw[e + n]) * factor - base);
          uint32_t lo[TERMS], hi[TERMS];
          const __half2 w0 = e4m3_terms_half<TERMS>(__floats2half2_rn(p[0], p[1]), lo);
          const __half2 w1 = e4m3_terms_half<TERMS>(__floats2half2_rn(p[2], p[3]), hi);
          // The sums are of the weights as they were rounded, so that they add up to one.
          s0 = ptx::add_halves(s0, *reinterpret_cast<const uint32_t*>(&w0));
          s1 = ptx::add_halves(s1, *reinterpret_cast<const uint32_t*>(&w1));
#pragma unroll
          for (int k = 0; k < TERMS; ++k) codes[k][e / 4] = __byte_perm(lo[k], hi[k], 0x5410);
        }
        // P of the tile before last (or of the last one) has been read.
        if (i >= C::kBuffers)
          wait(pvdone0 + 8 * buffer, (uint32_t)(i / C::kBuffers - 1) & 1u, 513);
        if constexpr (C::kTmemP) {
#pragma unroll
          for (int k = 0; k < TERMS; ++k)
            ptx::tmem_st_x8(lane_t + C::kPCol + 32 * k + 8 * block, codes[k]);
        } else {
          uint8_t* p_buffer = p_row + buffer * C::kPBytes;
#pragma unroll
          for (int k = 0; k < TERMS; ++k) {
#pragma unroll
            for (int c16 = 0; c16 < 2; ++c16) {
              const int chunk = block * 2 + c16;
              *reinterpret_cast<uint4*>(p_buffer + k * kRows * kKvTile + ((chunk ^ (row & 7)) << 4)) =
                  make_uint4(codes[k][c16 * 4], codes[k][c16 * 4 + 1], codes[k][c16 * 4 + 2],
                             codes[k][c16 * 4 + 3]);
            }
          }
        }
        wait(vsync, syncs & 1u, 514);
        ++syncs;
        if (!failed && *asked != 0) {
          row_top[block * kRows + row] = top;
          meet(515);
          if (block == 0 && lane == 0) *asked = 0;  // not used by the next vote, but the one after
          const float most = fmaxf(fmaxf(row_top[row], row_top[kRows + row]),
                                   fmaxf(row_top[2 * kRows + row], row_top[3 * kRows + row]));
          const bool up = most > ref + kMostLog2;
          const float f = up ? pow2_whole(ref - most) : 1.0f;
          if (up) ref = most;
          sum *= f;
          if (j > 0) {
            // What has been added up so far shrinks, once the last output has been added.
            wait(pvdone0 + 8 * ((i - 1) % C::kBuffers), (uint32_t)((i - 1) / C::kBuffers) & 1u, 516);
            if (failed) break;
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c0 = block * (D / 4); c0 < (block + 1) * (D / 4); c0 += 8) {
              uint32_t o[8];
              ptx::tmem_ld_x8(lane_t + C::kOCol + c0, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int n = 0; n < 8; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * f);
              ptx::tmem_st_x8(lane_t + C::kOCol + c0, o);
            }
            ptx::tmem_st_wait();
          }
          // The others read row_top of this meeting before the next one is written.
          meet(517);
        }
        if (failed) break;
        // Block scale of P: 2^(top - ref), the further terms 2^-4 and 2^-8 of it.
        const float power = pow2_whole(top == -INFINITY ? 0.0f : top - ref);
        sum += (s0 + s1) * power;
        const uint32_t code = __float_as_uint(power) >> 23;
#pragma unroll
        for (int k = 0; k < TERMS; ++k)
          p_sf_row[(buffer * TERMS + k) * 512] = (uint8_t)(code > 4u * k ? code - 4u * k : 0u);
        if constexpr (C::kTmemP) ptx::tmem_st_wait();
        ptx::fence_proxy_async();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(pfull0 + 8 * buffer);
      }
      // ---- the rows of this CTA's tiles of the item ----
      row_sum[block * kRows + row] = sum;
      const int i = i0 + tiles - 1;
      if (tiles > 0) wait(pvdone0 + 8 * (i % C::kBuffers), (uint32_t)(i / C::kBuffers) & 1u, 518);
      failed = ptx::barrier_any(1, kSoftmaxWarps * 32, failed);
      if (failed) break;
      ptx::tc_fence_after();
      const float l = (row_sum[row] + row_sum[kRows + row]) + (row_sum[2 * kRows + row] + row_sum[3 * kRows + row]);
      const int r = seg.row0 + row;
      const bool mine = r < seg.rows;
      // Through shared memory, so that a row's values leave together: each warp has 2 KB of its
      // rows in the first two terms of P, which no product reads any more, or 1 KB apart.
      const bool nans = *nan_seen != 0;
      constexpr int kMost = C::kStageWarp / 64;                 // 16-bit columns that fit
      constexpr int kCols = D / 4 < kMost ? D / 4 : kMost, kPieces = kCols / 8;  // a pass; 16-byte pieces
      constexpr int kPartCols = kMost / 2, kPartPieces = kPartCols / 4;          // of 32-bit columns
      uint8_t* stage = C::kTmemP ? stages + warp * C::kStageWarp
                                 : p_tiles + (block >> 1) * kRows * kKvTile + quarter * 4096 + (block & 1) * 2048;
      if (seg.whole) {
        const float scale = l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t own = (seg.row + r / a.group) * a.out_token_stride +
                            (int64_t)(seg.head * a.group + r % a.group) * a.out_head_stride;
        T* out = static_cast<T*>(a.out);
        const unsigned real = __ballot_sync(0xffffffffu, mine);
#pragma unroll 1
        for (int c0 = block * (D / 4); c0 < (block + 1) * (D / 4); c0 += kCols) {
          uint32_t o[kCols];
          ptx::tmem_ld_chunk<kCols>(lane_t + C::kOCol + c0, o);
          ptx::tmem_ld_wait();
          if (nans) {
#pragma unroll
            for (int n = 0; n < kCols; ++n)
              if (nan_from[c0 + n] < visible) o[n] = 0x7fc00000u;
          }
          uint32_t w[kCols / 2];
#pragma unroll
          for (int n = 0; n < kCols / 2; ++n) {
            const float x = __uint_as_float(o[2 * n]) * scale, y = __uint_as_float(o[2 * n + 1]) * scale;
            if constexpr (TERMS == 2) {
              const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
              w[n] = *reinterpret_cast<const uint32_t*>(&v);
            } else {
              const __half2 v = __floats2half2_rn(x, y);
              w[n] = *reinterpret_cast<const uint32_t*>(&v);
            }
          }
#pragma unroll
          for (int n = 0; n < kPieces; ++n)
            *reinterpret_cast<uint4*>(stage + lane * kCols * 2 + ((n ^ (lane * kPieces / 8 & (kPieces - 1))) << 4)) =
                make_uint4(w[4 * n], w[4 * n + 1], w[4 * n + 2], w[4 * n + 3]);
          __syncwarp();
#pragma unroll
          for (int n = 0; n < kPieces; ++n) {
            const int from = (n * 32 + lane) / kPieces, piece = lane % kPieces;
            const int64_t at = __shfl_sync(0xffffffffu, own, from);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + from * kCols * 2 +
                                                            ((piece ^ (from * kPieces / 8 & (kPieces - 1))) << 4));
            if ((real >> from & 1u) == 0) continue;
            T* dst = out + at + c0 + piece * 8;
            if (a.vector_out) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {
              const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                reinterpret_cast<uint16_t*>(dst)[2 * e] = (uint16_t)x[e];
                reinterpret_cast<uint16_t*>(dst)[2 * e + 1] = (uint16_t)(x[e] >> 16);
              }
            }
          }
          __syncwarp();
        }
      } else {
        // A share that begins inside an item uses the CTA's first partial slot for it, one that
        // ends inside the second.
        float* part = a.partials +
                      (int64_t)(2 * blockIdx.x + (seg.tile != 0 ? 0 : 1)) * C::kPartialFloats;
        if (block == 0) {
          part[kRows * D + 2 * row] = ref;
          part[kRows * D + 2 * row + 1] = l;
        }
#pragma unroll 1
        for (int c0 = block * (D / 4); c0 < (block + 1) * (D / 4); c0 += kPartCols) {
          uint32_t o[kPartCols];
          ptx::tmem_ld_chunk<kPartCols>(lane_t + C::kOCol + c0, o);
          ptx::tmem_ld_wait();
          if (nans) {
#pragma unroll
            for (int n = 0; n < kPartCols; ++n)
              if (nan_from[c0 + n] < visible) o[n] = 0x7fc00000u;
          }
#pragma unroll
          for (int n = 0; n < kPartPieces; ++n)
            *reinterpret_cast<uint4*>(stage + lane * kPartCols * 4 +
                                      ((n ^ (lane * kPartPieces / 8 & (kPartPieces - 1))) << 4)) =
                make_uint4(o[4 * n], o[4 * n + 1], o[4 * n + 2], o[4 * n + 3]);
          __syncwarp();
#pragma unroll
          for (int n = 0; n < kPartPieces; ++n) {
            const int from = (n * 32 + lane) / kPartPieces, piece = lane % kPartPieces;
            const uint4 v = *reinterpret_cast<const uint4*>(
                stage + from * kPartCols * 4 + ((piece ^ (from * kPartPieces / 8 & (kPartPieces - 1))) << 4));
            *reinterpret_cast<uint4*>(part + (quarter * 32 + from) * D + c0 + piece * 4) = v;
          }
          __syncwarp();
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(sdone0 + 8 * (segment & 1));
      // The warps of a quarter write P where they have staged their rows.
      meet(519);
      i0 += tiles;
      at0 += 2 * tiles;
      if (i0 < count) turn_rows(segment + 1);
      if (failed) break;
    }
  }

  if (warp == kTmaWarp && lane == 0 && blockIdx.x + 1 < gridDim.x) {
    // For the joining kernel, now that nothing waits for it: the item in which the next share begins,
    // and over how many CTAs it goes if its first tile is this CTA's.
    const Share s = share_of(share_smem[2], (int)gridDim.x);
    const int cta = (int)blockIdx.x;
    int parts = 1;
    if (cta + 1 < s.ctas && s.total > 0) {
      const Sequence q = load_sequence(a, next->b);
      const int64_t u0 = share_smem[3] + kItemUnits, u1 = u0 + tiles_of(a, q, next->t) - 1;
      // CTA of a unit: the last one whose share begins at or before it.
      if ((int)(((u0 + 1) * s.ctas - 1) / s.total) == cta)
        parts = (int)(((u1 + 1) * s.ctas - 1) / s.total) - cta + 1;
    }
    borders_of(a)[cta] = Border{next->b, next->t, next->head, parts};
  }

  // ---------------- teardown ----------------
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // Give copies and MMAs still in flight time to land before the CTA's shared
    // and tensor memory are handed back.
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Joins the partial rows of every item whose tiles went to more than one CTA, in the order of the
// tiles.  A border between two shares has kRows / kJoinRows CTAs; the first border inside an item
// has it.
constexpr int kJoinRows = 8;
constexpr int kJoinThreads = 256;

template <int D, int TERMS>
__global__ void __launch_bounds__(kJoinThreads)
kv_prefill_join_kernel(const AttentionArgs a) {
  using C = PrefillCfg<D, TERMS>;
  using T = typename std::conditional<TERMS == 2, __nv_bfloat16, __half>::type;
  constexpr int kColumns = D / 4;                   // four values a thread
  constexpr int kAtOnce = kJoinThreads / kColumns;  // rows
  const int c0 = (int)blockIdx.x, tid = threadIdx.x;
  ptx::grid_dependency_wait();
  const Border item = borders_of(a)[c0];
  const int parts = item.parts;
  if (parts == 1) return;
  const Sequence seq = load_sequence(a, item.b);
  const int column = tid % kColumns;
  // The first CTA began before this item or with it, the others inside it.
  const int64_t first = 2 * c0 + 1, later = 2 * c0;  // slot of part p: p == 0 ? first : later + 2 p
  for (int k = tid / kColumns; k < kJoinRows; k += kAtOnce) {
    const int row = (int)blockIdx.y * kJoinRows + k;
    const int r = item.t * kRows + row;
    if (r >= seq.rows) continue;
    float top = -INFINITY;
    for (int p = 0; p < parts; ++p)
      top = fmaxf(top, a.partials[(p == 0 ? first : later + 2 * p) * C::kPartialFloats + kRows * D + 2 * row]);
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float* part = a.partials + (p == 0 ? first : later + 2 * p) * C::kPartialFloats;
      const float2 tl = *reinterpret_cast<const float2*>(part + kRows * D + 2 * row);
      const float4 v = *reinterpret_cast<const float4*>(part + row * D + column * 4);
      const float f = tl.x == top ? 1.0f : pow2_whole(tl.x - top);
      l += f * tl.y;
      o.x += f * v.x;
      o.y += f * v.y;
      o.z += f * v.z;
      o.w += f * v.w;
    }
    const float scale = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.out) + (seq.row + r / a.group) * a.out_token_stride +
             (int64_t)(item.head * a.group + r % a.group) * a.out_head_stride + column * 4;
    const float v[4] = {o.x * scale, o.y * scale, o.z * scale, o.w * scale};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TERMS == 2) out[i] = __float2bfloat16_rn(v[i]);
      else out[i] = __float2half_rn(v[i]);
    }
  }
}

bool use_pdl() {
  static const bool enabled = []() {
    const char* env = std::getenv("MXFP6_B200_PDL");
    return env == nullptr || env[0] != '0';
  }();
  return enabled;
}

template <int D, int TERMS>
int launch(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttentionArgs& a, int grid,
           cudaStream_t stream) {
  using C = PrefillCfg<D, TERMS>;
  static bool configured[64] = {};
  int device = 0;
  MX_CUDA(cudaGetDevice(&device));
  if (device >= 64 || !configured[device]) {
    MX_CUDA(cudaFuncSetAttribute(kv_prefill_kernel<D, TERMS>,
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
  MX_CUDA(cudaLaunchKernelEx(&config, kv_prefill_kernel<D, TERMS>, tm_k, tm_v, a));
  if (grid == 1) return kOk;  // nothing was cut
  config.gridDim = dim3((unsigned)(grid - 1), kRows / kJoinRows);
  config.blockDim = dim3(kJoinThreads);
  config.dynamicSmemBytes = 0;
  MX_CUDA(cudaLaunchKernelEx(&config, kv_prefill_join_kernel<D, TERMS>, a));
  return kOk;
}

}  // namespace

// CTAs of a prefill launch: at most one per SM and no more than there can be work for.
int kv_prefill_grid(int64_t batch, int64_t tokens, int kv_heads, int group, int64_t max_context) {
  const int64_t items = (tokens * group / kRows + batch) * kv_heads;
  const int64_t units = items * (ceil_div64(max_context < 1 ? 1 : max_context, kKvTile) + kItemUnits);
  const int64_t want = ceil_div64(units, kMinUnits);
  return (int)(want < kSms ? want : kSms);
}

int64_t kv_prefill_workspace(int64_t batch, int64_t tokens, int kv_heads, int group, int head_dim,
                             int64_t max_context) {
  const int grid = kv_prefill_grid(batch, tokens, kv_heads, group, max_context);
  return grid == 1 ? 0 : kSms * (int64_t)sizeof(Border) +
                             (int64_t)grid * 2 * (kRows * head_dim + 2 * kRows) * 4;
}

// Sequences with more than a.min_rows rows (tokens x group).
int launch_kv_prefill(const AttentionArgs& args, int dtype, cudaStream_t stream) {
  AttentionArgs a = args;
  static_assert(sizeof(Border) % 16 == 0, "partial rows stay aligned");
  a.partials = reinterpret_cast<float*>(reinterpret_cast<Border*>(args.partials) + kSms);
  CUtensorMap tm_k, tm_v;
  if (int rc = make_kv_map(&tm_k, a.cache.k_values, a.cache)) return rc;
  if (int rc = make_kv_map(&tm_v, a.cache.v_values, a.cache)) return rc;
  const int grid = kv_prefill_grid(a.batch.batch, a.batch.tokens, a.cache.kv_heads, a.group,
                                   (int64_t)a.batch.table_width * a.cache.page_size);
  const int d = a.cache.head_dim;
  if (dtype == kBF16) {
    if (d == 64) return launch<64, 2>(tm_k, tm_v, a, grid, stream);
    if (d == 128) return launch<128, 2>(tm_k, tm_v, a, grid, stream);
    return launch<256, 2>(tm_k, tm_v, a, grid, stream);
  }
  if (d == 64) return launch<64, 3>(tm_k, tm_v, a, grid, stream);
  if (d == 128) return launch<128, 3>(tm_k, tm_v, a, grid, stream);
  return launch<256, 3>(tm_k, tm_v, a, grid, stream);
}

}  // namespace mx
