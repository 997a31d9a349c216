// What the attention kernels over the paged 8-bit cache share: arguments, number formats, and
// the walk of a CTA along its share of the (sequence, head, tile) work list.
//
// Numbers.  Keys and values enter the tensor cores as they lie in the cache (E4M3 under UE8M0
// block scales, kind::mxf8f6f4).  The other operand of each product, 16-bit queries and 32-bit
// weights, becomes a sum of E4M3 terms x = t0 + t1 / 16 (+ t2 / 256): a term keeps four
// significant bits, rounding to nearest makes the remainder at most half a step (2^-4 relative to
// the binade), so each further term takes four more.  Below E4M3's smallest normal number a term's
// step is fixed, so that two terms leave up to 2^-14 of a small x and three up to 2^-18.
//  * Queries are scaled so that a row's largest magnitude is in (224, 448].  Two terms hold a BF16
//    query (8 bits) exactly from 2^-6 on, three an FP16 one (11 bits) from 2^-7 on; what is smaller
//    is off by at most 2^-14 and 2^-18: 2^-21 and 2^-25 of the row's largest.
//  * Weights (largest of a block in (181, 363)) are rounded to FP16 first, where two of them become
//    terms with one instruction a step: off by up to 2^-11.  Two terms leave 2^-9 of the binade
//    beside it, three nothing.  2^-9 + 2^-11 for BF16 and 2^-11 for FP16 are chosen: no more than
//    the half step (2^-8, 2^-11) that the output is rounded by, and rows are divided by the sum of
//    the weights as they were rounded, so that a row is not off as a whole.  A third term for BF16
//    would be half as many matrix instructions again.
// The products of all terms accumulate in 32 bits, weights 2^8 times and, where a block exceeds its
// row's reference, 2^24 times their size: values up to 2^80 in magnitude cannot overflow.
#pragma once

#include "kv_cache.cuh"
#include "ptx.cuh"
#include "wait.cuh"

#include <cuda_fp8.h>
#include <type_traits>

namespace mx {

constexpr int kKvTile = 128;                       // cached tokens per tile
constexpr int kKvTileBlocks = kKvTile / kKvBlock;  // scale blocks per tile

struct AttentionArgs {
  KvCache cache;
  KvBatch batch;
  const void* q;
  void* out;
  float* partials;  // workspace, see the kernels
  int* status;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int q_heads;
  int group;        // query heads per key head
  float scale_log2; // softmax scale * log2(e)
  int causal;
  int max_rows;     // rows (tokens x group) a sequence may have to be the decode kernel's
  int min_rows;     // and has more of to be the prefill kernel's
  int vector;       // q rows can be read sixteen bytes at a time
  int vector_out;   // and output rows written so
  int item_units;   // what a (sequence, head) costs beside its tiles, in tiles
  int whole_items;  // a (sequence, head) is not cut between CTAs
};

int make_kv_map(CUtensorMap* map, const uint8_t* values, const KvCache& cache);

#ifdef __CUDACC__
// E4M3 terms of two FP16 numbers: codes[t] holds both in its low sixteen bits.  The remainders
// are exact in FP16.  Returns what the terms add up to, exact in FP16 as well: it is a multiple of
// x's last place, or of the second term's smallest step.  Three terms leave at most 2^-18 of x.
template <int kTerms>
__device__ __forceinline__ __half2 e4m3_terms_half(__half2 x, uint32_t (&codes)[kTerms]) {
  const __half2 whole = x;
  __half2 first{};
#pragma unroll
  for (int t = 0; t < kTerms; ++t) {
    codes[t] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(x), __NV_SATFINITE, __NV_E4M3);
    if (kTerms == 3 && t == 2) return whole;
    const __half2 v(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes[t], __NV_E4M3));
    if (t == 0) first = v;
    else if (kTerms == 2) return __hfma2(v, __float2half2_rn(0.0625f), first);
    x = __hmul2(__hsub2(x, v), __float2half2_rn(16.0f));
  }
  return whole;
}

// 2^v of a whole v up to 127 (below -126: 2^-126): adding 1.5 * 2^23 leaves v in the low bits.
__device__ __forceinline__ float pow2_whole(float v) {
  const uint32_t bits = __float_as_uint(fmaxf(v, -126.0f) + 12582912.0f);
  return __uint_as_float((bits + 127u) << 23);
}

// Words of kBatch query rows, kPer values a lane: row n is at `base` plus lane r0 + n's `offset`.
// All loads are issued before anything waits for one.
template <int kBatch, int kPer>
__device__ __forceinline__ void load_query_rows(const uint16_t* base, int64_t offset, int r0, int vector,
                                                uint32_t (&raw)[kBatch][kPer / 2]) {
  const uint16_t* src[kBatch];
#pragma unroll
  for (int n = 0; n < kBatch; ++n) src[n] = base + __shfl_sync(0xffffffffu, offset, r0 + n);
  if (vector) {
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      if constexpr (kPer == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(src[n]);
        raw[n][0] = v.x;
        raw[n][1] = v.y;
        raw[n][2] = v.z;
        raw[n][3] = v.w;
      } else if constexpr (kPer == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(src[n]);
        raw[n][0] = v.x;
        raw[n][1] = v.y;
      } else {
        raw[n][0] = *reinterpret_cast<const uint32_t*>(src[n]);
      }
    }
  } else {
#pragma unroll
    for (int n = 0; n < kBatch; ++n)
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) raw[n][i] = (uint32_t)src[n][2 * i] | (uint32_t)src[n][2 * i + 1] << 16;
  }
}

// Power of two that takes a row's largest magnitude (kPer values a lane, a row of zeros where
// `real` is false) to E4M3's largest; NaN where it has an infinity or NaN: it has no scale, and
// its scores become NaN.  By a full warp.
template <class T, int kPer>
__device__ __forceinline__ float query_scale(const uint32_t (&words)[kPer / 2], bool real) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kInf = kBf16 ? 0x7f80u : 0x7c00u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i)
    top = max(top, max(words[i] & 0x7fffu, (words[i] >> 16) & 0x7fffu));
  top = __reduce_max_sync(0xffffffffu, real ? top : 0u);
  const float most = kBf16 ? __uint_as_float(top << 16)
                           : __half2float(__ushort_as_half((unsigned short)top));
  return top < kInf ? __uint_as_float(ue8m0_scale_bits_shift<8>(most)) : NAN;
}

// E4M3 terms of the row over its scale, times `sign`.  The scaled values go through FP16, which
// holds them exactly down to 2^-14 (2^-23 of the row's largest) and rounds what is below.
template <class T, int kTerms, int kPer>
__device__ __forceinline__ void query_terms(const uint32_t (&words)[kPer / 2], bool real, float scale,
                                            float sign, uint32_t (&codes)[kTerms][kPer / 2]) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const float inverse = real && scale == scale ? ue8m0_inverse(__float_as_uint(scale)) * sign : 0.0f;
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i) {
    const uint32_t w = words[i];
    float lo, hi;
    if constexpr (kBf16) {
      lo = __uint_as_float(w << 16);
      hi = __uint_as_float(w & 0xffff0000u);
    } else {
      lo = __half2float(__ushort_as_half((unsigned short)w));
      hi = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
    }
    uint32_t t[kTerms];
    e4m3_terms_half<kTerms>(__floats2half2_rn(lo * inverse, hi * inverse), t);
#pragma unroll
    for (int k = 0; k < kTerms; ++k) codes[k][i] = t[k];
  }
}

// NaN among cached values.  A row's weight for a token that it does not see is zero, and the
// tensor cores would make 0 * NaN a NaN.  So where some rows do not see all of a tile, its NaN
// codes are cleared and `nan_from` remembers, per value of head_dim, the first such token: rows
// that see it get NaN there when they are written.  Tokens t0 .. t0 + count of a V tile in shared
// memory (sub-tiles of kRowBytes a token), by a full warp; `first` is the tile's first token.
template <int D>
__device__ __forceinline__ void clear_nan(uint8_t* tile, int t0, int count, int first, int* nan_from,
                                          volatile int* nan_seen, int lane) {
  constexpr int kRowBytes = D < 128 ? D : 128, kPieces = D / 16;
  for (int n = lane; n < count * kPieces; n += 32) {
    const int t = t0 + n / kPieces, piece = n % kPieces;
    const int sub = piece / (kRowBytes / 16), place = piece % (kRowBytes / 16);
    uint4* at = reinterpret_cast<uint4*>(tile + sub * kKvTile * kRowBytes + t * kRowBytes + place * 16);
    uint4 v = *at;
    // A byte of 0x7f or 0xff carries into bit 7.
    const uint32_t found = ((v.x & 0x7f7f7f7fu) + 0x01010101u) | ((v.y & 0x7f7f7f7fu) + 0x01010101u) |
                           ((v.z & 0x7f7f7f7fu) + 0x01010101u) | ((v.w & 0x7f7f7f7fu) + 0x01010101u);
    if ((found & 0x80808080u) == 0) continue;
    const int logical = place ^ (kRowBytes == 128 ? (t & 7) : ((t >> 1) & 3));
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((w[i / 4] >> (8 * (i % 4)) & 0x7fu) != 0x7fu) continue;
      atomicMin(nan_from + sub * kRowBytes + logical * 16 + i, first + t);
      w[i / 4] &= ~(0xffu << (8 * (i % 4)));
    }
    *at = make_uint4(w[0], w[1], w[2], w[3]);
    *nan_seen = 1;
  }
}

// A sequence as this kernel sees it: `tiles` is 0 when it has no rows or is another kernel's.
struct KvSequence {
  int64_t row;  // first token row
  int rows;     // new tokens
  int length;   // cached tokens that its rows may see
  int64_t last; // unclamped position of its last row
  int tiles;
};
__device__ __forceinline__ KvSequence kv_sequence(const AttentionArgs& a, int b) {
  const KvSpan s = kv_span(a.batch, a.cache.page_size, b);
  KvSequence q;
  q.row = s.row;
  q.rows = s.rows;
  q.length = s.length;
  q.last = (int64_t)a.batch.seq_lens[b] - 1;
  const bool mine = s.rows > 0 && (int64_t)s.rows * a.group <= a.max_rows;
  q.tiles = mine ? max(1, (s.length + kKvTile - 1) / kKvTile) : 0;
  return q;
}
#endif

}  // namespace mx
