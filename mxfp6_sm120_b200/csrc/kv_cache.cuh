// Layout of the paged 8-bit KV cache and the sequence bookkeeping its kernels share.
//
// Values are E4M3 bytes [pages, kv_heads, page_size, head_dim]; scales are UE8M0 bytes
// [pages, kv_heads, page_size / 32]: the 32 tokens x head_dim values of a block of one head
// share one power of two.  32 tokens is the MX block length along the contraction of the
// second attention product (weights x values), so tcgen05 applies the scale in hardware;
// along head_dim the scale is constant, so the first product can take it the same way.
#pragma once

#include "common.cuh"

namespace mx {

constexpr int kKvBlock = 32;  // tokens that share a scale

// Token rows [cu_seqlens[b], cu_seqlens[b + 1]) of q / k / v are the LAST positions of
// sequence b, whose cached length including them is seq_lens[b].  Without cu_seqlens every
// sequence has exactly one row.
struct KvBatch {
  const int32_t* block_table;  // [batch, table_width], page of every page_size tokens
  const int32_t* seq_lens;     // [batch]
  const int32_t* cu_seqlens;   // [batch + 1] or null
  int64_t table_stride;        // elements between sequences of the block table
  int64_t tokens;              // rows of q / k / v
  int table_width;
  int batch;
};

struct KvCache {
  uint8_t* k_values;
  uint8_t* v_values;
  uint8_t* k_scales;
  uint8_t* v_scales;
  int64_t pages;
  int kv_heads;
  int page_size;  // 32, 64 or 128
  int head_dim;   // 64, 128 or 256
};

int check_kv(const KvCache& cache, const KvBatch& batch);

#ifdef __CUDACC__
struct KvSpan {
  int64_t row;  // first token row
  int rows;     // token rows (new tokens)
  int length;   // cached length including them, at most what the block table can name
};

// What the device-side metadata says about sequence b, clamped to the extents of the launch so
// that no content of these arrays can send an access out of bounds.
__device__ __forceinline__ KvSpan kv_span(const KvBatch& batch, int page_size, int b) {
  KvSpan s;
  if (batch.cu_seqlens == nullptr) {
    s.row = b;
    s.rows = 1;
  } else {
    const int64_t first = batch.cu_seqlens[b], last = batch.cu_seqlens[b + 1];
    const int64_t lo = first < 0 ? 0 : (first > batch.tokens ? batch.tokens : first);
    const int64_t hi = last < lo ? lo : (last > batch.tokens ? batch.tokens : last);
    s.row = lo;
    s.rows = (int)(hi - lo);
  }
  const int64_t most = (int64_t)batch.table_width * page_size;
  const int64_t len = batch.seq_lens[b];
  s.length = (int)(len < 0 ? 0 : (len > most ? most : len));
  return s;
}

// Page that holds block `block` (32 tokens) of sequence b, or -1 when the table names none.
__device__ __forceinline__ int64_t kv_page(const KvBatch& batch, const KvCache& cache, int b,
                                           int block) {
  const int per_page = cache.page_size / kKvBlock;
  const int index = block / per_page;
  if (index < 0 || index >= batch.table_width) return -1;
  const int32_t page = batch.block_table[(int64_t)b * batch.table_stride + index];
  return page >= 0 && page < cache.pages ? page : -1;
}
#endif

}  // namespace mx
