// Quantising keys and values into the pages of the 8-bit cache, and reading them back.
//
// Write.  A block of 32 tokens and one head shares a scale 2^e.  For the tokens that a call
// adds to a block, `need` is the smallest power of two that takes their largest finite
// magnitude to 448 or less (the rule of the activation quantizer, floor 2^-99).  A block whose
// first token is new takes e = need; a block that already holds tokens takes
// e = max(stored e, need), and when that raises the scale the kept codes are rounded once more
// to it.  A scale never shrinks until the block's first token is written again.  Values are
// rounded to nearest even and saturate; NaN stays NaN; an infinity saturates to the largest
// code and does not enter the scale, so that it cannot flush the 31 tokens beside it.
//
// One CTA owns a (block, head, K or V), so no two CTAs touch the same bytes and the result
// does not depend on their order.  Both kernels move each byte once and compute next to
// nothing: HBM bounds them, launch latency at decode sizes.  Inside a CUDA graph (copy rate
// 6.57 TB/s): write of 8191 tokens, 4 heads of 256: 14 us, 3.6 TB/s (the first bytes come after
// the lengths and the page, three loads one after another); of one token for 32 sequences:
// 3.5 us; read of 12 sequences of up to 6000 tokens: 51 us, 5.4 TB/s; of 77 tokens: 2.7 us.
#include "kv_cache.cuh"

#include <cuda_fp8.h>

namespace mx {
namespace {

constexpr int kWriteThreads = 128;

struct KvRows {
  const void* k;
  const void* v;
  int64_t k_token_stride, k_head_stride;  // elements
  int64_t v_token_stride, v_head_stride;
};

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float2 values2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

template <class T>
__device__ __forceinline__ float half_bits_to_float(uint32_t bits) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
    return __uint_as_float(bits << 16);
  } else {
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
}

// Blocks that a call may touch: sequence b gets the slots [S_b, S_(b+1)) with
// S_b = cu[b] / 32 + 2 b.  n new tokens touch at most (n + 30) / 32 + 1 blocks, and
// cu[b+1] / 32 - cu[b] / 32 + 2 >= n / 32 + 2 is never less, so the slots suffice without any
// pass over the lengths.
__host__ __device__ __forceinline__ int64_t slots_before(int64_t cu, int64_t b) {
  return cu / kKvBlock + 2 * b;
}

template <class T, int D, bool kVector>
__global__ void __launch_bounds__(kWriteThreads)
kv_write_kernel(const KvCache cache, const KvBatch batch, const KvRows rows) {
  __shared__ uint32_t warp_top[kWriteThreads / 32];
  const int64_t slot = blockIdx.x;
  const int head = blockIdx.y;
  const bool is_v = blockIdx.z != 0;

  int b = (int)slot, nth = 0;
  if (batch.cu_seqlens != nullptr) {
    int lo = 0, hi = batch.batch - 1;  // last b whose first slot is not behind this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (slots_before(batch.cu_seqlens[mid], mid) <= slot) lo = mid; else hi = mid - 1;
    }
    b = lo;
    const int64_t at = slot - slots_before(batch.cu_seqlens[b], b);
    if (at < 0 || at > (1 << 26)) return;
    nth = (int)at;
  }
  const KvSpan span = kv_span(batch, cache.page_size, b);
  // The unclamped length places the rows; rows behind the table's reach are dropped.
  const int64_t start = (int64_t)batch.seq_lens[b] - span.rows;  // position of the first new row
  const int64_t from = start < 0 ? 0 : start;
  const int64_t block = from / kKvBlock + nth;
  const int64_t first = block * kKvBlock;
  if (span.rows <= 0 || first >= span.length || from >= span.length) return;
  const int kept = from > first ? (int)(from - first) : 0;
  const int filled = span.length - first < kKvBlock ? (int)(span.length - first) : kKvBlock;

  const T* src = static_cast<const T*>(is_v ? rows.v : rows.k);
  const int64_t token_stride = is_v ? rows.v_token_stride : rows.k_token_stride;
  src += head * (is_v ? rows.v_head_stride : rows.k_head_stride) +
         (span.row + first - start) * token_stride;  // row of the block's first token
  // Eight values per thread and row; the block's new rows stay in registers between the
  // maximum and the rounding.
  constexpr int kChunks = D / 8;
  constexpr int kRowsPerPass = kWriteThreads / kChunks;
  constexpr int kPasses = kKvBlock / kRowsPerPass;
  const int chunk = threadIdx.x % kChunks, row0 = threadIdx.x / kChunks;
  uint4 raw[kPasses];
  uint32_t top = 0;  // largest finite magnitude as a bit pattern (monotonic)
  constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = row0 + p * kRowsPerPass;
    raw[p] = make_uint4(0, 0, 0, 0);
    if (r >= kept && r < filled) {
      const T* at = src + r * token_stride + chunk * 8;
      if constexpr (kVector) {
        raw[p] = __ldcs(reinterpret_cast<const uint4*>(at));
      } else {
        uint16_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = reinterpret_cast<const uint16_t*>(at)[i];
        raw[p] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
      }
    }
  }
  // The page is looked up while the rows are on their way.
  const int64_t page = kv_page(batch, cache, b, (int)block);
  if (page < 0) return;
  const int per_page = cache.page_size / kKvBlock;
  const int64_t block_index = (page * cache.kv_heads + head) * per_page + block % per_page;
  uint8_t* dst = (is_v ? cache.v_values : cache.k_values) + block_index * kKvBlock * D;
  uint8_t* scale = (is_v ? cache.v_scales : cache.k_scales) + block_index;

#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const uint32_t w[4] = {raw[p].x, raw[p].y, raw[p].z, raw[p].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
      top = max(top, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWriteThreads / 32; ++w) top = max(top, warp_top[w]);

  uint32_t code = ue8m0_scale_bits_shift<8>(half_bits_to_float<T>(top)) >> 23;
  const uint32_t before = kept > 0 ? min((uint32_t)*scale, 253u) : 0u;
  code = max(code, before);
  const float inverse = ue8m0_inverse(code << 23);
  // Factor of the kept codes; differences of more than 100 flush them all the same.
  const uint32_t moved = min(code - before, 100u);
  const float shrink = __uint_as_float((127u - moved) << 23);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = row0 + p * kRowsPerPass;
    uint2* out = reinterpret_cast<uint2*>(dst + r * D + chunk * 8);
    if (r >= kept && r < filled) {
      const uint32_t w[4] = {raw[p].x, raw[p].y, raw[p].z, raw[p].w};
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = half_bits_to_float<T>(w[i] & 0xffffu) * inverse;
        f[2 * i + 1] = half_bits_to_float<T>(w[i] >> 16) * inverse;
      }
      *out = make_uint2(codes4(f[0], f[1], f[2], f[3]), codes4(f[4], f[5], f[6], f[7]));
    } else if (r < kept && code > before) {
      const uint2 old = *out;
      const float2 a = values2(old.x), c = values2(old.x >> 16);
      const float2 e = values2(old.y), g = values2(old.y >> 16);
      *out = make_uint2(codes4(a.x * shrink, a.y * shrink, c.x * shrink, c.y * shrink),
                        codes4(e.x * shrink, e.y * shrink, g.x * shrink, g.y * shrink));
    }
  }
  // Every thread has read the stored scale before the barrier below orders its replacement.
  __syncthreads();
  if (threadIdx.x == 0) *scale = (uint8_t)code;
}

// ------------------------------------------------------------------------------- read

constexpr int kReadThreads = 256;
constexpr int kReadRows = 16;  // token rows per CTA at most

struct KvOut {
  void* k;
  void* v;
};

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// out[row] = code * 2^(scale - 127), rounded once: exact in BF16 (three fraction bits), exact in
// FP16 wherever FP16 has the exponent.  A CTA looks its rows' pages up once, then streams
// 16-byte pieces of codes to 32-byte pieces of values.
template <class T>
__global__ void __launch_bounds__(kReadThreads)
kv_read_kernel(const KvCache cache, const KvBatch batch, const KvOut out, int cta_rows) {
  __shared__ int64_t block_of[kReadRows];  // (page * heads) * blocks + block, -1: zeros, -2: untouched
  __shared__ int token_of[kReadRows];      // token within the block
  const int64_t row0 = (int64_t)blockIdx.x * cta_rows;
  const int per_page = cache.page_size / kKvBlock;
  if (threadIdx.x < cta_rows) {
    const int64_t row = row0 + threadIdx.x;
    int64_t where = -2;
    int token = 0;
    if (row < batch.tokens) {
      int b = (int)row;
      if (batch.cu_seqlens != nullptr) {
        int lo = 0, hi = batch.batch - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (batch.cu_seqlens[mid] <= row) lo = mid; else hi = mid - 1;
        }
        b = lo;
      }
      const KvSpan span = kv_span(batch, cache.page_size, b);
      if (row >= span.row && row < span.row + span.rows) {
        where = -1;
        const int64_t position = (int64_t)batch.seq_lens[b] - span.rows + (row - span.row);
        if (position >= 0 && position < span.length) {
          const int block = (int)(position / kKvBlock);
          const int64_t page = kv_page(batch, cache, b, block);
          if (page >= 0) {
            where = page * cache.kv_heads * per_page + block % per_page;
            token = (int)(position % kKvBlock);
          }
        }
      }
    }
    block_of[threadIdx.x] = where;
    token_of[threadIdx.x] = token;
  }
  __syncthreads();
  const int pieces = cache.head_dim / 16;            // per head
  const int per_row = cache.kv_heads * pieces;       // per row of K or V
  const int total = cta_rows * 2 * per_row;
  for (int i = threadIdx.x; i < total; i += kReadThreads) {
    const int piece = i % per_row, r = (i / per_row) % cta_rows;
    const bool is_v = i / per_row >= cta_rows;
    const int64_t where = block_of[r];
    if (where == -2) continue;
    const int head = piece / pieces, chunk = piece % pieces;
    uint4 codes = make_uint4(0, 0, 0, 0);
    float scale = 0.0f;
    if (where >= 0) {
      const int64_t block_index = where + (int64_t)head * per_page;
      codes = *reinterpret_cast<const uint4*>(
          (is_v ? cache.v_values : cache.k_values) +
          (block_index * kKvBlock + token_of[r]) * cache.head_dim + chunk * 16);
      // UE8M0: 255 is NaN, 0 is 2^-127 (a subnormal).
      const uint32_t code = (is_v ? cache.v_scales : cache.k_scales)[block_index];
      scale = code == 0 ? __uint_as_float(0x00400000u)
                        : __uint_as_float(code == 255u ? 0x7fc00000u : code << 23);
    }
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = values2(w[j]), c = values2(w[j] >> 16);
      o[2 * j] = pack2<T>(a.x * scale, a.y * scale);
      o[2 * j + 1] = pack2<T>(c.x * scale, c.y * scale);
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(is_v ? out.v : out.k) +
                                          (row0 + r) * per_row * 16 + (int64_t)piece * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

template <class T, int D>
void launch_write(const KvCache& cache, const KvBatch& batch, const KvRows& rows, bool vector,
                  dim3 grid, cudaStream_t stream) {
  if (vector) {
    kv_write_kernel<T, D, true><<<grid, kWriteThreads, 0, stream>>>(cache, batch, rows);
  } else {
    kv_write_kernel<T, D, false><<<grid, kWriteThreads, 0, stream>>>(cache, batch, rows);
  }
}

template <class T>
void launch_write_dim(const KvCache& cache, const KvBatch& batch, const KvRows& rows, bool vector,
                      dim3 grid, cudaStream_t stream) {
  if (cache.head_dim == 64) launch_write<T, 64>(cache, batch, rows, vector, grid, stream);
  if (cache.head_dim == 128) launch_write<T, 128>(cache, batch, rows, vector, grid, stream);
  if (cache.head_dim == 256) launch_write<T, 256>(cache, batch, rows, vector, grid, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int check_kv(const KvCache& cache, const KvBatch& batch) {
  MX_REQUIRE(cache.k_values && cache.v_values && cache.k_scales && cache.v_scales,
             "cache pointers must not be null");
  MX_REQUIRE(cache.head_dim == 64 || cache.head_dim == 128 || cache.head_dim == 256,
             "head_dim must be 64, 128 or 256; got %d", cache.head_dim);
  MX_REQUIRE(cache.page_size == 32 || cache.page_size == 64 || cache.page_size == 128,
             "page_size must be 32, 64 or 128; got %d", cache.page_size);
  MX_REQUIRE(cache.pages > 0 && cache.kv_heads > 0 && cache.kv_heads <= 65535,
             "the cache needs pages and 1 to 65535 heads");
  MX_REQUIRE(cache.pages * cache.kv_heads <= (int64_t(1) << 31) / cache.page_size - 1,
             "pages * kv_heads * page_size must stay below 2^31");
  MX_REQUIRE(aligned16(cache.k_values) && aligned16(cache.v_values),
             "cache values must be 16-byte aligned");
  MX_REQUIRE(batch.batch > 0 && batch.tokens >= 0, "batch must be positive");
  MX_REQUIRE(batch.block_table && batch.seq_lens, "block_table and seq_lens must not be null");
  MX_REQUIRE(batch.table_width > 0 &&
                 (int64_t)batch.table_width * cache.page_size <= (int64_t(1) << 30),
             "block_table must have columns, for at most 2^30 tokens a sequence");
  MX_REQUIRE(batch.cu_seqlens != nullptr || batch.tokens == batch.batch,
             "without cu_seqlens every sequence has exactly one row");
  MX_REQUIRE(batch.tokens <= (int64_t(1) << 30), "at most 2^30 token rows a call");
  return kOk;
}

int kv_cache_write(const KvCache& cache, const KvBatch& batch, const void* k, const void* v,
                   int dtype, const int64_t strides[4], cudaStream_t stream) {
  if (int rc = check_kv(cache, batch)) return rc;
  MX_REQUIRE(dtype == kF16 || dtype == kBF16, "k and v must be float16 or bfloat16");
  if (batch.tokens == 0) return kOk;
  MX_REQUIRE(k != nullptr && v != nullptr, "k and v must not be null");
  const KvRows rows{k, v, strides[0], strides[1], strides[2], strides[3]};
  bool vector = aligned16(k) && aligned16(v);
  for (int i = 0; i < 4; ++i) vector = vector && strides[i] % 8 == 0;
  const int64_t slots = batch.cu_seqlens == nullptr
                            ? batch.batch
                            : slots_before(batch.tokens, batch.batch) + 1;
  const dim3 grid((unsigned)slots, (unsigned)cache.kv_heads, 2);
  if (dtype == kBF16) {
    launch_write_dim<__nv_bfloat16>(cache, batch, rows, vector, grid, stream);
  } else {
    launch_write_dim<__half>(cache, batch, rows, vector, grid, stream);
  }
  MX_CUDA(cudaGetLastError());
  return kOk;
}

int kv_cache_read(const KvCache& cache, const KvBatch& batch, void* k, void* v, int dtype,
                  cudaStream_t stream) {
  if (int rc = check_kv(cache, batch)) return rc;
  MX_REQUIRE(dtype == kF16 || dtype == kBF16, "outputs must be float16 or bfloat16");
  if (batch.tokens == 0) return kOk;
  MX_REQUIRE(k != nullptr && v != nullptr && aligned16(k) && aligned16(v),
             "outputs must be 16-byte aligned");
  const KvOut out{k, v};
  // Few rows are dealt out thin: 77 rows of 8 heads took 5.9 us at 16 a CTA.
  int cta_rows = kReadRows;
  while (cta_rows > 1 && batch.tokens < (int64_t)cta_rows * 2 * 148) cta_rows /= 2;
  const unsigned grid = (unsigned)ceil_div64(batch.tokens, cta_rows);
  if (dtype == kBF16) {
    kv_read_kernel<__nv_bfloat16><<<grid, kReadThreads, 0, stream>>>(cache, batch, out, cta_rows);
  } else {
    kv_read_kernel<__half><<<grid, kReadThreads, 0, stream>>>(cache, batch, out, cta_rows);
  }
  MX_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace mx
