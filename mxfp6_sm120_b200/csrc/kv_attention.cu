// Grouped-query attention of new tokens over the paged 8-bit cache.
//
//   out_i = sum_j p_ij v_j,  p_ij = softmax_j(scale * q_i . k_j)
// over the cached tokens j < seq_len of the sequence, and j <= position of i when causal.  A row
// that may see no token is zero.
//
// First form: four warps per (token row, query head); each walks every fourth block of 32 tokens
// with a running maximum and sum, and the four results are joined in a fixed order.
#include "kv_cache.cuh"

#include <cuda_fp8.h>
#include <type_traits>

namespace mx {
namespace {

constexpr int kWarps = 4;

struct AttentionArgs {
  KvCache cache;
  KvBatch batch;
  const void* q;
  void* out;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int q_heads;
  float scale_log2;  // softmax scale * log2(e)
  int causal;
};

__device__ __forceinline__ float2 values2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}
__device__ __forceinline__ float scale_of(uint32_t code) {
  return code == 0 ? __uint_as_float(0x00400000u)
                   : __uint_as_float(code == 255u ? 0x7fc00000u : code << 23);
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) kv_attention_rows_kernel(const AttentionArgs a) {
  __shared__ float q_s[D];
  __shared__ float p_s[kWarps][32];
  __shared__ float acc_s[kWarps][D];
  __shared__ float max_s[kWarps], sum_s[kWarps];
  const int64_t row = blockIdx.x;
  const int head = blockIdx.y;
  const int kv_head = head / (a.q_heads / a.cache.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b = (int)row;
  if (a.batch.cu_seqlens != nullptr) {
    int lo = 0, hi = a.batch.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.batch.cu_seqlens[mid] <= row) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  const KvSpan span = kv_span(a.batch, a.cache.page_size, b);
  if (row < span.row || row >= span.row + span.rows) return;
  const int64_t position = (int64_t)a.batch.seq_lens[b] - span.rows + (row - span.row);
  int64_t end = span.length;
  if (a.causal && position + 1 < end) end = position + 1;
  const T* q = static_cast<const T*>(a.q) + row * a.q_token_stride + head * a.q_head_stride;
  for (int i = threadIdx.x; i < D; i += kWarps * 32) q_s[i] = to_float<T>(q[i]) * a.scale_log2;
  __syncthreads();
  const int per_page = a.cache.page_size / kKvBlock;
  float top = -INFINITY, sum = 0.0f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
  for (int64_t block = warp; block * kKvBlock < end; block += kWarps) {
    const int64_t page = kv_page(a.batch, a.cache, b, (int)block);
    if (page < 0) continue;
    const int64_t index = (page * a.cache.kv_heads + kv_head) * per_page + block % per_page;
    const int held = end - block * kKvBlock < kKvBlock ? (int)(end - block * kKvBlock) : kKvBlock;
    const uint8_t* k = a.cache.k_values + index * kKvBlock * D;
    const uint8_t* v = a.cache.v_values + index * kKvBlock * D;
    float s = -INFINITY;
    if (lane < held) {
      s = 0.0f;
      const uint4* kr = reinterpret_cast<const uint4*>(k + lane * D);
      for (int c = 0; c < D / 16; ++c) {
        const uint4 raw = kr[c];
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = values2(w[j]), y = values2(w[j] >> 16);
          const float* qq = q_s + c * 16 + j * 4;
          s += qq[0] * x.x + qq[1] * x.y + qq[2] * y.x + qq[3] * y.y;
        }
      }
      s *= scale_of(a.cache.k_scales[index]);
    }
    float block_top = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) block_top = fmaxf(block_top, __shfl_xor_sync(~0u, block_top, o));
    const float next = fmaxf(top, block_top);
    const float base = next == -INFINITY ? 0.0f : next;
    const float fade = exp2f(top - base);
    const float p = lane < held ? exp2f(s - base) : 0.0f;
    float block_sum = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) block_sum += __shfl_xor_sync(~0u, block_sum, o);
    sum = sum * fade + block_sum;
    top = next;
    p_s[warp][lane] = p;
    __syncwarp();
    const float vs = scale_of(a.cache.v_scales[index]);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] *= fade;
    for (int t = 0; t < held; ++t) {
      const float w = p_s[warp][t] * vs;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const float2 x = values2(*reinterpret_cast<const uint16_t*>(v + t * D + i * 64 + lane * 2));
        acc[2 * i] += w * x.x;
        acc[2 * i + 1] += w * x.y;
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    acc_s[warp][i * 64 + lane * 2] = acc[2 * i];
    acc_s[warp][i * 64 + lane * 2 + 1] = acc[2 * i + 1];
  }
  if (lane == 0) {
    max_s[warp] = top;
    sum_s[warp] = sum;
  }
  __syncthreads();
  float all = -INFINITY;
  for (int w = 0; w < kWarps; ++w) all = fmaxf(all, max_s[w]);
  const float base = all == -INFINITY ? 0.0f : all;
  float total = 0.0f, factor[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    factor[w] = exp2f(max_s[w] - base);
    total += factor[w] * sum_s[w];
  }
  T* out = static_cast<T*>(a.out) + row * a.out_token_stride + head * a.out_head_stride;
  for (int i = threadIdx.x; i < D; i += kWarps * 32) {
    float o = 0.0f;
    for (int w = 0; w < kWarps; ++w) o += factor[w] * acc_s[w][i];
    o = total == 0.0f ? 0.0f : o / total;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) out[i] = __float2bfloat16_rn(o);
    else out[i] = __float2half_rn(o);
  }
}

template <class T>
void launch_rows(const AttentionArgs& a, cudaStream_t stream) {
  const dim3 grid((unsigned)a.batch.tokens, (unsigned)a.q_heads);
  if (a.cache.head_dim == 64) kv_attention_rows_kernel<T, 64><<<grid, kWarps * 32, 0, stream>>>(a);
  if (a.cache.head_dim == 128) kv_attention_rows_kernel<T, 128><<<grid, kWarps * 32, 0, stream>>>(a);
  if (a.cache.head_dim == 256) kv_attention_rows_kernel<T, 256><<<grid, kWarps * 32, 0, stream>>>(a);
}

}  // namespace

int kv_cache_attention(const KvCache& cache, const KvBatch& batch, const void* q, void* out,
                       int dtype, int q_heads, const int64_t strides[4], int64_t max_query_len,
                       float scale, int causal, void* workspace, int64_t workspace_bytes,
                       cudaStream_t stream) {
  if (int rc = check_kv(cache, batch)) return rc;
  MX_REQUIRE(dtype == kF16 || dtype == kBF16, "q must be float16 or bfloat16");
  MX_REQUIRE(q_heads > 0 && q_heads <= 65535 && q_heads % cache.kv_heads == 0,
             "q_heads (%d) must be a multiple of the cache's %d heads", q_heads, cache.kv_heads);
  MX_REQUIRE(max_query_len >= 1, "max_query_len must be positive");
  if (batch.tokens == 0) return kOk;
  MX_REQUIRE(q != nullptr && out != nullptr, "q and out must not be null");
  (void)workspace;
  (void)workspace_bytes;
  AttentionArgs a{cache, batch, q, out, strides[0], strides[1], strides[2], strides[3], q_heads,
                  scale * 1.4426950408889634f, causal};
  if (dtype == kBF16) launch_rows<__nv_bfloat16>(a, stream);
  else launch_rows<__half>(a, stream);
  MX_CUDA(cudaGetLastError());
  return kOk;
}

int64_t kv_cache_attention_workspace(int64_t, int64_t, int64_t, int, int, int, int, int64_t) {
  return 0;
}

}  // namespace mx
