// Grouped-query attention of new tokens over the paged 8-bit cache.
//
//   out_i = sum_j p_ij v_j,  p_ij = softmax_j(scale * q_i . k_j)
// over the cached tokens j < seq_len of the sequence, and j <= position of i when causal.  A row
// that may see no token is zero.
//
// First form: four warps per (token row, query head); each walks every fourth block of 32 tokens
// with a running maximum and sum, and the four results are joined in a fixed order.
#include "kv_attention.cuh"

namespace mx {

int launch_kv_decode(const AttentionArgs& a, int dtype, cudaStream_t stream);
int kv_decode_rows(int head_dim, int dtype);
int64_t kv_decode_workspace(int64_t batch, int kv_heads, int head_dim, int dtype, int rows,
                            int64_t max_context);
int* device_status_word(int device);

namespace {

constexpr int kWarps = 4;

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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = []() -> EncodeFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      return nullptr;
    }
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

}  // namespace

// The cache's values as rows of head_dim bytes, copied one page x 128 (64) columns at a time.
int make_kv_map(CUtensorMap* map, const uint8_t* values, const KvCache& cache) {
  EncodeFn fn = encode_fn();
  if (fn == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from the CUDA driver");
    return kCudaError;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cache.head_dim,
                              (cuuint64_t)(cache.pages * cache.kv_heads * cache.page_size)};
  const cuuint64_t strides[1] = {(cuuint64_t)cache.head_dim};
  const cuuint32_t inner = cache.head_dim < 128 ? cache.head_dim : 128;
  const cuuint32_t box[2] = {inner, (cuuint32_t)cache.page_size};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(values), dims,
                         strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with CUresult %d for the cache", (int)rc);
    return kCudaError;
  }
  return kOk;
}

int64_t kv_cache_attention_workspace(int64_t batch, int64_t tokens, int64_t max_query_len,
                                     int q_heads, int kv_heads, int head_dim, int dtype,
                                     int64_t max_context) {
  (void)tokens;
  if (batch < 1 || max_query_len < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || max_context < 1) {
    return -1;
  }
  const int64_t rows = max_query_len * (q_heads / kv_heads);
  if (rows > kv_decode_rows(head_dim, dtype)) return 0;
  return kv_decode_workspace(batch, kv_heads, head_dim, dtype, (int)rows, max_context);
}

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
  const int64_t need = kv_cache_attention_workspace(
      batch.batch, batch.tokens, max_query_len, q_heads, cache.kv_heads, cache.head_dim, dtype,
      (int64_t)batch.table_width * cache.page_size);
  MX_REQUIRE(workspace_bytes >= need && (need == 0 || aligned16(workspace)) &&
                 (need == 0 || workspace != nullptr),
             "the workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
  int device = 0;
  MX_CUDA(cudaGetDevice(&device));
  AttentionArgs a{};
  a.cache = cache;
  a.batch = batch;
  a.q = q;
  a.out = out;
  a.partials = static_cast<float*>(workspace);
  a.status = device_status_word(device);
  if (a.status == nullptr) return kCudaError;
  a.q_token_stride = strides[0];
  a.q_head_stride = strides[1];
  a.out_token_stride = strides[2];
  a.out_head_stride = strides[3];
  a.q_heads = q_heads;
  a.group = q_heads / cache.kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.causal = causal;
  a.vector = aligned16(q) && strides[0] % 8 == 0 && strides[1] % 8 == 0;
  const int64_t rows = max_query_len * a.group;
  if (rows <= kv_decode_rows(cache.head_dim, dtype)) {
    a.max_rows = (int)rows;
    return launch_kv_decode(a, dtype, stream);
  }
  if (dtype == kBF16) launch_rows<__nv_bfloat16>(a, stream);
  else launch_rows<__half>(a, stream);
  MX_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace mx
