// Grouped-query attention of new tokens over the paged 8-bit cache: the entry points.
//
//   out_i = sum_j p_ij v_j,  p_ij = softmax_j(scale * q_i . k_j)
// over the cached tokens j < seq_len of the sequence, and j <= position of i when causal.  A row
// that may see no token is zero.
//
// Two kernels share the sequences of a batch by their rows (new tokens x query heads per key
// head): up to kv_decode_rows() go to the decode kernel, whose tiles have the cached tokens as
// their long side, the others to the prefill kernel, which has 128 rows to a tile.  The border is
// what the decode kernel's tensor memory holds: it is still the faster one there (65536 tokens, 8
// key heads of 128: 49 us with 32 rows, the other 76 us with 36; 4 key heads of 256: 50 us with 24,
// 65 us with 32).
#include "kv_attention.cuh"

#include <climits>
#include <cmath>

namespace mx {

int launch_kv_decode(const AttentionArgs& a, int dtype, cudaStream_t stream);
int kv_decode_rows(int head_dim, int dtype);
int64_t kv_decode_workspace(int64_t batch, int kv_heads, int head_dim, int dtype, int rows,
                            int64_t max_context);
int launch_kv_prefill(const AttentionArgs& a, int dtype, cudaStream_t stream);
int64_t kv_prefill_workspace(int64_t batch, int64_t tokens, int kv_heads, int group, int head_dim,
                             int64_t max_context);
int* device_status_word(int device);

namespace {

// Limits of a call: query heads, rows (token rows, and times the query heads of a key head), and cached
// tokens that a block table can name (check_kv).
constexpr int kMostHeads = 65535;
constexpr int64_t kMostRows = int64_t(1) << 30, kMostContext = int64_t(1) << 30;

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

// A call's launches: `decode_rows` > 0 runs the decode kernel for sequences of up to that many
// rows, `prefill` the other one for those with more.
struct AttentionPlan {
  int decode_rows;
  bool prefill;
  int64_t decode_bytes, prefill_bytes;
};
static AttentionPlan plan_attention(int64_t batch, int64_t tokens, int64_t max_query_len, int group,
                                    int kv_heads, int head_dim, int dtype, int64_t max_context) {
  AttentionPlan p{};
  const int most = kv_decode_rows(head_dim, dtype);
  const int64_t rows = (max_query_len < tokens ? max_query_len : tokens) * group;
  if (rows <= most) {
    p.decode_rows = (int)rows;
  } else {
    p.prefill = true;
    // In a batch of several sequences some may have few rows; a lone one has all of them.
    if (batch > 1 && group <= most) p.decode_rows = most;
  }
  if (p.decode_rows > 0)
    p.decode_bytes = kv_decode_workspace(batch, kv_heads, head_dim, dtype, p.decode_rows, max_context);
  if (p.prefill)
    p.prefill_bytes = kv_prefill_workspace(batch, tokens, kv_heads, group, head_dim, max_context);
  return p;
}

int64_t kv_cache_attention_workspace(int64_t batch, int64_t tokens, int64_t max_query_len,
                                     int q_heads, int kv_heads, int head_dim, int dtype,
                                     int64_t max_context) {
  // The call's own limits.
  if (batch < 1 || batch > INT_MAX || tokens < 0 || tokens > kMostRows || max_query_len < 1 ||
      q_heads < 1 || q_heads > kMostHeads || kv_heads < 1 || q_heads % kv_heads != 0 ||
      tokens * (q_heads / kv_heads) > kMostRows ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || (dtype != kF16 && dtype != kBF16) ||
      max_context < 1 || max_context > kMostContext) {
    return -1;
  }
  if (tokens == 0) return 0;
  const AttentionPlan p = plan_attention(batch, tokens, max_query_len, q_heads / kv_heads, kv_heads,
                                         head_dim, dtype, max_context);
  return p.decode_bytes + p.prefill_bytes;
}

int kv_cache_attention(const KvCache& cache, const KvBatch& batch, const void* q, void* out,
                       int dtype, int q_heads, const int64_t strides[4], int64_t max_query_len,
                       float scale, int causal, void* workspace, int64_t workspace_bytes,
                       cudaStream_t stream) {
  if (int rc = check_kv(cache, batch)) return rc;
  MX_REQUIRE(dtype == kF16 || dtype == kBF16, "q must be float16 or bfloat16");
  MX_REQUIRE(q_heads > 0 && q_heads <= kMostHeads && q_heads % cache.kv_heads == 0,
             "q_heads (%d) must be a multiple of the cache's %d heads", q_heads, cache.kv_heads);
  MX_REQUIRE(max_query_len >= 1, "max_query_len must be positive");
  const float scale_log2 = scale * 1.4426950408889634f;
  MX_REQUIRE(std::isfinite(scale_log2), "scale must be finite, and still be so times log2(e)");
  if (batch.tokens == 0) return kOk;
  MX_REQUIRE(q != nullptr && out != nullptr, "q and out must not be null");
  const int group = q_heads / cache.kv_heads;
  MX_REQUIRE(batch.tokens * group <= kMostRows, "at most 2^30 rows (tokens x group) a call");
  const AttentionPlan plan =
      plan_attention(batch.batch, batch.tokens, max_query_len, group, cache.kv_heads,
                     cache.head_dim, dtype, (int64_t)batch.table_width * cache.page_size);
  const int64_t need = plan.decode_bytes + plan.prefill_bytes;
  MX_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && aligned16(workspace))),
             "the workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
  int device = 0;
  MX_CUDA(cudaGetDevice(&device));
  AttentionArgs a{};
  a.cache = cache;
  a.batch = batch;
  a.q = q;
  a.out = out;
  a.status = device_status_word(device);
  if (a.status == nullptr) return kCudaError;
  a.q_token_stride = strides[0];
  a.q_head_stride = strides[1];
  a.out_token_stride = strides[2];
  a.out_head_stride = strides[3];
  a.q_heads = q_heads;
  a.group = group;
  a.scale_log2 = scale_log2;
  a.causal = causal;
  a.vector = aligned16(q) && strides[0] % 8 == 0 && strides[1] % 8 == 0;
  a.vector_out = aligned16(out) && strides[2] % 8 == 0 && strides[3] % 8 == 0;
  a.max_rows = plan.decode_rows;
  a.min_rows = plan.decode_rows;
  if (plan.prefill) {
    a.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.decode_bytes);
    if (int rc = launch_kv_prefill(a, dtype, stream)) return rc;
  }
  a.partials = static_cast<float*>(workspace);
  return plan.decode_rows > 0 ? launch_kv_decode(a, dtype, stream) : kOk;
}

}  // namespace mx
