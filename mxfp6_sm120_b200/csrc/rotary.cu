// Rotary positions with several axes (time, height, width of image and video tokens).
//
// Frequency i of a head turns the pair (x[i], x[i + half]) by
//   angle(t, i) = positions[axis[i]][t] * inv_freq[i].
// A position of 10^6 times a frequency near 1 leaves a 32-bit product only four fraction bits of
// a turn's radians, so the product is taken in 64 bits, in turns (inv_freq / 2 pi), and reduced
// to half a turn there; sine and cosine of what is left are 32-bit, the rotation is a 32-bit
// multiply-add, rounded once.  All heads of a token share the angles: a CTA computes them once
// into shared memory and then streams its heads, sixteen bytes a thread and half.
// Every byte is read and written once: HBM bounds it, launch latency at decode sizes.  Inside a
// CUDA graph: 8192 tokens, 32 + 8 heads of 128: 32 us, 5.3 TB/s of a copy's 6.57; 17 tokens: 2.7 us.
#include "common.cuh"

#include <type_traits>

namespace mx {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;
constexpr int kMaxAxes = 8;
constexpr int kMostTokens = 4;  // tokens of a CTA

struct RotaryArgs {
  const void* x[2];  // query and key heads
  void* out[2];
  int64_t x_token[2], x_head[2];      // strides in elements
  int64_t out_token[2], out_head[2];
  int heads[2];
  const void* positions;  // [axes, tokens] int32 or int64
  int64_t position_stride;
  const double* inv_freq;  // [half]
  const int32_t* axis;     // [half]
  int64_t tokens;
  int axes;
  int half;
  int dim;
  int wide_positions;  // 1: int64
  int adjacent;        // 1: pairs (2 i, 2 i + 1) instead of (i, i + half)
  int cta_tokens;      // tokens a CTA takes
};

template <class T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Whole vectors when every stride and pointer allows it, single values otherwise.
template <class T, bool kVector>
__device__ __forceinline__ uint4 load8(const T* at) {
  if constexpr (kVector) return *reinterpret_cast<const uint4*>(at);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(at) + 2 * i;
    w[i] = (uint32_t)u[0] | (uint32_t)u[1] << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T, bool kVector>
__device__ __forceinline__ void store8(T* at, const uint4& v) {
  if constexpr (kVector) {
    *reinterpret_cast<uint4*>(at) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint16_t* u = reinterpret_cast<uint16_t*>(at) + 2 * i;
      u[0] = (uint16_t)w[i];
      u[1] = (uint16_t)(w[i] >> 16);
    }
  }
}

__host__ __device__ __forceinline__ int kept_items(int dim, int half) { return (dim - 2 * half + 15) / 16; }

template <class T, bool kVector>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  __shared__ __align__(16) float cosines[kMostTokens * kMaxHalf];
  __shared__ __align__(16) float sines[kMostTokens * kMaxHalf];
  const int64_t token0 = (int64_t)blockIdx.x * a.cta_tokens;
  const int tokens = (int)(a.tokens - token0 < a.cta_tokens ? a.tokens - token0 : a.cta_tokens);
  for (int n = threadIdx.x; n < tokens * a.half; n += kThreads) {
    const int i = n % a.half;
    const int axis = a.axis[i];
    float s = NAN, c = NAN;  // no row of positions for the axis: no angle to turn by
    if (axis >= 0 && axis < a.axes) {
      const int64_t at = axis * a.position_stride + token0 + n / a.half;
      const int64_t position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[at]
                                                : static_cast<const int32_t*>(a.positions)[at];
      const double turns = (double)position * (a.inv_freq[i] * 0.15915494309189533577);
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    }
    sines[n] = s;
    cosines[n] = c;
  }
  __syncthreads();
  // Work items: eight pairs of a head, then up to sixteen untouched values behind rotary_dim.
  const int turned = a.half / 8;
  const int per_head = turned + kept_items(a.dim, a.half);
  const int total = (a.heads[0] + a.heads[1]) * per_head;
#pragma unroll 2
  for (int n = blockIdx.y * kThreads + threadIdx.x; n < total * tokens; n += gridDim.y * kThreads) {
    const int which_token = n / total, i = n % total;
    const int64_t token = token0 + which_token;
    const float* cosine = cosines + which_token * a.half;
    const float* sine = sines + which_token * a.half;
    const int all = i / per_head, item = i % per_head;
    const int which = all >= a.heads[0] ? 1 : 0;
    const int head = which ? all - a.heads[0] : all;
    const T* x = static_cast<const T*>(a.x[which]) + token * a.x_token[which] +
                 head * a.x_head[which];
    T* y = static_cast<T*>(a.out[which]) + token * a.out_token[which] + head * a.out_head[which];
    if (item >= turned) {
      if (x != y) {
        const int at = 2 * a.half + (item - turned) * 16;
        const bool two = at + 8 < a.dim;
        const uint4 u = load8<T, kVector>(x + at), v = load8<T, kVector>(x + (two ? at + 8 : at));
        store8<T, kVector>(y + at, u);
        if (two) store8<T, kVector>(y + at + 8, v);
      }
      continue;
    }
    const int lo_at = a.adjacent ? item * 16 : item * 8;
    const int hi_at = a.adjacent ? item * 16 + 8 : item * 8 + a.half;
    float lo[8], hi[8];
    unpack8<T>(load8<T, kVector>(x + lo_at), lo);
    unpack8<T>(load8<T, kVector>(x + hi_at), hi);
    if (a.adjacent) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float c = cosine[item * 8 + j], s = sine[item * 8 + j];
        const float u = lo[2 * j], v = lo[2 * j + 1];
        lo[2 * j] = u * c - v * s;
        lo[2 * j + 1] = v * c + u * s;
        const float d = cosine[item * 8 + 4 + j], t = sine[item * 8 + 4 + j];
        const float p = hi[2 * j], q = hi[2 * j + 1];
        hi[2 * j] = p * d - q * t;
        hi[2 * j + 1] = q * d + p * t;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = cosine[item * 8 + j], s = sine[item * 8 + j];
        const float u = lo[j], v = hi[j];
        lo[j] = u * c - v * s;
        hi[j] = v * c + u * s;
      }
    }
    store8<T, kVector>(y + lo_at, pack8<T>(lo));
    store8<T, kVector>(y + hi_at, pack8<T>(hi));
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int rotary_multi_axis(const void* q, void* q_out, int q_heads, const int64_t q_strides[4],
                      const void* k, void* k_out, int k_heads, const int64_t k_strides[4],
                      int dtype, int64_t tokens, int dim, const void* positions,
                      int64_t position_stride, int axes, int wide_positions,
                      const double* inv_freq, const int32_t* axis, int half, int adjacent,
                      cudaStream_t stream) {
  MX_REQUIRE(dtype == kF16 || dtype == kBF16, "q and k must be float16 or bfloat16");
  MX_REQUIRE(dim > 0 && dim % 8 == 0, "head_dim must be a positive multiple of 8; got %d", dim);
  MX_REQUIRE(half > 0 && half % 8 == 0 && half <= kMaxHalf && 2 * half <= dim,
             "rotary_dim must be a multiple of 16, at most head_dim and %d; got %d", 2 * kMaxHalf,
             2 * half);
  MX_REQUIRE(axes >= 1 && axes <= kMaxAxes, "1 to %d position axes; got %d", kMaxAxes, axes);
  MX_REQUIRE(q_heads >= 0 && k_heads >= 0 && tokens >= 0, "sizes must not be negative");
  MX_REQUIRE(tokens <= 0x7fffffff && (int64_t)(q_heads + k_heads) * dim <= (int64_t(1) << 30),
             "at most 2^31 - 1 tokens and 2^30 values a token");
  if (tokens == 0 || q_heads + k_heads == 0) return kOk;
  MX_REQUIRE((q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)) && positions &&
                 inv_freq && axis,
             "pointers must not be null");
  RotaryArgs a{};
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* strides[2] = {q_strides, k_strides};
  bool vector = true;
  for (int w = 0; w < 2; ++w) {
    a.heads[w] = w ? k_heads : q_heads;
    if (a.heads[w] == 0) continue;
    a.x[w] = in[w];
    a.out[w] = out[w];
    a.x_token[w] = strides[w][0];
    a.x_head[w] = strides[w][1];
    a.out_token[w] = strides[w][2];
    a.out_head[w] = strides[w][3];
    vector = vector && aligned16(in[w]) && aligned16(out[w]);
    for (int i = 0; i < 4; ++i) vector = vector && strides[w][i] % 8 == 0;
  }
  a.positions = positions;
  a.position_stride = position_stride;
  a.inv_freq = inv_freq;
  a.axis = axis;
  a.tokens = tokens;
  a.axes = axes;
  a.half = half;
  a.dim = dim;
  a.wide_positions = wide_positions;
  a.adjacent = adjacent;
  // Four tokens share a CTA where there are enough, so that its angles and its last items fill the
  // threads (8192 tokens x 40 heads of 128: 34.9 us with one).  A CTA's items are dealt to several
  // while CTAs alone leave SMs idle, and, in shares of two passes or more, while there are fewer than
  // eight an SM (1924 tokens x 28 heads of 256, 64 turned: 15 us, with a CTA for four tokens 26).
  const int items = (q_heads + k_heads) * (half / 8 + kept_items(dim, half));
  a.cta_tokens = tokens >= 8 * 148 ? kMostTokens : 1;
  const int64_t groups = ceil_div64(tokens, a.cta_tokens);
  const int64_t cta_items = (int64_t)items * a.cta_tokens;
  int64_t parts = ceil_div64(cta_items, kThreads);
  if (groups * parts > 2 * 148) {
    const int64_t most = cta_items / (2 * kThreads), want = ceil_div64(8 * 148, groups);
    parts = most < want ? most : want;
    if (parts < 1) parts = 1;
  }
  const dim3 grid((unsigned)groups, (unsigned)parts);
  if (dtype == kBF16) {
    if (vector) rotary_kernel<__nv_bfloat16, true><<<grid, kThreads, 0, stream>>>(a);
    else rotary_kernel<__nv_bfloat16, false><<<grid, kThreads, 0, stream>>>(a);
  } else {
    if (vector) rotary_kernel<__half, true><<<grid, kThreads, 0, stream>>>(a);
    else rotary_kernel<__half, false><<<grid, kThreads, 0, stream>>>(a);
  }
  MX_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace mx
