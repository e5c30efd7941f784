// Rounding to 8-bit floating point (e4m3) with a scale for each block of 128, and the
// entry points of its products (fp8_tc.cu).
//
// A block's scale is the smallest power of two s with max |x| <= 448 s (at least 2^-126),
// so that x / s is exact and q = e4m3(x / s) is x rounded once, to 4 significant bits,
// whatever the block's largest value; a scale of max / 448 would use at most one more of
// the type's 15 powers of two and round twice. A block with an infinity or NaN has scale
// and values NaN. Rows: 128 consecutive values of a row (the last block may be
// shorter). Weights: 128 x 128 of a matrix.
// Bound by memory's latency and the conversions alike (B200: 8191 x 4096 bf16 22 us, 4.6 TB/s
// with 72% of the issue slots; 16400 x 1408 with silu 27 us, 4.4 TB/s, 75%): a thread has
// the eight values of one block (sixteen with an activation) in flight and no other load.
// Weights are rounded once: 4096 x 8192 bf16 60 us where they lie along K, 196 us with the
// transposing copy before it.
#include <cuda_fp8.h>

#include "activation.cuh"
#include "experts.cuh"
#include "fp8.cuh"

namespace es {
namespace {

constexpr int kFp8Threads = 256;

// The larger of two magnitudes; NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A block's scale from its largest magnitude, and 1 / scale. 448 = 1.75 * 2^8.
__device__ __forceinline__ float block_scale(float peak, float& inverse) {
  const uint32_t bits = __float_as_uint(peak);
  int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased by 127
  e = e < 1 ? 1 : e;
  const bool finite = bits < 0x7f800000u;
  inverse = finite ? __uint_as_float(static_cast<uint32_t>(254 - e) << 23) : NAN;
  return finite ? __uint_as_float(static_cast<uint32_t>(e) << 23) : NAN;
}

__device__ __forceinline__ uint32_t round4(const float* v, float inverse) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0] * inverse, v[1] * inverse), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2] * inverse, v[3] * inverse), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// Eight values from p (8 elements aligned to 16 bytes).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  constexpr int LOADS = 8 * sizeof(T) / 16;
  alignas(16) T t[8];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
}

// Sixteen threads a block, eight consecutive values each. WIDE: whole pieces at 16-byte
// addresses. ACT: the value is act(x[i]) * x[K + i], in fp32 (-1: x[i]); the fast exp's
// error is far below 8 bits' rounding. I: the type that holds every block's number (64-bit
// divisions are a fifth of the time).
template <typename T, int ACT, bool WIDE, typename I>
__global__ void __launch_bounds__(kFp8Threads) quantize_blocks_kernel(const T* x, I n, I blocks, int64_t K,
                                                                      int64_t stride, uint8_t* q, float* scale) {
  let_next_grid_start();
  const I at = static_cast<I>(blockIdx.x) * (kFp8Threads / 16) + (threadIdx.x >> 4);
  const bool live = at < n;
  const I row = at / blocks;
  const int64_t r = row, c = static_cast<int64_t>(at - row * blocks) * kScaleBlock + (threadIdx.x & 15) * 8;
  const T* from = x + r * stride + c;
  float v[8];
  auto load = [&](const T* p, float (&t)[8]) {
    if (WIDE && live && c < K) {
      load8(p, t);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = !WIDE && live && c + i < K ? to_f32(p[i]) : 0.0f;
    }
  };
  load(from, v);
  if constexpr (ACT >= 0) {
    float u[8];
    load(from + K, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a, s;
      activate<ACT, false>(v[i], a, s);
      v[i] = a * u[i];
    }
  }
  float peak = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) peak = max_nan(peak, fabsf(v[i]));
#pragma unroll
  for (int o = 8; o; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
  if (!live) return;
  float inverse;
  const float s = block_scale(peak, inverse);
  if ((threadIdx.x & 15) == 0) scale[at] = s;
  const uint2 o = make_uint2(round4(v, inverse), round4(v + 4, inverse));
  uint8_t* to = q + r * K + c;
  if constexpr (WIDE) {
    if (c < K) *reinterpret_cast<uint2*>(to) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) to[i] = static_cast<uint8_t>((i < 4 ? o.x : o.y) >> (i & 3) * 8);
  }
}

// A CTA for a block of 128 x 128 of a contiguous (matrices, N, K) tensor.
template <typename T>
__global__ void __launch_bounds__(kFp8Threads) quantize_weights_kernel(const T* w, int64_t N, int64_t K, uint8_t* q,
                                                                       float* scale) {
  const int64_t kb = (K + kScaleBlock - 1) / kScaleBlock, nb = (N + kScaleBlock - 1) / kScaleBlock;
  const int64_t at = blockIdx.x, m = at / (nb * kb), n0 = at / kb % nb * kScaleBlock, k0 = at % kb * kScaleBlock;
  const int rows = static_cast<int>(min(N - n0, static_cast<int64_t>(kScaleBlock)));
  const int cols = static_cast<int>(min(K - k0, static_cast<int64_t>(kScaleBlock)));
  const int64_t base = (m * N + n0) * K + k0;
  const int c = threadIdx.x & (kScaleBlock - 1);
  __shared__ float part[kFp8Threads / 32];
  float peak = 0.0f;
  for (int r = threadIdx.x / kScaleBlock; r < rows; r += kFp8Threads / kScaleBlock)
    if (c < cols) peak = max_nan(peak, fabsf(to_f32(w[base + r * K + c])));
#pragma unroll
  for (int o = 16; o; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = peak;
  __syncthreads();
  peak = part[0];
#pragma unroll
  for (int i = 1; i < kFp8Threads / 32; ++i) peak = max_nan(peak, part[i]);
  float inverse;
  const float s = block_scale(peak, inverse);
  if (threadIdx.x == 0) scale[at] = s;
  for (int r = threadIdx.x / kScaleBlock; r < rows; r += kFp8Threads / kScaleBlock)
    if (c < cols)
      q[base + r * K + c] = __nv_cvt_float_to_fp8(to_f32(w[base + r * K + c]) * inverse, __NV_SATFINITE, __NV_E4M3);
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

template <typename T, int ACT, typename I>
int quantize_indexed(const void* x, int64_t rows, int64_t K, int64_t stride, uint8_t* q, float* scale,
                     cudaStream_t s) {
  const int64_t blocks = (K + kScaleBlock - 1) / kScaleBlock, n = rows * blocks, per = kFp8Threads / 16;
  if ((n + per - 1) / per > 0x7fffffffLL) return ES_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>((n + per - 1) / per);
  if (K % 8 == 0 && stride * sizeof(T) % 16 == 0 && aligned(x, 16) && aligned(q, 8))
    ES_LAUNCH((quantize_blocks_kernel<T, ACT, true, I>), grid, kFp8Threads, 0, s, static_cast<const T*>(x),
              static_cast<I>(n), static_cast<I>(blocks), K, stride, q, scale);
  else
    ES_LAUNCH((quantize_blocks_kernel<T, ACT, false, I>), grid, kFp8Threads, 0, s, static_cast<const T*>(x),
              static_cast<I>(n), static_cast<I>(blocks), K, stride, q, scale);
  return ES_OK;
}

template <typename T, int ACT>
int quantize_launch(const void* x, int64_t rows, int64_t K, int64_t stride, uint8_t* q, float* scale, cudaStream_t s) {
  if (rows * ((K + kScaleBlock - 1) / kScaleBlock) < 0x7fffff00LL)
    return quantize_indexed<T, ACT, uint32_t>(x, rows, K, stride, q, scale, s);
  return quantize_indexed<T, ACT, int64_t>(x, rows, K, stride, q, scale, s);
}

GroupedArgs args_of(const float* x_scale, int64_t x_rows, int64_t x_stride, const float* w_scale, int num_experts,
                    int64_t K, int64_t N, int64_t w_expert_stride, int64_t w_n_stride, const int32_t* offsets,
                    const int32_t* order, int top_k, int64_t num_rows) {
  return GroupedArgs{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride, 1,
                     w_n_stride, x_scale, w_scale};
}

}  // namespace
}  // namespace es

using namespace es;

extern "C" int es_quantize_blocks(const void* x, int dtype, int64_t num_rows, int64_t width, int64_t row_stride,
                                  int activation, uint8_t* q, float* scale, void* stream) {
  if (num_rows < 0 || width < 0 || activation < -1 || activation > ES_ACT_RELU) return ES_ERR_INVALID;
  if (num_rows > 0x7fffff00LL || width > 0x3fffff00LL) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || width == 0) return ES_OK;
  if (!x || !q || !scale) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (activation < 0)
    ES_BY_TYPE(dtype, return (quantize_launch<T, -1>(x, num_rows, width, row_stride, q, scale, s)));
  else
    ES_BY_TYPE(dtype, ES_BY_ACT(activation,
                                return (quantize_launch<T, ACT>(x, num_rows, width, row_stride, q, scale, s))));
  return ES_ERR_UNSUPPORTED;
}

extern "C" int es_quantize_block_weights(const void* w, int dtype, int64_t matrices, int64_t N, int64_t K, uint8_t* q,
                                         float* scale, void* stream) {
  if (matrices < 0 || N < 0 || K < 0) return ES_ERR_INVALID;
  if (N > 0x7fffff00LL || K > 0x7fffff00LL || matrices > 0x7fffff00LL) return ES_ERR_UNSUPPORTED;
  if (matrices == 0 || N == 0 || K == 0) return ES_OK;
  if (!w || !q || !scale) return ES_ERR_INVALID;
  const int64_t per = ((N + kScaleBlock - 1) / kScaleBlock) * ((K + kScaleBlock - 1) / kScaleBlock);
  if (per > 0x7fffffffLL / matrices) return ES_ERR_UNSUPPORTED;
  ES_BY_TYPE(dtype, {
    ES_LAUNCH((quantize_weights_kernel<T>), static_cast<unsigned>(matrices * per), kFp8Threads, 0, as_stream(stream),
              static_cast<const T*>(w), N, K, q, scale);
    return ES_OK;
  });
  return ES_ERR_UNSUPPORTED;
}

extern "C" size_t es_fp8_matmul_workspace_size(const uint8_t* q, const float* x_scale, int64_t x_rows,
                                               int64_t x_stride, const uint8_t* wq, const float* w_scale,
                                               int num_experts, int64_t K, int64_t N, int64_t w_expert_stride,
                                               int64_t w_n_stride, const int32_t* offsets, const int32_t* order,
                                               int top_k, int64_t num_rows) {
  const GroupedArgs g = args_of(x_scale, x_rows, x_stride, w_scale, num_experts, K, N, w_expert_stride, w_n_stride,
                                offsets, order, top_k, num_rows);
  return check_grouped(g) == ES_OK && fp8_tc_ok(g) ? fp8_tc_workspace(g, q, wq) : 0;
}

extern "C" int es_fp8_matmul(const uint8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride,
                             const uint8_t* wq, const float* w_scale, int num_experts, int64_t K, int64_t N,
                             int64_t w_expert_stride, int64_t w_n_stride, const int32_t* offsets,
                             const int32_t* order, int top_k, int64_t num_rows, void* y, int out_dtype,
                             void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const GroupedArgs g = args_of(x_scale, x_rows, x_stride, w_scale, num_experts, K, N, w_expert_stride, w_n_stride,
                                offsets, order, top_k, num_rows);
  ES_TRY(check_grouped(g));
  if (out_dtype != ES_F32 && out_dtype != ES_BF16 && out_dtype != ES_F16) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || N == 0) return ES_OK;
  if (!y) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (K == 0 || x_rows == 0) {
    const size_t bytes = static_cast<size_t>(num_rows) * N * (out_dtype == ES_F32 ? 4 : 2);
    count_launch();
    return cudaMemsetAsync(y, 0, bytes, s) == cudaSuccess ? ES_OK : ES_ERR_CUDA;
  }
  if (!q || !x_scale || !wq || !w_scale) return ES_ERR_INVALID;
  if (!fp8_tc_ok(g)) return ES_ERR_UNSUPPORTED;
  if (workspace_bytes < fp8_tc_workspace(g, q, wq)) return ES_ERR_WORKSPACE;
  return fp8_tc(g, q, wq, y, out_dtype, workspace, status, s);
}

extern "C" int es_fp8_matmul_path(int num_experts, int64_t K, int64_t N, int64_t num_rows) {
  const GroupedArgs g = args_of(nullptr, num_rows, K, nullptr, num_experts, K, N, K * N, K, nullptr, nullptr, 1,
                                num_rows);
  return num_experts >= 0 && num_experts <= kMaxExperts && fp8_tc_ok(g) ? fp8_tc_path(g) : -1;
}
