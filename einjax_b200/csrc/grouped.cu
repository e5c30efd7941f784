// Products grouped by expert with ragged group sizes, and their gradient of
// the weights, on the CUDA cores: every type, size, stride and alignment.
//
// One CTA of 256 threads computes a 64 x 64 tile of one expert's product in
// 16-deep steps through shared memory, 4 x 4 results a thread.
// fp32 sums are folded into a second accumulator every 64 steps, so that a
// long sum's rounding error grows with the root of its blocks.
#include "experts.cuh"
#include "grouped.cuh"

namespace es {
namespace {

constexpr int kTile = 64;
constexpr int kStep = 16;
constexpr int kThreads = 256;
constexpr int kFold = 4;  // steps between folds

template <typename T>
struct Acc {
  using type = float;
};
template <>
struct Acc<int8_t> {
  using type = int;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ int widen(int8_t x) { return x; }

// The tile product: a(i, s), b(s, j) give operands (zero outside). AI, BJ:
// whether neighbouring threads walk a's i (b's j) or the depth s.
template <typename A, bool AI, bool BJ, typename FA, typename FB>
__device__ __forceinline__ void tile_product(int64_t depth, FA a, FB b, A (&out)[4][4]) {
  __shared__ A as[kStep][kTile + 4];
  __shared__ A bs[kStep][kTile + 4];
  const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
  A acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) out[i][j] = acc[i][j] = A(0);
  int fold = 0;
  for (int64_t s0 = 0; s0 < depth; s0 += kStep) {
#pragma unroll
    for (int n = 0; n < kTile * kStep / kThreads; ++n) {
      const int l = threadIdx.x + n * kThreads;
      const int ia = AI ? l % kTile : l / kStep, sa = AI ? l / kTile : l % kStep;
      const int jb = BJ ? l % kTile : l / kStep, sb = BJ ? l / kTile : l % kStep;
      as[sa][ia] = s0 + sa < depth ? a(ia, s0 + sa) : A(0);
      bs[sb][jb] = s0 + sb < depth ? b(s0 + sb, jb) : A(0);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kStep; ++s) {
      A x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = as[s][ti * 4 + i];
        y[i] = bs[s][tj * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += x[i] * y[j];
    }
    __syncthreads();
    if (++fold == kFold) {
      fold = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          out[i][j] += acc[i][j];
          acc[i][j] = A(0);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) out[i][j] += acc[i][j];
}

// The expert and first row of this CTA's row tile: warp 0 counts the tiles of
// 32 experts at a time. Returns false past the last tile.
__device__ __forceinline__ bool find_tile(const GroupedArgs& g, int64_t tile, int& expert, int64_t& row0,
                                          int64_t& row1) {
  __shared__ int64_t found[3];
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int64_t run = 0, at = -1, a = 0, b = 0;
    for (int e0 = 0; e0 < g.groups() && at < 0; e0 += 32) {
      const int e = e0 + lane;
      int64_t lo = 0, hi = 0;
      if (e < g.groups()) g.bounds(e, lo, hi);
      const int64_t n = (hi - lo + kTile - 1) / kTile;
      int64_t s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      const bool hit = tile >= run + s - n && tile < run + s;
      const unsigned m = __ballot_sync(0xffffffffu, hit);
      if (m) {
        const int src = __ffs(m) - 1;
        at = e0 + src;
        a = __shfl_sync(0xffffffffu, lo + (tile - (run + s - n)) * kTile, src);
        b = __shfl_sync(0xffffffffu, hi, src);
      }
      run += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) {
      found[0] = at;
      found[1] = a;
      found[2] = b;
    }
  }
  __syncthreads();
  expert = static_cast<int>(found[0]);
  row0 = found[1];
  row1 = min(found[2], row0 + kTile);
  return expert >= 0;
}

template <typename T, typename U, bool NCONTIG>
__global__ void __launch_bounds__(kThreads) rows_kernel(GroupedArgs g, const T* x, const T* w, U* y) {
  using A = typename Acc<T>::type;
  const int64_t n0 = blockIdx.y * static_cast<int64_t>(kTile);
  const int64_t kept = g.kept();
  for (int64_t r = kept + blockIdx.x; r < g.rows; r += gridDim.x)  // rows of no expert
    if (threadIdx.x < kTile && n0 + threadIdx.x < g.N) y[r * g.N + n0 + threadIdx.x] = from_f32<U>(0.0f);
  int e;
  int64_t r0, r1;
  if (!find_tile(g, blockIdx.x, e, r0, r1)) return;
  __shared__ int64_t src[kTile];
  if (threadIdx.x < kTile) src[threadIdx.x] = r0 + threadIdx.x < r1 ? g.source(r0 + threadIdx.x) : -1;
  __syncthreads();
  const T* we = w + e * g.w_e;
  A out[4][4];
  tile_product<A, false, NCONTIG>(
      g.K, [&](int i, int64_t k) { return src[i] >= 0 ? A(widen(x[src[i] * g.x_stride + k])) : A(0); },
      [&](int64_t k, int j) { return n0 + j < g.N ? A(widen(we[k * g.w_k + (n0 + j) * g.w_n])) : A(0); }, out);
  const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + ti * 4 + i;
    if (r >= r1) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tj * 4 + j;
      if (n >= g.N) continue;
      float v = static_cast<float>(out[i][j]);
      if constexpr (std::is_same<T, int8_t>::value) {
        const int64_t t = src[ti * 4 + i];
        v = t >= 0 ? v * g.x_scale[t] * g.w_scale[e * g.N + n] : 0.0f;
      }
      y[r * g.N + n] = from_f32<U>(v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) wgrad_kernel(GroupedArgs g, const T* x, const T* dy, int64_t dy_stride,
                                                         T* dw) {
  const int e = blockIdx.z;
  const int64_t k0 = blockIdx.x * static_cast<int64_t>(kTile), n0 = blockIdx.y * static_cast<int64_t>(kTile);
  int64_t lo, hi;
  g.bounds(e, lo, hi);
  float out[4][4];
  tile_product<float, true, true>(
      hi - lo,
      [&](int i, int64_t s) {
        const int64_t t = k0 + i < g.K ? g.source(lo + s) : -1;
        return t >= 0 ? to_f32(x[t * g.x_stride + k0 + i]) : 0.0f;
      },
      [&](int64_t s, int j) { return n0 + j < g.N ? to_f32(dy[(lo + s) * dy_stride + n0 + j]) : 0.0f; }, out);
  const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t k = k0 + ti * 4 + i, n = n0 + tj * 4 + j;
      if (k < g.K && n < g.N) dw[e * g.w_e + k * g.w_k + n * g.w_n] = from_f32<T>(out[i][j]);
    }
}

template <typename T, typename U>
int rows_simt(const GroupedArgs& g, const void* x, const void* w, void* y, cudaStream_t s) {
  const int64_t tiles = g.rows / kTile + min(static_cast<int64_t>(g.groups()), g.rows);
  const int64_t cols = (g.N + kTile - 1) / kTile;
  if (cols > 65535) return ES_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(cols));
  if (g.w_n == 1)
    ES_LAUNCH((rows_kernel<T, U, true>), grid, kThreads, 0, s, g, static_cast<const T*>(x), static_cast<const T*>(w),
              static_cast<U*>(y));
  else
    ES_LAUNCH((rows_kernel<T, U, false>), grid, kThreads, 0, s, g, static_cast<const T*>(x),
              static_cast<const T*>(w), static_cast<U*>(y));
  return ES_OK;
}

int check_args(const GroupedArgs& g) {
  if (g.num_experts < 0 || g.K < 0 || g.N < 0 || g.rows < 0 || g.x_rows < 0) return ES_ERR_INVALID;
  if (g.num_experts > 0 && !g.offsets) return ES_ERR_INVALID;
  if (g.num_experts == 0 && (g.order || g.offsets || g.x_rows != g.rows)) return ES_ERR_INVALID;
  if (!g.order && g.x_rows != g.rows) return ES_ERR_INVALID;
  if (g.order && g.top_k < 1) return ES_ERR_INVALID;
  if (g.num_experts > kMaxExperts || g.rows > 0x7fffff00LL || g.x_rows > 0x7fffff00LL || g.K > 0x7fffff00LL ||
      g.N > 0x7fffff00LL)
    return ES_ERR_UNSUPPORTED;
  return ES_OK;
}

bool value_type(int dtype) { return dtype == ES_F32 || dtype == ES_BF16 || dtype == ES_F16; }

bool use_tc(const GroupedArgs& g, int dtype, const void* x, const void* w) { return grouped_rows_tc_ok(g, dtype); }

}  // namespace
}  // namespace es

using namespace es;

extern "C" size_t es_grouped_matmul_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride,
                                                   const void* w, int num_experts, int64_t K, int64_t N,
                                                   int64_t w_expert_stride, int64_t w_k_stride, int64_t w_n_stride,
                                                   const int32_t* offsets, const int32_t* order, int top_k,
                                                   int64_t num_rows) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride,
                      w_k_stride, w_n_stride, nullptr, nullptr};
  return check_args(g) == ES_OK && use_tc(g, dtype, x, w) ? grouped_rows_tc_workspace(g, dtype, x, w) : 0;
}

extern "C" int es_grouped_matmul(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w,
                                 int num_experts, int64_t K, int64_t N, int64_t w_expert_stride, int64_t w_k_stride,
                                 int64_t w_n_stride, const int32_t* offsets, const int32_t* order, int top_k,
                                 int64_t num_rows, void* y, int out_dtype, void* workspace, size_t workspace_bytes,
                                 int32_t* status, void* stream) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride,
                      w_k_stride, w_n_stride, nullptr, nullptr};
  if (num_experts < 1) return ES_ERR_INVALID;
  ES_TRY(check_args(g));
  if (!value_type(dtype) || (out_dtype != dtype && out_dtype != ES_F32)) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || N == 0) return ES_OK;
  if (!y || (K && ((x_rows && !x) || !w))) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (use_tc(g, dtype, x, w)) {
    if (workspace_bytes < grouped_rows_tc_workspace(g, dtype, x, w)) return ES_ERR_WORKSPACE;
    return grouped_rows_tc(g, dtype, x, w, y, out_dtype, workspace, status, s);
  }
  if (out_dtype == dtype) ES_BY_TYPE(dtype, return (rows_simt<T, T>(g, x, w, y, s)));
  ES_BY_TYPE(dtype, return (rows_simt<T, float>(g, x, w, y, s)));
  return ES_ERR_UNSUPPORTED;
}

extern "C" size_t es_grouped_matmul_wgrad_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride,
                                                         const void* dy, int64_t dy_stride, int num_experts, int64_t K,
                                                         int64_t N, const int32_t* offsets, const int32_t* order,
                                                         int top_k, int64_t num_rows, void* dw,
                                                         int64_t dw_expert_stride, int64_t dw_k_stride,
                                                         int64_t dw_n_stride) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, dw_expert_stride,
                      dw_k_stride, dw_n_stride, nullptr, nullptr};
  return check_args(g) == ES_OK && grouped_wgrad_tc_ok(g, dtype)
             ? grouped_wgrad_tc_workspace(g, dtype, x, dy, dy_stride) : 0;
}

extern "C" int es_grouped_matmul_wgrad(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* dy,
                                       int64_t dy_stride, int num_experts, int64_t K, int64_t N,
                                       const int32_t* offsets, const int32_t* order, int top_k, int64_t num_rows,
                                       void* dw, int64_t dw_expert_stride, int64_t dw_k_stride, int64_t dw_n_stride,
                                       void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, dw_expert_stride,
                      dw_k_stride, dw_n_stride, nullptr, nullptr};
  if (num_experts < 1) return ES_ERR_INVALID;
  ES_TRY(check_args(g));
  if (!value_type(dtype)) return ES_ERR_UNSUPPORTED;
  if (K == 0 || N == 0) return ES_OK;
  if (!dw || (num_rows && (!dy || (x_rows && !x)))) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (grouped_wgrad_tc_ok(g, dtype)) {
    if (workspace_bytes < grouped_wgrad_tc_workspace(g, dtype, x, dy, dy_stride)) return ES_ERR_WORKSPACE;
    return grouped_wgrad_tc(g, dtype, x, dy, dy_stride, dw, workspace, status, s);
  }
  const int64_t kt = (K + kTile - 1) / kTile, nt = (N + kTile - 1) / kTile;
  if (nt > 65535) return ES_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(kt), static_cast<unsigned>(nt), static_cast<unsigned>(num_experts));
  ES_BY_TYPE(dtype, {
    ES_LAUNCH((wgrad_kernel<T>), grid, kThreads, 0, s, g, static_cast<const T*>(x), static_cast<const T*>(dy),
              dy_stride, static_cast<T*>(dw));
    return ES_OK;
  });
  return ES_ERR_UNSUPPORTED;
}

extern "C" size_t es_int8_matmul_workspace_size(const int8_t* q, const float* x_scale, int64_t x_rows,
                                                int64_t x_stride, const int8_t* wq, const float* w_scale,
                                                int num_experts, int64_t K, int64_t N, int64_t w_expert_stride,
                                                int64_t w_n_stride, const int32_t* offsets, const int32_t* order,
                                                int top_k, int64_t num_rows) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride, 1,
                      w_n_stride, x_scale, w_scale};
  return check_args(g) == ES_OK && use_tc(g, kInt8, q, wq) ? grouped_rows_tc_workspace(g, kInt8, q, wq) : 0;
}

extern "C" int es_int8_matmul(const int8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride,
                              const int8_t* wq, const float* w_scale, int num_experts, int64_t K, int64_t N,
                              int64_t w_expert_stride, int64_t w_n_stride, const int32_t* offsets,
                              const int32_t* order, int top_k, int64_t num_rows, void* y, int out_dtype,
                              void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride, 1,
                      w_n_stride, x_scale, w_scale};
  ES_TRY(check_args(g));
  if (K > kMaxInt8Depth || !value_type(out_dtype)) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || N == 0) return ES_OK;
  if (!y || !w_scale || (x_rows && !x_scale) || (K && ((x_rows && !q) || !wq))) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (use_tc(g, kInt8, q, wq)) {
    if (workspace_bytes < grouped_rows_tc_workspace(g, kInt8, q, wq)) return ES_ERR_WORKSPACE;
    return grouped_rows_tc(g, kInt8, q, wq, y, out_dtype, workspace, status, s);
  }
  ES_BY_TYPE(out_dtype, return (rows_simt<int8_t, T>(g, q, wq, y, s)));
  return ES_ERR_UNSUPPORTED;
}
