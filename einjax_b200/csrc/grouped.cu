// Entry points of the products grouped by expert: checks of arguments, and the
// cases that have no product (no depth, no rows). The kernels are in
// grouped_tc.cu, and in grouped_few.cu for fp32 groups of a few rows. A first,
// general form on the CUDA cores is gone: with operands that TMA cannot read
// copied first, the tensor cores were faster for all but products of some 2^18
// steps, and there slower by 2 us.
#include "experts.cuh"
#include "grouped.cuh"

namespace es {
namespace {

constexpr int kClearThreads = 256;

// Zeros in an (experts, K, N) tensor of any strides.
template <typename T>
__global__ void __launch_bounds__(kClearThreads) clear_kernel(GroupedArgs g, T* out) {
  const int64_t n = g.groups() * g.K * g.N, step = gridDim.x * static_cast<int64_t>(kClearThreads);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kClearThreads) + threadIdx.x; i < n; i += step) {
    const int64_t col = i % g.N, row = i / g.N % g.K, e = i / g.N / g.K;
    out[e * g.w_e + row * g.w_k + col * g.w_n] = T(0);
  }
}

int clear_rows_of(const GroupedArgs& g, void* y, int out_dtype, cudaStream_t s) {
  const size_t bytes = static_cast<size_t>(g.rows) * g.N * (out_dtype == ES_F32 ? 4 : 2);
  count_launch();
  return cudaMemsetAsync(y, 0, bytes, s) == cudaSuccess ? ES_OK : ES_ERR_CUDA;
}

bool value_type(int dtype) { return dtype == ES_F32 || dtype == ES_BF16 || dtype == ES_F16; }

bool empty(const GroupedArgs& g) { return g.K == 0 || g.N == 0 || g.rows == 0 || g.x_rows == 0; }

}  // namespace

int check_grouped(const GroupedArgs& g) {
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

}  // namespace es

using namespace es;

extern "C" size_t es_grouped_matmul_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride,
                                                   const void* w, int num_experts, int64_t K, int64_t N,
                                                   int64_t w_expert_stride, int64_t w_k_stride, int64_t w_n_stride,
                                                   const int32_t* offsets, const int32_t* order, int top_k,
                                                   int64_t num_rows) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride,
                      w_k_stride, w_n_stride, nullptr, nullptr};
  if (check_grouped(g) != ES_OK || empty(g) || grouped_rows_few_ok(g, dtype, w)) return 0;
  return grouped_rows_tc_workspace(g, dtype, x, w);
}

extern "C" int es_grouped_matmul(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w,
                                 int num_experts, int64_t K, int64_t N, int64_t w_expert_stride, int64_t w_k_stride,
                                 int64_t w_n_stride, const int32_t* offsets, const int32_t* order, int top_k,
                                 int64_t num_rows, void* y, int out_dtype, void* workspace, size_t workspace_bytes,
                                 int32_t* status, void* stream) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride,
                      w_k_stride, w_n_stride, nullptr, nullptr};
  ES_TRY(check_grouped(g));
  if (!value_type(dtype) || (out_dtype != dtype && out_dtype != ES_F32)) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || N == 0) return ES_OK;
  if (!y || (K && ((x_rows && !x) || !w))) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (empty(g)) return clear_rows_of(g, y, out_dtype, s);
  if (grouped_rows_few_ok(g, dtype, w)) return grouped_rows_few(g, x, w, y, s);
  if (!grouped_rows_tc_ok(g, dtype)) return ES_ERR_UNSUPPORTED;
  if (workspace_bytes < grouped_rows_tc_workspace(g, dtype, x, w)) return ES_ERR_WORKSPACE;
  return grouped_rows_tc(g, dtype, x, w, y, out_dtype, workspace, status, s);
}

extern "C" int es_grouped_matmul_path(int dtype, int num_experts, int64_t K, int64_t N, int64_t num_rows) {
  const GroupedArgs g{num_experts, K, N, num_rows, num_rows, K, 1, nullptr, nullptr, K * N, N, 1, nullptr, nullptr};
  if (num_experts < 1 || num_experts > kMaxExperts || !value_type(dtype) || empty(g)) return -1;
  if (grouped_rows_few_ok(g, dtype, nullptr)) return ES_GROUPED_FEW;
  return grouped_rows_tc_ok(g, dtype) ? grouped_rows_tc_path(g, dtype) : -1;
}

extern "C" int es_int8_matmul_path(int num_experts, int64_t K, int64_t N, int64_t num_rows) {
  const GroupedArgs g{num_experts, K, N, num_rows, num_rows, K, 1, nullptr, nullptr, K * N, 1, K, nullptr, nullptr};
  if (num_experts < 0 || num_experts > kMaxExperts || K > kMaxInt8Depth || empty(g)) return -1;
  return grouped_rows_tc_ok(g, kInt8) ? grouped_rows_tc_path(g, kInt8) : -1;
}

extern "C" size_t es_grouped_matmul_wgrad_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride,
                                                         const void* dy, int64_t dy_stride, int num_experts, int64_t K,
                                                         int64_t N, const int32_t* offsets, const int32_t* order,
                                                         int top_k, int64_t num_rows, void* dw,
                                                         int64_t dw_expert_stride, int64_t dw_k_stride,
                                                         int64_t dw_n_stride) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, dw_expert_stride,
                      dw_k_stride, dw_n_stride, nullptr, nullptr};
  return check_grouped(g) == ES_OK && !empty(g) ? grouped_wgrad_tc_workspace(g, dtype, x, dy, dy_stride) : 0;
}

extern "C" int es_grouped_matmul_wgrad(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* dy,
                                       int64_t dy_stride, int num_experts, int64_t K, int64_t N,
                                       const int32_t* offsets, const int32_t* order, int top_k, int64_t num_rows,
                                       void* dw, int64_t dw_expert_stride, int64_t dw_k_stride, int64_t dw_n_stride,
                                       void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, dw_expert_stride,
                      dw_k_stride, dw_n_stride, nullptr, nullptr};
  ES_TRY(check_grouped(g));
  if (!value_type(dtype)) return ES_ERR_UNSUPPORTED;
  if (K == 0 || N == 0) return ES_OK;
  if (!dw || (num_rows && (!dy || (x_rows && !x)))) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (empty(g)) {
    const int blocks = grid_for(g.groups() * K * N, kClearThreads);
    ES_BY_TYPE(dtype, {
      ES_LAUNCH((clear_kernel<T>), blocks, kClearThreads, 0, s, g, static_cast<T*>(dw));
      return ES_OK;
    });
  }
  if (!grouped_wgrad_tc_ok(g, dtype)) return ES_ERR_UNSUPPORTED;
  if (workspace_bytes < grouped_wgrad_tc_workspace(g, dtype, x, dy, dy_stride)) return ES_ERR_WORKSPACE;
  return grouped_wgrad_tc(g, dtype, x, dy, dy_stride, dw, workspace, status, s);
}

extern "C" size_t es_int8_matmul_workspace_size(const int8_t* q, const float* x_scale, int64_t x_rows,
                                                int64_t x_stride, const int8_t* wq, const float* w_scale,
                                                int num_experts, int64_t K, int64_t N, int64_t w_expert_stride,
                                                int64_t w_n_stride, const int32_t* offsets, const int32_t* order,
                                                int top_k, int64_t num_rows) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride, 1,
                      w_n_stride, x_scale, w_scale};
  return check_grouped(g) == ES_OK && !empty(g) ? grouped_rows_tc_workspace(g, kInt8, q, wq) : 0;
}

extern "C" int es_int8_matmul(const int8_t* q, const float* x_scale, int64_t x_rows, int64_t x_stride,
                              const int8_t* wq, const float* w_scale, int num_experts, int64_t K, int64_t N,
                              int64_t w_expert_stride, int64_t w_n_stride, const int32_t* offsets,
                              const int32_t* order, int top_k, int64_t num_rows, void* y, int out_dtype,
                              void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const GroupedArgs g{num_experts, K, N, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride, 1,
                      w_n_stride, x_scale, w_scale};
  ES_TRY(check_grouped(g));
  if (K > kMaxInt8Depth || !value_type(out_dtype)) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || N == 0) return ES_OK;
  if (!y || !w_scale || (x_rows && !x_scale) || (K && ((x_rows && !q) || !wq))) return ES_ERR_INVALID;
  cudaStream_t s = as_stream(stream);
  if (empty(g)) return clear_rows_of(g, y, out_dtype, s);
  if (!grouped_rows_tc_ok(g, kInt8)) return ES_ERR_UNSUPPORTED;
  if (workspace_bytes < grouped_rows_tc_workspace(g, kInt8, q, wq)) return ES_ERR_WORKSPACE;
  return grouped_rows_tc(g, kInt8, q, wq, y, out_dtype, workspace, status, s);
}
