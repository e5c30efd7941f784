// Gated products: h[r] = act(x[r] gate[e]) * (x[r] up[e]) with w[e] = [gate | up]
// (K, 2F), dense or grouped by expert, and their gradients.
//
//   dh/d(x gate) = act'(x gate) * (x up),   dh/d(x up) = act(x gate)
//
// A training step keeps these two slopes (num_rows, 2F) instead of the products
// themselves: the backward pass multiplies each by dh and calls no exp. They are kept in
// fp32: what the tensor cores read has to be rounded to 16 bits, but only once (with
// 16-bit slopes the gradients of a bf16 step were 0.0029 off in the norm where one
// rounding fewer gives 0.0024; the writes and reads cost 3% of the step). With dy = dh times the
// slopes the rest are the products that are there already: dx = dy w^T, dw = x^T dy.
#include "activation.cuh"
#include "experts.cuh"
#include "grouped.cuh"

namespace es {
namespace {

constexpr int kGatedThreads = 256;

template <typename T, int VEC>
struct alignas(VEC * sizeof(T) >= 16 ? 16 : VEC * sizeof(T)) Values {
  T v[VEC];
};

// h and slopes from the fp32 product (rows, 2F). A thread makes VEC values of h.
// Rows of no expert are zero in the product and in h.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGatedThreads) gated_act_kernel(const float* y, int64_t rows, int64_t F, T* h,
                                                                  float* slopes) {
  using V = Values<T, VEC>;
  using Y = Values<float, VEC>;
  const int64_t pieces = F / VEC, n = rows * pieces;
  for (int64_t at = blockIdx.x * static_cast<int64_t>(kGatedThreads) + threadIdx.x; at < n;
       at += gridDim.x * static_cast<int64_t>(kGatedThreads)) {
    const int64_t r = at / pieces, c = at - r * pieces;
    const Y g = reinterpret_cast<const Y*>(y + r * 2 * F)[c], u = reinterpret_cast<const Y*>(y + (r * 2 + 1) * F)[c];
    V out;
    Y sg, su;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float a, s;
      activate<ACT, std::is_same<T, float>::value>(g.v[i], a, s);
      out.v[i] = from_f32<T>(a * u.v[i]);
      sg.v[i] = s * u.v[i];
      su.v[i] = a;
    }
    reinterpret_cast<V*>(h + r * F)[c] = out;
    if (slopes) {
      reinterpret_cast<Y*>(slopes + r * 2 * F)[c] = sg;
      reinterpret_cast<Y*>(slopes + (r * 2 + 1) * F)[c] = su;
    }
  }
}

// Bound by memory: 0.94 GB in 128 us (8192 rows, F 8192, bf16).
// dy = dh times the slopes; zero for the rows of no expert, whose slopes are not read.
template <typename T, int VEC>
__global__ void __launch_bounds__(kGatedThreads) gated_grad_kernel(const T* dh, int64_t stride, const float* slopes,
                                                                   int64_t rows, int64_t F, const int32_t* kept,
                                                                   T* dy) {
  using V = Values<T, VEC>;
  using Y = Values<float, VEC>;
  const int64_t pieces = F / VEC, n = rows * pieces, live = kept ? *kept : rows;
  for (int64_t at = blockIdx.x * static_cast<int64_t>(kGatedThreads) + threadIdx.x; at < n;
       at += gridDim.x * static_cast<int64_t>(kGatedThreads)) {
    const int64_t r = at / pieces, c = at - r * pieces;
    V g{}, u{};
    if (r < live) {
      const V d = reinterpret_cast<const V*>(dh + r * stride)[c];
      const Y sg = reinterpret_cast<const Y*>(slopes + r * 2 * F)[c];
      const Y su = reinterpret_cast<const Y*>(slopes + (r * 2 + 1) * F)[c];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        g.v[i] = from_f32<T>(to_f32(d.v[i]) * sg.v[i]);
        u.v[i] = from_f32<T>(to_f32(d.v[i]) * su.v[i]);
      }
    }
    reinterpret_cast<V*>(dy + r * 2 * F)[c] = g;
    reinterpret_cast<V*>(dy + (r * 2 + 1) * F)[c] = u;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int ACT>
int act_launch(const float* y, int64_t rows, int64_t F, void* h, float* slopes, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (F % VEC == 0 && aligned16(y) && aligned16(h) && aligned16(slopes))
    ES_LAUNCH((gated_act_kernel<T, VEC, ACT>), grid_for(rows * F / VEC, kGatedThreads), kGatedThreads, 0, s, y, rows, F,
              static_cast<T*>(h), slopes);
  else
    ES_LAUNCH((gated_act_kernel<T, 1, ACT>), grid_for(rows * F, kGatedThreads), kGatedThreads, 0, s, y, rows, F,
              static_cast<T*>(h), slopes);
  return ES_OK;
}

template <typename T>
int grad_launch(const void* dh, int64_t stride, const float* slopes, int64_t rows, int64_t F, const int32_t* kept,
                void* dy, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (F % VEC == 0 && stride % VEC == 0 && aligned16(dh) && aligned16(slopes) && aligned16(dy))
    ES_LAUNCH((gated_grad_kernel<T, VEC>), grid_for(rows * F / VEC, kGatedThreads), kGatedThreads, 0, s,
              static_cast<const T*>(dh), stride, slopes, rows, F, kept, static_cast<T*>(dy));
  else
    ES_LAUNCH((gated_grad_kernel<T, 1>), grid_for(rows * F, kGatedThreads), kGatedThreads, 0, s,
              static_cast<const T*>(dh), stride, slopes, rows, F, kept, static_cast<T*>(dy));
  return ES_OK;
}

// 16 bits up to a depth that is summed in one chain: the activation is the product's
// epilogue. Else (fp32, whose planes take the accumulators; deep sums; empty products)
// the product is made in fp32 and read again.
bool one_kernel(const GroupedArgs& g, int dtype) {
  return check_grouped(g) == ES_OK && grouped_gated_tc_ok(g, dtype);
}

size_t product_bytes(int64_t rows, int64_t F) {
  return (static_cast<size_t>(rows) * 2 * F * sizeof(float) + 255) / 256 * 256;
}

}  // namespace
}  // namespace es

using namespace es;

extern "C" size_t es_gated_matmul_workspace_size(const void* x, int dtype, int64_t x_rows, int64_t x_stride,
                                                 const void* w, int num_experts, int64_t K, int64_t F,
                                                 int64_t w_expert_stride, int64_t w_k_stride, int64_t w_n_stride,
                                                 const int32_t* offsets, const int32_t* order, int top_k,
                                                 int64_t num_rows) {
  if (num_rows <= 0 || F <= 0) return 0;
  const GroupedArgs g{num_experts, K, F, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride,
                      w_k_stride, w_n_stride, nullptr, nullptr};
  if (one_kernel(g, dtype)) return grouped_gated_tc_workspace(g, dtype, x, w);
  return product_bytes(num_rows, F) +
         es_grouped_matmul_workspace_size(x, dtype, x_rows, x_stride, w, num_experts, K, 2 * F, w_expert_stride,
                                          w_k_stride, w_n_stride, offsets, order, top_k, num_rows);
}

extern "C" int es_gated_matmul(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* w,
                               int num_experts, int64_t K, int64_t F, int64_t w_expert_stride, int64_t w_k_stride,
                               int64_t w_n_stride, const int32_t* offsets, const int32_t* order, int top_k,
                               int64_t num_rows, int activation, void* h, float* slopes, void* workspace,
                               size_t workspace_bytes, int32_t* status, void* stream) {
  if (activation < ES_ACT_SILU || activation > ES_ACT_RELU || F < 0 || num_rows < 0) return ES_ERR_INVALID;
  if (F > 0x3fffff00LL) return ES_ERR_UNSUPPORTED;
  if (F > 0 && num_rows > 0 && !h) return ES_ERR_INVALID;
  const GroupedArgs g{num_experts, K, F, num_rows, x_rows, x_stride, top_k, offsets, order, w_expert_stride,
                      w_k_stride, w_n_stride, nullptr, nullptr};
  ES_TRY(check_grouped(g));
  if (one_kernel(g, dtype)) {
    if (!h || !x || !w) return ES_ERR_INVALID;
    if (workspace_bytes < grouped_gated_tc_workspace(g, dtype, x, w)) return ES_ERR_WORKSPACE;
    return grouped_gated_tc(g, dtype, x, w, activation, h, slopes, workspace, status, as_stream(stream));
  }
  const size_t own = num_rows > 0 && F > 0 ? product_bytes(num_rows, F) : 0;
  if (workspace_bytes < own) return ES_ERR_WORKSPACE;
  float* y = static_cast<float*>(workspace);
  ES_TRY(es_grouped_matmul(x, dtype, x_rows, x_stride, w, num_experts, K, 2 * F, w_expert_stride, w_k_stride,
                           w_n_stride, offsets, order, top_k, num_rows, y, ES_F32,
                           static_cast<char*>(workspace) + own, workspace_bytes - own, status, stream));
  if (num_rows == 0 || F == 0) return ES_OK;
  ES_BY_TYPE(dtype, ES_BY_ACT(activation, return (act_launch<T, ACT>(y, num_rows, F, h, slopes, as_stream(stream)))));
  return ES_ERR_UNSUPPORTED;
}

extern "C" int es_gated_matmul_path(int dtype, int num_experts, int64_t K, int64_t F, int64_t num_rows) {
  const GroupedArgs g{num_experts, K, F, num_rows, num_rows, K, 1, nullptr, nullptr, 2 * K * F, 2 * F, 1, nullptr,
                      nullptr};
  if (num_experts < 0 || num_experts > kMaxExperts || num_rows <= 0 || K <= 0 || F <= 0) return -1;
  if (dtype != ES_F32 && dtype != ES_BF16 && dtype != ES_F16) return -1;
  return grouped_gated_tc_ok(g, dtype) ? grouped_gated_tc_path(g) : ES_GATED_TWO;
}

extern "C" int es_gated_matmul_grad(const void* dh, int dtype, int64_t dh_stride, const float* slopes,
                                    int64_t num_rows, int64_t F, const int32_t* kept_rows, void* dy, void* stream) {
  if (num_rows < 0 || F < 0) return ES_ERR_INVALID;
  if (num_rows > 0x7fffff00LL || F > 0x3fffff00LL) return ES_ERR_UNSUPPORTED;
  if (num_rows == 0 || F == 0) return ES_OK;
  if (!dh || !slopes || !dy) return ES_ERR_INVALID;
  ES_BY_TYPE(dtype, return grad_launch<T>(dh, dh_stride, slopes, num_rows, F, kept_rows, dy, as_stream(stream)));
  return ES_ERR_UNSUPPORTED;
}
