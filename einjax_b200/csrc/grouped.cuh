// Arguments of the products grouped by expert, and how a kernel reads the
// groups: offsets and orders come from the device and are bounded here.
#pragma once

#include <type_traits>

#include "experts.cuh"

namespace es {

// |sum| <= 128^2 K stays inside int32
constexpr int64_t kMaxInt8Depth = 131071;

struct GroupedArgs {
  int num_experts;  // 0: one group of all rows
  int64_t K, N;
  int64_t rows;     // grouped rows
  int64_t x_rows, x_stride;
  int top_k;
  const int32_t* offsets;
  const int32_t* order;  // nullptr: x is in grouped order
  int64_t w_e, w_k, w_n;
  const float* x_scale;  // 8-bit operands only
  const float* w_scale;

  __host__ __device__ __forceinline__ int groups() const { return num_experts > 0 ? num_experts : 1; }
  __device__ __forceinline__ int64_t bound(int e) const {
    const int64_t v = offsets[e];
    return v < 0 ? 0 : v > rows ? rows : v;
  }
  // Rows [lo, hi) of a group; empty for offsets that fall.
  __device__ __forceinline__ void bounds(int e, int64_t& lo, int64_t& hi) const {
    if (num_experts == 0) {
      lo = 0;
      hi = rows;
      return;
    }
    lo = bound(e);
    hi = bound(e + 1);
    if (hi < lo) hi = lo;
  }
  __device__ __forceinline__ int64_t kept() const { return num_experts > 0 ? bound(num_experts) : rows; }
  // Row of x behind grouped row r, -1 for none.
  __device__ __forceinline__ int64_t source(int64_t r) const {
    if (!order) return r;
    const int64_t a = order[r];
    const int64_t t = a < 0 ? -1 : a / top_k;
    return t < x_rows ? t : -1;
  }
};

int check_grouped(const GroupedArgs& g);  // an es_status for sizes and orders that do not belong together

constexpr int kInt8 = 0x100;  // operand type of the 8-bit product

// The fp32 rows' product for groups of a few rows (grouped_few.cu): no workspace.
bool grouped_rows_few_ok(const GroupedArgs& g, int dtype, const void* w);
int grouped_rows_few(const GroupedArgs& g, const void* x, const void* w, void* y, cudaStream_t stream);

// Tensor-core forms (grouped_tc.cu). The workspace holds copies of what TMA
// cannot read as it lies.
bool grouped_rows_tc_ok(const GroupedArgs& g, int dtype);
int grouped_rows_tc_path(const GroupedArgs& g, int dtype);  // an es_grouped_path
size_t grouped_rows_tc_workspace(const GroupedArgs& g, int dtype, const void* x, const void* w);
int grouped_rows_tc(const GroupedArgs& g, int dtype, const void* x, const void* w, void* y, int out_dtype,
                    void* workspace, int32_t* status, cudaStream_t stream);
// Gated products of 16-bit operands in one kernel: N is the channels of h, up lies N
// columns behind gate.
bool grouped_gated_tc_ok(const GroupedArgs& g, int dtype);
int grouped_gated_tc_path(const GroupedArgs& g);
size_t grouped_gated_tc_workspace(const GroupedArgs& g, int dtype, const void* x, const void* w);
int grouped_gated_tc(const GroupedArgs& g, int dtype, const void* x, const void* w, int activation, void* h,
                     float* slopes, void* workspace, int32_t* status, cudaStream_t stream);
bool grouped_wgrad_tc_ok(const GroupedArgs& g, int dtype);
size_t grouped_wgrad_tc_workspace(const GroupedArgs& g, int dtype, const void* x, const void* dy, int64_t dy_stride);
int grouped_wgrad_tc(const GroupedArgs& g, int dtype, const void* x, const void* dy, int64_t dy_stride, void* dw,
                     void* workspace, int32_t* status, cudaStream_t stream);

}  // namespace es
