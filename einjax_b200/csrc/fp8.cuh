// Products of 8-bit floating point with block scales on the tensor cores (fp8_tc.cu).
#pragma once

#include "grouped.cuh"

namespace es {

constexpr int kScaleBlock = 128;  // values that share a scale

bool fp8_tc_ok(const GroupedArgs& g);
int fp8_tc_path(const GroupedArgs& g);  // an es_grouped_path
size_t fp8_tc_workspace(const GroupedArgs& g, const void* x, const void* w);
int fp8_tc(const GroupedArgs& g, const void* x, const void* w, void* y, int out_dtype, void* workspace,
           int32_t* status, cudaStream_t stream);

}  // namespace es
