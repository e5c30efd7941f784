// Value types and limits that the expert operators share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace es {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;

// Programmatic dependent launch: the next kernel of the stream, if it was
// launched for it, may start before this one is done; it waits for the earlier
// ones' results before it touches memory.
__device__ __forceinline__ void let_next_grid_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_earlier_grids() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half(x);
}

// Runs the statement with T as the value type of an es_dtype; falls through
// for a type that these operators do not take.
#define ES_BY_TYPE(dtype, ...)  \
  do {                          \
    if ((dtype) == ES_F32) {    \
      using T = float;          \
      __VA_ARGS__;              \
    }                           \
    if ((dtype) == ES_BF16) {   \
      using T = __nv_bfloat16;  \
      __VA_ARGS__;              \
    }                           \
    if ((dtype) == ES_F16) {    \
      using T = __half;         \
      __VA_ARGS__;              \
    }                           \
  } while (0)

}  // namespace es
