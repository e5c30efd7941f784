// Activations of the gated products and their derivatives, in fp32.
#pragma once

#include <cuda_runtime.h>

#include "einsparse.h"

namespace es {

// a = act(g), s = act'(g). EXACT: for fp32 results, the full-precision functions; else exp
// and the division by the fast ones: __expf(x) is within (2 + 1.173 |x|) 2^-23 of its value
// and __fdividef within 2^-22 of its, together less than 2^-15 at |g| = 88, far below the
// rounding to 16 bits. Past 2^126 __fdividef returns zero: silu is zero from about -87.3 on
// (where it is above -1.1e-36), gelu by tanh where its logistic function is that small.
// Written so that no tail cancels: 1 + erf is an erfc, 1 + tanh a logistic function.
template <int ACT, bool EXACT>
__device__ __forceinline__ void activate(float g, float& a, float& s) {
  auto logistic = [](float v) {
    if constexpr (EXACT) return 1.0f / (1.0f + expf(-v));
    return __fdividef(1.0f, 1.0f + __expf(-v));
  };
  if constexpr (ACT == ES_ACT_SILU) {
    const float p = logistic(g);
    a = g * p;
    s = p * fmaf(g, 1.0f - p, 1.0f);
  } else if constexpr (ACT == ES_ACT_GELU) {
    const float p = 0.5f * erfcf(-0.70710678118654752f * g);
    a = g * p;
    const float e = -0.5f * g * g;
    s = fmaf(g, 0.39894228040143268f * (EXACT ? expf(e) : __expf(e)), p);
  } else if constexpr (ACT == ES_ACT_GELU_TANH) {
    constexpr float b = 1.5957691216057308f, c = 0.044715f;  // 2 sqrt(2 / pi)
    const float p = logistic(b * g * fmaf(c, g * g, 1.0f));
    const float q = p * (1.0f - p);
    a = g * p;
    s = q > 0.0f ? fmaf(g * q, b * fmaf(3.0f * c, g * g, 1.0f), p) : p;  // far out g * g may be infinite
  } else {
    a = g <= 0.0f ? 0.0f : g;  // NaN stays
    s = g > 0.0f ? 1.0f : 0.0f;
  }
}

// Runs the statement with ACT as the constant of an es_activation.
#define ES_BY_ACT(activation, ...)                \
  do {                                            \
    if ((activation) == ES_ACT_SILU) {            \
      constexpr int ACT = ES_ACT_SILU;            \
      __VA_ARGS__;                                \
    }                                             \
    if ((activation) == ES_ACT_GELU) {            \
      constexpr int ACT = ES_ACT_GELU;            \
      __VA_ARGS__;                                \
    }                                             \
    if ((activation) == ES_ACT_GELU_TANH) {       \
      constexpr int ACT = ES_ACT_GELU_TANH;       \
      __VA_ARGS__;                                \
    }                                             \
    if ((activation) == ES_ACT_RELU) {            \
      constexpr int ACT = ES_ACT_RELU;            \
      __VA_ARGS__;                                \
    }                                             \
  } while (0)

}  // namespace es
