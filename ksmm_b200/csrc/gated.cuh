// The gate's function and its derivative.
#pragma once

#include "common.cuh"

namespace ksmm {

// 1 / (1 + exp(-x)).  B16: for results rounded to 16 bits, one exponential and one reciprocal of the special-function
// unit (relative error about 2^-21); fp32 results take the library's expf and a rounded division.
template <bool B16>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (B16) return __fdividef(1.f, 1.f + __expf(-x));
  else return 1.f / (1.f + expf(-x));
}

template <bool B16>
__device__ __forceinline__ float gate_value(float g, int act) {
  switch (act) {
    case KSMM_ACT_SILU: return g * sigmoid<B16>(g);
    case KSMM_ACT_SIGMOID: return sigmoid<B16>(g);
    case KSMM_ACT_GELU: return B16 ? gelu_16bit(g) : g * normcdff(g);
    case KSMM_ACT_RELU: return g < 0.f ? 0.f : g;  // (a NaN stays one)
    default: return g;
  }
}

// value and derivative
template <bool B16>
__device__ __forceinline__ void gate_slope(float g, int act, float& value, float& slope) {
  value = g;
  slope = 1.f;
  if (act == KSMM_ACT_SILU) {
    const float s = sigmoid<B16>(g);
    value = g * s;
    slope = s * fmaf(g, 1.f - s, 1.f);
  } else if (act == KSMM_ACT_SIGMOID) {
    value = sigmoid<B16>(g);
    slope = value * (1.f - value);
  } else if (act == KSMM_ACT_GELU) {
    // (beyond |g| = 15 the density is 0 in fp32; g times it would be inf * 0 for an infinite g)
    const float cdf = normcdff(g), t = fminf(fmaxf(g, -15.f), 15.f);
    value = g * cdf;
    slope = fmaf(t * 0.3989422804f, __expf(-0.5f * t * t), cdf);
  } else if (act == KSMM_ACT_RELU) {
    value = g < 0.f ? 0.f : g;
    slope = g <= 0.f ? 0.f : 1.f;
  }
}

}  // namespace ksmm
