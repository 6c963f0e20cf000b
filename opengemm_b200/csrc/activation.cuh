// Activations of the fused epilogues and their derivatives, in float32.
//
// silu and the tanh form of gelu are one expression, x * sigmoid(a x + b x^3):
// (a, b) = (1, 0) and 2 sqrt(2/pi) (1, 0.044715), since (1 + tanh u) / 2 =
// sigmoid(2u).  The epilogues therefore carry the two coefficients at run time
// and compile one code path for both.  gelu itself is x * Phi(x); Phi(-|x|)
// comes from Abramowitz and Stegun, Handbook of Mathematical Functions,
// 7.1.26 (|error| <= 1.5e-7 in erf), whose exponential the derivative shares.
// Both need two special-function instructions a value; a call of erff or tanhf
// would be two to three times the instructions, and the four epilogue warps
// have to keep up with the tensor pipe.
#pragma once

#include <cstdint>

namespace og {

// What the host fills in; the codes of og_b200_* entry points.
enum Activation : int {
  ACT_NONE = 0,
  ACT_RELU = 1,
  ACT_GELU = 2,
  ACT_GELU_TANH = 3,
  ACT_SILU = 4,
  ACT_SWIGLU = 5,  // silu(gate) * up, gate and up the halves of the columns (experts' products only)
  ACT_GEGLU = 6,   // gelu(gate) * up, likewise
};

constexpr float SIGMOID_TANH_A = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float SIGMOID_TANH_B = 0.07135481282553488f;  // 2 sqrt(2 / pi) * 0.044715

#ifdef __CUDACC__

// Shape of the code an activation runs: none, relu, x * Phi(x), x * sigmoid(a x + b x^3).
enum ActShape : int { SHAPE_NONE = 0, SHAPE_RELU = 1, SHAPE_PHI = 2, SHAPE_SIGMOID = 3 };

__device__ __forceinline__ float sigmoid_of(float t) { return __fdividef(1.0f, 1.0f + __expf(-t)); }

// Phi(-|x|) and, through `density`, exp(-x^2 / 2).
__device__ __forceinline__ float lower_tail(float x, float* density) {
  const float y = fabsf(x) * 0.7071067811865476f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, y, 1.0f));
  const float e = __expf(-0.5f * x * x);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  *density = e;
  return 0.5f * p * t * e;
}

__device__ __forceinline__ float act_phi(float x) {
  float e;
  const float tail = lower_tail(x, &e);
  return x * (x > 0.0f ? 1.0f - tail : tail);
}

// sigmoid(a x + b x^3).  The square is capped far past saturation, so that an infinite x
// times b = 0 makes no NaN.
__device__ __forceinline__ float gate_of(float x, float a, float b) { return sigmoid_of(x * fmaf(b, fminf(x * x, 1e8f), a)); }

template <int SHAPE>
__device__ __forceinline__ float act_value(float x, float a, float b) {
  if constexpr (SHAPE == SHAPE_RELU) return x < 0.0f ? 0.0f : x;  // keeps a NaN
  else if constexpr (SHAPE == SHAPE_PHI) return act_phi(x);
  else if constexpr (SHAPE == SHAPE_SIGMOID) return x * gate_of(x, a, b);
  else return x;
}

// The activation and its derivative at x.
template <int SHAPE>
__device__ __forceinline__ void act_both(float x, float a, float b, float* value, float* slope) {
  if constexpr (SHAPE == SHAPE_RELU) {
    *value = x < 0.0f ? 0.0f : x;
    *slope = x > 0.0f ? 1.0f : (x == x ? 0.0f : x);
  } else if constexpr (SHAPE == SHAPE_PHI) {
    float e;
    const float tail = lower_tail(x, &e);
    const float cdf = x > 0.0f ? 1.0f - tail : tail;
    *value = x * cdf;
    *slope = fmaf(x * 0.3989422804014327f, e, cdf);
  } else if constexpr (SHAPE == SHAPE_SIGMOID) {
    const float p = gate_of(x, a, b);
    *value = x * p;
    *slope = fmaf(x * p * (1.0f - p), fmaf(3.0f * b, fminf(x * x, 1e8f), a), p);
  } else {
    *value = x;
    *slope = 1.0f;
  }
}

#endif  // __CUDACC__

// The code path and the coefficients of an activation (the inner one, for a gated pair).
inline void act_constants(int activation, int* shape, float* a, float* b) {
  *a = 0.0f, *b = 0.0f;
  switch (activation) {
    case ACT_RELU: *shape = 1; break;
    case ACT_GELU: case ACT_GEGLU: *shape = 2; break;
    case ACT_GELU_TANH: *shape = 3, *a = SIGMOID_TANH_A, *b = SIGMOID_TANH_B; break;
    case ACT_SILU: case ACT_SWIGLU: *shape = 3, *a = 1.0f; break;
    default: *shape = 0;
  }
}

}  // namespace og
