// Activations of the fused epilogues and their derivatives, in float32.
//
// silu and the tanh form of gelu are one expression, x * sigmoid(a x + b x^3):
// (a, b) = (1, 0) and 2 sqrt(2/pi) (1, 0.044715), since (1 + tanh u) / 2 =
// sigmoid(2u).  The epilogues therefore carry the two coefficients at run time
// (times -log2(e), for the base-2 exponential) and compile one code path for
// both.  gelu itself is x * Phi(x), and Phi(-u) = exp(-u^2 / 2) R(u) with
// R(u) = erfcx(u / sqrt 2) / 2, which falls from 1/2 like 1 / u: t P(t) with
// t = 1 / (1 + 0.305 u) and P of degree 7, the coefficients a least-maximum fit
// of the relative error over 0 <= u <= 14 (9.4e-8; 6.5 units of 2^-24 with
// float32 coefficients in float32).  So the tail is good relative to itself, to
// (1.5 u^2 + 20) 2^-24 with the exponential's argument rounded: 1.3e-6 at -1,
// 3.4e-6 at -5, 6.9e-6 at -8 (an absolute approximation of erf to 1.5e-7 has
// 1 % there).  The derivative shares the exponential.  Each needs two
// special-function instructions and 6 to 15 others a value: the epilogue's warps
// have to keep up with the tensor pipe, and a call of erff or tanhf is two to
// three times that.
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

// Rows that a block of an activation's gradient (routing.cu) works on: 64, or 16
// where such blocks of 256 columns would leave most of the GPU idle (1001 x 520
// values: 5.6 us in blocks of 64 rows).
inline int gradient_block_rows(long long rows, int width) { return (rows + 63) / 64 * ((width + 255) / 256) >= 2 * 148 ? 64 : 16; }

constexpr double LOG2_E = 1.4426950408889634;
constexpr double TANH_A = 1.5957691216057308;  // 2 sqrt(2 / pi)

#ifdef __CUDACC__

// Shape of the code an activation runs: none, relu, x * Phi(x), x * sigmoid(a x + b x^3).
enum ActShape : int { SHAPE_NONE = 0, SHAPE_RELU = 1, SHAPE_PHI = 2, SHAPE_SIGMOID = 3 };

// 2^x and 1 / x to within 2 units and 1 unit of the last place; results and
// arguments below the normal range are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// sigmoid(t) for the coefficients of -log2(e) t = a x + b x^3.  The square is capped
// far past saturation, so that an infinite x times b = 0 makes no NaN.
__device__ __forceinline__ float gate_of(float x, float a, float b) {
  return reciprocal_fast(1.0f + exp2_fast(x * fmaf(b, fminf(x * x, 1e8f), a)));
}

// P's coefficients, from the constant term on.
constexpr float TAIL_SLOPE = 0.305f;
constexpr float TAIL_0 = 0.121639736f, TAIL_1 = 0.122466817f, TAIL_2 = 0.103420876f, TAIL_3 = 0.121021658f;
constexpr float TAIL_4 = -0.0379767939f, TAIL_5 = 0.185716867f, TAIL_6 = -0.1529883f, TAIL_7 = 0.0366991907f;

// Phi(-|x|), and exp(-x^2 / 2) through `density`.
__device__ __forceinline__ float lower_tail(float x, float* density) {
  const float t = reciprocal_fast(fmaf(TAIL_SLOPE, fabsf(x), 1.0f));
  const float e = exp2_fast(x * x * -0.7213475204444817f);  // -log2(e) / 2
  float p = fmaf(TAIL_7, t, TAIL_6);
  p = fmaf(p, t, TAIL_5);
  p = fmaf(p, t, TAIL_4);
  p = fmaf(p, t, TAIL_3);
  p = fmaf(p, t, TAIL_2);
  p = fmaf(p, t, TAIL_1);
  p = fmaf(p, t, TAIL_0);
  *density = e;
  return p * t * e;
}

template <int SHAPE>
__device__ __forceinline__ float act_value(float x, float a, float b) {
  if constexpr (SHAPE == SHAPE_RELU) {
    return x < 0.0f ? 0.0f : x;  // keeps a NaN
  } else if constexpr (SHAPE == SHAPE_PHI) {
    // x Phi(x) = max(x, 0) - |x| Phi(-|x|); the cap keeps infinity times zero out
    float e;
    return fmaf(-fminf(fabsf(x), 1e4f), lower_tail(x, &e), fmaxf(x, 0.0f));
  } else if constexpr (SHAPE == SHAPE_SIGMOID) {
    return x * gate_of(x, a, b);
  } else {
    return x;
  }
}

// Two float32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// act_value of two values; the same operations, two at a time where there are such instructions.
template <int SHAPE>
__device__ __forceinline__ float2 act_value2(float2 x, float a, float b) {
  if constexpr (SHAPE == SHAPE_SIGMOID) {
    float2 q = mul2(x, x);
    q = make_float2(fminf(q.x, 1e8f), fminf(q.y, 1e8f));
    const float2 t = mul2(x, fma2(both(b), q, both(a)));
    const float2 e = make_float2(1.0f + exp2_fast(t.x), 1.0f + exp2_fast(t.y));
    return mul2(x, make_float2(reciprocal_fast(e.x), reciprocal_fast(e.y)));
  } else if constexpr (SHAPE == SHAPE_PHI) {
    const float2 m = make_float2(fabsf(x.x), fabsf(x.y));
    const float2 d = fma2(both(TAIL_SLOPE), m, both(1.0f));
    const float2 t = make_float2(reciprocal_fast(d.x), reciprocal_fast(d.y));
    const float2 q = mul2(mul2(x, x), both(-0.7213475204444817f));
    const float2 e = make_float2(exp2_fast(q.x), exp2_fast(q.y));
    float2 p = fma2(both(TAIL_7), t, both(TAIL_6));
    p = fma2(p, t, both(TAIL_5));
    p = fma2(p, t, both(TAIL_4));
    p = fma2(p, t, both(TAIL_3));
    p = fma2(p, t, both(TAIL_2));
    p = fma2(p, t, both(TAIL_1));
    p = fma2(p, t, both(TAIL_0));
    return fma2(make_float2(-fminf(m.x, 1e4f), -fminf(m.y, 1e4f)), mul2(mul2(p, t), e), make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
  } else {
    return make_float2(act_value<SHAPE>(x.x, a, b), act_value<SHAPE>(x.y, a, b));
  }
}

template <int SHAPE, int COUNT>
__device__ __forceinline__ void activate_all(float* v, float a, float b) {
#pragma unroll
  for (int j = 0; j < COUNT; j += 2) {
    const float2 y = act_value2<SHAPE>(make_float2(v[j], v[j + 1]), a, b);
    v[j] = y.x, v[j + 1] = y.y;
  }
}

// The activation and its derivative at two values.
template <int SHAPE>
__device__ __forceinline__ void act_both2(float2 x, float a, float b, float2* value, float2* slope) {
  if constexpr (SHAPE == SHAPE_RELU) {
    *value = make_float2(x.x < 0.0f ? 0.0f : x.x, x.y < 0.0f ? 0.0f : x.y);
    *slope = make_float2(x.x > 0.0f ? 1.0f : (x.x == x.x ? 0.0f : x.x), x.y > 0.0f ? 1.0f : (x.y == x.y ? 0.0f : x.y));
  } else if constexpr (SHAPE == SHAPE_PHI) {
    float2 e;
    const float2 tail = make_float2(lower_tail(x.x, &e.x), lower_tail(x.y, &e.y));
    const float2 cdf = make_float2(x.x > 0.0f ? 1.0f - tail.x : tail.x, x.y > 0.0f ? 1.0f - tail.y : tail.y);
    *value = mul2(x, cdf);
    *slope = fma2(mul2(x, both(0.3989422804014327f)), e, cdf);
  } else {
    // p' = p (1 - p) t' with t = -ln(2) (a x + b x^3)
    float2 q = mul2(x, x);
    q = make_float2(fminf(q.x, 1e8f), fminf(q.y, 1e8f));
    const float2 t = mul2(x, fma2(both(b), q, both(a)));
    const float2 p = make_float2(reciprocal_fast(1.0f + exp2_fast(t.x)), reciprocal_fast(1.0f + exp2_fast(t.y)));
    constexpr float LN2 = 0.6931471805599453f;
    const float2 d = fma2(both(-3.0f * LN2 * b), q, both(-LN2 * a));
    *value = mul2(x, p);
    *slope = fma2(mul2(*value, fma2(p, both(-1.0f), both(1.0f))), d, p);
  }
}

#endif  // __CUDACC__

// The code path and the coefficients of an activation (the inner one, for a gated pair).
inline void act_constants(int activation, int* shape, float* a, float* b) {
  *a = 0.0f, *b = 0.0f;
  switch (activation) {
    case ACT_RELU: *shape = 1; break;
    case ACT_GELU: case ACT_GEGLU: *shape = 2; break;
    case ACT_GELU_TANH: *shape = 3, *a = float(-LOG2_E * TANH_A), *b = float(-LOG2_E * TANH_A * 0.044715); break;
    case ACT_SILU: case ACT_SWIGLU: *shape = 3, *a = float(-LOG2_E); break;
    default: *shape = 0;
  }
}

}  // namespace og
