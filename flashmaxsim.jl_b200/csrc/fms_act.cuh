// fms_act.cuh -- activations of the gated feed-forward block and their
// derivatives, two values at a time in float32.
//
// All of them are one exponential, one reciprocal and a few products per value
// (packed f32x2 where both values take the same operation): the error function's
// float32 routine alone would cost more issue slots than the matrix product leaves
// an epilogue.  The approximate exponential and reciprocal are off by about 2^-21 of
// their values here, the error function's side of gelu by 2^-14 of its own where it is
// small; the results are rounded to 11 or 8 bits afterwards.
#pragma once
#include "fms_common.cuh"

namespace fms {

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }

// 1 / (1 + 2^x) of both values.
__device__ __forceinline__ float2 logistic2(float2 x) {
  const float2 e = __fadd2_rn(make_float2(ex2_approx(x.x), ex2_approx(x.y)), pair(1.f));
  return make_float2(rcp_approx(e.x), rcp_approx(e.y));
}

// a(g) and, when DERIV, a'(g).
template <int ACT, bool DERIV>
__device__ __forceinline__ void act_eval2(float2 g, float2& a, float2& da) {
  constexpr float LOG2E = 1.4426950408889634f;
  if (ACT == FMS_ACT_SILU) {
    const float2 s = logistic2(__fmul2_rn(g, pair(-LOG2E)));
    a = __fmul2_rn(g, s);
    // s (1 + g (1 - s)) = s + a (1 - s); with 1 - s taken first, s + a does not round to a
    if (DERIV) da = __ffma2_rn(a, __fadd2_rn(pair(1.f), make_float2(-s.x, -s.y)), s);
  } else if (ACT == FMS_ACT_GELU) {
    // Phi(-|g|) = q = t (c1 + t (c2 + ...)) e^(-g^2/2), t = 1 / (1 + p |g|): the form of
    // Abramowitz and Stegun 7.1.26 with one term more.  The coefficients are a minimax fit
    // (linear programming over 1800 points of [0, 13.2]): off by 6.1e-8 and by 6.1e-5 of q at
    // most, so that the far side of the activation is right to below its rounding; in float32
    // |g| q is off by 1.6e-7.  Past 30 it is zero.
    const float2 m = make_float2(fminf(fabsf(g.x), 30.f), fminf(fabsf(g.y), 30.f));
    const float2 w = __ffma2_rn(m, pair(0.292f), pair(1.f));
    const float2 t = make_float2(rcp_approx(w.x), rcp_approx(w.y));
    const float2 x = __fmul2_rn(__fmul2_rn(m, m), pair(-0.5f * LOG2E));
    const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    float2 q = __ffma2_rn(t, pair(-0.086761039f), pair(0.270794447f));
    q = __ffma2_rn(t, q, pair(-0.076288227f));
    q = __ffma2_rn(t, q, pair(0.170907308f));
    q = __ffma2_rn(t, q, pair(0.103905974f));
    q = __ffma2_rn(t, q, pair(0.117441477f));
    q = __fmul2_rn(__fmul2_rn(t, q), e);
    // g Phi(g) = max(g, 0) - |g| q on both sides
    a = __ffma2_rn(make_float2(-m.x, -m.y), q, make_float2(max_nan(g.x, 0.f), max_nan(g.y, 0.f)));
    if (DERIV) {
      // Phi(g) + g phi(g): h = q - |g| phi for g < 0, and 1 - h on the other side
      const float2 h = __ffma2_rn(__fmul2_rn(m, pair(-0.3989422804f)), e, q);
      const float2 r = __fadd2_rn(pair(1.f), make_float2(-h.x, -h.y));
      da = make_float2(g.x < 0.f ? h.x : r.x, g.y < 0.f ? h.y : r.y);
      da = __ffma2_rn(g, pair(0.f), da);  // a NaN stays one
    }
  } else if (ACT == FMS_ACT_GELU_TANH) {
    // (1 + tanh y) / 2 = 1 / (1 + e^(-2y)), y = k (g + c g^3)
    constexpr float K = 0.7978845608028654f, C = 0.044715f;
    const float2 g2 = __fmul2_rn(g, g);
    const float2 y = __fmul2_rn(g, __ffma2_rn(g2, pair(-2.f * LOG2E * K * C), pair(-2.f * LOG2E * K)));
    const float2 s = logistic2(y);
    a = __fmul2_rn(g, s);
    if (DERIV) {
      // s + g s (1 - s) 2 y',  y' = k (1 + 3 c g^2).  From |g| = 10 on s (1 - s) is
      // below 2^-125 or zero: g^2 may end at 100, so that no infinity meets that zero.
      const float2 d = __ffma2_rn(make_float2(fminf(g2.x, 100.f), fminf(g2.y, 100.f)), pair(6.f * K * C), pair(2.f * K));
      da = __ffma2_rn(__fmul2_rn(a, __fadd2_rn(pair(1.f), make_float2(-s.x, -s.y))), d, s);
    }
  } else {  // FMS_ACT_RELU; a NaN stays one
    a = make_float2(max_nan(g.x, 0.f), max_nan(g.y, 0.f));
    if (DERIV) da = make_float2(g.x > 0.f ? 1.f : 0.f, g.y > 0.f ? 1.f : 0.f);
  }
}

}  // namespace fms
