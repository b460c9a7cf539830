// fms_act.cuh -- activations of the gated feed-forward block and their
// derivatives, in float32.
#pragma once
#include "fms_common.cuh"

namespace fms {

// a(g) and, when DERIV, a'(g).  The exponentials are the fast ones (relative
// error about 2^-21 here): the results are rounded to 11 or 8 bits afterwards.
template <int ACT, bool DERIV>
__device__ __forceinline__ void act_eval(float g, float& a, float& da) {
  if (ACT == FMS_ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    a = g * s;
    if (DERIV) da = s * (1.f + g * (1.f - s));
  } else if (ACT == FMS_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    if (DERIV) da = cdf + g * 0.3989422804014327f * __expf(-0.5f * g * g);
  } else if (ACT == FMS_ACT_GELU_TANH) {
    const float k = 0.7978845608028654f, c = 0.044715f;
    const float y = k * (g + c * g * g * g);
    const float t = 1.f - __fdividef(2.f, 1.f + __expf(2.f * y));  // tanh(y)
    a = 0.5f * g * (1.f + t);
    if (DERIV) da = 0.5f * (1.f + t) + 0.5f * g * (1.f - t * t) * k * (1.f + 3.f * c * g * g);
  } else {  // FMS_ACT_RELU; a NaN stays one
    a = g > 0.f || g != g ? g : 0.f;
    if (DERIV) da = g > 0.f ? 1.f : 0.f;
  }
}

}  // namespace fms
