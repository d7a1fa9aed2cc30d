// Gate activations of the gated feed-forward kernels, in fp32, with their derivatives.
//   0  silu      g * s(g), s(g) = 1 / (1 + exp(-g));           slope  s * (1 + g * (1 - s))
//   1  gelu      tanh form, written with the same logistic function: 0.5 * (1 + tanh(z)) = s(2 z), so
//                gelu(g) = g * s(2 z), z = sqrt(2/pi) * (g + 0.044715 g^3);
//                slope  s + g * s * (1 - s) * 2 z'
// One exponential and one reciprocal per value serve both the value and the slope.  __expf errs by 2 + 1.2 |x| units in
// the last place of fp32: at |x| = 80, where s has long become 0 or 1 to the bits that are kept, 2^-17, still below
// the rounding to 16 bits that follows.  For a large negative argument exp overflows to infinity and 1 / (1 + inf)
// is the 0 it should be.  gelu's argument is taken at |g| <= 30, beyond which s is exactly 0 or 1, so that its
// cube and its slope cannot overflow.
#pragma once

#include <cuda_runtime.h>

namespace b200 {

constexpr int kNumActivations = 2;
enum : int { kActSilu = 0, kActGeluTanh = 1 };

__device__ __forceinline__ float logistic(float x) { return __frcp_rn(1.f + __expf(-x)); }

__device__ __forceinline__ float gate_value(float g, int act) {
  float arg = g;
  if (act == kActGeluTanh) {
    const float c = fminf(fmaxf(g, -30.f), 30.f);
    arg = 1.5957691216f * c * fmaf(0.044715f * c, c, 1.f);
  }
  return g * logistic(arg);
}

// value and slope
__device__ __forceinline__ void gate_value_slope(float g, int act, float& value, float& slope) {
  float arg = g, darg = 1.f;
  if (act == kActGeluTanh) {
    const float c = fminf(fmaxf(g, -30.f), 30.f);
    const float g2 = 0.044715f * c * c;
    arg = 1.5957691216f * c * (g2 + 1.f);
    darg = 1.5957691216f * fmaf(3.f, g2, 1.f);
  }
  const float s = logistic(arg);
  value = g * s;
  slope = fmaf(value * (1.f - s), darg, s);
}

}  // namespace b200
