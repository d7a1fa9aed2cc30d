// Gate activations of the gated feed-forward kernels, in fp32, with their derivatives.
//   0  silu      g * s(g), s(g) = 1 / (1 + exp(-g));           slope  s * (1 + g * (1 - s))
//   1  gelu      tanh form, written with the same logistic function: 0.5 * (1 + tanh(z)) = s(2 z), so
//                gelu(g) = g * s(2 z), z = sqrt(2/pi) * (g + 0.044715 g^3);
//                slope  s + g * s * (1 - s) * 2 z'
// One exponential and one reciprocal (the hardware's approximations) serve both the value and the slope: the
// exponential errs by about 2 + 1.2 |x| units in the last place of fp32, 2^-17 at |x| = 80, where s has long become 0
// or 1 to the bits that are kept; the rounding to 16 bits that follows is larger.  For a large negative argument
// exp overflows to infinity and 1 / (1 + inf) is the 0 it should be.  gelu's argument is taken at |g| <= 30, beyond
// which s is exactly 0 or 1, so that its cube and its slope cannot overflow.
#pragma once

#include <cuda_runtime.h>

namespace b200 {

constexpr int kNumActivations = 2;
enum : int { kActSilu = 0, kActGeluTanh = 1 };

// 1 / (1 + 2^y)
__device__ __forceinline__ float logistic2(float y) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kGeluArg = 2.f * 0.7978845608028654f * kLog2E;  // 2 sqrt(2/pi) log2(e)

template <int kAct>
__device__ __forceinline__ float gate_value(float g) {
  if constexpr (kAct == kActSilu) return g * logistic2(-kLog2E * g);
  const float c = fminf(fmaxf(g, -30.f), 30.f);
  return g * logistic2(-kGeluArg * c * fmaf(0.044715f * c, c, 1.f));
}

// value and slope
template <int kAct>
__device__ __forceinline__ void gate_value_slope(float g, float& value, float& slope) {
  if constexpr (kAct == kActSilu) {
    const float s = logistic2(-kLog2E * g);
    value = g * s;
    slope = fmaf(value, 1.f - s, s);
  } else {
    const float c = fminf(fmaxf(g, -30.f), 30.f);
    const float c2 = 0.044715f * c * c;
    const float s = logistic2(-kGeluArg * c * (c2 + 1.f));
    value = g * s;
    slope = fmaf(value * (1.f - s), (kGeluArg / kLog2E) * fmaf(3.f, c2, 1.f), s);
  }
}

}  // namespace b200
