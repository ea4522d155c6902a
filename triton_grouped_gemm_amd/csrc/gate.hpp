// The activations of the gated feed-forward block, shared by the kernels that apply them.
//
// Both are x sigma(z(x)) with z = x (silu) or z = 2 sqrt(2/pi) (x + 0.044715 x^3) (the tanh form of gelu: (1 + tanh(y)) / 2 = sigma(2 y)), so a value
// costs one exponential and one reciprocal.  Everything is fp32: the hardware's exp2 and reciprocal are good to an ulp, far below the rounding of a
// 16-bit result.  A gate of -inf gives NaN, as x / (1 + exp(-x)) does.
#pragma once
#include "common.hpp"

namespace tgg {

enum : int { GATE_SILU = 0, GATE_GELU_TANH = 1 };

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGelu1 = 1.5957691216057308f;             // 2 sqrt(2 / pi)
constexpr float kGelu3 = 1.5957691216057308f * 0.044715f;

// sigma(z(x))
template <int ACT> TGG_DEV float gate_sigma(float x) {
  const float z2 = ACT == GATE_SILU ? x * -kLog2e : x * (-kLog2e * kGelu1 - kLog2e * kGelu3 * (x * x));  // -z log2(e)
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z2));
}
template <int ACT> TGG_DEV float gate_act(float x) { return x * gate_sigma<ACT>(x); }

// Activation and its slope at x: sigma + x sigma (1 - sigma) z'(x)
template <int ACT> TGG_DEV void gate_act_slope(float x, float& act, float& slope) {
  const float s = gate_sigma<ACT>(x);
  // (the square kept finite: for |x| beyond 1.8e19 the slope of sigma is an exact 0 and must stay one)
  const float dz = ACT == GATE_SILU ? 1.0f : kGelu1 + 3.0f * kGelu3 * fminf(x * x, 1e30f);
  act = x * s;
  slope = s + act * (1.0f - s) * dz;
}

}  // namespace tgg
