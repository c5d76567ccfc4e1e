// The activations of the gated projections: act(g) = g sigma(t), with t = g for silu and
// t = sqrt(8 / pi) (g + 0.044715 g^3) for gelu in its tanh form (g / 2 (1 + tanh(t / 2))).
// All in fp32: an exponential and a reciprocal, each good to some 1e-7 of its argument's
// size, far below the half steps of the 16 bits that the results are rounded to.
#pragma once
#include <hip/hip_runtime.h>

namespace w4a16 {

constexpr int kActNone = 0, kActSilu = 1, kActGelu = 2;
__host__ __device__ __forceinline__ bool act_known(int act) { return act == kActSilu || act == kActGelu; }

constexpr float kGeluA = 1.5957691216057308f;   // sqrt(8 / pi)
constexpr float kGeluB = 0.07135481627260025f;  // 0.044715 of that

__device__ __forceinline__ float act_sigma(float g, int act) {
  const float t = act == kActGelu ? g * __builtin_fmaf(kGeluB * g, g, kGeluA) : g;
  // (exp(-t) beyond the largest float is infinity, and its reciprocal zero)
  return __builtin_amdgcn_rcpf(1.f + __expf(-t));
}

// act(g) u
__device__ __forceinline__ float act_mul(float g, float u, int act) { return g * act_sigma(g, act) * u; }

// act(g) and act'(g) = sigma + g sigma (1 - sigma) t'
__device__ __forceinline__ void act_slope(float g, int act, float* value, float* slope) {
  const float s = act_sigma(g, act);
  const float dt = act == kActGelu ? __builtin_fmaf(3.f * kGeluB * g, g, kGeluA) : 1.f;
  *value = g * s;
  // (far out, where 1 - sigma is 0 and g t' may be infinite, the product is 0)
  const float bend = s * (1.f - s);
  *slope = bend == 0.f ? s : __builtin_fmaf(g * dt, bend, s);
}

}  // namespace w4a16
