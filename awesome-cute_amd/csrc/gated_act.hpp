// The activations of the products: act(g) = g sigma(t), with t = g for silu and
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

// The same for a product with one sum, in as few instructions: the epilogue of a tile computes them for
// 256 values a lane with nothing to hide behind.  exp(-t) = 2^u, u = -log2(e) t.
template <int ACT>
__device__ __forceinline__ float act_sigma_of(float g, float g2) {
  constexpr float kLog2e = 1.4426950408889634f;
  const float u = ACT == kActGelu ? g * __builtin_fmaf(-kLog2e * kGeluB, g2, -kLog2e * kGeluA) : g * -kLog2e;
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u));
}
template <int ACT>
__device__ __forceinline__ float act_value(float g) { return g * act_sigma_of<ACT>(g, g * g); }

// Where such a product keeps anything for its backward pass, it is the slope, in 16 bits: slopes
// lie between -0.13 and 1.13, and a step of 2^-15 leaves them off by at most 2^-16, a thirtieth of what the
// rounding of dy act' to 16 bits adds where slopes are near one, and zero and one are exact.  The sums
// in 32 bits would take twice the bytes: 2048 x 10752 x 4096 12 us of 168 forward, and 14 of 40 backward.
// A slope's code is 8192 more than its steps, a NaN's zero.
constexpr float kSlopeSteps = 32768.f;
constexpr int kSlopeZero = 8192;
template <int ACT>
__device__ __forceinline__ float act_coded(float g, unsigned* code) {
  const float g2 = g * g, s = act_sigma_of<ACT>(g, g2);
  // sigma + g t' sigma (1 - sigma); far out, where the last factor is 0, g t' must not be infinite
  const float gt = ACT == kActGelu ? g * __builtin_fmaf(3.f * kGeluB, g2, kGeluA) : g;
  const float slope = __builtin_fmaf(__builtin_amdgcn_fmed3f(gt, -3e38f, 3e38f), __builtin_fmaf(-s, s, s), s);
  // the steps, rounded, are the low bits of a number as large as this (NaN: the maximum's other operand)
  constexpr float kLarge = 8388608.f;  // 2^23
  *code = __builtin_bit_cast(unsigned, __builtin_fmaxf(__builtin_fmaf(slope, kSlopeSteps, kLarge + kSlopeZero), kLarge));
  return g * s;
}
__device__ __forceinline__ float slope_of(unsigned code) {
  return code == 0 ? __builtin_nanf("") : (float)((int)code - kSlopeZero) * (1.f / kSlopeSteps);
}

}  // namespace w4a16
