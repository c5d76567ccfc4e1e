// The activations of the products: act(g) = g sigma(t), with t = g for silu and
// t = sqrt(8 / pi) (g + 0.044715 g^3) for gelu in its tanh form (g / 2 (1 + tanh(t / 2))).
// All in fp32: an exponential and a reciprocal, each good to some 1e-7 of its argument's
// size, far below the half steps of the 16 bits that the results are rounded to.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

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

// Where such a product keeps anything for its backward pass, it is the slope, in 16 bits.  Slopes lie between
// -0.13 and 1.13, so that a step of 2^-15 leaves them off by at most 2^-16, a thirtieth of what the rounding
// of dy act' to fp16 adds where slopes are near one; but of a unit that is far on the negative side,
// where slopes are 2^-14 and less, such steps leave little or nothing.  So slopes below a border B in size,
// 2^-5 in fp16 and 2^-7 in bfloat16, are numbers of the type itself, brought by a power of two to where its
// exponents begin, and steps of 2^-15 go on from there, as fine as these are at the border:
//   code = the number's bits of min(s, B)  +  (s - B) 2^15, if that is positive,
// of a slope's size; 65535 less this for negative ones, and 49151, between the two, for NaN.  bfloat16: good to 2^-8
// of a slope, what dy act' is rounded to, down to 2^-102.  fp16: to 2^-11 down to 2^-16, from there in
// steps of 2^-26, no coarser than fp16 holds dy act' where dy is up to 4.  Nowhere off by more than 2^-16; zero and one
// are exact.  Both passes of 2048 x 10752 x 4096 take 477 us, with steps alone 473; the sums in 32 bits, twice the
// bytes, took 12 more forward and 14 more backward.
constexpr float kSlopeSteps = 32768.f;
constexpr unsigned kSlopeBorder = 12288, kSlopeNan = 49151;  // codes
template <bool BF>
struct SlopeForm {
  static constexpr float kBorder = BF ? 0x1p-7f : 0x1p-5f;
  static constexpr float kUnit = BF ? 0x1p-24f : 4.f;  // (brings the border to the number whose bits are kSlopeBorder)
};

// Steps of 2^-15 alone (feedforward_linear's form): a code is 8192 more than a slope's steps, a NaN's is zero.
constexpr int kSlopeZero = 8192;

// act(g), and the slope
template <int ACT>
__device__ __forceinline__ float act_value_slope(float g, float* slope) {
  const float g2 = g * g, s = act_sigma_of<ACT>(g, g2);
  // sigma + g t' sigma (1 - sigma); far out, where the last factor is 0, g t' must not be infinite
  const float gt = ACT == kActGelu ? g * __builtin_fmaf(3.f * kGeluB, g2, kGeluA) : g;
  *slope = __builtin_fmaf(__builtin_amdgcn_fmed3f(gt, -3e38f, 3e38f), __builtin_fmaf(-s, s, s), s);
  return g * s;
}

// the low halves of two numbers
__device__ __forceinline__ unsigned low_halves(float first, float second) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, second), __builtin_bit_cast(unsigned, first), 0x05040100);
}

// the codes of two slopes
template <bool BF>
__device__ __forceinline__ unsigned slope_codes(float a, float b) {
  typedef short S2 __attribute__((ext_vector_type(2)));
  typedef unsigned short U2 __attribute__((ext_vector_type(2)));
  using Number = std::conditional_t<BF, __bf16, _Float16>;
  typedef Number N2 __attribute__((ext_vector_type(2)));
  using Form = SlopeForm<BF>;
  const auto inside = [](float s) { return __builtin_amdgcn_fmed3f(s, -Form::kBorder, Form::kBorder); };
  const float ia = inside(a), ib = inside(b);
  unsigned number = __builtin_bit_cast(unsigned, (N2){(Number)(ia * Form::kUnit), (Number)(ib * Form::kUnit)});
#if defined(__HIP_DEVICE_COMPILE__)
  asm("" : "+v"(number));  // (one register: otherwise each half is converted once more for its sign)
#endif
  const unsigned negative = __builtin_bit_cast(unsigned, __builtin_bit_cast(S2, number) >> 15);
  // What is left in steps of 2^-15, rounded, a negative slope's negative: the low bits of a number as large as 384.  (NaN:
  // the maximum's other operand, and its inside is -B, the least of the median's others: their sum is kSlopeNan.)
  const auto steps = [](float left) { return __builtin_fmaxf(left + 384.f, 384.f - 4096.f / kSlopeSteps); };
  static_assert((0xffffu - kSlopeBorder) - 4096 == kSlopeNan, "");
  return __builtin_bit_cast(unsigned, (U2)(__builtin_bit_cast(U2, (number & 0x7fff7fffu) ^ negative) +
                                           __builtin_bit_cast(U2, low_halves(steps(a - ia), steps(b - ib)))));
}
template <bool BF>
__device__ __forceinline__ float slope_of(unsigned code) {
  using Number = std::conditional_t<BF, __bf16, _Float16>;
  const bool negative = code > kSlopeNan;
  const unsigned size = negative ? 0xffffu - code : code, number = size < kSlopeBorder ? size : kSlopeBorder;
  const float inside = (float)__builtin_bit_cast(Number, (unsigned short)number) * (1.f / SlopeForm<BF>::kUnit);
  const float s = __builtin_fmaf((float)(size - number), 1.f / kSlopeSteps, inside);
  return code == kSlopeNan ? __builtin_nanf("") : negative ? -s : s;
}

// ... and in steps alone
__device__ __forceinline__ unsigned slope_step_codes(float a, float b) {
  // (likewise; NaN: the maximum's other operand)
  const auto steps = [](float s) { return __builtin_fmaxf(s + (256.f + kSlopeZero / kSlopeSteps), 256.f); };
  return low_halves(steps(a), steps(b));
}
__device__ __forceinline__ float slope_of_steps(unsigned code) {
  return code == 0 ? __builtin_nanf("") : (float)((int)code - kSlopeZero) * (1.f / kSlopeSteps);
}

}  // namespace w4a16
