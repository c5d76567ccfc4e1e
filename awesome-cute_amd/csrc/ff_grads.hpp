// Launches of ff_grads.hip.
#pragma once
#include <hip/hip_runtime.h>

#include "dropout.hpp"

namespace w4a16 {

struct GatedGradArgs {
  const void* dh;    // (m x n)
  const float* pre;  // (m x ldpre), the forward pass's sums
  void* dgu;         // (m x 2n): [dg | du]
  long long lddh, ldpre, lddgu;
  int m, n, act;
};
void launch_gated_grad(const GatedGradArgs& a, bool bf, hipStream_t stream);

struct LinearGradArgs {
  const void* dy;    // (m x n)
  const unsigned short* slopes;  // null (no activation), or the forward pass's (m x n)
  void* dz;          // null, or (m x n)
  void* dbias;       // null, or n elements
  float* partials;   // linear_grad_parts(m, n) rows of n, where dbias is wanted and these are more than one
  long long lddy, ldslopes, lddz;
  int m, n, rows_per_part;
  bool slope_steps;  // their form (gated_act.hpp)
  DropArgs drop;
  float bias_factor;  // of dbias (of what is kept, where dz is without it)
};
int linear_grad_parts(int m, int n);
void launch_linear_grad(LinearGradArgs a, bool bf, hipStream_t stream);

// y = residual (or null) + drop(x), `count` elements that lie as one row
struct DropoutArgs {
  const void* x;
  const void* residual;
  void* y;
  long long count;
  DropArgs drop;
};
void launch_dropout(const DropoutArgs& a, int type, hipStream_t stream);  // FEEDFORWARD_FP16 ...

}  // namespace w4a16
