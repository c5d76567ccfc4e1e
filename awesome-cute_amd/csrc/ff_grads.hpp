// Launches of ff_grads.hip.
#pragma once
#include <hip/hip_runtime.h>

namespace w4a16 {

struct GatedGradArgs {
  const void* dh;    // (m x n)
  const float* pre;  // (m x ldpre), the forward pass's sums
  void* dgu;         // (m x 2n): [dg | du]
  long long lddh, ldpre, lddgu;
  int m, n, act;
};
void launch_gated_grad(const GatedGradArgs& a, bool bf, hipStream_t stream);

}  // namespace w4a16
