// Dropout, with the residual's addition or without, and its gradient, which is the same of dy: the
// mask is made from the seed both times (dropout.hpp) and never stored.
//
// A thread has one group of eight elements: 16 bytes of 16-bit elements, one run of the generator.
// Inside fp32, rounded once.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/feedforward_amd.h"
#include "dropout.hpp"
#include "ff_grads.hpp"

namespace w4a16 {

namespace {

constexpr int kThreads = 256;

template <class T>
struct Eight {
  T v[8];
};

}  // namespace

// WHOLE: every matrix starts on 16 bytes, the count is a multiple of eight
template <class T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs p) {
  const unsigned long long group = (unsigned long long)blockIdx.x * kThreads + threadIdx.x;
  const long long left = p.count - (long long)(8 * group);
  if (left <= 0) return;
  const T* const x = (const T*)p.x + 8 * group;
  const T* const residual = (const T*)p.residual + 8 * group;
  T* const y = (T*)p.y + 8 * group;
  __attribute__((aligned(16))) Eight<T> a, r;
  if constexpr (WHOLE) {
    a = *(const Eight<T>*)__builtin_assume_aligned(x, 16);
    if (p.residual) r = *(const Eight<T>*)__builtin_assume_aligned(residual, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      a.v[e] = e < left ? x[e] : (T)0.f;
      if (p.residual) r.v[e] = e < left ? residual[e] : (T)0.f;
    }
  }
  const i4 bits = drop_bits(group, DropKey(p.drop));
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float v = drop_one((float)a.v[e], bits, e, p.drop);
    a.v[e] = (T)(p.residual ? (float)r.v[e] + v : v);
  }
  if constexpr (WHOLE) {
    *(Eight<T>*)__builtin_assume_aligned(y, 16) = a;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < left) y[e] = a.v[e];
  }
}

template <class T>
static void launch_of(const DropoutArgs& a, hipStream_t stream) {
  const bool whole = a.count % 8 == 0 && ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.residual & 15) == 0 &&
                     ((uintptr_t)a.y & 15) == 0;
  const dim3 grid((unsigned)((a.count + 8 * kThreads - 1) / (8 * kThreads)));
  if (whole)
    hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
}

void launch_dropout(const DropoutArgs& a, int type, hipStream_t stream) {
  if (type == FEEDFORWARD_FP16) launch_of<half_t>(a, stream);
  if (type == FEEDFORWARD_BF16) launch_of<__bf16>(a, stream);
  if (type == FEEDFORWARD_FP32) launch_of<float>(a, stream);
}

}  // namespace w4a16
