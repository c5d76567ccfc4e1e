// What stands between the products of a gated projection's backward pass: the gradients of its
// two sums, dg = dh u act'(g) and du = dh act(g), in fp32 from the sums that the forward pass
// kept in fp32, rounded to 16 bits, as matrix instructions take them.  Rows of [dg | du]: both
// products of the backward pass read them as they are (ff_tile.hpp).
//
// Bound: HBM: 14 bytes for every element of dh.  2048 x 10752: 308 MB, 48 us, 6.4 TB/s.
#include <hip/hip_runtime.h>

#include "ff_grads.hpp"
#include "ff_products.hpp"

namespace w4a16 {

namespace {

template <bool BF>
__device__ __forceinline__ float widen(unsigned bits) {
  if constexpr (BF) return __builtin_bit_cast(float, bits << 16);
  return (float)__builtin_bit_cast(half_t, (unsigned short)bits);
}

}  // namespace

// eight columns of a row a thread
template <bool BF>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedGradArgs p) {
  const int pieces = p.n / 8;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(at / pieces), c = (int)(at - (long long)r * pieces);
  if (r >= p.m) return;
  half_t* const out = (half_t*)p.dgu + (size_t)r * p.lddgu;
  const i4 dh = *(const i4*)((const half_t*)p.dh + (size_t)r * p.lddh + 8 * c);
  const float* const pre = p.pre + (size_t)r * p.ldpre + pre_col(8 * c);
  i4 dg, du;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const f4 g = *(const f4*)(pre + 2 * i), u = *(const f4*)(pre + 2 * i + 16);
    f4 a, b;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float d = widen<BF>((unsigned)dh[i + (e >> 1)] >> (16 * (e & 1)) & 0xffffu);
      float value, slope;
      act_slope(g[e], p.act, &value, &slope);
      a[e] = d * u[e] * slope;
      b[e] = d * value;
    }
    const i2 ra = product_round<BF>(a), rb = product_round<BF>(b);
    dg[i] = ra[0];
    dg[i + 1] = ra[1];
    du[i] = rb[0];
    du[i + 1] = rb[1];
  }
  *(i4*)(out + 8 * c) = dg;
  *(i4*)(out + p.n + 8 * c) = du;
}

void launch_gated_grad(const GatedGradArgs& a, bool bf, hipStream_t stream) {
  const dim3 grid((unsigned)(((long long)a.m * (a.n / 8) + 255) / 256));
  if (bf)
    hipLaunchKernelGGL(gated_grad_kernel<true>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(gated_grad_kernel<false>, grid, dim3(256), 0, stream, a);
}

}  // namespace w4a16
