// What stands between the products of a backward pass: the gradients of a gated product's two
// sums, and transposes.  The products themselves (ff_tiles.hip) take both operands with the
// summed dimension along a row, so the gradient of a weight, a sum over tokens, is a product of
// transposed operands.
//
// Bound: HBM.  A workgroup takes 64 x 64 elements, two rows of eight columns a thread; turned
// over, pairs of rows go through LDS as words, pitch 33 of them, so that a wave's 64 words
// meet no bank twice.
#include <hip/hip_runtime.h>

#include "ff_grads.hpp"
#include "ff_products.hpp"

namespace w4a16 {

namespace {

constexpr int kTile = 64, kThreads = 256;
constexpr int kPitch = kTile / 2 + 1;  // words: 32 pairs of rows of a column

struct Pieces {  // eight columns of two rows
  i4 row[2];
};

// the words (row 2 rp, row 2 rp + 1) of columns 8 c ... 8 c + 7
__device__ __forceinline__ void put_pairs(int* lds, const Pieces& v, int rp, int c) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const unsigned a = v.row[0][i], b = v.row[1][i];
    lds[(8 * c + 2 * i) * kPitch + rp] = (int)((a & 0xffffu) | (b << 16));
    lds[(8 * c + 2 * i + 1) * kPitch + rp] = (int)((a >> 16) | (b & 0xffff0000u));
  }
}
// 64 columns turned into rows of `out`: columns below `cols`, all 64 rows of the tile
__device__ __forceinline__ void store_turned(const int* lds, half_t* out, size_t ld, int cols) {
#pragma unroll
  for (int it = 0; it < 2; it++) {
    const int at = it * kThreads + (int)threadIdx.x;
    const int col = at >> 3, q = at & 7;
    if (col >= cols) continue;
    const int* const w = lds + col * kPitch + 4 * q;
    *(i4*)(out + (size_t)col * ld + 8 * q) = (i4){w[0], w[1], w[2], w[3]};
  }
}

template <bool BF>
__device__ __forceinline__ float widen(unsigned bits) {
  if constexpr (BF) return __builtin_bit_cast(float, bits << 16);
  return (float)__builtin_bit_cast(half_t, (unsigned short)bits);
}

}  // namespace

// out (cols x rows, rows of out ld_out apart) = in^T; columns of out from `rows` up to the next
// multiple of 64 are zeros
__global__ __launch_bounds__(kThreads) void transpose_kernel(const half_t* in, long long ld_in, half_t* out,
                                                             long long ld_out, int rows, int cols) {
  __shared__ int lds[kTile * kPitch];
  const int c0 = kTile * blockIdx.x, r0 = kTile * blockIdx.y;
  const int c = threadIdx.x & 7, rp = threadIdx.x >> 3;
  Pieces v;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = r0 + 2 * rp + h;
    v.row[h] = (i4){0, 0, 0, 0};
    if (r < rows && c0 + 8 * c < cols) v.row[h] = *(const i4*)(in + (size_t)r * ld_in + c0 + 8 * c);
  }
  put_pairs(lds, v, rp, c);
  __syncthreads();
  store_turned(lds, out + (size_t)c0 * ld_out + r0, ld_out, min(kTile, cols - c0));
}

// dg = dh u act'(g), du = dh act(g) of a gated product, in fp32 from the sums that the forward
// pass kept in fp32, rounded to 16 bits, as matrix instructions take them: as rows of
// [dg | du] for the product with the weights, and turned over for that with the inputs.
template <bool BF>
__global__ __launch_bounds__(kThreads) void gated_grad_kernel(GatedGradArgs p) {
  __shared__ int lds[2][kTile * kPitch];
  const int c0 = kTile * blockIdx.x, r0 = kTile * blockIdx.y;
  const int c = threadIdx.x & 7, rp = threadIdx.x >> 3;
  Pieces dg, du;
  const bool in = c0 + 8 * c < p.n;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = r0 + 2 * rp + h;
    dg.row[h] = du.row[h] = (i4){0, 0, 0, 0};
    if (!in || r >= p.m) continue;
    const i4 dh = *(const i4*)((const half_t*)p.dh + (size_t)r * p.lddh + c0 + 8 * c);
    const float* const pre = p.pre + (size_t)r * p.ldpre + pre_col(c0 + 8 * c);
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
      dg.row[h][i] = ra[0];
      dg.row[h][i + 1] = ra[1];
      du.row[h][i] = rb[0];
      du.row[h][i + 1] = rb[1];
    }
    if (p.dgu) {
      half_t* const out = (half_t*)p.dgu + (size_t)r * p.lddgu + c0 + 8 * c;
      *(i4*)out = dg.row[h];
      *(i4*)(out + p.n) = du.row[h];
    }
  }
  if (p.dgu && blockIdx.x == 0) {  // what a row has behind its 2n columns up to a multiple of 64
    const int r = r0 + 2 * rp + (c & 1), pieces = ((2 * p.n + 63) / 64 * 64 - 2 * p.n) / 8;
    if (r < p.m)
      for (int i = c >> 1; i < pieces; i += 4)
        *(i4*)((half_t*)p.dgu + (size_t)r * p.lddgu + 2 * p.n + 8 * i) = (i4){0, 0, 0, 0};
  }
  if (!p.dgu_t) return;
  put_pairs(lds[0], dg, rp, c);
  put_pairs(lds[1], du, rp, c);
  __syncthreads();
  half_t* const out = (half_t*)p.dgu_t + (size_t)c0 * p.lddgu_t + r0;
  const int cols = min(kTile, p.n - c0);
  store_turned(lds[0], out, p.lddgu_t, cols);
  store_turned(lds[1], out + (size_t)p.n * p.lddgu_t, p.lddgu_t, cols);
}

void launch_transpose(const void* in, long long ld_in, void* out, long long ld_out, int rows, int cols,
                      hipStream_t stream) {
  hipLaunchKernelGGL(transpose_kernel, dim3(ceil_div(cols, kTile), ceil_div(rows, kTile)), dim3(kThreads), 0, stream,
                     (const half_t*)in, ld_in, (half_t*)out, ld_out, rows, cols);
}

void launch_gated_grad(const GatedGradArgs& a, bool bf, hipStream_t stream) {
  const dim3 grid(ceil_div(a.n, kTile), ceil_div(a.m, kTile));
  if (bf)
    hipLaunchKernelGGL(gated_grad_kernel<true>, grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(gated_grad_kernel<false>, grid, dim3(kThreads), 0, stream, a);
}

}  // namespace w4a16
