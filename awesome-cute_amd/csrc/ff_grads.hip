// What stands between the products of a backward pass.
//
// Of a gated projection: the gradients of its
// two sums, dg = dh u act'(g) and du = dh act(g), in fp32 from the sums that the forward pass
// kept in fp32, rounded to 16 bits, as matrix instructions take them.  Rows of [dg | du]: both
// products of the backward pass read them as they are (ff_tile.hpp).  Bound: HBM: 14 bytes for every element of dh.  2048 x 10752: 308 MB, 48 us, 6.4 TB/s.
//
// Of a full product, y = residual + drop(act(z)) with z = x W^T + bias: dz = drop(dy) act'(z), rounded to
// 16 bits for the products, without the factor of what is kept, by which these multiply their sums in fp32: so it is,
// without an activation, dy or zero, exactly (rounded with the factor, gradients were 1.4 times as far off as their
// own rounding makes them), and stays in fp16's range whatever the factor, and the bias's gradient, its sum over rows, of the unrounded values in
// fp32.  A workgroup takes 256 columns (fewer where there are fewer) of a run of rows, 16 bytes a
// thread; its column sums meet in LDS and go to `partials`, and a second launch adds the runs' in their
// order, unless there is one.  Bound: HBM, of small ones the launches: 2048 x 10752 with slopes 132 MB, 23.4 us,
// 5.8 TB/s, and 4 us for the sums; four rows a thread at least and half the workgroups 25, eight rows 30.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ff_grads.hpp"
#include "ff_products.hpp"

namespace w4a16 {

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
    const f4 d = widen4<BF>((i2){dh[i], dh[i + 1]});
    f4 a, b;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float value, slope;
      act_slope(g[e], p.act, &value, &slope);
      a[e] = d[e] * u[e] * slope;
      b[e] = d[e] * value;
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

namespace {

constexpr int kRunThreads = 256;
constexpr int kRunGroups = 4096;  // workgroups that the runs make up, at most
constexpr int kRunRows = 2;       // rows that a thread has, at least

// threads beside each other along a row, eight columns each
__host__ __device__ __forceinline__ int run_width(int n) {
  int width = 32;
  while (width > 1 && 4 * width >= n) width /= 2;
  return width;
}

template <bool BF>
__device__ __forceinline__ void store_bias(void* dbias, int column, float sum) {
  if constexpr (BF)
    ((__bf16*)dbias)[column] = (__bf16)sum;
  else
    ((half_t*)dbias)[column] = (half_t)sum;
}

}  // namespace

// STEPS: slopes in steps alone
template <bool BF, bool STEPS>
__global__ __launch_bounds__(kRunThreads) void linear_grad_kernel(LinearGradArgs p) {
  __shared__ float room[kRunThreads][8 + 1];
  const int width = run_width(p.n), high = kRunThreads / width;
  const int c = threadIdx.x % width, r0 = threadIdx.x / width;
  const int col = 8 * ((int)blockIdx.x * width + c);
  const bool in = col < p.n;
  const int part = blockIdx.y;
  const long long first = (long long)part * p.rows_per_part;
  const long long end = min(first + p.rows_per_part, (long long)p.m);
  const DropKey key(p.drop);
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (in) {
#pragma unroll 2
    for (long long r = first + r0; r < end; r += high) {
      const i4 dy = *(const i4*)((const half_t*)p.dy + (size_t)r * p.lddy + col);
      i4 slopes, bits;
      // (read this once, and written a forward pass ago)
      if (p.slopes) slopes = __builtin_nontemporal_load((const i4*)(p.slopes + (size_t)r * p.ldslopes + col));
      if (p.drop.below) bits = drop_bits((unsigned long long)r * (unsigned)(p.n >> 3) + (unsigned)(col >> 3), key);
      i4 dz;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        f4 d = widen4<BF>((i2){dy[2 * h], dy[2 * h + 1]});
        if (p.slopes)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned code = (unsigned)slopes[2 * h + (e >> 1)] >> (16 * (e & 1)) & 0xffffu;
            d[e] *= STEPS ? slope_of_steps(code) : slope_of<BF>(code);
          }
        // (last: what is dropped has no gradient, whatever its slope)
        if (p.drop.below) d = drop4(d, (i2){bits[2 * h], bits[2 * h + 1]}, p.drop);
#pragma unroll
        for (int e = 0; e < 4; e++) sum[4 * h + e] += d[e];
        const i2 rounded = product_round<BF>(d);
        dz[2 * h] = rounded[0];
        dz[2 * h + 1] = rounded[1];
      }
      if (p.dz) *(i4*)((half_t*)p.dz + (size_t)r * p.lddz + col) = dz;
    }
  }
  if (!p.dbias) return;
#pragma unroll
  for (int e = 0; e < 8; e++) room[threadIdx.x][e] = sum[e];
  __syncthreads();
  // a thread a column, the rows' sums in their order
  for (int at = threadIdx.x; at < 8 * width; at += kRunThreads) {
    const int column = 8 * (int)blockIdx.x * width + at;
    if (column >= p.n) continue;
    float s = room[at / 8][at % 8];
    for (int r = 1; r < high; r++) s += room[r * width + at / 8][at % 8];
    if (p.partials)
      p.partials[(size_t)part * p.n + column] = s;
    else
      store_bias<BF>(p.dbias, column, s * p.bias_factor);
  }
}

// the runs' sums: 64 columns and 16 waves a workgroup, a wave every sixteenth run
template <bool BF>
__global__ __launch_bounds__(1024) void bias_sums_kernel(LinearGradArgs p, int parts) {
  __shared__ float room[16][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = 64 * blockIdx.x + lane;
  const float* const from = p.partials + (c < p.n ? c : 0);
  float s = 0.f;
#pragma unroll 8
  for (int i = wave; i < parts; i += 16) s += from[(size_t)i * p.n];
  room[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= p.n) return;
  s = room[0][lane];
#pragma unroll
  for (int i = 1; i < 16; i++) s += room[i][lane];
  store_bias<BF>(p.dbias, c, s * p.bias_factor);
}

// (rows count in 64 bits: with what rounds them up they may pass an int)
static int runs_of(int m, long long rows) { return (int)((m + rows - 1) / rows); }
int linear_grad_parts(int m, int n) {
  const int width = run_width(n), across = ceil_div(n, 8 * width), high = kRunThreads / width;
  return std::max(1, std::min(kRunGroups / across, runs_of(m, kRunRows * high)));
}

void launch_linear_grad(LinearGradArgs a, bool bf, hipStream_t stream) {
  const int width = run_width(a.n);
  a.rows_per_part = runs_of(a.m, linear_grad_parts(a.m, a.n));
  const int parts = runs_of(a.m, a.rows_per_part);
  if (parts == 1) a.partials = nullptr;  // (its sums are the bias's)
  const dim3 grid(ceil_div(a.n, 8 * width), parts), sums(ceil_div(a.n, 64));
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kRunThreads), 0, stream, a); };
  if (bf)
    a.slope_steps ? launch(linear_grad_kernel<true, true>) : launch(linear_grad_kernel<true, false>);
  else
    a.slope_steps ? launch(linear_grad_kernel<false, true>) : launch(linear_grad_kernel<false, false>);
  if (!a.partials) return;
  if (bf)
    hipLaunchKernelGGL(bias_sums_kernel<true>, sums, dim3(1024), 0, stream, a, parts);
  else
    hipLaunchKernelGGL(bias_sums_kernel<false>, sums, dim3(1024), 0, stream, a, parts);
}

}  // namespace w4a16
