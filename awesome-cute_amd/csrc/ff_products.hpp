// What the dense products of the feed-forward block share: their arguments, the two 16-bit
// types, the gated column order, and what becomes of a product's sums.
#pragma once
#include <hip/hip_runtime.h>

#include "buffer_loads.hpp"
#include "dropout.hpp"
#include "f16_dense.hpp"
#include "gated_act.hpp"
#include "w4a16_common.hpp"

namespace w4a16 {

// How the operands of a product lie: as rows along the summed dimension, or turned over, B as K
// rows of N and A as K rows of M (the gradients' products: dx = dy w, dw = dy^T x)
enum Layout { kRows, kTurnB, kTurnBoth };

// What becomes of the sums: times a number, they are C; or, gated, C (M x n) = act(A G^T) * (A U^T), B given as the n
// rows of G and then the n of U; or C = residual + drop(act(A B^T + bias)), whatever of these there is
enum Finish { kPlain, kGated, kFull };

// C (M x N) = A (M x K) B^T, rows `lda`, `ldb`, `ldc` elements apart, finished one way or another
struct ProductArgs {
  const void* A;
  const void* B;
  void* C;
  float* pre;   // gated: null, or both sums for the backward pass, (M x ldpre) in the product's order
  float* part;  // null, or what the k range is cut into slices for: (slices x M x ldpart) partial sums
                // in the product's order, which sum_parts turns into C; or, with words, a tile of
                // sums as the waves hold them for every workgroup, which finish it together
  unsigned long long* words;  // big tiles: null, or one for every tile, kWordStride apart, whatever is in them
  unsigned long long token;   // this launch's, a multiple of eight (meet_arrive)
  int M, N, K;  // N: columns of C
  int lda, ldb, ldc, ldpre, ldpart;
  Finish finish;
  float scale;  // plain: of the sums
  int act;
  int tiles_m, tiles_n, slices, polls;  // polls: looks at a tile's other slice before leaving it a share
  // full alone
  const void* bias;      // null, or N elements
  const void* residual;  // null, or rows ldr elements apart
  unsigned short* slopes;  // null, or act' of the sums for the backward pass, rows ldslopes apart
  int ldr, ldslopes;
  bool slope_steps;      // their form (gated_act.hpp)
  DropArgs drop;
};

typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <bool BF>
__device__ __forceinline__ f4 product_mfma(i4 a, i4 b, f4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// four sums rounded to nearest
template <bool BF>
__device__ __forceinline__ i2 product_round(f4 v) {
  if constexpr (BF)
    return __builtin_bit_cast(i2, (b4){(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]});
  else
    return __builtin_bit_cast(i2, (h4){(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]});
}

// four elements of memory
template <bool BF>
__device__ __forceinline__ f4 widen4(i2 v) {
  if constexpr (BF) {
    const unsigned lo = (unsigned)v[0], hi = (unsigned)v[1];
    return (f4){__builtin_bit_cast(float, lo << 16), __builtin_bit_cast(float, lo & 0xffff0000u),
                __builtin_bit_cast(float, hi << 16), __builtin_bit_cast(float, hi & 0xffff0000u)};
  } else {
    const h4 h = __builtin_bit_cast(h4, v);
    return (f4){(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
  }
}

template <int ACT>
__device__ __forceinline__ f4 act4(f4 v) {
  return (f4){act_value<ACT>(v[0]), act_value<ACT>(v[1]), act_value<ACT>(v[2]), act_value<ACT>(v[3])};
}
// ... and their slopes as the backward pass takes them; STEPS: in steps alone
template <bool BF, int ACT, bool STEPS>
__device__ __forceinline__ f4 act4(f4 v, i2* slopes) {
  f4 s;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    float slope;
    v[e] = act_value_slope<ACT>(v[e], &slope);
    s[e] = slope;
  }
#pragma unroll
  for (int h = 0; h < 2; h++)
    (*slopes)[h] = (int)(STEPS ? slope_step_codes(s[2 * h], s[2 * h + 1]) : slope_codes<BF>(s[2 * h], s[2 * h + 1]));
  return v;
}
__device__ __forceinline__ f4 drop4(f4 v, i2 bits, const DropArgs& a) {
  return (f4){drop_one(v[0], bits, 0, a), drop_one(v[1], bits, 1, a), drop_one(v[2], bits, 2, a),
              drop_one(v[3], bits, 3, a)};
}

// the random bits of four columns of a row of C, of which their group of eight has as many again
__device__ __forceinline__ i2 own_bits(const ProductArgs& p, const DropKey& key, int row, int col) {
  const i4 w = drop_bits((unsigned long long)(unsigned)row * (unsigned)(p.N >> 3) + (unsigned)(col >> 3), key);
  return col & 4 ? (i2){w[2], w[3]} : (i2){w[0], w[1]};
}

// kFull, four columns of a row of C by themselves: where a lane has no others of their group of
// eight, and makes its bits alone.  Bias and residual are fetched ahead of the sums.
struct FullOperands {
  i2 bias, residual;
  __device__ __forceinline__ void fetch(const ProductArgs& p, int row, int col) {
    if (p.bias) bias = *(const i2*)((const half_t*)p.bias + col);
    if (p.residual) residual = *(const i2*)((const half_t*)p.residual + (size_t)row * p.ldr + col);
  }
};
template <bool BF>
__device__ __forceinline__ void finish_full(const ProductArgs& p, int row, int col, f4 v, const FullOperands& o) {
  if (p.bias) v += widen4<BF>(o.bias);
  if (p.act != kActNone) {
    i2 slopes;
    if (p.slope_steps)
      v = p.act == kActGelu ? act4<BF, kActGelu, true>(v, &slopes) : act4<BF, kActSilu, true>(v, &slopes);
    else
      v = p.act == kActGelu ? act4<BF, kActGelu, false>(v, &slopes) : act4<BF, kActSilu, false>(v, &slopes);
    if (p.slopes) *(i2*)(p.slopes + (size_t)row * p.ldslopes + col) = slopes;
  }
  if (p.drop.below) v = drop4(v, own_bits(p, DropKey(p.drop), row, col), p.drop);
  if (p.residual) v += widen4<BF>(o.residual);
  *(i2*)((half_t*)p.C + (size_t)row * p.ldc + col) = product_round<BF>(v);
}

__device__ __forceinline__ f4 act_mul4(f4 g, f4 u, int act) {
  return (f4){act_mul(g[0], u[0], act), act_mul(g[1], u[1], act), act_mul(g[2], u[2], act), act_mul(g[3], u[3], act)};
}

// Gated, the product's columns are gates and ups in turns of sixteen, an MFMA operand each, so
// that neighbouring operands of a wave hold a gate's sum and its partner's in the same lane and
// register: nothing is exchanged.  The order exists in the addresses of B's rows alone.  Column
// `col`, counted from `first` (a multiple of 32): its row of B as an offset in elements from
// row first / 2 of G.  Rows past the last repeat it (their columns are not stored).
__device__ __forceinline__ int gated_row(int first, int col, int n, int ldb) {
  const int at = first + col;
  int row = ((at >> 5) << 4) + (at & 15);
  if (row >= n) row = n - 1;
  return (row - (first >> 1)) * ldb + (at & 16 ? n * ldb : 0);
}

// where column `col` of C has its gate's sum in a row of `pre`; its partner's is 16 further on
__host__ __device__ __forceinline__ int pre_col(int col) { return ((col >> 4) << 5) + (col & 15); }

// columns of the product, which are C's, or gates and ups
__host__ __device__ __forceinline__ int product_columns(int n, bool gated) { return gated ? (n + 15) / 16 * 32 : n; }

// Tiles: rows x columns of the product.  256 columns and 160, 192, 224 or 256 rows are
// ff_big.hpp's, 16 and 32 columns of products of up to kProductRows rows ff_rows.hip's, the others
// ff_tiles.hip's.
struct FfTile {
  int rows, cols;
};
constexpr int kProductRows = 64;
constexpr int kSlicesMost = 8;  // of the k range
constexpr int kWordStride = 8;  // a tile's slices meet in a cache line of their own
// bytes of a big tile's sums
constexpr size_t big_sums(int rows) { return (size_t)rows * 256 * 4; }
constexpr bool big_tile(const FfTile& t) { return t.cols == 256 && t.rows >= 160; }
// a tile's workgroup
constexpr int tile_threads(const FfTile& t) { return t.cols <= 64 || big_tile(t) ? 256 : 512; }
constexpr long long kLaunchThreads = 0xffffffffLL;  // of all workgroups of a launch
hipError_t configure_product_tiles();
hipError_t configure_product_big_f16();
hipError_t configure_product_big_bf16();
hipError_t configure_product_rows();
// launches of any kind; bf: bfloat16 operands
void launch_product_tiles(ProductArgs a, const FfTile& t, Layout layout, bool bf, hipStream_t stream);
void launch_product_big_f16(const ProductArgs& a, int rows, Layout layout, hipStream_t stream);
void launch_product_big_bf16(const ProductArgs& a, int rows, Layout layout, hipStream_t stream);
void launch_product_rows(const ProductArgs& a, int blocks, bool bf, hipStream_t stream);  // of 16 columns
void launch_sum_parts(const ProductArgs& a, bool bf, hipStream_t stream);

}  // namespace w4a16
