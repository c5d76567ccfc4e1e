// What the dense products of the feed-forward block share: their arguments, the two 16-bit
// types, and the gated column order.
#pragma once
#include <hip/hip_runtime.h>

#include "buffer_loads.hpp"
#include "f16_dense.hpp"
#include "gated_act.hpp"
#include "w4a16_common.hpp"

namespace w4a16 {

// How the operands of a product lie: as rows along the summed dimension, or turned over, B as K
// rows of N and A as K rows of M (the gradients' products: dx = dy w, dw = dy^T x)
enum Layout { kRows, kTurnB, kTurnBoth };

// C (M x N) = A (M x K) B^T, rows `lda`, `ldb`, `ldc` elements apart; or, gated, C (M x n) =
// act(A G^T) * (A U^T), B given as the n rows of G and then the n of U.
struct ProductArgs {
  const void* A;
  const void* B;
  void* C;
  float* pre;   // gated: null, or both sums for the backward pass, (M x ldpre) in the product's order
  float* part;  // null, or what the k range is cut into slices for: (slices x M x ldpart) partial sums
                // in the product's order, which sum_parts turns into C
  int M, N, K;  // N: columns of C
  int lda, ldb, ldc, ldpre, ldpart;
  int act;  // kActNone: not gated
  int tiles_m, tiles_n, slices;
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
// ff_big.hip's, 16 and 32 columns, of up to kProductRows rows, ff_rows.hip's, the others
// ff_tiles.hip's.
struct FfTile {
  int rows, cols;
};
constexpr int kProductRows = 64;
constexpr int kSlicesMost = 8;  // of the k range
inline bool big_tile(const FfTile& t) { return t.cols == 256 && t.rows >= 160; }
inline bool few_tile(const FfTile& t) { return t.cols <= 32; }
hipError_t configure_product_tiles();
hipError_t configure_product_big();
hipError_t configure_product_rows();
// launches of any kind; bf: bfloat16 operands
void launch_product_tiles(ProductArgs a, const FfTile& t, Layout layout, bool bf, hipStream_t stream);
void launch_product_big(ProductArgs a, int rows, Layout layout, bool bf, hipStream_t stream);
void launch_product_rows(const ProductArgs& a, int blocks, bool bf, hipStream_t stream);  // of 16 columns
void launch_sum_parts(const ProductArgs& a, bool bf, hipStream_t stream);

}  // namespace w4a16
