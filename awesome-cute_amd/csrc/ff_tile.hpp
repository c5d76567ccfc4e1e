// What the product tiles of ff_tiles.hip and ff_big.hip share: where a tile's operands lie and
// how its results leave.
#pragma once
#include <hip/hip_runtime.h>

#include "ff_products.hpp"

namespace w4a16 {

// ---- operands.  By rows: a tile's rows along the summed dimension, as in f16_streamk.hip, 128
// bytes of each per 64-deep stage.  Turned over: 64 rows per stage, of all the tile's columns; a
// stage's window ends with its last row, so that what lies past the end of the sum reads as
// zeros, and the window moves on by its base, so that the sum may be any length.

// The tile of a workgroup: (tile, slice), the slices of one k range neighbours
struct TileAt {
  int m0, n0, slice;
  __device__ __forceinline__ TileAt(const ProductArgs& p, int tm_rows, int tn_cols) {
    const int tiles = p.tiles_m * p.tiles_n;
    const int work = xcd_work_index((int)blockIdx.x, tiles * p.slices);
    slice = work / tiles;
    int tm, tn;
    dn_tile_coord(work - slice * tiles, p.tiles_m, p.tiles_n, &tm, &tn);
    m0 = tm_rows * tm;
    n0 = tn_cols * tn;
  }
  // my stages [first, last) of all
  __device__ __forceinline__ int stage(const ProductArgs& p, int all, int more) const {
    return (int)((long long)(slice + more) * all / p.slices);
  }
};

// Turned over, sixteen columns of a row are 32 bytes, an MFMA operand's share of it.  Chunk c of
// row r sits at position c ^ turned_swizzle(r), so that the eight rows which half a wave reads
// together, r0 ... r0 + 3 and eight further on, meet no bank twice.
template <int COLS>
__host__ __device__ __forceinline__ int turned_swizzle(int r) {
  return COLS >= 128 ? (r & 3) | ((r >> 1) & 4) : ((r >> 1) & 1) | ((r >> 2) & 2);
}

__device__ __forceinline__ unsigned rows_bytes(int rows, int ld, int width) {
  return (unsigned)(rows - 1) * (unsigned)ld * 2u + (unsigned)width * 2u;
}

// ---- results

// ROWS x COLS tile of 16-bit results on its way through LDS: a row holds COLS columns, or,
// gated, COLS / 2
template <int COLS, bool GATED>
constexpr int out_pitch() {
  return (GATED ? COLS : 2 * COLS) + 16;
}

// 16-byte pieces of ROWS rows (at smem) to C, rows below `rows`, columns below `cols`
template <int ROWS, int COLS, bool GATED, int THREADS, class RowOf>
__device__ __forceinline__ void store_rows(const ProductArgs& p, const char* smem, int m0, int c0, int rows, int cols,
                                           RowOf row_of) {
  constexpr int kPitch = out_pitch<COLS, GATED>();
  constexpr int kPieces = (GATED ? COLS / 2 : COLS) / 8;
#pragma unroll 8
  for (int at = threadIdx.x; at < ROWS * kPieces; at += THREADS) {
    const int r = at / kPieces, c = at % kPieces;
    const int m = row_of(r);
    if (m < rows && 8 * c < cols)
      // nobody reads it again in this launch: keep it out of the way of A and B in L2
      __builtin_nontemporal_store(*(const i4*)(smem + r * kPitch + 16 * c),
                                  (i4*)((half_t*)p.C + (size_t)(m0 + m) * p.ldc + c0 + 8 * c));
  }
}

// What a lane puts into row `m` of the tile's LDS image, of operands j and (gated) j + 1 of a
// row block: their sums at column `col` of the product's tile.  The sums that the backward pass
// takes go to memory from here, in fp32 -- rounded to 16 bits they made the gradients 1.8
// times as far off as the products' own roundings do; they cost 17 us of a forward pass of 313 (2048
// x 2 x 10752 x 4096) and some 15 of a backward pass -- and in the product's order, in which a
// gate's sixteen columns and its partner's fill a cache line of a row.
template <int COLS, bool GATED, bool BF>
__device__ __forceinline__ void put(const ProductArgs& p, char* row, int m0, int n0, int m, int col, int rows, int cols,
                                    f4 v, f4 next) {
  if constexpr (!GATED) {
    *(i2*)(row + 2 * col) = product_round<BF>(v);
  } else {
    const int at = ((col >> 5) << 4) + (col & 15);  // (col: 16 of gates, 16 of ups)
    *(i2*)(row + 2 * at) = product_round<BF>(act_mul4(v, next, p.act));
    if (p.pre && m < rows && at < cols) {
      float* const pre = p.pre + (size_t)(m0 + m) * p.ldpre + n0 + col;
      __builtin_nontemporal_store(v, (f4*)pre);
      __builtin_nontemporal_store(next, (f4*)(pre + 16));
    }
  }
}
// ... and of a slice: the sums as they are (columns in the product's order)
__device__ __forceinline__ void put_part(const ProductArgs& p, int slice, int m, int col, int rows_end, int cols_end,
                                         f4 v) {
  if (m < rows_end && col < cols_end)
    *(f4*)(p.part + ((size_t)slice * p.M + m) * p.ldpart + col) = v;
}

// the rows of B by rows: the base of a tile's, and how many columns of C it computes
template <bool GATED>
__device__ __forceinline__ const char* b_base(const ProductArgs& p, int n0, int tile_cols, unsigned* bytes, int* cols) {
  if constexpr (!GATED) {
    *cols = min(tile_cols, p.N - n0);
    *bytes = rows_bytes(*cols, p.ldb, p.K);
    return (const char*)p.B + (size_t)n0 * p.ldb * 2;
  } else {
    *cols = min(tile_cols / 2, p.N - (n0 >> 1));
    *bytes = rows_bytes(2 * p.N - (n0 >> 1), p.ldb, p.K);
    return (const char*)p.B + (size_t)(n0 >> 1) * p.ldb * 2;
  }
}
// bytes from there to the row of column c of the tile (columns past the last repeat it)
template <bool GATED>
__device__ __forceinline__ int b_offset(const ProductArgs& p, int n0, int c, int cols) {
  if constexpr (!GATED) return (c < cols ? c : cols - 1) * p.ldb * 2;
  return gated_row(n0, c, p.N, p.ldb) * 2;
}

}  // namespace w4a16
