// What the product tiles of ff_tiles.hip and ff_big.hpp share: where a tile's operands lie and
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
  int m0, n0, slice, tile;
  __device__ __forceinline__ TileAt(const ProductArgs& p, int tm_rows, int tn_cols) {
    const int tiles = p.tiles_m * p.tiles_n;
    const int work = xcd_work_index((int)blockIdx.x, tiles * p.slices);
    slice = work / tiles;
    tile = work - slice * tiles;
    int tm, tn;
    dn_tile_coord(tile, p.tiles_m, p.tiles_n, &tm, &tn);
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

// 16-byte pieces of ROWS rows (at smem) to `to`, which is C or of its shape, rows below `rows`, columns
// below `cols`
template <int ROWS, int COLS, bool GATED, int THREADS, class RowOf>
__device__ __forceinline__ void store_rows(void* to, int ld, const char* smem, int m0, int c0, int rows, int cols,
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
                                  (i4*)((half_t*)to + (size_t)(m0 + m) * ld + c0 + 8 * c));
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

// The 128 bits of a group of eight columns are those of two lanes sixteen apart, each with four of
// them.  Of a pair of operands' two groups the even lane group makes the first one's, the odd one the
// second's, and they swap what is the other's: one generator's run for eight elements.  `row`, `col`: of C
// and the first operand's.
__device__ __forceinline__ void full_bits(const ProductArgs& p, const DropKey& key, int row, int col, int kg, i2* first,
                                          i2* second) {
  const int at = col - 4 * kg + (kg & 1 ? 16 : 0) + 8 * (kg >> 1);
  const i4 w = drop_bits((unsigned long long)(unsigned)row * (unsigned)(p.N >> 3) + (unsigned)(at >> 3), key);
#if defined(__HIP_DEVICE_COMPILE__)
  // (the odd rows of sixteen lanes of one with the even rows of the other)
  const auto a = __builtin_amdgcn_permlane16_swap((unsigned)w[0], (unsigned)w[2], false, false);
  const auto b = __builtin_amdgcn_permlane16_swap((unsigned)w[1], (unsigned)w[3], false, false);
  *first = (i2){(int)a[0], (int)b[0]};
  *second = (i2){(int)a[1], (int)b[1]};
#else
  *first = *second = (i2){w[0], w[1]};
#endif
}

// kFull: what a wave brings to the tile's LDS image, of NI row blocks and NJ operands, from their sums v.
// `out`: this lane's row of the image in the first block, `slopes_at` bytes further on that of the slopes
// (stored from the registers, 8 bytes of a row a lane: 2048 x 10752 x 4096 174 us, so 169); m, col:
// its row and first column of the tile, of which rows x cols are there.  Bias and residual, fetched ahead,
// are past them the last ones, and are not stored.  (The bias ahead of the residual, and of the main loop: loads come
// back in order, and what waits for a bias behind a residual waits for both.)
//
// One pass over the registers for each of what there may be: a branch for each of them at every
// operand spreads what a call executes over 127 KB of instructions, twice the cache that two compute
// units share, and took 8192 x 4096 x 4096 with a bias from 212 us to 232.
template <int NJ>
__device__ __forceinline__ void fetch_bias(const ProductArgs& p, int n0, int col, int cols, i2 (&bias)[NJ]) {
  if (p.bias)
    for_each<NJ>([&](auto J) {
      constexpr int j = decltype(J)::value;
      bias[j] = *(const i2*)((const half_t*)p.bias + n0 + min(col + 16 * j, cols - 4));
    });
}
template <int NI, int NJ>
__device__ __forceinline__ void fetch_residual(const ProductArgs& p, int m0, int n0, int m, int col, int rows, int cols,
                                               i2 (&residual)[NI][NJ]) {
  if (p.residual)
    for_each<NI>([&](auto I) {
      constexpr int i = decltype(I)::value;
      const half_t* const row = (const half_t*)p.residual + (size_t)(m0 + min(m + 16 * i, rows - 1)) * p.ldr + n0;
      for_each<NJ>([&](auto J) {
        constexpr int j = decltype(J)::value;
        residual[i][j] = *(const i2*)(row + min(col + 16 * j, cols - 4));
      });
    });
}
template <bool BF, int NI, int NJ, int PITCH>
__device__ __forceinline__ void put_full(const ProductArgs& p, char* out, int slopes_at, int m0, int n0, int m, int col,
                                         int kg, const i2 (&bias)[NJ], const i2 (&residual)[NI][NJ], f4 (&v)[NI][NJ]) {
  if (p.bias)
    for_each<NJ>([&](auto J) {
      constexpr int j = decltype(J)::value;
      const f4 add = widen4<BF>(bias[j]);
      for_each<NI>([&](auto I) { v[decltype(I)::value][j] += add; });
    });
  const auto activate = [&](auto Act) {
    constexpr int act = decltype(Act)::value;
    for_each<NI>([&](auto I) {
      for_each<NJ>([&](auto J) {
        constexpr int i = decltype(I)::value, j = decltype(J)::value;
        v[i][j] = act4<act>(v[i][j]);
      });
    });
  };
  const auto activate_slopes = [&](auto Act, auto Steps) {
    constexpr int act = decltype(Act)::value;
    for_each<NI>([&](auto I) {
      for_each<NJ>([&](auto J) {
        constexpr int i = decltype(I)::value, j = decltype(J)::value;
        i2 slopes;
#if defined(__HIP_DEVICE_COMPILE__)
        // (what both forms have in common stays behind the branch to either: ahead of it, it spills)
        if constexpr (decltype(Steps)::value) asm("" : "+v"(v[i][j]));
#endif
        v[i][j] = act4<BF, act, decltype(Steps)::value>(v[i][j], &slopes);
        *(i2*)(out + slopes_at + 16 * i * PITCH + 2 * (col + 16 * j)) = slopes;
        // (four operands by themselves: more at once take registers that the big tiles do not have)
        if constexpr (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      });
    });
  };
  const auto activated = [&](auto Act) {
    if (!p.slopes)
      activate(Act);
    else if (p.slope_steps)
      activate_slopes(Act, std::true_type{});
    else
      activate_slopes(Act, std::false_type{});
  };
  if (p.act == kActGelu)
    activated(std::integral_constant<int, kActGelu>{});
  else if (p.act == kActSilu)
    activated(std::integral_constant<int, kActSilu>{});
  if (p.drop.below) {
    const DropKey key(p.drop);
    for_each<NI>([&](auto I) {
      constexpr int i = decltype(I)::value;
      const int row = m0 + m + 16 * i;
      for_each<NJ / 2>([&](auto J) {
        constexpr int j = 2 * decltype(J)::value;
        i2 first, second;
        full_bits(p, key, row, n0 + col + 16 * j, kg, &first, &second);
        v[i][j] = drop4(v[i][j], first, p.drop);
        v[i][j + 1] = drop4(v[i][j + 1], second, p.drop);
      });
      if constexpr (NJ % 2)  // (one without a partner)
        v[i][NJ - 1] = drop4(v[i][NJ - 1], own_bits(p, key, row, n0 + col + 16 * (NJ - 1)), p.drop);
    });
  }
  if (p.residual)
    for_each<NI * NJ>([&](auto At) {
      constexpr int i = decltype(At)::value / NJ, j = decltype(At)::value % NJ;
      v[i][j] += widen4<BF>(residual[i][j]);
    });
  for_each<NI * NJ>([&](auto At) {
    constexpr int i = decltype(At)::value / NJ, j = decltype(At)::value % NJ;
    *(i2*)(out + 16 * i * PITCH + 2 * (col + 16 * j)) = product_round<BF>(v[i][j]);
  });
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
