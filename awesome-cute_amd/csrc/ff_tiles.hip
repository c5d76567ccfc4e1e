// Dense products in fp16 or bfloat16 by tiles, with a gated epilogue: more than kProductRows
// rows, and what ff_rows.hip does not take.  Operands, slabs, swizzle, order of MFMA operands
// and the loops are those of f16_streamk.hip and f16_tiles.hip, where they are explained and
// measured; here
//   - rows of A, B and C may lie further apart than they are long,
//   - C may have any number of columns that is a multiple of 8, and k any such depth: what is
//     past the end of a row in its last 64-deep stage is requested at an offset past
//     everything, and so reads as zeros, in A and in B,
//   - gated, a tile's columns are gates and ups in turns of sixteen (gated_row), and its
//     epilogue writes act(g) u, for the backward pass both sums as well.
//
// What bounds them: as there, the board's power for large products of 256 x 256 tiles, the way
// into LDS for the others.
#include <hip/hip_runtime.h>

#include "ff_products.hpp"

namespace w4a16 {

namespace {

enum Form { kPlain, kGated, kGatedPre };

// ROWS x COLS tile of 16-bit results on its way through LDS: a row holds COLS columns, or,
// gated, COLS / 2
template <int COLS, Form FORM>
constexpr int out_pitch() {
  return (FORM == kPlain ? 2 * COLS : COLS) + 16;
}

// 16-byte pieces of ROWS rows (of the tile from `row0` on, at smem) to C, rows below `rows`,
// columns below `cols`
template <int ROWS, int COLS, Form FORM, int THREADS, class RowOf>
__device__ __forceinline__ void store_rows(const ProductArgs& p, const char* smem, int m0, int c0, int rows, int cols,
                                           RowOf row_of) {
  constexpr int kPitch = out_pitch<COLS, FORM>();
  constexpr int kPieces = (FORM == kPlain ? COLS : COLS / 2) / 8;
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
// times as far off as the products' own roundings do, for 35 us less of 1030 (2048 x 2 x 10752
// x 4096, forward and backward) -- and in the product's order, in which a gate's sixteen
// columns and its partner's fill a cache line of a row.
template <int COLS, Form FORM, bool BF>
__device__ __forceinline__ void put(const ProductArgs& p, char* image, int m0, int n0, int m, int col, int rows,
                                    int cols, f4 v, f4 next) {
  char* const row = image;
  if constexpr (FORM == kPlain) {
    *(i2*)(row + 2 * col) = product_round<BF>(v);
  } else {
    const int at = ((col >> 5) << 4) + (col & 15);  // (col: 16 of gates, 16 of ups)
    *(i2*)(row + 2 * at) = product_round<BF>(act_mul4(v, next, p.act));
    if (FORM == kGatedPre && m < rows && at < cols) {
      float* const pre = p.pre + (size_t)(m0 + m) * p.ldpre + n0 + col;
      __builtin_nontemporal_store(v, (f4*)pre);
      __builtin_nontemporal_store(next, (f4*)(pre + 16));
    }
  }
}

__device__ __forceinline__ unsigned rows_bytes(int rows, int ld, int k) {
  return (unsigned)(rows - 1) * (unsigned)ld * 2u + (unsigned)k * 2u;
}

// the resource of a tile's rows of B, and how many columns of C it computes
template <Form FORM>
__device__ __forceinline__ const char* b_base(const ProductArgs& p, int n0, int tile_cols, unsigned* bytes, int* cols) {
  if constexpr (FORM == kPlain) {
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
template <Form FORM>
__device__ __forceinline__ int b_offset(const ProductArgs& p, int n0, int c, int cols) {
  if constexpr (FORM == kPlain) return (c < cols ? c : cols - 1) * p.ldb * 2;
  return gated_row(n0, c, p.N, p.ldb) * 2;
}

// TM x TN tiles, WM x WN waves
template <int TM, int TN, int WM, int WN, int RING, Form FORM>
struct FfShape {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kRB = TM / 16 / WM, kNJ = TN / 16 / WN;  // operands of a wave per k step
  static constexpr int kOps = 2 * (kRB + kNJ);                  // ... per stage
  static constexpr int kTA = (TM / 8 + kWaves - 1) / kWaves, kTB = TN / 8 / kWaves;  // loads per wave and slab
  static constexpr int kSlabA = kTA * kWaves * 1024, kSlab = kSlabA + TN * 128;
  static constexpr int kLoads = kTA + kTB;
  static constexpr int kRingBytes = RING * kSlab, kTileBytes = TM * out_pitch<TN, FORM>();
  static constexpr int kLds = kRingBytes > kTileBytes ? kRingBytes : kTileBytes;
  static_assert(kTB * 8 * kWaves == TN && TM % (16 * WM) == 0 && TN % (16 * WN) == 0, "whole blocks");
  static_assert(FORM == kPlain || kNJ % 2 == 0, "a gate's operand and its partner's in one wave");
  static_assert(kLds <= 160 * 1024 - 256, "LDS of a compute unit");
};

template <int N>
__device__ __forceinline__ void ff_landed(i4 (&v)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#pragma unroll
  for (int i = 4; i < N; i++) asm volatile("" : "+v"(v[i]));
#endif
}
template <int COUNT>
__device__ __forceinline__ void ff_read_blocks(unsigned at, i4* v) {
  if constexpr (COUNT > 0) {
    ff_read_blocks<COUNT - 1>(at, v);
    read_lds16<2048 * (COUNT - 1)>(at, v[COUNT - 1]);
  }
}

}  // namespace

// One barrier per 64-deep stage; the loop is dense_tile_kernel's (f16_tiles.hip).
template <bool BF, Form FORM, int TM, int TN, int WM, int WN, int RING>
__global__ __launch_bounds__(64 * WM * WN) void product_tile_kernel(ProductArgs p) {
  using Sh = FfShape<TM, TN, WM, WN, RING, FORM>;
  constexpr int RB = Sh::kRB, NJ = Sh::kNJ, TA = Sh::kTA, TB = Sh::kTB;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // Sh::kLds
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int kg = lane >> 4;
  const int nu = lane & 15;
  const int wm = wave / WN;
  const int wn = wave % WN;

  int tm, tn;
  dn_tile_coord(xcd_work_index((int)blockIdx.x, p.tiles_m * p.tiles_n), p.tiles_m, p.tiles_n, &tm, &tn);
  const int m0 = TM * tm, n0 = TN * tn;
  const int rows = min(TM, p.M - m0);
  const __amdgpu_buffer_rsrc_t rA =
      make_rsrc((const char*)p.A + (size_t)m0 * p.lda * 2, rows_bytes(rows, p.lda, p.K));
  unsigned b_bytes;
  int cols;
  const char* const b_at = b_base<FORM>(p, n0, TN, &b_bytes, &cols);
  const __amdgpu_buffer_rsrc_t rB = make_rsrc(b_at, b_bytes);

  const int stages = (p.K + kDnStageK - 1) / kDnStageK;
  int a_src[TA], b_src[TB];
  int past;  // this lane's 16 bytes of a row in the last stage: kOob where the row has ended
  {
    const int r8 = lane >> 3, c = (lane & 7) ^ r8;
#pragma unroll
    for (int t = 0; t < TA; t++) {
      const int r = 8 * (TA * wave + t) + r8;
      a_src[t] = r >= TM ? kOob : (r < rows ? r : rows - 1) * p.lda * 2 + 16 * c;
    }
#pragma unroll
    for (int t = 0; t < TB; t++) b_src[t] = b_offset<FORM>(p, n0, 8 * (TB * wave + t) + r8, cols) + 16 * c;
    past = (stages - 1) * kDnStageK + 8 * c < p.K ? 0 : kOob;
  }

  auto issue_slab = [&](int s, int slot) {
    const int inv = s < stages - 1 ? 0 : s == stages - 1 ? past : kOob;
    const int at = s * (kDnStageK * 2);
    char* const base = smem + slot * Sh::kSlab;
#pragma unroll
    for (int t = 0; t < TA; t++) load_to_lds16(rA, base + (TA * wave + t) * 1024, a_src[t] | inv, at);
#pragma unroll
    for (int t = 0; t < TB; t++)
      load_to_lds16(rB, base + Sh::kSlabA + (TB * wave + t) * 1024, b_src[t] | inv, at);
  };

  unsigned a_rd[2], b_rd[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const unsigned sw = 16 * ((4 * h + kg) ^ (nu & 7));
    a_rd[h] = (unsigned)(size_t)smem + (16 * RB * wm + nu) * 128 + sw;
    b_rd[h] = (unsigned)(size_t)smem + Sh::kSlabA + (16 * NJ * wn + nu) * 128 + sw;
  }
  auto read = [&](i4 (&o)[Sh::kOps], unsigned slab) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      ff_read_blocks<NJ>(b_rd[h] + slab, o + h * (RB + NJ));
      ff_read_blocks<RB>(a_rd[h] + slab, o + h * (RB + NJ) + NJ);
    }
  };

  f4 acc[RB][NJ];
#pragma unroll
  for (int i = 0; i < RB; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[i][j] = (f4){0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](i4 (&o)[Sh::kOps]) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
          acc[i][j] = product_mfma<BF>(o[h * (RB + NJ) + j], o[h * (RB + NJ) + NJ + i], acc[i][j]);
  };

  // Every slot requested; slab 0 landed (loads complete in order), its operands read.
  // Between the reads into a set of registers and the wait that names them stand the MFMAs
  // of the other set and nothing else.
  i4 even[Sh::kOps], odd[Sh::kOps];
#pragma unroll
  for (int r = 0; r < RING; r++) issue_slab(r, r);
  __builtin_amdgcn_s_waitcnt(vmcnt((RING - 1) * Sh::kLoads));
  __builtin_amdgcn_s_barrier();
  read(even, 0);
  ff_landed(even);
  int slot = 0;
  auto stage = [&](int s, i4 (&cur)[Sh::kOps], i4 (&next)[Sh::kOps]) {
    __builtin_amdgcn_s_waitcnt(vmcnt((RING - 2) * Sh::kLoads));
    __builtin_amdgcn_s_barrier();
    const int slot_next = slot == RING - 1 ? 0 : slot + 1;
    __builtin_amdgcn_sched_barrier(0);
    read(next, slot_next * Sh::kSlab);
    issue_slab(s + RING, slot);
    __builtin_amdgcn_sched_barrier(0);
    multiply(cur);
    __builtin_amdgcn_sched_barrier(0);
    ff_landed(next);
    slot = slot_next;
  };
  int s = 0;
  for (; s + 1 < stages; s += 2) {
    stage(s, even, odd);
    stage(s + 1, odd, even);
  }
  if (s < stages) multiply(even);
  // nothing of the ring may still be on its way when LDS is reused
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  // a lane holds, per (i, j), row 16i + nu and four consecutive columns; the tile leaves
  // through LDS as whole rows
  char* const out = smem + (16 * RB * wm + nu) * out_pitch<TN, FORM>();
#pragma unroll
  for (int i = 0; i < RB; i++)
#pragma unroll
    for (int j = 0; j < NJ; j += FORM == kPlain ? 1 : 2)
      put<TN, FORM, BF>(p, out + 16 * i * out_pitch<TN, FORM>(), m0, n0, 16 * RB * wm + 16 * i + nu,
                        16 * NJ * wn + 16 * j + 4 * kg, rows, cols, acc[i][j], acc[i][FORM == kPlain ? j : j + 1]);
  __syncthreads();
  store_rows<TM, TN, FORM, Sh::kThreads>(p, smem, m0, FORM == kPlain ? n0 : n0 >> 1, rows, cols,
                                         [](int r) { return r; });
}

namespace {

struct BigShape {
  static constexpr int kSlabA = 256 * 128, kSlab = 2 * kSlabA;
  static constexpr int kTA = 8, kTB = 8;  // load instructions per wave and slab
  static constexpr int kLds = 2 * kSlab;  // (half a tile of results is less)
  static_assert(128 * out_pitch<256, kPlain>() <= kLds, "");
};

}  // namespace

// 256 x 256 tiles by four waves of 128 x 128, the main loop one assembly statement
// (gen_dense.py); k is a multiple of 64.
template <bool BF, Form FORM>
__global__ __launch_bounds__(256) void product_big_kernel(ProductArgs p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // BigShape::kLds
  constexpr int TA = BigShape::kTA, TB = BigShape::kTB;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int kg = lane >> 4;
  const int nu = lane & 15;
  const int wm = wave >> 1;  // 128-row half of the tile
  const int wn = wave & 1;   // 128-column half

  int tm, tn;
  dn_tile_coord(xcd_work_index((int)blockIdx.x, p.tiles_m * p.tiles_n), p.tiles_m, p.tiles_n, &tm, &tn);
  const int m0 = tm * 256, n0 = tn * 256;
  const int rows = min(256, p.M - m0);
  unsigned b_bytes;
  int cols;
  const char* const b_at = b_base<FORM>(p, n0, 256, &b_bytes, &cols);
  i4 ra_words = rsrc_words((const char*)p.A + (size_t)m0 * p.lda * 2, rows_bytes(rows, p.lda, p.K));
  i4 rb_words = rsrc_words(b_at, b_bytes);
  int src[TA + TB];
  {
    const int r8 = lane >> 3, c = (lane & 7) ^ r8;
#pragma unroll
    for (int t = 0; t < TA; t++) {
      const int r = 8 * (TA * wave + t) + r8;
      src[t] = (r < rows ? r : rows - 1) * p.lda * 2 + 16 * c;
    }
#pragma unroll
    for (int t = 0; t < TB; t++) src[TA + t] = b_offset<FORM>(p, n0, 8 * (TB * wave + t) + r8, cols) + 16 * c;
  }
  const int slabs = p.K / kDnStageK;
  int s_at = 0;  // byte offset of the next slab to request
  const int lds = (int)(size_t)smem;
  const int lds_a = lds + wave * TA * 1024, lds_b = lds + BigShape::kSlabA + wave * TB * 1024;
  int a_rd[4], b_rd[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int at = lds + j / 2 * BigShape::kSlab + nu * 128 + 16 * ((4 * (j % 2) + kg) ^ (nu & 7));
    a_rd[j] = at + 128 * wm * 128;
    b_rd[j] = at + BigShape::kSlabA + 128 * wn * 128;
  }

  f4 acc[8][8];
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (BF) {
#include "bf16_dense_256x256.inc"
  } else {
#include "f16_dense_256x256.inc"
  }
#else  // the host pass only needs the launch stub
  (void)slabs, (void)s_at, (void)lds_a, (void)lds_b, (void)src;
  (void)a_rd, (void)b_rd, (void)ra_words, (void)rb_words;
  for (auto& r : acc)
    for (auto& v : r) v = (f4){0.f, 0.f, 0.f, 0.f};
#endif
  // The tile leaves through LDS in two halves, 64 rows of either wave row each; where both
  // have room, the second is written to LDS while the first is on its way to memory.
  constexpr int kPitch = out_pitch<256, FORM>();
  constexpr bool kBoth = 256 * kPitch <= BigShape::kLds;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    char* const base = smem + (kBoth ? half * 128 * kPitch : 0);
    if (half == 0 || !kBoth) __syncthreads();  // (nothing is on its way into LDS, and nobody reads it)
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int o = 0; o < 8; o += FORM == kPlain ? 1 : 2)
        put<256, FORM, BF>(p, base + (64 * wm + 16 * i + nu) * kPitch, m0, n0, 128 * wm + 16 * (4 * half + i) + nu,
                           128 * wn + 16 * o + 4 * kg, rows, cols, acc[4 * half + i][o],
                           acc[4 * half + i][FORM == kPlain ? o : o + 1]);
    __syncthreads();
    store_rows<128, 256, FORM, 256>(p, base, m0, FORM == kPlain ? n0 : n0 >> 1, rows, cols,
                                    [&](int r) { return (r >> 6) * 128 + half * 64 + (r & 63); });
  }
}

namespace {

// calls f(kernel, LDS bytes, threads) for a tile, a form and a type
template <bool BF, Form FORM, class F>
void with_tile(const FfTile& t, F f) {
#define FF_TILE(TM, TN, WM, WN, RING) \
  if (t.rows == TM && t.cols == TN)   \
  return f(product_tile_kernel<BF, FORM, TM, TN, WM, WN, RING>, FfShape<TM, TN, WM, WN, RING, FORM>::kLds, 64 * WM * WN)
  FF_TILE(64, 64, 2, 2, 4);
  FF_TILE(64, 128, 2, 4, 6);
  FF_TILE(96, 128, 2, 4, 4);
  FF_TILE(128, 128, 2, 4, 4);
  FF_TILE(96, 256, 2, 4, 3);
  FF_TILE(128, 256, 2, 4, 3);
#undef FF_TILE
  if (t.rows == 256 && t.cols == 256) return f(product_big_kernel<BF, FORM>, BigShape::kLds, 256);
}
template <class F>
void with_product(const FfTile& t, bool bf, Form form, F f) {
  if (bf) {
    if (form == kPlain) return with_tile<true, kPlain>(t, f);
    if (form == kGated) return with_tile<true, kGated>(t, f);
    return with_tile<true, kGatedPre>(t, f);
  }
  if (form == kPlain) return with_tile<false, kPlain>(t, f);
  if (form == kGated) return with_tile<false, kGated>(t, f);
  return with_tile<false, kGatedPre>(t, f);
}

}  // namespace

hipError_t configure_product_tiles() {
  hipError_t e = hipSuccess;
  for (const int rows : {64, 96, 128, 256})
    for (const int cols : {64, 128, 256})
      for (const bool bf : {false, true})
        for (const Form form : {kPlain, kGated, kGatedPre})
          with_product({rows, cols}, bf, form, [&](auto kernel, int lds, int) {
            if (e == hipSuccess)
              e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
          });
  return e;
}

void launch_product_tiles(ProductArgs a, const FfTile& t, bool bf, hipStream_t stream) {
  const int columns = a.act == kActNone ? a.N : 2 * ((a.N + 15) / 16 * 16);
  a.tiles_m = ceil_div(a.M, t.rows);
  a.tiles_n = ceil_div(columns, t.cols);
  const Form form = a.act == kActNone ? kPlain : a.pre ? kGatedPre : kGated;
  with_product(t, bf, form, [&](auto kernel, int lds, int threads) {
    hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n), dim3(threads), lds, stream, a);
  });
}

}  // namespace w4a16
