// Dense products in fp16 or bfloat16 by tiles of 160, 192, 224 or 256 rows x 256 columns: four
// waves, two by two, the main loop one assembly statement (gen_products.py).  Operands by rows
// or turned over, any depth, slices and the gated epilogue as in ff_tiles.hip.
//
// Bound: how evenly the tiles fill the compute units, hence the heights (777 x 2 x 5208 x 4160: 164
// tiles of 256 rows, 205 of 160), some 12 us of a tile outside its loop (the first slabs' way, and
// results that all compute units write at once), and in the loop the board's power.  bfloat16, operands
// from memory, us and TFLOP/s: 2048 x 2 x 10752 x 4096 296, 1220 (with the sums kept 313); its backward
// pass 2048 x 4096 x 21504 277, 1300, of which 14 the slices' sums, and 21504 x 4096 x 2048 307, 1170;
// 8192 x 4096 x 4096 205, 1340.  The matrix pipe is in use for 57 to 72 % of these.  Results past the
// caches or through them: level.
#include <hip/hip_runtime.h>

#include "ff_tile.hpp"

namespace w4a16 {

namespace {

template <int RB, Layout LAYOUT>
struct BigShape {
  static constexpr bool kTurnA = LAYOUT == kTurnBoth, kTurnedB = LAYOUT != kRows;
  static constexpr int kTM = 32 * RB;
  static constexpr int kTA = kTurnA ? 8 : RB, kTB = 8;  // load instructions per wave and slab
  static constexpr int kSlabA = kTA * 4 * 1024, kSlabB = 256 * 128;
  // the results leave in two halves: RB / 2 (rounded up) row blocks of either wave row, and the rest
  static constexpr int kHalf = (RB + 1) / 2;
  static constexpr int kOut = 32 * kHalf * out_pitch<256, false>();
  static constexpr int kRingA = 3 * (kSlabA + kSlabB) <= 160 * 1024 ? 3 : 2, kRingB = 3;  // slabs in LDS
  static constexpr int kRings = kRingA * kSlabA + kRingB * kSlabB;
  static constexpr int kLds = kRings > kOut ? kRings : kOut;
  static_assert(kLds <= 160 * 1024, "LDS of a compute unit");
};

}  // namespace

template <bool BF, Finish FINISH, Layout LAYOUT, int RB>
__global__ __launch_bounds__(256) void product_big_kernel(ProductArgs p) {
  constexpr bool GATED = FINISH == kGated;
  using Sh = BigShape<RB, LAYOUT>;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // Sh::kLds
  constexpr int TA = Sh::kTA, TB = Sh::kTB, TM = Sh::kTM;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int kg = lane >> 4;
  const int nu = lane & 15;
  const int wm = wave >> 1;  // half of the tile's rows
  const int wn = wave & 1;   // ... of its columns

  const TileAt at(p, TM, 256);
  const int m0 = at.m0, n0 = at.n0;
  const int rows = min(TM, p.M - m0);
  int cols = min(GATED ? 128 : 256, p.N - (GATED ? n0 >> 1 : n0));
  const int all = (p.K + kDnStageK - 1) / kDnStageK;
  const int first = at.stage(p, all, 0), end = at.stage(p, all, 1);
  const int slabs = end - first;
  const int last_k = end == all ? p.K - kDnStageK * (all - 1) : kDnStageK;  // k-values of my last slab

  // by rows: lane (r = lane / 8, c = lane % 8) fetches chunk c ^ r of a row; turned over: two rows
  // of 256 columns a load
  int src[TA + TB];
  i4 ra_words, rb_words;
  unsigned full_a, last_a, step_a, full_b, last_b, step_b;
  const int r8 = lane >> 3, c8 = (lane & 7) ^ r8;
  const int past = 8 * c8 < last_k ? 0 : kOob;  // this lane's k-values of a row, in my last slab
  const int r2 = lane >> 5, piece = lane & 31;
  if constexpr (Sh::kTurnA) {
    step_a = 128u * (unsigned)p.lda;
    full_a = rows_bytes(kDnStageK, p.lda, p.M - m0);
    last_a = rows_bytes(last_k, p.lda, p.M - m0);
    ra_words = rsrc_words((const char*)p.A + ((size_t)first * kDnStageK * p.lda + m0) * 2, full_a);
#pragma unroll
    for (int t = 0; t < TA; t++) {
      const int r = 2 * (TA * wave + t) + r2;
      src[t] = r * p.lda * 2 + 16 * (piece ^ (2 * turned_swizzle<256>(r)));
    }
  } else {
    step_a = kDnStageK * 2;
    full_a = rows_bytes(rows, p.lda, kDnStageK);
    last_a = rows_bytes(rows, p.lda, last_k);
    ra_words = rsrc_words((const char*)p.A + ((size_t)m0 * p.lda + (size_t)first * kDnStageK) * 2, full_a);
#pragma unroll
    for (int t = 0; t < TA; t++) {
      const int r = 8 * (TA * wave + t) + r8;
      src[t] = (r < rows ? r : rows - 1) * p.lda * 2 + 16 * c8;
    }
  }
  if constexpr (Sh::kTurnedB) {
    step_b = 128u * (unsigned)p.ldb;
    full_b = rows_bytes(kDnStageK, p.ldb, p.N - n0);
    last_b = rows_bytes(last_k, p.ldb, p.N - n0);
    rb_words = rsrc_words((const char*)p.B + ((size_t)first * kDnStageK * p.ldb + n0) * 2, full_b);
#pragma unroll
    for (int t = 0; t < TB; t++) {
      const int r = 2 * (TB * wave + t) + r2;
      src[TA + t] = r * p.ldb * 2 + 16 * (piece ^ (2 * turned_swizzle<256>(r)));
    }
  } else {
    unsigned b_bytes;
    const char* const b_at = b_base<GATED>(p, n0, 256, &b_bytes, &cols);
    step_b = kDnStageK * 2;
    full_b = b_bytes - (unsigned)p.K * 2u + kDnStageK * 2;
    last_b = full_b - 2u * (unsigned)(kDnStageK - last_k);
    rb_words = rsrc_words(b_at + (size_t)first * kDnStageK * 2, full_b);
#pragma unroll
    for (int t = 0; t < TB; t++) src[TA + t] = b_offset<GATED>(p, n0, 8 * (TB * wave + t) + r8, cols) + 16 * c8;
  }

  // LDS: where this wave's loads of slot 0 go, and where its operands of every slot are read
  const int lds = (int)(size_t)smem;
  const int lds_a = lds + wave * TA * 1024, lds_b = lds + Sh::kRingA * Sh::kSlabA + wave * TB * 1024;
  int a_rd[(Sh::kTurnA ? 8 : 2) * Sh::kRingA], b_rd[(Sh::kTurnedB ? 8 : 2) * Sh::kRingB];
  const int turned_at = (8 * kg + (nu >> 2)) * 512 + 8 * (nu & 3), swizzle = turned_swizzle<256>(8 * kg + (nu >> 2));
#pragma unroll
  for (int slot = 0; slot < Sh::kRingA; slot++) {
    const int slab = lds + slot * Sh::kSlabA;
    if constexpr (Sh::kTurnA) {
#pragma unroll
      for (int i = 0; i < 8; i++) a_rd[8 * slot + i] = slab + turned_at + 32 * ((RB * wm + i) ^ swizzle);
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++)
        a_rd[2 * slot + h] = slab + (16 * RB * wm + nu) * 128 + 16 * ((4 * h + kg) ^ (nu & 7));
    }
  }
#pragma unroll
  for (int slot = 0; slot < Sh::kRingB; slot++) {
    const int slab = lds + Sh::kRingA * Sh::kSlabA + slot * Sh::kSlabB;
    if constexpr (Sh::kTurnedB) {
#pragma unroll
      for (int o = 0; o < 8; o++) b_rd[8 * slot + o] = slab + turned_at + 32 * ((8 * wn + o) ^ swizzle);
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++) b_rd[2 * slot + h] = slab + (128 * wn + nu) * 128 + 16 * ((4 * h + kg) ^ (nu & 7));
    }
  }

  f4 acc[RB][8];
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (BF == false && LAYOUT == kRows && RB == 5) {
#include "ff_f16_rows_5.inc"
  }
  if constexpr (BF == false && LAYOUT == kRows && RB == 6) {
#include "ff_f16_rows_6.inc"
  }
  if constexpr (BF == false && LAYOUT == kRows && RB == 7) {
#include "ff_f16_rows_7.inc"
  }
  if constexpr (BF == false && LAYOUT == kRows && RB == 8) {
#include "ff_f16_rows_8.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnB && RB == 5) {
#include "ff_f16_b_5.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnB && RB == 6) {
#include "ff_f16_b_6.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnB && RB == 7) {
#include "ff_f16_b_7.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnB && RB == 8) {
#include "ff_f16_b_8.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnBoth && RB == 5) {
#include "ff_f16_both_5.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnBoth && RB == 6) {
#include "ff_f16_both_6.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnBoth && RB == 7) {
#include "ff_f16_both_7.inc"
  }
  if constexpr (BF == false && LAYOUT == kTurnBoth && RB == 8) {
#include "ff_f16_both_8.inc"
  }
  if constexpr (BF == true && LAYOUT == kRows && RB == 5) {
#include "ff_bf16_rows_5.inc"
  }
  if constexpr (BF == true && LAYOUT == kRows && RB == 6) {
#include "ff_bf16_rows_6.inc"
  }
  if constexpr (BF == true && LAYOUT == kRows && RB == 7) {
#include "ff_bf16_rows_7.inc"
  }
  if constexpr (BF == true && LAYOUT == kRows && RB == 8) {
#include "ff_bf16_rows_8.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnB && RB == 5) {
#include "ff_bf16_b_5.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnB && RB == 6) {
#include "ff_bf16_b_6.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnB && RB == 7) {
#include "ff_bf16_b_7.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnB && RB == 8) {
#include "ff_bf16_b_8.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnBoth && RB == 5) {
#include "ff_bf16_both_5.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnBoth && RB == 6) {
#include "ff_bf16_both_6.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnBoth && RB == 7) {
#include "ff_bf16_both_7.inc"
  }
  if constexpr (BF == true && LAYOUT == kTurnBoth && RB == 8) {
#include "ff_bf16_both_8.inc"
  }
#else  // the host pass only needs the launch stub
  (void)slabs, (void)lds_a, (void)lds_b, (void)src, (void)a_rd, (void)b_rd, (void)ra_words, (void)rb_words;
  (void)full_a, (void)last_a, (void)step_a, (void)full_b, (void)last_b, (void)step_b, (void)past;
  for (auto& r : acc)
    for (auto& v : r) v = (f4){0.f, 0.f, 0.f, 0.f};
#endif
  // a lane holds, per (i, o), row 16i + nu and four consecutive columns
  if (p.part) {
    const int columns = product_columns(p.N, GATED);
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int o = 0; o < 8; o++)
        put_part(p, at.slice, m0 + 16 * RB * wm + 16 * i + nu, n0 + 128 * wn + 16 * o + 4 * kg, p.M, columns,
                        acc[i][o]);
    return;
  }
  // The tile leaves through LDS in two halves; where both have room, the second is written to
  // LDS while the first is on its way to memory.
  constexpr int kPitch = out_pitch<256, GATED>(), kHalf = Sh::kHalf;
  constexpr bool kBoth = 64 * kHalf * kPitch <= Sh::kLds;
  const DropKey key(p.drop);
  const int col0 = 128 * wn + 4 * kg;
  i2 bias[8];
  if (FINISH == kFull && p.bias)
#pragma unroll
    for (int o = 0; o < 8; o++) bias[o] = full_bias(p, n0, col0 + 16 * o, cols);
#pragma unroll
  for (int half = 0; half < 2; half++) {
    char* const base = smem + (kBoth ? half * 32 * kHalf * kPitch : 0);
    if (half == 0 || !kBoth) __syncthreads();  // (nothing is on its way into LDS, and nobody reads it)
    if constexpr (FINISH == kFull) {
      i2 residual[kHalf][8];
      if (p.residual)
#pragma unroll
        for (int i = 0; i < kHalf; i++)
#pragma unroll
          for (int o = 0; o < 8; o++)
            if (kHalf * half + i < RB)
              residual[i][o] =
                  full_residual(p, m0, n0, 16 * RB * wm + 16 * (kHalf * half + i) + nu, col0 + 16 * o, rows, cols);
#pragma unroll
      for (int i = 0; i < kHalf; i++) {
        if (kHalf * half + i >= RB) continue;
#pragma unroll
        for (int o = 0; o < 8; o += 2)
          put_full<BF>(p, key, base + (16 * kHalf * wm + 16 * i + nu) * kPitch, m0, n0,
                       16 * RB * wm + 16 * (kHalf * half + i) + nu, col0 + 16 * o, kg, rows, cols, bias + o,
                       residual[i] + o, acc[(kHalf * half + i) % RB][o], acc[(kHalf * half + i) % RB][o + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kHalf; i++) {
        if (kHalf * half + i >= RB) continue;
#pragma unroll
        for (int o = 0; o < 8; o += GATED ? 2 : 1)
          put<256, GATED, BF>(p, base + (16 * kHalf * wm + 16 * i + nu) * kPitch, m0, n0,
                              16 * RB * wm + 16 * (kHalf * half + i) + nu, 128 * wn + 16 * o + 4 * kg, rows, cols,
                              acc[(kHalf * half + i) % RB][o],
                              acc[(kHalf * half + i) % RB][GATED ? o + 1 : o]);
      }
    }
    __syncthreads();
    store_rows<32 * kHalf, 256, GATED, 256>(p, base, m0, GATED ? n0 >> 1 : n0, rows, cols, [&](int r) {
      const int up = r / (16 * kHalf), at_row = 16 * kHalf * half + r % (16 * kHalf);
      return at_row < 16 * RB ? 16 * RB * up + at_row : TM;  // (an odd number of row blocks: the second half has one fewer)
    });
  }
}

namespace {

// calls f(kernel, LDS bytes) for a height, a layout and a type
template <bool BF, Finish FINISH, Layout LAYOUT, class F>
void with_height(int rows, F f) {
  if (rows == 256) f(product_big_kernel<BF, FINISH, LAYOUT, 8>, BigShape<8, LAYOUT>::kLds);
  if (rows == 224) f(product_big_kernel<BF, FINISH, LAYOUT, 7>, BigShape<7, LAYOUT>::kLds);
  if (rows == 192) f(product_big_kernel<BF, FINISH, LAYOUT, 6>, BigShape<6, LAYOUT>::kLds);
  if (rows == 160) f(product_big_kernel<BF, FINISH, LAYOUT, 5>, BigShape<5, LAYOUT>::kLds);
}
template <bool BF, class F>
void with_finish(int rows, Finish finish, Layout layout, F f) {
  if (finish == kGated) return with_height<BF, kGated, kRows>(rows, f);
  if (finish == kFull) return with_height<BF, kFull, kRows>(rows, f);
  if (layout == kRows) return with_height<BF, kPlain, kRows>(rows, f);
  if (layout == kTurnB) return with_height<BF, kPlain, kTurnB>(rows, f);
  return with_height<BF, kPlain, kTurnBoth>(rows, f);
}
template <class F>
void with_big(int rows, Finish finish, Layout layout, bool bf, F f) {
  bf ? with_finish<true>(rows, finish, layout, f) : with_finish<false>(rows, finish, layout, f);
}

}  // namespace

hipError_t configure_product_big() {
  hipError_t e = hipSuccess;
  for (const int rows : {160, 192, 224, 256})
    for (const bool bf : {false, true})
      for (const int form : {0, 1, 2, 3, 4})
        with_big(rows, form > 2 ? (Finish)(form - 2) : kPlain, form > 2 ? kRows : (Layout)form, bf, [&](auto kernel, int lds) {
          if (e == hipSuccess)
            e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        });
  return e;
}

void launch_product_big(ProductArgs a, int rows, Layout layout, bool bf, hipStream_t stream) {
  a.tiles_m = ceil_div(a.M, rows);
  a.tiles_n = ceil_div(product_columns(a.N, a.finish == kGated), 256);
  with_big(rows, a.finish, layout, bf, [&](auto kernel, int lds) {
    hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n * a.slices), dim3(256), lds, stream, a);
  });
}

}  // namespace w4a16
