// Dense products in fp16 or bfloat16 by tiles of 160, 192, 224 or 256 rows x 256 columns: four
// waves, two by two, the main loop one assembly statement (gen_products.py).  Operands by rows
// or turned over, any depth, slices and the gated epilogue as in ff_tiles.hip.
//
// Bound: how evenly the tiles fill the compute units, hence the heights (777 x 2 x 5208 x 4160: 164
// tiles of 256 rows, 205 of 160), some 12 us of a tile outside its loop (the first slabs' way, and
// results that all compute units write at once), and in the loop the board's power.  bfloat16, operands
// from memory, us and TFLOP/s: 2048 x 2 x 10752 x 4096 296, 1220 (with the sums kept 313); its backward
// pass 2048 x 4096 x 21504 267, 1350, in two slices that meet, and 21504 x 4096 x 2048 307, 1170;
// 8192 x 4096 x 4096 205, 1340, with bias and residual 226 to 230.  The matrix pipe is in use for 53 to 72 % of these.  Results
// past the caches or through them: level, with what reads them next too (two products one after the other, an Mlp's
// training step: 2 % to either side).
//
// A source for each type includes this: the kernels of one take the compiler a minute and more.
#pragma once
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
  static constexpr int kOut = 2 * 32 * kHalf * out_pitch<256, false>();  // (a half of the results, and of the slopes)
  static constexpr int kRingA = 3 * (kSlabA + kSlabB) <= 160 * 1024 ? 3 : 2, kRingB = 3;  // slabs in LDS
  static constexpr int kRings = kRingA * kSlabA + kRingB * kSlabB;
  static constexpr int kLds = kRings > kOut ? kRings : kOut;
  static_assert(kLds <= 160 * 1024, "LDS of a compute unit");
};

// How two slices of a tile meet, at a word of which nothing is known but that it is not this launch's: it
// counts as empty unless it holds the launch's token, a number of 61 bits that no other launch of the
// process has, and it is left as zero, so that a captured launch, whose token is always the same, finds
// none of its own either.  (What memory held before could be the token by chance, once in 2^61
// tiles.  Zeros ahead of the launch, from a kernel of their own, took 2 to 4 us.)
//
// Bits 0 and 1 of the word: slice 0, 1 has arrived; bit 2: it has left.  Thread 0 calls meet_arrive once the
// workgroup's sums of the other's half have been acknowledged: the halves to finish as a bit mask, or 0 if the
// other has not come within some 50 us -- the slices are equally long and start together, but nothing
// promises that they run at the same time --, and then meet_abandon, once those of its own half are out as well:
// the same, 0 meaning that the other finishes both.
__device__ __forceinline__ bool meet_swap(unsigned long long* word, unsigned long long* seen, unsigned long long next) {
  return __hip_atomic_compare_exchange_strong(word, seen, next, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ int meet_arrive(unsigned long long* word, unsigned long long token, int slice, int max_polls) {
  const unsigned long long other = token | (2 >> slice), both = token | 3;
  unsigned long long v = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (;;) {  // (the other slice alone writes the word, twice at most)
    const unsigned long long next = v == other ? both : v == (other | 4) ? 0 : token | (1 << slice);
    if (!meet_swap(word, &v, next)) continue;
    if (v == other) return 1 << slice;
    if (v == (other | 4)) return 3;
    break;
  }
  for (int polls = 0; polls < max_polls; polls++) {
    __builtin_amdgcn_s_sleep(2);
    v = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (v != both) continue;
    __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return 1 << slice;
  }
  return 0;
}
__device__ __forceinline__ int meet_abandon(unsigned long long* word, unsigned long long token, int slice) {
  unsigned long long v = token | (1 << slice);
  if (meet_swap(word, &v, v | 4)) return 0;
  __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // (it is `both`)
  return 1 << slice;
}

}  // namespace

// MEET: two slices of a tile finish it together
template <bool BF, Finish FINISH, Layout LAYOUT, int RB, bool MEET>
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

  const int m_at = 16 * RB * wm + nu, col = 128 * wn + 4 * kg;
  i2 bias[8];
  // (where two slices meet their meeting hides its way, and in registers for the loop's length it spills)
  if constexpr (FINISH == kFull && !MEET) fetch_bias(p, n0, col, cols, bias);

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
  constexpr int kHalf = Sh::kHalf;
  int halves = 3;  // of the tile's row blocks that this workgroup finishes, kHalf and the rest
  const __amdgpu_buffer_rsrc_t rP = make_rsrc(p.part, 0x7fffffffu);
  const int lane_at = wave * (RB * 8 * 1024) + lane * 16;
  const auto part = [&](int slice) { return (2 * at.tile + slice) * (int)big_sums(TM); };
  if constexpr (MEET) {
    if constexpr (FINISH == kFull) fetch_bias(p, n0, col, cols, bias);
    // Two slices that finish their tile together (meet_arrive): each writes its sums of the other's
    // half through to memory, waits for the acknowledgement and arrives, and adds the other's sums to its
    // own, in whichever order the same bits as sum_parts.  (Nobody waits for long, whatever runs when.)  A
    // launch that adds up both slices' sums of everything takes 14 us of 145 (2048 x 4096 x 10752, B turned
    // over), and 21 of 165 with a residual.
    unsigned long long* const word = p.words + at.tile * kWordStride;
    const auto write_out = [&](int which) {
      for_each<RB>([&](auto I) {
        constexpr int i = decltype(I)::value;
        if (which >> (i >= kHalf) & 1)
          for_each<8>([&](auto O) {
            constexpr int o = decltype(O)::value;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, acc[i][o]), rP, lane_at + (8 * i + o) * 1024,
                                                   part(at.slice), 16 /* sc1 */);
          });
      });
      __builtin_amdgcn_s_waitcnt(vmcnt(0));  // my stores have been acknowledged
      __syncthreads();                       // so have everybody's, and LDS is free
    };
    volatile int* const shares = (volatile int*)smem;
    write_out(2 >> at.slice);
    if (tid == 0) *shares = meet_arrive(word, p.token, at.slice, p.polls);
    __syncthreads();
    halves = __builtin_amdgcn_readfirstlane(*shares);
    if (halves == 0) {
      write_out(1 << at.slice);
      if (tid == 0) *shares = meet_abandon(word, p.token, at.slice);
      __syncthreads();
      halves = __builtin_amdgcn_readfirstlane(*shares);
    }
  } else if (p.part) {
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
  // LDS while the first is on its way to memory.  (Full, the slopes' image is the second half's.)
  constexpr int kPitch = out_pitch<256, GATED>(), kImage = 32 * kHalf * kPitch;
  const bool both = !MEET && 2 * kImage <= Sh::kLds && !(FINISH == kFull && p.slopes);
  for_each<2>([&](auto Half) {
    constexpr int half = decltype(Half)::value, first_block = half * kHalf, kBlocks = half ? RB - kHalf : kHalf;
    if (MEET && !(halves >> half & 1)) return;
    char* const base = smem + (both ? half * kImage : 0);
    if (half == 0 || !both) __syncthreads();  // (nothing is on its way into LDS, and nobody reads it)
    char* const out = base + (16 * kHalf * wm + nu) * kPitch;
    // four row blocks two at a time: with the residual, or the other slice's sums, registers spill otherwise
    constexpr int kChunk = kHalf > 3 ? 2 : kHalf;
    for_each<(kBlocks + kChunk - 1) / kChunk>([&](auto At) {
      constexpr int i0 = kChunk * decltype(At)::value, block = first_block + i0;
      constexpr int count = kBlocks - i0 < kChunk ? kBlocks - i0 : kChunk;
      const int m = m_at + 16 * block;
      f4 v[count][8];
      for_each<count * 8>([&](auto At) {
        constexpr int i = decltype(At)::value / 8, o = decltype(At)::value % 8;
        if constexpr (MEET)
          v[i][o] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rP, lane_at + (8 * (block + i) + o) * 1024,
                                                                                 part(1 - at.slice), 16 /* sc1 */));
        else
          v[i][o] = acc[block + i][o];
      });
      i2 residual[count][8];
      if constexpr (FINISH == kFull) fetch_residual(p, m0, n0, m, col, rows, cols, residual);
      if constexpr (MEET)
        for_each<count * 8>([&](auto At) {
          constexpr int i = decltype(At)::value / 8, o = decltype(At)::value % 8;
          v[i][o] += acc[block + i][o];
        });
      if constexpr (FINISH == kPlain)
        if (p.scale != 1.f)
          for_each<count * 8>([&](auto At) { v[decltype(At)::value / 8][decltype(At)::value % 8] *= p.scale; });
      if constexpr (FINISH == kFull)
        put_full<BF, count, 8, kPitch>(p, out + 16 * i0 * kPitch, kImage, m0, n0, m, col, kg, bias, residual, v);
      else
        for_each<count>([&](auto I) {
          constexpr int i = decltype(I)::value, step = GATED ? 2 : 1;
          for_each<8 / step>([&](auto O) {
            constexpr int o = step * decltype(O)::value;
            put<256, GATED, BF>(p, out + 16 * (i0 + i) * kPitch, m0, n0, m + 16 * i, col + 16 * o, rows, cols, v[i][o],
                                v[i][GATED ? o + 1 : o]);
          });
        });
    });
    __syncthreads();
    const auto row_of = [&](int r) {
      const int up = r / (16 * kHalf), at_row = 16 * kHalf * half + r % (16 * kHalf);
      return at_row < 16 * RB ? 16 * RB * up + at_row : TM;  // (an odd number of row blocks: the second half has one fewer)
    };
    store_rows<32 * kHalf, 256, GATED, 256>(p.C, p.ldc, base, m0, GATED ? n0 >> 1 : n0, rows, cols, row_of);
    if constexpr (FINISH == kFull)
      if (p.slopes)
        store_rows<32 * kHalf, 256, false, 256>(p.slopes, p.ldslopes, base + kImage, m0, n0, rows, cols, row_of);
  });
}

namespace {

// calls f(kernel, LDS bytes) for a height, a layout, a type and whether two slices meet
template <bool BF, Finish FINISH, Layout LAYOUT, bool MEET, class F>
void with_height(int rows, F f) {
  if (rows == 256) f(product_big_kernel<BF, FINISH, LAYOUT, 8, MEET>, BigShape<8, LAYOUT>::kLds);
  if (rows == 224) f(product_big_kernel<BF, FINISH, LAYOUT, 7, MEET>, BigShape<7, LAYOUT>::kLds);
  if (rows == 192) f(product_big_kernel<BF, FINISH, LAYOUT, 6, MEET>, BigShape<6, LAYOUT>::kLds);
  if (rows == 160) f(product_big_kernel<BF, FINISH, LAYOUT, 5, MEET>, BigShape<5, LAYOUT>::kLds);
}
template <bool BF, bool MEET, class F>
void with_finish(int rows, Finish finish, Layout layout, F f) {
  if (finish == kGated) return with_height<BF, kGated, kRows, MEET>(rows, f);
  if (finish == kFull) return with_height<BF, kFull, kRows, MEET>(rows, f);
  if (layout == kRows) return with_height<BF, kPlain, kRows, MEET>(rows, f);
  if (layout == kTurnB) return with_height<BF, kPlain, kTurnB, MEET>(rows, f);
  return with_height<BF, kPlain, kTurnBoth, MEET>(rows, f);
}
template <bool BF, class F>
void with_big(int rows, Finish finish, Layout layout, bool meet, F f) {
  meet ? with_finish<BF, true>(rows, finish, layout, f) : with_finish<BF, false>(rows, finish, layout, f);
}

}  // namespace

template <bool BF>
hipError_t configure_big() {
  hipError_t e = hipSuccess;
  for (const int rows : {160, 192, 224, 256})
    for (const bool meet : {false, true})
      for (const int form : {0, 1, 2, 3, 4})
        with_big<BF>(rows, form > 2 ? (Finish)(form - 2) : kPlain, form > 2 ? kRows : (Layout)form, meet,
                     [&](auto kernel, int lds) {
                       if (e == hipSuccess)
                         e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
                     });
  return e;
}

template <bool BF>
void launch_big(ProductArgs a, int rows, Layout layout, hipStream_t stream) {
  a.tiles_m = ceil_div(a.M, rows);
  a.tiles_n = ceil_div(product_columns(a.N, a.finish == kGated), 256);
  with_big<BF>(rows, a.finish, layout, a.words != nullptr, [&](auto kernel, int lds) {
    hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n * a.slices), dim3(256), lds, stream, a);
  });
}

}  // namespace w4a16
