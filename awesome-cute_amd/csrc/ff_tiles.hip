// Dense products in fp16 or bfloat16 by tiles, with a gated epilogue: what
// ff_rows.hip and ff_big.hip do not compute.  Slabs, swizzle, order of MFMA operands and the
// loop are those of f16_tiles.hip, where they are explained and measured; here
//   - rows of A, B and C may lie further apart than they are long,
//   - C may have any number of columns that is a multiple of 8, and k any such depth: what is
//     past the end of a row in its last 64-deep stage is requested at an offset past
//     everything, and so reads as zeros, in A and in B,
//   - an operand may lie turned over (ff_tile.hpp); its reads from LDS turn it back
//     (ds_read_b64_tr_b16), so that no transposed copy of a weight or of activations is made:
//     those took 75 us of 1060 of a forward and backward pass of 2048 x 2 x 10752 x 4096,
//   - gated, a tile's columns are gates and ups in turns of sixteen (gated_row), and its
//     epilogue writes act(g) u, for the backward pass both sums as well,
//   - the k range may be cut into slices, whose sums meet in memory (sum_parts): problems of few
//     tiles over a deep k.
//
// What bounds them: the way into LDS, and where a problem's tiles are about one to a compute unit
// the stages' latency (eight waves hide more of it than four with twice the operands each, which
// read a third less from LDS and take 1.0 to 1.2 of the time).  1237 x 1032 x 2744: 19 us by 117
// tiles of 96 x 128 in two slices, and 4 for their sums; 2744 x 1237 x 1032 of its backward pass
// 16 us, 440 TFLOP/s, 28 % of the matrix pipe's time in use.
#include <hip/hip_runtime.h>

#include "ff_tile.hpp"

namespace w4a16 {

namespace {

// TM x TN tiles, WM x WN waves
template <int TM, int TN, int WM, int WN, int RING, bool GATED>
struct FfShape {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kRB = TM / 16 / WM, kNJ = TN / 16 / WN;  // operands of a wave per k step
  static constexpr int kTA = (TM / 8 + kWaves - 1) / kWaves, kTB = TN / 8 / kWaves;  // loads per wave and slab
  static constexpr int kSlabA = kTA * kWaves * 1024, kSlab = kSlabA + TN * 128;
  static constexpr int kLoads = kTA + kTB;
  static constexpr int kRingBytes = RING * kSlab, kTileBytes = TM * out_pitch<TN, GATED>();
  static constexpr int kLds = kRingBytes > kTileBytes ? kRingBytes : kTileBytes;
  static_assert(kTB * 8 * kWaves == TN && TM % (16 * WM) == 0 && TN % (16 * WN) == 0, "whole blocks");
  static_assert(!GATED || kNJ % 2 == 0, "a gate's operand and its partner's in one wave");
  static_assert(kLds <= 160 * 1024 - 256, "LDS of a compute unit");
};

// An operand in LDS registers: by rows one read of 16 bytes, turned over two of 8
struct Operand {
  i2 half[2];
};
__device__ __forceinline__ i4 whole(const Operand& o) { return (i4){o.half[0][0], o.half[0][1], o.half[1][0], o.half[1][1]}; }

template <int OFF>
__device__ __forceinline__ void read_turned(unsigned at, i2& v) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(at), "n"(OFF) : "memory");
#endif
}
// wait for every LDS read in flight; the registers are named so that they count as in use up to
// here
template <int N>
__device__ __forceinline__ void ff_landed(i4 (&v)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0]));
#pragma unroll
  for (int i = 1; i < N; i++) asm volatile("" : "+v"(v[i]));
#endif
}
template <int N>
__device__ __forceinline__ void ff_landed(Operand (&v)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0].half[0]), "+v"(v[0].half[1]));
#pragma unroll
  for (int i = 1; i < N; i++) asm volatile("" : "+v"(v[i].half[0]), "+v"(v[i].half[1]));
#endif
}
__device__ __forceinline__ i4 whole(const i4& o) { return o; }

// ROWS_OR_COLS rows (by rows) or columns (turned over) of one operand of the tile
template <bool TURNED, int WIDTH, int WAVES, int LOADS, int BLOCKS>
struct Side {
  using Reg = std::conditional_t<TURNED, Operand, i4>;
  static constexpr int kPitch = 2 * WIDTH;             // turned over: bytes of a row in LDS
  static constexpr int kPerLoad = 1024 / kPitch;       // ... rows of a load
  static constexpr int kAddresses = TURNED ? BLOCKS : 2;
  static_assert(!TURNED || (64 % kPerLoad == 0 && LOADS * WAVES * kPerLoad == 64), "whole rows");
  int src[LOADS];
  unsigned rd[kAddresses];
  const char* base;
  long long step;      // turned over: bytes from one stage to the next
  int ld, width, depth;

  // where this wave's operands of slab 0 are read, their first block `first`
  __device__ __forceinline__ void read_from(unsigned slab, int first, int lane) {
    const int kg = lane >> 4, x = lane & 15;
    if constexpr (TURNED) {
      const unsigned at = slab + (8 * kg + (x >> 2)) * kPitch + 8 * (x & 3);
      const int s = turned_swizzle<WIDTH>(8 * kg + (x >> 2));
#pragma unroll
      for (int b = 0; b < BLOCKS; b++) rd[b] = at + 32 * ((first + b) ^ s);
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++) rd[h] = slab + (16 * first + x) * 128 + 16 * ((4 * h + kg) ^ (x & 7));
    }
  }
  // what this wave's loads fetch of a stage, turned over
  __device__ __forceinline__ void fetch_turned(const void* p, int c0, int ld_, int width_, int depth_, int wave, int lane) {
    base = (const char*)p + (size_t)c0 * 2;
    ld = ld_;
    width = width_ - c0;
    depth = depth_;
    step = (long long)kDnStageK * ld * 2;
    constexpr int kPieces = WIDTH / 8;
#pragma unroll
    for (int t = 0; t < LOADS; t++) {
      const int r = (LOADS * wave + t) * kPerLoad + lane / kPieces, piece = lane % kPieces;
      src[t] = r * ld * 2 + 16 * (piece ^ (2 * turned_swizzle<WIDTH>(r)));
    }
  }
  // the window of stage s
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t window(int s) const {
    const int left = depth - kDnStageK * s;
    const unsigned bytes = left <= 0 ? 0u : rows_bytes(min(left, kDnStageK), ld, width);
    return make_rsrc(base + s * step, bytes);
  }
  // operand block b of k step h from the slab at `slab`
  template <int H, int B>
  __device__ __forceinline__ void read(unsigned slab, Reg& v) const {
    if constexpr (TURNED) {
      read_turned<32 * H * kPitch>(rd[B] + slab, v.half[0]);
      read_turned<(32 * H + 4) * kPitch>(rd[B] + slab, v.half[1]);
    } else {
      read_lds16<2048 * B>(rd[H] + slab, v);
    }
  }
};

}  // namespace

// One barrier per 64-deep stage; the loop is dense_tile_kernel's (f16_tiles.hip).  ONCE: B's rows
// are requested as read once, as the kernel for few rows requests them: where one tile is as high
// as C.  56 problems of 9 to 64 rows that take tiles, weights from memory: 0.90 to 0.95 of the
// time; the same weights over and over, from the last-level cache, 1.00 to 1.08, but the weights
// of a model pass that cache.  With more tiles above each other it is slower either way (777 x 2
// x 5208 x 4160 60 -> 69 us, 1237 x 1032 x 2744 21 -> 30).
template <bool BF, bool GATED, Layout LAYOUT, int TM, int TN, int WM, int WN, int RING, bool ONCE>
__global__ __launch_bounds__(64 * WM * WN) void product_tile_kernel(ProductArgs p) {
  static_assert(!GATED || LAYOUT == kRows, "");
  using Sh = FfShape<TM, TN, WM, WN, RING, GATED>;
  constexpr int RB = Sh::kRB, NJ = Sh::kNJ, TA = Sh::kTA, TB = Sh::kTB;
  constexpr bool kTurnA = LAYOUT == kTurnBoth, kTurnedB = LAYOUT != kRows;
  using SideA = Side<kTurnA, TM, Sh::kWaves, TA, RB>;
  using SideB = Side<kTurnedB, TN, Sh::kWaves, TB, NJ>;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // Sh::kLds
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int kg = lane >> 4;
  const int nu = lane & 15;
  const int wm = wave / WN;
  const int wn = wave % WN;

  const TileAt at(p, TM, TN);
  const int m0 = at.m0, n0 = at.n0;
  const int rows = min(TM, p.M - m0);
  const int all = (p.K + kDnStageK - 1) / kDnStageK;
  const int first = at.stage(p, all, 0), end = at.stage(p, all, 1);

  SideA sa;
  SideB sb;
  __amdgpu_buffer_rsrc_t rA, rB;
  int cols = min(GATED ? TN / 2 : TN, p.N - (GATED ? n0 >> 1 : n0));
  int past;  // this lane's 16 bytes of a row in the last stage: kOob where the row has ended
  {
    const int r8 = lane >> 3, c = (lane & 7) ^ r8;
    past = (all - 1) * kDnStageK + 8 * c < p.K ? 0 : kOob;
    if constexpr (kTurnA) {
      sa.fetch_turned(p.A, m0, p.lda, p.M, p.K, wave, lane);
    } else {
      rA = make_rsrc((const char*)p.A + (size_t)m0 * p.lda * 2, rows_bytes(rows, p.lda, p.K));
#pragma unroll
      for (int t = 0; t < TA; t++) {
        const int r = 8 * (TA * wave + t) + r8;
        sa.src[t] = r >= TM ? kOob : (r < rows ? r : rows - 1) * p.lda * 2 + 16 * c;
      }
    }
    if constexpr (kTurnedB) {
      sb.fetch_turned(p.B, n0, p.ldb, p.N, p.K, wave, lane);
    } else {
      unsigned b_bytes;
      const char* const b_at = b_base<GATED>(p, n0, TN, &b_bytes, &cols);
      rB = make_rsrc(b_at, b_bytes);
#pragma unroll
      for (int t = 0; t < TB; t++) sb.src[t] = b_offset<GATED>(p, n0, 8 * (TB * wave + t) + r8, cols) + 16 * c;
    }
  }
  sa.read_from((unsigned)(size_t)smem, RB * wm, lane);
  sb.read_from((unsigned)(size_t)smem + Sh::kSlabA, NJ * wn, lane);

  // stage s of all into a slot; one past my last fetches zeros
  auto issue_slab = [&](int s, int slot) {
    const int inv = s >= end ? kOob : s == all - 1 ? past : 0, gone = s >= end ? kOob : 0;
    const int k_at = s * (kDnStageK * 2);
    char* const base = smem + slot * Sh::kSlab;
    if constexpr (kTurnA) {
      const __amdgpu_buffer_rsrc_t r = sa.window(s);
#pragma unroll
      for (int t = 0; t < TA; t++) load_to_lds16(r, base + (TA * wave + t) * 1024, sa.src[t] | gone, 0);
    } else {
#pragma unroll
      for (int t = 0; t < TA; t++) load_to_lds16(rA, base + (TA * wave + t) * 1024, sa.src[t] | inv, k_at);
    }
    if constexpr (kTurnedB) {
      const __amdgpu_buffer_rsrc_t r = sb.window(s);
#pragma unroll
      for (int t = 0; t < TB; t++) load_to_lds16(r, base + Sh::kSlabA + (TB * wave + t) * 1024, sb.src[t] | gone, 0);
    } else {
#pragma unroll
      for (int t = 0; t < TB; t++)
        load_to_lds16<ONCE ? 2 : 0>(rB, base + Sh::kSlabA + (TB * wave + t) * 1024, sb.src[t] | inv, k_at);
    }
  };

  // the operands of a stage
  struct Set {
    typename SideB::Reg b[2 * NJ];
    typename SideA::Reg a[2 * RB];
  };
  auto read = [&](Set& o, unsigned slab) {
    for_each<2>([&](auto H) {
      constexpr int h = decltype(H)::value;
      for_each<NJ>([&](auto J) {
        constexpr int j = decltype(J)::value;
        sb.template read<h, j>(slab, o.b[h * NJ + j]);
      });
      for_each<RB>([&](auto I) {
        constexpr int i = decltype(I)::value;
        sa.template read<h, i>(slab, o.a[h * RB + i]);
      });
    });
  };
  auto landed = [&](Set& o) {
    ff_landed(o.b);
    ff_landed(o.a);
  };

  f4 acc[RB][NJ];
#pragma unroll
  for (int i = 0; i < RB; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[i][j] = (f4){0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](Set& o) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
          acc[i][j] = product_mfma<BF>(whole(o.b[h * NJ + j]), whole(o.a[h * RB + i]), acc[i][j]);
  };

  // Every slot requested; slab 0 landed (loads complete in order), its operands read.
  // Between the reads into a set of registers and the wait that names them stand the MFMAs
  // of the other set and nothing else.
  Set even, odd;
#pragma unroll
  for (int r = 0; r < RING; r++) issue_slab(first + r, r);
  __builtin_amdgcn_s_waitcnt(vmcnt((RING - 1) * Sh::kLoads));
  __builtin_amdgcn_s_barrier();
  read(even, 0);
  landed(even);
  int slot = 0;
  auto stage = [&](int s, Set& cur, Set& next) {
    __builtin_amdgcn_s_waitcnt(vmcnt((RING - 2) * Sh::kLoads));
    __builtin_amdgcn_s_barrier();
    const int slot_next = slot == RING - 1 ? 0 : slot + 1;
    __builtin_amdgcn_sched_barrier(0);
    read(next, slot_next * Sh::kSlab);
    issue_slab(s + RING, slot);
    __builtin_amdgcn_sched_barrier(0);
    multiply(cur);
    __builtin_amdgcn_sched_barrier(0);
    landed(next);
    slot = slot_next;
  };
  int s = first;
  for (; s + 1 < end; s += 2) {
    stage(s, even, odd);
    stage(s + 1, odd, even);
  }
  if (s < end) multiply(even);
  // nothing of the ring may still be on its way when LDS is reused
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  // a lane holds, per (i, j), row 16i + nu and four consecutive columns; the tile leaves
  // through LDS as whole rows
  if (p.part) {
    const int columns = product_columns(p.N, GATED);
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int j = 0; j < NJ; j++)
        put_part(p, at.slice, m0 + 16 * RB * wm + 16 * i + nu, n0 + 16 * NJ * wn + 16 * j + 4 * kg, p.M, columns,
                        acc[i][j]);
    return;
  }
  char* const out = smem + (16 * RB * wm + nu) * out_pitch<TN, GATED>();
#pragma unroll
  for (int i = 0; i < RB; i++)
#pragma unroll
    for (int j = 0; j < NJ; j += GATED ? 2 : 1)
      put<TN, GATED, BF>(p, out + 16 * i * out_pitch<TN, GATED>(), m0, n0, 16 * RB * wm + 16 * i + nu,
                         16 * NJ * wn + 16 * j + 4 * kg, rows, cols, acc[i][j], acc[i][GATED ? j + 1 : j]);
  __syncthreads();
  store_rows<TM, TN, GATED, Sh::kThreads>(p, smem, m0, GATED ? n0 >> 1 : n0, rows, cols, [](int r) { return r; });
}

// The slices' sums in their order, and what a tile's epilogue does with them; four columns of C
// a thread.  All SLICES are on their way together: fetched one after the other, eight cost 1.2 us
// of 13.5 where C is small (64 x 2048 x 8192).
template <bool BF, bool GATED, int SLICES>
__global__ __launch_bounds__(256) void sum_parts_kernel(ProductArgs p) {
  const int quads = p.N / 4;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(at / quads), col = 4 * (int)(at - (long long)m * quads);
  if (m >= p.M) return;
  const float* const from = p.part + (size_t)m * p.ldpart + (GATED ? pre_col(col) : col);
  f4 part[SLICES], part_up[GATED ? SLICES : 1];
#pragma unroll
  for (int s = 0; s < SLICES; s++) {
    const float* const at_slice = from + (size_t)s * p.M * p.ldpart;
    part[s] = *(const f4*)at_slice;
    if constexpr (GATED) part_up[s] = *(const f4*)(at_slice + 16);
  }
  f4 v = part[0], up = GATED ? part_up[0] : v;
#pragma unroll
  for (int s = 1; s < SLICES; s++) {
    v += part[s];
    if constexpr (GATED) up += part_up[s];
  }
  if constexpr (GATED) {
    if (p.pre) {
      float* const pre = p.pre + (size_t)m * p.ldpre + pre_col(col);
      *(f4*)pre = v;
      *(f4*)(pre + 16) = up;
    }
    v = act_mul4(v, up, p.act);
  }
  *(i2*)((half_t*)p.C + (size_t)m * p.ldc + col) = product_round<BF>(v);
}

namespace {

// calls f(kernel, LDS bytes, threads) for a tile, a layout and a type; once: one tile is as high as C
template <bool BF, bool GATED, Layout LAYOUT, class F>
void with_tile(const FfTile& t, bool once, F f) {
#define FF_TILE_OF(TM, TN, WM, WN, RING, ONCE)                                    \
  if (t.rows == TM && t.cols == TN && once == ONCE)                               \
  return f(product_tile_kernel<BF, GATED, LAYOUT, TM, TN, WM, WN, RING, ONCE>,    \
           FfShape<TM, TN, WM, WN, RING, GATED>::kLds, 64 * WM * WN)
#define FF_TILE(TM, TN, WM, WN, RING) FF_TILE_OF(TM, TN, WM, WN, RING, false)
  if constexpr (LAYOUT == kRows) {
    FF_TILE_OF(64, 64, 2, 2, 4, true);
    FF_TILE_OF(64, 128, 2, 4, 6, true);
  }
  once = false;
  FF_TILE(64, 64, 2, 2, 4);
  FF_TILE(64, 128, 2, 4, 6);
  FF_TILE(128, 128, 2, 4, 4);
  FF_TILE(128, 256, 2, 4, 3);
  if constexpr (LAYOUT != kTurnBoth) {
    FF_TILE(96, 128, 2, 4, 4);
    FF_TILE(96, 256, 2, 4, 3);
  }
#undef FF_TILE
#undef FF_TILE_OF
}
template <class F>
void with_product(const FfTile& t, bool gated, Layout layout, bool once, bool bf, F f) {
  if (gated) return bf ? with_tile<true, true, kRows>(t, once, f) : with_tile<false, true, kRows>(t, once, f);
  if (layout == kRows) return bf ? with_tile<true, false, kRows>(t, once, f) : with_tile<false, false, kRows>(t, once, f);
  if (layout == kTurnB) return bf ? with_tile<true, false, kTurnB>(t, once, f) : with_tile<false, false, kTurnB>(t, once, f);
  return bf ? with_tile<true, false, kTurnBoth>(t, once, f) : with_tile<false, false, kTurnBoth>(t, once, f);
}

}  // namespace

hipError_t configure_product_tiles() {
  hipError_t e = hipSuccess;
  for (const int rows : {64, 96, 128})
    for (const int cols : {64, 128, 256})
      for (const bool bf : {false, true})
        for (const bool once : {false, true})
          for (const int form : {0, 1, 2, 3})
            with_product({rows, cols}, form == 3, form == 3 ? kRows : (Layout)form, once, bf,
                         [&](auto kernel, int lds, int) {
                           if (e == hipSuccess)
                             e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
                         });
  return e;
}

void launch_product_tiles(ProductArgs a, const FfTile& t, Layout layout, bool bf, hipStream_t stream) {
  const bool gated = a.act != kActNone;
  a.tiles_m = ceil_div(a.M, t.rows);
  a.tiles_n = ceil_div(product_columns(a.N, gated), t.cols);
  with_product(t, gated, layout, a.tiles_m == 1, bf, [&](auto kernel, int lds, int threads) {
    hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n * a.slices), dim3(threads), lds, stream, a);
  });
}

template <int SLICES>
static void launch_sum_of(const ProductArgs& a, bool bf, hipStream_t stream) {
  if constexpr (SLICES > 1) {
    if (a.slices != SLICES) return launch_sum_of<SLICES - 1>(a, bf, stream);
    const bool gated = a.act != kActNone;
    const dim3 grid((unsigned)(((long long)a.M * (a.N / 4) + 255) / 256)), block(256);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
    if (bf)
      gated ? launch(sum_parts_kernel<true, true, SLICES>) : launch(sum_parts_kernel<true, false, SLICES>);
    else
      gated ? launch(sum_parts_kernel<false, true, SLICES>) : launch(sum_parts_kernel<false, false, SLICES>);
  }
}
void launch_sum_parts(const ProductArgs& a, bool bf, hipStream_t stream) { launch_sum_of<kSlicesMost>(a, bf, stream); }

}  // namespace w4a16
