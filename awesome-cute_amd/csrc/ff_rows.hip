// Dense products of up to 64 rows, with a gated epilogue: one token to a decoding batch, where
// the weights are read once and nothing else counts.
//
// A workgroup owns S blocks of 16 rows of B over the whole k range -- gated, of eight gates and
// their eight ups, so that eight columns of C are whole in it -- and all rows of A: no
// partial sums in memory, nothing exchanged between workgroups.  Its four waves take every
// fourth 64-deep chunk of k by themselves, each with a ring of LDS slots of its own (no barrier
// in the loop), and their sums meet in LDS once, at the end.
//
// Weights and activations go straight into LDS, eight rows of 128 bytes per instruction, whole
// cache lines: an MFMA operand wants sixteen rows of 64 bytes, which as loads take two to three
// times as long.  Chunk c of row r sits at position c ^ (r % 8), so that the operand reads meet
// no bank twice.
//
// Bound: HBM, by the weights, and below some 10 us the launch and the first loads' way.  Four waves
// and a ring of two or three stages leave room for several workgroups on a compute unit: one's
// sums meet while another's weights come.  Eight waves with as much in flight take a compute unit
// to themselves: on 20000 problems with weights from memory 1.10 of the best variant's time or
// more up to 16 rows, four waves 1.08, and where more than 48 rows meet 1.24 and 1.21.
// 1 x 2 x 10752 x 4096: 28 us, 6.2 TB/s.
#include <hip/hip_runtime.h>

#include "ff_products.hpp"

namespace w4a16 {

namespace {

constexpr int kFewWaves = 4;

template <int S, int MB, int DEPTH>
struct FewShape {
  static constexpr int kLoads = 2 * (S + MB);  // of 1 KiB per wave and chunk
  static constexpr int kSlot = 1024 * kLoads;
  static constexpr int kRing = kFewWaves * DEPTH * kSlot;
  static constexpr int kReduce = kFewWaves * S * MB * 1024;
  static constexpr int kLds = kRing > kReduce ? kRing : kReduce;
  static_assert(kLds <= 160 * 1024, "LDS of a compute unit");
};

template <int COUNT>
__device__ __forceinline__ void few_read(unsigned at, i4* v) {
  if constexpr (COUNT > 0) {
    few_read<COUNT - 1>(at, v);
    read_lds16<2048 * (COUNT - 1)>(at, v[COUNT - 1]);
  }
}

}  // namespace

template <bool BF, bool GATED, int S, int MB, int DEPTH>
__global__ __launch_bounds__(64 * kFewWaves) void product_rows_kernel(ProductArgs p) {
  using Sh = FewShape<S, MB, DEPTH>;
  constexpr int kCols = GATED ? 8 : 16;  // columns of C per block
  extern __shared__ __attribute__((aligned(16))) char smem[];  // Sh::kLds
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int kg = lane >> 4;
  const int nu = lane & 15;
  const int col0 = S * kCols * xcd_work_index((int)blockIdx.x, p.tiles_n);  // (the grid)
  const int last = p.N - 1;

  const int chunks = (p.K + 63) / 64;
  const int mine = (chunks - wave + kFewWaves - 1) / kFewWaves;
  const __amdgpu_buffer_rsrc_t rA =
      make_rsrc(p.A, (unsigned)(p.M - 1) * (unsigned)p.lda * 2u + (unsigned)p.K * 2u);
  const int b_rows = min(S * kCols, p.N - col0) + (GATED ? p.N : 0);  // from my first row to my last
  const __amdgpu_buffer_rsrc_t rB = make_rsrc((const char*)p.B + (size_t)col0 * p.ldb * 2,
                                              (unsigned)(b_rows - 1) * (unsigned)p.ldb * 2u + (unsigned)p.K * 2u);
  int a_src[2 * MB], b_src[2 * S];
  int past;  // this lane's 16 bytes in the last chunk: kOob where the row has ended
  {
    const int r8 = lane >> 3, c = (lane & 7) ^ r8;
#pragma unroll
    for (int t = 0; t < 2 * MB; t++) {
      const int r = 8 * t + r8;
      a_src[t] = r < p.M ? r * p.lda * 2 + 16 * c : kOob;  // rows past the last are zeros
    }
#pragma unroll
    for (int t = 0; t < 2 * S; t++) {
      // (columns past the last repeat it and are not stored)
      const int col = min(GATED ? col0 + 8 * (t >> 1) + r8 : col0 + 8 * t + r8, last) - col0;
      b_src[t] = (GATED && (t & 1) ? col + p.N : col) * p.ldb * 2 + 16 * c;
    }
    past = (chunks - 1) * 64 + 8 * c < p.K ? 0 : kOob;
  }
  char* const stage = smem + wave * (DEPTH * Sh::kSlot);
  // my i-th chunk
  auto issue = [&](int i, int slot) {
    const int c = wave + kFewWaves * i;
    const int inv = i >= mine ? kOob : c == chunks - 1 ? past : 0;
    char* const base = stage + slot * Sh::kSlot;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2 * S; t++) load_to_lds16<2>(rB, base + 1024 * t, b_src[t] | inv, 128 * c);
#pragma unroll
    for (int t = 0; t < 2 * MB; t++) load_to_lds16(rA, base + 2048 * S + 1024 * t, a_src[t] | inv, 128 * c);
    __builtin_amdgcn_sched_barrier(0);
  };

  f4 acc[S][MB];
#pragma unroll
  for (int s = 0; s < S; s++)
#pragma unroll
    for (int m = 0; m < MB; m++) acc[s][m] = (f4){0.f, 0.f, 0.f, 0.f};
  unsigned rd[2];
#pragma unroll
  for (int h = 0; h < 2; h++) rd[h] = (unsigned)(size_t)stage + nu * 128 + 16 * ((4 * h + kg) ^ (nu & 7));

#pragma unroll
  for (int d = 0; d < DEPTH; d++) issue(d, d);
  int slot = 0;
  for (int i = 0; i < mine; i++) {
    // chunk i has landed (loads complete in order); its operands read, by hand, since the
    // compiler would wait for every load in flight
    __builtin_amdgcn_s_waitcnt(vmcnt((DEPTH - 1) * Sh::kLoads));
    __builtin_amdgcn_sched_barrier(0);
    i4 o[2][S + MB];
#pragma unroll
    for (int h = 0; h < 2; h++) few_read<S + MB>(rd[h] + slot * Sh::kSlot, o[h]);
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(o[0][0]), "+v"(o[1][0]));
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int x = 1; x < S + MB; x++) asm volatile("" : "+v"(o[h][x]));
#endif
    issue(i + DEPTH, slot);
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int s = 0; s < S; s++)
#pragma unroll
        for (int m = 0; m < MB; m++) acc[s][m] = product_mfma<BF>(o[h][s], o[h][S + m], acc[s][m]);
  }
  // nothing may still be on its way into LDS when it is reused
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  // ---- sum the waves, a block of 16 product columns x 16 rows to a wave.  A lane holds
  // columns 4 kg ... 4 kg + 3 of row nu; gated, lanes 32 apart a gate and its partner.
  f4* const red = (f4*)smem;
#pragma unroll
  for (int s = 0; s < S; s++)
#pragma unroll
    for (int m = 0; m < MB; m++) red[((wave * S + s) * MB + m) * 64 + lane] = acc[s][m];
  __syncthreads();
  for (int b = wave; b < S * MB; b += kFewWaves) {
    f4 v = red[b * 64 + lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) v += red[(w * S * MB + b) * 64 + lane];
    const int row = 16 * (b % MB) + nu;
    const int col = col0 + kCols * (b / MB) + 4 * (GATED ? kg & 1 : kg);
    f4 up = v;
    if constexpr (GATED) {
#pragma unroll
      for (int r = 0; r < 4; r++) up[r] = __shfl_xor(v[r], 32);
    }
    if (row >= p.M || col >= p.N) continue;
    if constexpr (GATED) {
      if (p.pre)
        *(f4*)(p.pre + (size_t)row * p.ldpre + pre_col(col) + (kg >> 1 ? 16 : 0)) = v;
      if (kg < 2) *(i2*)((half_t*)p.C + (size_t)row * p.ldc + col) = product_round<BF>(act_mul4(v, up, p.act));
    } else {
      *(i2*)((half_t*)p.C + (size_t)row * p.ldc + col) = product_round<BF>(v);
    }
  }
}

namespace {

template <class F>
void with_rows(int s, int mb, bool bf, bool gated, F f) {
#define FF_ROWS(S, MB, DEPTH)                                                         \
  if (s == S && mb == MB) {                                                           \
    constexpr int lds = FewShape<S, MB, DEPTH>::kLds;                                 \
    if (bf)                                                                           \
      return f(gated ? product_rows_kernel<true, true, S, MB, DEPTH>                  \
                     : product_rows_kernel<true, false, S, MB, DEPTH>, lds);          \
    return f(gated ? product_rows_kernel<false, true, S, MB, DEPTH>                   \
                   : product_rows_kernel<false, false, S, MB, DEPTH>, lds);           \
  }
  FF_ROWS(1, 1, 3)
  FF_ROWS(2, 1, 2)
  FF_ROWS(1, 2, 2)
  FF_ROWS(2, 2, 2)
  FF_ROWS(1, 3, 2)
  FF_ROWS(2, 3, 2)
  FF_ROWS(1, 4, 2)
  FF_ROWS(2, 4, 2)
#undef FF_ROWS
}

}  // namespace

hipError_t configure_product_rows() {
  hipError_t e = hipSuccess;
  for (const int s : {1, 2})
    for (const int mb : {1, 2, 3, 4})
      for (const bool bf : {false, true})
        for (const bool gated : {false, true})
          with_rows(s, mb, bf, gated, [&](auto kernel, int lds) {
            if (e == hipSuccess)
              e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
          });
  return e;
}

void launch_product_rows(const ProductArgs& a, int blocks, bool bf, hipStream_t stream) {
  const bool gated = a.act != kActNone;
  ProductArgs b = a;
  b.tiles_n = ceil_div(a.N, (gated ? 8 : 16) * blocks);
  with_rows(blocks, ceil_div(a.M, 16), bf, gated, [&](auto kernel, int lds) {
    hipLaunchKernelGGL(kernel, dim3(b.tiles_n), dim3(64 * kFewWaves), lds, stream, b);
  });
}

}  // namespace w4a16
