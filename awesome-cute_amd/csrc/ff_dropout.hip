// Dropout, with the residual's addition or without, and its gradient, which is the same of dy: the
// mask is made from the seed both times (dropout.hpp) and never stored.
//
// A lane has eight elements: a group of 16-bit ones, 16 bytes and one run of the generator; of 32-bit
// ones four of one group and four of another, so that a wave's loads are of neighbouring bytes.  Inside
// fp32, rounded once.
//
// Bound: HBM, or the last-level cache, which holds up to 256 MB of a call.  Operands are requested as read once
// (nontemporal) where a call moves more than that cache holds: 16384 x 4096 bfloat16 with a residual, 403 MB, 61.2 us,
// 6.6 TB/s (otherwise 70.3).  Where it moves less they are mostly there, and such requests would pass it by: 2048 x 10752 13.8 us, 6.4
// TB/s (16.2; of an operand that the call before has just written 13.9 and 14.2).  Results are
// stored past the caches where they alone are more than the last one holds: 65536 x 4096 with a residual 249 us (261), and the norm that
// reads it 222 (227).  Smaller ones are read from there next, and stored past it cost their reader more than they save
// here: 2048 x 10752 13.6 us in place of 13.9, but with a product behind it 162 in place of 151, 16384 x 4096
// 44.0 in place of 41.0, and 480 in place of 442.  The generator costs nothing visible; two or four groups
// a lane, or a grid of eight workgroups a compute unit, 2 to 10 % more.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/feedforward_amd.h"
#include "dropout.hpp"
#include "ff_grads.hpp"

namespace w4a16 {

namespace {

constexpr int kThreads = 256;
constexpr long long kLastLevel = 256LL << 20;  // bytes of the last-level cache

template <class T>
using Piece16 = T __attribute__((ext_vector_type(16 / sizeof(T))));

// 16 bytes of elements at `at`, of which `left` are there
template <bool WHOLE, bool ONCE, class T>
__device__ __forceinline__ Piece16<T> load_piece(const T* at, long long left) {
  constexpr int kN = 16 / sizeof(T);
  if (WHOLE && left >= kN) {
    const i4* const p = (const i4*)at;
    return __builtin_bit_cast(Piece16<T>, ONCE ? __builtin_nontemporal_load(p) : *p);
  }
  Piece16<T> out = {};
#pragma unroll
  for (int e = 0; e < kN; e++)
    if (e < left) out[e] = at[e];
  return out;
}
template <bool WHOLE, bool PAST, class T>
__device__ __forceinline__ void store_piece16(T* at, long long left, Piece16<T> v) {
  constexpr int kN = 16 / sizeof(T);
  if (WHOLE && left >= kN) {
    if constexpr (PAST)
      __builtin_nontemporal_store(__builtin_bit_cast(i4, v), (i4*)at);
    else
      *(i4*)at = __builtin_bit_cast(i4, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < kN; e++)
    if (e < left) at[e] = v[e];
}

}  // namespace

// WHOLE: every matrix starts on 16 bytes; ONCE: operands are requested as read once; PAST: results are stored past the caches
template <class T, bool WHOLE, bool ONCE, bool PAST>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs p) {
  constexpr int kN = 16 / sizeof(T), kPieces = 8 / kN;
  const int lane = threadIdx.x & 63;
  const unsigned long long wave = (unsigned long long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  Piece16<T> x[kPieces], residual[kPieces];
  long long at[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; i++) {
    at[i] = (long long)(512 * wave) + 64 * kN * i + kN * lane;
    x[i] = load_piece<WHOLE, ONCE>((const T*)p.x + at[i], p.count - at[i]);
    if (p.residual) residual[i] = load_piece<WHOLE, ONCE>((const T*)p.residual + at[i], p.count - at[i]);
  }
  i4 bits;
  if constexpr (kPieces == 1) {
    bits = drop_bits(64 * wave + lane, DropKey(p.drop));
  } else {
    // lanes 2 i and 2 i + 1 have group i of the first piece and group 32 + i of the second, a half each: the
    // even one makes the bits of the first, the odd one of the second, and they exchange halves
    const i4 w = drop_bits(64 * wave + (lane >> 1) + (lane & 1 ? 32 : 0), DropKey(p.drop));
    const bool odd = lane & 1;
    int mine[2], other[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      mine[h] = odd ? w[2 + h] : w[h];
      other[h] = __builtin_amdgcn_mov_dpp(odd ? w[h] : w[2 + h], 0xb1 /* quads 1, 0, 3, 2 */, 0xf, 0xf, true);
    }
    bits = odd ? (i4){other[0], other[1], mine[0], mine[1]} : (i4){mine[0], mine[1], other[0], other[1]};
  }
#pragma unroll
  for (int i = 0; i < kPieces; i++) {
#pragma unroll
    for (int e = 0; e < kN; e++) {
      const float v = drop_one((float)x[i][e], bits, kN * i + e, p.drop);
      x[i][e] = (T)(p.residual ? (float)residual[i][e] + v : v);
    }
    store_piece16<WHOLE, PAST, T>((T*)p.y + at[i], p.count - at[i], x[i]);
  }
}

template <class T>
static void launch_of(const DropoutArgs& a, hipStream_t stream) {
  const bool whole = (((uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.y) & 15) == 0;
  const long long bytes = a.count * (long long)sizeof(T);
  const dim3 grid((unsigned)((a.count + 8 * kThreads - 1) / (8 * kThreads)));
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a); };
  if (!whole)
    launch(dropout_kernel<T, false, false, false>);
  else if (bytes > kLastLevel)
    launch(dropout_kernel<T, true, true, true>);
  else if (bytes * (a.residual ? 3 : 2) > kLastLevel)
    launch(dropout_kernel<T, true, true, false>);
  else
    launch(dropout_kernel<T, true, false, false>);
}

void launch_dropout(const DropoutArgs& a, int type, hipStream_t stream) {
  if (type == FEEDFORWARD_FP16) launch_of<half_t>(a, stream);
  if (type == FEEDFORWARD_BF16) launch_of<__bf16>(a, stream);
  if (type == FEEDFORWARD_FP32) launch_of<float>(a, stream);
}

}  // namespace w4a16
