// The norms after a block and before the next one, with the block's gate and the residual's
// scale, and their gradients: per row b (the block's output) and r0 (the residual)
//
//   p = b rstd(b) post      rstd(v) = 1 / sqrt(mean(v^2) + eps)      (p = b without `post`)
//   r = scale r0 + gate p                                            (r = r0 without a block)
//   y = r rstd(r) pre
//
// in fp32 from inputs in 16 or 32 bits, r and y rounded once (y from the unrounded r).  With
// bh = b rstd(b), rh = r rstd(r) and the gradients dy and dr of y and r
//
//   dt = dr + rstd(r) (dy pre - rh mean(dy pre rh))       dr0 = scale dt      dpre = sum dy rh
//   db = rstd(b) (w - bh mean(w bh)),  w = dt gate post   q = sum dt bh: dgate = post q, dpost = gate q
//
// the sums over the rows that share a weight or a gate.
//
// Bound: HBM; every row is read and written once.  A row is kept in the registers of W waves, one
// or two 16-byte pieces a lane, so that the second pass over it that a norm needs costs nothing;
// the waves' sums meet in LDS, two meetings a row forward.  Backward one: mean(w bh) is put
// together from four sums, of dy pre rh, and of gate post bh times dr, dy pre and rh.
//
// Sums over rows: every part (a run of rows) adds up its own in registers, in the order of its
// rows, and leaves them in memory; a second launch adds the parts in their order.  No atomics,
// so the same call gives the same bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ff_norm.hpp"
#include "w4a16_common.hpp"

namespace w4a16 {

namespace {

typedef __bf16 bf;

// VEC elements of type T as they come from memory, and as floats
template <class T, int VEC>
struct Piece {
  T v[VEC];
  __device__ __forceinline__ float at(int i) const { return (float)v[i]; }
};
template <class T, int VEC>
__device__ __forceinline__ Piece<T, VEC> load_piece(const void* p, size_t at) {
  Piece<T, VEC> r;
  if constexpr (VEC * sizeof(T) == 16)
    *(i4*)&r = *(const i4*)((const T*)p + at);
  else
    r.v[0] = ((const T*)p)[at];
  return r;
}
template <class T, int VEC>
__device__ __forceinline__ void store_piece(void* p, size_t at, const float* f) {
  Piece<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; i++) r.v[i] = (T)f[i];
  if constexpr (VEC * sizeof(T) == 16)
    *(i4*)((T*)p + at) = *(const i4*)&r;
  else
    ((T*)p)[at] = r.v[0];
}

// The sums of N values over the W waves of a row, the same in every lane.  `room` is N x waves
// floats per set, used in turns: a set is written again only after another meeting.
template <int W, int N>
__device__ __forceinline__ void add_up(float (&v)[N], float* room, int wave_in_wg, int& turn) {
#pragma unroll
  for (int n = 0; n < N; n++)
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v[n] += __shfl_xor(v[n], d);
  if constexpr (W > 1) {
    float* const set = room + (turn & 1) * (N * 16);
    turn++;
    const int first = wave_in_wg / W * W;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int n = 0; n < N; n++) set[n * 16 + wave_in_wg] = v[n];
    }
    __syncthreads();
    // (a lane a value and wave: all N sums by log W exchanges)
    static_assert(N * W <= 64, "");
    const int l = threadIdx.x & 63;
    float s = l < N * W ? set[l / W * 16 + first + l % W] : 0.f;
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) s += __shfl_xor(s, d);
#pragma unroll
    for (int n = 0; n < N; n++) v[n] = __shfl(s, n * W);
  }
}

constexpr int wg_waves(int w) { return w < 4 ? 4 : w; }

}  // namespace

// W waves a row, NV pieces a lane; a workgroup of four waves or more takes 4 / W rows at once
template <class T, int VEC, int NV, int W>
__global__ __launch_bounds__(64 * wg_waves(W)) void norm_kernel(NormArgs p) {
  constexpr int kRows = wg_waves(W) / W;  // rows of a workgroup
  __shared__ float room[2 * 16];
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & (64 * W - 1);  // in the row
  const float mean = 1.f / (float)p.d;
  int turn = 0;
  // (all sets of waves of a workgroup go round equally often: they meet at barriers)
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < p.rows; r0 += (long long)gridDim.x * kRows) {
    const long long row = r0 + wave / W;
    const bool live = row < p.rows;
    float r[NV][VEC];
    if (p.block) {
      Piece<T, VEC> b[NV], r_in[NV];
      float sum[1] = {0.f};
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = VEC * (64 * W * i + lane);
        if (live && c < p.d) {
          b[i] = load_piece<T, VEC>(p.block, (size_t)row * p.ld_block + c);
          r_in[i] = load_piece<T, VEC>(p.residual, (size_t)row * p.ld_residual + c);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e++) b[i].v[e] = r_in[i].v[e] = (T)0.f;
        }
      }
      float rstd = 1.f;
      if (p.post) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
          for (int e = 0; e < VEC; e++) sum[0] = __builtin_fmaf(b[i].at(e), b[i].at(e), sum[0]);
        add_up<W, 1>(sum, room, wave, turn);
        rstd = 1.f / __builtin_sqrtf(__builtin_fmaf(sum[0], mean, p.eps));
        if (p.stats && live && lane == 0) p.stats[2 * row] = rstd;
      }
      const size_t gate_row = p.gate && live ? (size_t)(row / p.rows_per_gate) * p.ld_gate : 0;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = VEC * (64 * W * i + lane);
        if (!live || c >= p.d) {
#pragma unroll
          for (int e = 0; e < VEC; e++) r[i][e] = 0.f;
          continue;
        }
        Piece<T, VEC> post, gate;
        if (p.post) post = load_piece<T, VEC>(p.post, c);
        if (p.gate) gate = load_piece<T, VEC>(p.gate, gate_row + c);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          float x = b[i].at(e);
          if (p.post) x *= rstd * post.at(e);
          if (p.gate) x *= gate.at(e);
          r[i][e] = __builtin_fmaf(p.scale, r_in[i].at(e), x);
        }
        store_piece<T, VEC>(p.r, (size_t)row * p.d + c, r[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = VEC * (64 * W * i + lane);
        const bool in = live && c < p.d;
        Piece<T, VEC> x;
        if (in) x = load_piece<T, VEC>(p.residual, (size_t)row * p.ld_residual + c);
#pragma unroll
        for (int e = 0; e < VEC; e++) r[i][e] = in ? x.at(e) : 0.f;
      }
    }
    if (!p.pre) continue;
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < VEC; e++) sum[0] = __builtin_fmaf(r[i][e], r[i][e], sum[0]);
    add_up<W, 1>(sum, room, wave, turn);
    const float rstd = 1.f / __builtin_sqrtf(__builtin_fmaf(sum[0], mean, p.eps));
    if (p.stats && live && lane == 0) p.stats[2 * row + 1] = rstd;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = VEC * (64 * W * i + lane);
      if (!live || c >= p.d) continue;
      const Piece<T, VEC> pre = load_piece<T, VEC>(p.pre, c);
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) y[e] = r[i][e] * rstd * pre.at(e);
      store_piece<T, VEC>(p.y, (size_t)row * p.d + c, y);
    }
  }
}

// What a lane holds over all its rows stays as it came from memory: without this the compiler
// keeps every weight as a float from before the loop, twice the registers, and with sixteen
// waves a row the sums are then spilled.
template <class T, int VEC>
__device__ __forceinline__ void as_stored(Piece<T, VEC>& v) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (VEC * sizeof(T) == 16) {
    i4 x = *(i4*)&v;
    asm volatile("" : "+v"(x));
    *(i4*)&v = x;
  }
#endif
}

// Sums over rows that a backward pass keeps: none; of dy rh and dt bh over a part of a gate's
// rows; or over whole gates, and then that of gate dt bh as well
enum Sums { kNoSums, kPartSums, kGateSums };

// A set of W waves takes one part.
template <class T, int VEC, int NV, int W, Sums SUMS>
__global__ __launch_bounds__(64 * wg_waves(W)) void norm_grad_kernel(NormGradArgs p, NormParts parts) {
  constexpr int kSets = wg_waves(W) / W;
  // (weights of more than eight elements a lane are read again for every row)
  constexpr bool kKeep = NV * VEC <= 8;
  __shared__ float room[2 * 4 * 16];
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & (64 * W - 1);
  const float mean = 1.f / (float)p.d;
  const long long part = (long long)blockIdx.x * kSets + wave / W;
  // my rows
  long long first = 0, last = 0;
  if (part < parts.parts) {
    if (parts.whole) {
      first = part * parts.rows_per_part;
      last = first + parts.rows_per_part;
      if (last > p.rows) last = p.rows;
    } else {
      const long long gate = part / parts.parts_per_gate, at = part - gate * parts.parts_per_gate;
      const long long of_gate = parts.gates == 1 ? p.rows : p.rows_per_gate;
      first = at * parts.rows_per_part;
      last = first + parts.rows_per_part;
      if (last > of_gate) last = of_gate;
      if (first > last) first = last;
      first += gate * of_gate;
      last += gate * of_gate;
    }
  }
  auto in = [&](int i) { return VEC * (64 * W * i + lane) < p.d; };
  auto column = [&](int i) { return VEC * (64 * W * i + lane); };
  auto weight = [&](const void* from, int i, size_t row_at) {
    Piece<T, VEC> v;
#pragma unroll
    for (int e = 0; e < VEC; e++) v.v[e] = (T)1.f;
    if (from && in(i)) v = load_piece<T, VEC>(from, row_at + column(i));
    return v;
  };
  Piece<T, VEC> post[kKeep ? NV : 1], pre[kKeep ? NV : 1], gate[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      post[i] = weight(p.post, i, 0);
      pre[i] = weight(p.pre, i, 0);
      gate[i] = weight(nullptr, i, 0);
    }
  }
  constexpr int kHeld = SUMS == kNoSums ? 1 : NV;
  float sum_pre[kHeld][VEC], q[kHeld][VEC], sum_post[SUMS == kGateSums ? NV : 1][VEC];
  if constexpr (SUMS != kNoSums) {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        sum_pre[i][e] = q[i][e] = 0.f;
        if constexpr (SUMS == kGateSums) sum_post[i][e] = 0.f;
      }
  }
  long long held = -1;  // the row of `gate` that q belongs to
  // a gate's sums are complete: where parts hold whole gates, its gradient is written here
  auto close_gate = [&] {
    if constexpr (SUMS == kGateSums) {
      if (held < 0) return;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const Piece<T, VEC> w = weight(p.post, i, 0), g = weight(p.gate, i, (size_t)held * p.ld_gate);
        float dgate[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          dgate[e] = w.at(e) * q[i][e];
          sum_post[i][e] = __builtin_fmaf(g.at(e), q[i][e], sum_post[i][e]);
          q[i][e] = 0.f;
        }
        if (p.dgate && in(i)) store_piece<T, VEC>(p.dgate, (size_t)held * p.d + column(i), dgate);
      }
    }
  };
  int turn = 0;
  // every set of a workgroup goes round equally often: they meet at barriers
  for (long long at = 0; at < parts.rows_per_part; at++) {
    const long long row = first + at;
    const bool live = row < last;
    if (kSets == 1 && !live) break;
    Piece<T, VEC> dy[NV], dr[NV], r[NV], b[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
#pragma unroll
      for (int e = 0; e < VEC; e++) dy[i].v[e] = dr[i].v[e] = r[i].v[e] = b[i].v[e] = (T)0.f;
      if (!live || !in(i)) continue;
      if (p.pre) {
        dy[i] = load_piece<T, VEC>(p.dy, (size_t)row * p.ld_dy + column(i));
        r[i] = load_piece<T, VEC>(p.r, (size_t)row * p.ld_r + column(i));
      }
      if (p.dr) dr[i] = load_piece<T, VEC>(p.dr, (size_t)row * p.ld_dr + column(i));
      if (p.block) b[i] = load_piece<T, VEC>(p.block, (size_t)row * p.ld_block + column(i));
    }
    const float rstd1 = live && p.post ? p.stats[2 * row] : 1.f;
    const float rstd2 = live && p.pre ? p.stats[2 * row + 1] : 0.f;
    if (live && p.block) {
      const long long g = row / p.rows_per_gate;
      if (g != held) {
        close_gate();
        held = g;
        if constexpr (kKeep) {
#pragma unroll
          for (int i = 0; i < NV; i++) gate[i] = weight(p.gate, i, (size_t)g * p.ld_gate);
        }
      }
    }
    // this row's weights of piece i
    struct Weights {
      Piece<T, VEC> post, pre, gate;
    };
    auto weights = [&](int i) {
      Weights w;
      if constexpr (kKeep) {
        as_stored(post[i]);
        as_stored(pre[i]);
        as_stored(gate[i]);
        w = {post[i], pre[i], gate[i]};
      } else {
        w = {weight(p.post, i, 0), weight(p.pre, i, 0), weight(p.gate, i, held < 0 ? 0 : (size_t)held * p.ld_gate)};
      }
      return w;
    };
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Weights w = weights(i);
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const float dyp = dy[i].at(e) * w.pre.at(e), rh = r[i].at(e) * rstd2;
        const float gpb = w.gate.at(e) * w.post.at(e) * (b[i].at(e) * rstd1);
        s[0] = __builtin_fmaf(dyp, rh, s[0]);
        s[1] = __builtin_fmaf(gpb, dr[i].at(e), s[1]);
        s[2] = __builtin_fmaf(gpb, dyp, s[2]);
        s[3] = __builtin_fmaf(gpb, rh, s[3]);
      }
    }
    add_up<W, 4>(s, room, wave, turn);
    const float m1 = s[0] * mean;
    const float m2 = p.post ? mean * (s[1] + rstd2 * (s[2] - m1 * s[3])) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (!live || !in(i)) continue;
      as_stored(dy[i]);
      as_stored(dr[i]);
      as_stored(r[i]);
      as_stored(b[i]);
      const Weights w = weights(i);
      float d0[VEC], db[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const float rh = r[i].at(e) * rstd2, bh = b[i].at(e) * rstd1;
        const float dt = __builtin_fmaf(rstd2, dy[i].at(e) * w.pre.at(e) - rh * m1, dr[i].at(e));
        d0[e] = p.scale * dt;
        db[e] = rstd1 * (dt * w.gate.at(e) * w.post.at(e) - bh * m2);
        if constexpr (SUMS != kNoSums) {
          sum_pre[i][e] = __builtin_fmaf(dy[i].at(e), rh, sum_pre[i][e]);
          q[i][e] = __builtin_fmaf(dt, bh, q[i][e]);
        }
      }
      if (p.dresidual) store_piece<T, VEC>(p.dresidual, (size_t)row * p.d + column(i), d0);
      if (p.dblock) store_piece<T, VEC>(p.dblock, (size_t)row * p.d + column(i), db);
    }
  }
  if constexpr (SUMS != kNoSums) {
    close_gate();
    if (part >= parts.parts) return;
    float* const out = p.partials + (size_t)part * 2 * p.d;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (!in(i)) continue;
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        out[column(i) + e] = sum_pre[i][e];
        out[p.d + column(i) + e] = SUMS == kGateSums ? sum_post[i % (SUMS == kGateSums ? NV : 1)][e] : q[i][e];
      }
    }
  }
}

// The parts' sums added in their order: 16 columns a workgroup, 16 lanes a column, lane l taking
// every 16th part.  q of a gate's parts gives its gradient and its share of dpost.
template <class T>
__global__ __launch_bounds__(256) void norm_sums_kernel(NormGradArgs p, NormParts parts) {
  __shared__ float room[2][16][17];
  const int x = threadIdx.x & 15, l = threadIdx.x >> 4;
  const int c = 16 * blockIdx.x + x;
  const bool in = c < p.d;
  const float post = in && p.post ? (float)((const T*)p.post)[c] : 1.f;
  float dpost = 0.f, dpre = 0.f;
  const long long runs = parts.whole ? 1 : parts.gates;
  const long long run = parts.whole ? parts.parts : parts.parts_per_gate;
  for (long long g = 0; g < runs; g++) {
    float a = 0.f, b = 0.f;
    if (in)
      for (long long i = l; i < run; i += 16) {
        const float* const from = p.partials + (size_t)(g * run + i) * 2 * p.d + c;
        a += from[0];
        b += from[p.d];
      }
    __syncthreads();
    room[0][l][x] = a;
    room[1][l][x] = b;
    __syncthreads();
    if (l == 0) {
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        a += room[0][i][x];
        b += room[1][i][x];
      }
      dpre += a;
      if (parts.whole) {
        dpost += b;
      } else {
        const float gate = in && p.gate ? (float)((const T*)p.gate)[(size_t)g * p.ld_gate + c] : 1.f;
        dpost = __builtin_fmaf(gate, b, dpost);
        if (in && p.dgate) ((T*)p.dgate)[(size_t)g * p.d + c] = (T)(post * b);
      }
    }
  }
  if (l == 0 && in) {
    if (p.dpre) ((T*)p.dpre)[c] = (T)dpre;
    if (p.dpost) ((T*)p.dpost)[c] = (T)dpost;
  }
}

namespace {

bool whole16(const void* p, long long ld, int per) { return ((uintptr_t)p & 15) == 0 && ld % per == 0; }

// Pieces of a lane and waves of a row: one piece as long as sixteen waves hold the row
struct NormShape {
  int nv, waves;
};
NormShape norm_shape(int d, int vec) {
  const int pieces = (d + vec - 1) / vec;
  int waves = 1;
  while (waves < 16 && 64 * waves < pieces) waves *= 2;
  int nv = 1;
  while (64 * waves * nv < pieces) nv *= 2;
  return {nv, waves};
}

template <class T, int VEC, class F>
void with_shape(int d, F f) {
  const NormShape s = norm_shape(d, VEC);
  using std::integral_constant;
#define SHAPE(NV, W) \
  if (s.nv == NV && s.waves == W) return f(integral_constant<int, NV>{}, integral_constant<int, W>{});
  SHAPE(1, 1)
  SHAPE(1, 2)
  SHAPE(1, 4)
  SHAPE(1, 8)
  SHAPE(1, 16)
  SHAPE(2, 16)
  if constexpr (VEC <= 4) { SHAPE(4, 16) }
  if constexpr (VEC == 1) { SHAPE(8, 16) SHAPE(16, 16) }
#undef SHAPE
}

template <class T, class F>
void with_vectors(bool vectors, F f) {
  if (vectors)
    f(std::integral_constant<int, 16 / sizeof(T)>{});
  else
    f(std::integral_constant<int, 1>{});
}

template <class F>
void with_type(NormType type, F f) {
  if (type == kNormFp16) f((half_t)0);
  if (type == kNormBf16) f((bf)0);
  if (type == kNormFp32) f(0.f);
}

constexpr int kPartWaves = 4096;  // waves that the parts of a backward pass make up

}  // namespace

bool norm_vectors(const NormArgs& a, int size) {
  const int per = 16 / size;
  return a.d % per == 0 && whole16(a.residual, a.ld_residual, per) && whole16(a.block, a.ld_block, per) &&
         whole16(a.gate, a.ld_gate, per) && whole16(a.post, 0, per) && whole16(a.pre, 0, per) &&
         whole16(a.r, 0, per) && whole16(a.y, 0, per);
}
bool norm_vectors(const NormGradArgs& a, int size) {
  const int per = 16 / size;
  return a.d % per == 0 && whole16(a.dy, a.ld_dy, per) && whole16(a.dr, a.ld_dr, per) && whole16(a.r, a.ld_r, per) &&
         whole16(a.block, a.ld_block, per) && whole16(a.gate, a.ld_gate, per) && whole16(a.post, 0, per) &&
         whole16(a.pre, 0, per) && whole16(a.dresidual, 0, per) && whole16(a.dblock, 0, per) && whole16(a.dgate, 0, per);
}

NormParts norm_parts(long long rows, int rows_per_gate, int d, int size, bool vectors) {
  NormParts p = {};
  p.waves = norm_shape(d, vectors ? 16 / size : 1).waves;
  const long long most = kPartWaves / p.waves;
  p.gates = (rows + rows_per_gate - 1) / rows_per_gate;
  p.whole = p.gates > most;
  if (p.whole) {
    const long long gates_per_part = (p.gates + most - 1) / most;
    p.rows_per_part = gates_per_part * rows_per_gate;
    p.parts = (p.gates + gates_per_part - 1) / gates_per_part;
    p.parts_per_gate = 0;
  } else {
    const long long of_gate = p.gates <= 1 ? rows : rows_per_gate;
    p.parts_per_gate = std::max<long long>(1, std::min<long long>(most / std::max<long long>(p.gates, 1), of_gate));
    p.rows_per_part = (of_gate + p.parts_per_gate - 1) / p.parts_per_gate;
    p.parts_per_gate = (of_gate + p.rows_per_part - 1) / std::max<long long>(p.rows_per_part, 1);
    p.parts = p.gates * p.parts_per_gate;
  }
  p.bytes = (size_t)p.parts * 2 * d * sizeof(float);
  return p;
}

void launch_norm(const NormArgs& a, NormType type, int cus, hipStream_t stream) {
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    with_vectors<T>(norm_vectors(a, sizeof(T)), [&](auto vec) {
      with_shape<T, decltype(vec)::value>(a.d, [&](auto nv, auto w) {
        constexpr int VEC = decltype(vec)::value, NV = decltype(nv)::value, W = decltype(w)::value;
        constexpr int rows = wg_waves(W) / W;
        const long long groups = (a.rows + rows - 1) / rows, most = 0x7fffffff;
        hipLaunchKernelGGL((norm_kernel<T, VEC, NV, W>), dim3((unsigned)std::min(groups, most)),
                           dim3(64 * wg_waves(W)), 0, stream, a);
      });
    });
  });
}

void launch_norm_grad(const NormGradArgs& a, NormType type, hipStream_t stream) {
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    const bool vectors = norm_vectors(a, sizeof(T));
    const NormParts parts = norm_parts(a.rows, a.rows_per_gate, a.d, sizeof(T), vectors);
    with_vectors<T>(vectors, [&](auto vec) {
      with_shape<T, decltype(vec)::value>(a.d, [&](auto nv, auto w) {
        constexpr int VEC = decltype(vec)::value, NV = decltype(nv)::value, W = decltype(w)::value;
        constexpr int sets = wg_waves(W) / W;
        const dim3 grid((unsigned)((parts.parts + sets - 1) / sets)), block(64 * wg_waves(W));
        if (!a.partials)
          hipLaunchKernelGGL((norm_grad_kernel<T, VEC, NV, W, kNoSums>), grid, block, 0, stream, a, parts);
        else if (parts.whole)
          hipLaunchKernelGGL((norm_grad_kernel<T, VEC, NV, W, kGateSums>), grid, block, 0, stream, a, parts);
        else
          hipLaunchKernelGGL((norm_grad_kernel<T, VEC, NV, W, kPartSums>), grid, block, 0, stream, a, parts);
      });
    });
    if (a.partials)
      hipLaunchKernelGGL(norm_sums_kernel<T>, dim3((a.d + 15) / 16), dim3(256), 0, stream, a, parts);
  });
}

}  // namespace w4a16
