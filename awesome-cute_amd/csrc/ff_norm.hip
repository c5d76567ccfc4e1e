// The norms after a block and before the next one, with the block's gate and the residual's
// scale, and their gradients: per row b (the block's output) and r0 (the residual)
//
//   p = b rstd(b) post      rstd(v) = 1 / sqrt(mean(v^2) + eps)      (p = b without `post`)
//   r = scale r0 + gate p                                            (r = r0 without a block)
//   y = r rstd(r) pre
//
// in fp32 from inputs in 16 or 32 bits, r and y rounded once (y from the unrounded r).  The backward
// pass takes r as it was rounded, the value that the model goes on with: it is kept anyhow, where
// one in fp32 would be twice the bytes; the gradients are off by 0.0023 of their length instead of
// the 0.0017 that their own rounding makes (bfloat16).  With
// bh = b rstd(b), rh = r rstd(r) and the gradients dy and dr of y and r
//
//   dt = dr + rstd(r) (dy pre - rh mean(dy pre rh))       dr0 = scale dt      dpre = sum dy rh
//   db = rstd(b) (w - bh mean(w bh)),  w = dt gate post   q = sum dt bh: dgate = post q, dpost = gate q
//
// the sums over the rows that share a weight or a gate.
//
// Bound: HBM; every row is read and written once.  8192 rows of 8192 in bfloat16 110 us, 4.9 TB/s, by
// one norm alone 48, 5.6; 4096 rows of 4096 26 us and backward 45, 4.5 TB/s, and 6 for the sums over
// parts; one row 3.7.  A wave is the least that takes a row: of 64 elements in 16 bits eight lanes
// hold some, and 262144 such rows take 99 us, 1.4 TB/s.
// A row is kept in the registers of W waves, a 16-byte piece a lane, of the longest rows two or (fp32)
// four, so that the second pass over it that a norm needs costs nothing; the waves' sums meet in
// LDS, two meetings a row forward.  Backward one: mean(w bh) is put together from four sums, of dy
// pre rh, and of gate post bh times dr, dy pre and rh.
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
typedef int i4_anywhere __attribute__((ext_vector_type(4), aligned(2)));

// 16 bytes of a row as they come from memory, and as floats
template <class T>
struct Piece {
  static constexpr int kN = 16 / sizeof(T);
  T v[kN];
  __device__ __forceinline__ float at(int i) const { return (float)v[i]; }
};
template <class T>
__device__ __forceinline__ Piece<T> piece_of(float x) {
  Piece<T> r;
#pragma unroll
  for (int i = 0; i < Piece<T>::kN; i++) r.v[i] = (T)x;
  return r;
}
// WHOLE: rows are whole pieces that start on 16 bytes.  Otherwise a piece may lie anywhere (the
// hardware's 16-byte loads to registers take any address), and the last of a row holds `left`
// elements, fetched one by one, zeros behind them.
template <bool WHOLE, class T>
__device__ __forceinline__ Piece<T> load_piece(const T* p, int left) {
  Piece<T> r;
  if constexpr (WHOLE) {
    *(i4*)&r = *(const i4*)p;
  } else if (left >= Piece<T>::kN) {
    *(i4*)&r = *(const i4_anywhere*)p;
  } else {
    r = piece_of<T>(0.f);
#pragma unroll
    for (int i = 0; i < Piece<T>::kN - 1; i++)
      if (i < left) r.v[i] = p[i];
  }
  return r;
}
template <bool WHOLE, class T>
__device__ __forceinline__ void store_piece(T* p, int left, const float* f) {
  Piece<T> r;
#pragma unroll
  for (int i = 0; i < Piece<T>::kN; i++) r.v[i] = (T)f[i];
  if constexpr (WHOLE) {
    *(i4*)p = *(const i4*)&r;
  } else if (left >= Piece<T>::kN) {
    *(i4_anywhere*)p = *(const i4*)&r;
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::kN - 1; i++)
      if (i < left) p[i] = r.v[i];
  }
}

// What a lane holds over all its rows stays as it came from memory: without this the compiler
// keeps every weight as a float from before the loop, twice the registers.
template <class T>
__device__ __forceinline__ void as_stored(Piece<T>& v) {
#if defined(__HIP_DEVICE_COMPILE__)
  i4 x = *(i4*)&v;
  asm volatile("" : "+v"(x));
  *(i4*)&v = x;
#endif
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
    const int l = threadIdx.x & 63;
    if (l == 0) {
#pragma unroll
      for (int n = 0; n < N; n++) set[n * 16 + wave_in_wg] = v[n];
    }
#if defined(__HIP_DEVICE_COMPILE__)
    // (only LDS is exchanged: the next row stays on its way)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
    // a lane a value and wave: all N sums by log W exchanges
    static_assert(N * W <= 64, "");
    float s = l < N * W ? set[l / W * 16 + first + l % W] : 0.f;
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) s += __shfl_xor(s, d);
#pragma unroll
    for (int n = 0; n < N; n++) v[n] = __shfl(s, n * W);
  }
}

__device__ __forceinline__ float rstd_of(float sum, float mean, float eps) {
  return 1.f / __builtin_sqrtf(__builtin_fmaf(sum, mean, eps));
}

constexpr int wg_waves(int w) { return w < 4 ? 4 : w; }

// Where a lane's pieces lie in a row
template <class T, int NV, int W>
struct Lane {
  int d, lane;
  __device__ __forceinline__ Lane(int d_) : d(d_), lane((int)threadIdx.x & (64 * W - 1)) {}
  __device__ __forceinline__ int column(int i) const { return Piece<T>::kN * (64 * W * i + lane); }
  __device__ __forceinline__ int left(int i) const { return d - column(i); }
  __device__ __forceinline__ bool in(int i) const { return column(i) < d; }
};

}  // namespace

// W waves a row, NV pieces a lane; a workgroup of four waves or more takes 4 / W rows at once.
// A set of W waves takes a run of rows; the next row is requested before this one's lengths are
// known, and the weights stay in registers where a lane holds few of them.
template <class T, bool WHOLE, int NV, int W>
__global__ __launch_bounds__(64 * wg_waves(W)) void norm_kernel(NormArgs p, int sets) {
  constexpr int kSets = wg_waves(W) / W, kN = Piece<T>::kN;
  constexpr bool kKeep = NV * kN <= 8;
  __shared__ float room[2 * 16];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Lane<T, NV, W> me(p.d);
  const float mean = 1.f / (float)p.d;
  const int set = (int)blockIdx.x * kSets + wave / W, rows = (int)p.rows;
  const int longest = (rows + sets - 1) / sets;
  const int first = (int)((long long)rows * set / sets);
  const int last = set < sets ? (int)((long long)rows * (set + 1) / sets) : first;
  auto load = [&](const void* base, long long at, int i) {
    return load_piece<WHOLE>((const T*)base + at + me.column(i), me.left(i));
  };
  Piece<T> post[kKeep ? NV : 1], gate[kKeep ? NV : 1], pre[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      post[i] = gate[i] = pre[i] = piece_of<T>(1.f);
      if (p.post && me.in(i)) post[i] = load(p.post, 0, i);
      if (p.pre && me.in(i)) pre[i] = load(p.pre, 0, i);
    }
  }
  Piece<T> b[NV], x[NV];
  auto fetch = [&](int row) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      b[i] = x[i] = piece_of<T>(0.f);
      if (row >= last || !me.in(i)) continue;
      if (p.block) b[i] = load(p.block, row * p.ld_block, i);
      x[i] = load(p.residual, row * p.ld_residual, i);
    }
  };
  int turn = 0, held = -1;
  fetch(first);
  // (all sets of a workgroup go round equally often: they meet at barriers)
  for (int at = 0; at < longest; at++) {
    const int row = first + at;
    const bool live = row < last;
    float r[NV][kN];
    if (p.block) {
      float sum[1] = {0.f}, rstd = 1.f;
      if (p.post) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
          for (int e = 0; e < kN; e++) sum[0] = __builtin_fmaf(b[i].at(e), b[i].at(e), sum[0]);
      }
      const int g = p.gate && live ? (int)((unsigned)row / (unsigned)p.rows_per_gate) : held;
      if (kKeep && g != held) {
#pragma unroll
        for (int i = 0; i < NV; i++)
          if (me.in(i)) gate[kKeep ? i : 0] = load(p.gate, g * p.ld_gate, i);
      }
      held = g;
      if (p.post) {
        add_up<W, 1>(sum, room, wave, turn);
        rstd = rstd_of(sum[0], mean, p.eps);
        if (p.stats && live && me.lane == 0) p.stats[2 * (size_t)row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        Piece<T> w = piece_of<T>(1.f), gt = w;
        if constexpr (kKeep) {
          as_stored(post[i]);
          as_stored(gate[i]);
          w = post[i];
          gt = gate[i];
        } else if (me.in(i)) {
          if (p.post) w = load(p.post, 0, i);
          if (p.gate && held >= 0) gt = load(p.gate, held * p.ld_gate, i);
        }
#pragma unroll
        for (int e = 0; e < kN; e++)
          r[i][e] = __builtin_fmaf(p.scale, x[i].at(e), b[i].at(e) * (rstd * w.at(e)) * gt.at(e));
        if (live && me.in(i))
          store_piece<WHOLE>((T*)p.r + (long long)row * p.d + me.column(i), me.left(i), r[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < kN; e++) r[i][e] = x[i].at(e);
    }
    fetch(row + 1);
    if (!p.pre) continue;
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < kN; e++) sum[0] = __builtin_fmaf(r[i][e], r[i][e], sum[0]);
    add_up<W, 1>(sum, room, wave, turn);
    const float rstd = rstd_of(sum[0], mean, p.eps);
    if (p.stats && live && me.lane == 0) p.stats[2 * (size_t)row + 1] = rstd;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (!live || !me.in(i)) continue;
      Piece<T> w;
      if constexpr (kKeep) {
        as_stored(pre[i]);
        w = pre[i];
      } else {
        w = load(p.pre, 0, i);
      }
      float y[kN];
#pragma unroll
      for (int e = 0; e < kN; e++) y[e] = r[i][e] * rstd * w.at(e);
      store_piece<WHOLE>((T*)p.y + (long long)row * p.d + me.column(i), me.left(i), y);
    }
  }
}

// Sums over rows that a backward pass keeps: none; of dy rh and dt bh over a part of a gate's
// rows; or over whole gates, and then that of gate dt bh as well
enum Sums { kNoSums, kPartSums, kGateSums };

// A set of W waves takes one part.
template <class T, bool WHOLE, int NV, int W, Sums SUMS>
__global__ __launch_bounds__(64 * wg_waves(W)) void norm_grad_kernel(NormGradArgs p, NormParts parts) {
  constexpr int kSets = wg_waves(W) / W, kN = Piece<T>::kN;
  // (of more than eight elements a lane the weights are read again for every row, and no row is
  // requested ahead: sixteen waves have 128 registers each, and the sums take most of them)
  constexpr bool kKeep = NV * kN <= 8;
  __shared__ float room[2 * 4 * 16];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Lane<T, NV, W> me(p.d);
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
  auto load = [&](const void* base, long long at, int i) {
    return load_piece<WHOLE>((const T*)base + at + me.column(i), me.left(i));
  };
  auto weight = [&](const void* from, int i, long long row_at) {
    return from && me.in(i) ? load(from, row_at, i) : piece_of<T>(1.f);
  };
  Piece<T> post[kKeep ? NV : 1], pre[kKeep ? NV : 1], gate[kKeep ? NV : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      post[i] = weight(p.post, i, 0);
      pre[i] = weight(p.pre, i, 0);
      gate[i] = piece_of<T>(1.f);
    }
  }
  constexpr int kHeld = SUMS == kNoSums ? 1 : NV;
  float sum_pre[kHeld][kN], q[kHeld][kN], sum_post[SUMS == kGateSums ? NV : 1][kN];
  if constexpr (SUMS != kNoSums) {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < kN; e++) {
        sum_pre[i][e] = q[i][e] = 0.f;
        if constexpr (SUMS == kGateSums) sum_post[i][e] = 0.f;
      }
  }
  int held = -1;  // the row of `gate` that q belongs to
  // a gate's sums are complete: where parts hold whole gates, its gradient is written here
  auto close_gate = [&] {
    if constexpr (SUMS == kGateSums) {
      if (held < 0) return;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const Piece<T> w = weight(p.post, i, 0), g = weight(p.gate, i, held * p.ld_gate);
        float dgate[kN];
#pragma unroll
        for (int e = 0; e < kN; e++) {
          dgate[e] = w.at(e) * q[i][e];
          sum_post[i][e] = __builtin_fmaf(g.at(e), q[i][e], sum_post[i][e]);
          q[i][e] = 0.f;
        }
        if (p.dgate && me.in(i))
          store_piece<WHOLE>((T*)p.dgate + (long long)held * p.d + me.column(i), me.left(i), dgate);
      }
    }
  };
  Piece<T> dy[NV], dr[NV], r[NV], b[NV];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      dy[i] = dr[i] = r[i] = b[i] = piece_of<T>(0.f);
      if (row >= last || !me.in(i)) continue;
      if (p.pre) {
        dy[i] = load(p.dy, row * p.ld_dy, i);
        r[i] = load(p.r, row * p.ld_r, i);
      }
      if (p.dr) dr[i] = load(p.dr, row * p.ld_dr, i);
      if (p.block) b[i] = load(p.block, row * p.ld_block, i);
    }
  };
  int turn = 0;
  if (kKeep) fetch(first);
  // every set of a workgroup goes round equally often: they meet at barriers
  for (long long at = 0; at < parts.rows_per_part; at++) {
    const long long row = first + at;
    const bool live = row < last;
    if (kSets == 1 && !live) break;
    if (!kKeep) fetch(row);
    const float rstd1 = live && p.post ? p.stats[2 * row] : 1.f;
    const float rstd2 = live && p.pre ? p.stats[2 * row + 1] : 0.f;
    if (live && p.block) {
      const int g = (int)((unsigned)row / (unsigned)p.rows_per_gate);
      if (g != held) {
        close_gate();
        held = g;
        if constexpr (kKeep) {
#pragma unroll
          for (int i = 0; i < NV; i++) gate[i] = weight(p.gate, i, g * p.ld_gate);
        }
      }
    }
    // this row's weights of piece i
    struct Weights {
      Piece<T> post, pre, gate;
    };
    auto weights = [&](int i) {
      Weights w;
      if constexpr (kKeep) {
        as_stored(post[i]);
        as_stored(pre[i]);
        as_stored(gate[i]);
        w = {post[i], pre[i], gate[i]};
      } else {
        w = {weight(p.post, i, 0), weight(p.pre, i, 0), weight(p.gate, i, held < 0 ? 0 : held * p.ld_gate)};
      }
      return w;
    };
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const Weights w = weights(i);
#pragma unroll
      for (int e = 0; e < kN; e++) {
        const float dyp = dy[i].at(e) * w.pre.at(e), rh = r[i].at(e) * rstd2;
        const float gpb = w.gate.at(e) * w.post.at(e) * (b[i].at(e) * rstd1);
        s[0] = __builtin_fmaf(dyp, rh, s[0]);
        s[1] = __builtin_fmaf(gpb, dr[i].at(e), s[1]);
        s[2] = __builtin_fmaf(gpb, dyp, s[2]);
        s[3] = __builtin_fmaf(gpb, rh, s[3]);
      }
    }
    Piece<T> this_dy[NV], this_dr[NV], this_r[NV], this_b[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      this_dy[i] = dy[i];
      this_dr[i] = dr[i];
      this_r[i] = r[i];
      this_b[i] = b[i];
    }
    if (kKeep) fetch(row + 1);
    add_up<W, 4>(s, room, wave, turn);
    const float m1 = s[0] * mean;
    const float m2 = p.post ? mean * (s[1] + rstd2 * (s[2] - m1 * s[3])) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (!live || !me.in(i)) continue;
      as_stored(this_dy[i]);
      as_stored(this_dr[i]);
      as_stored(this_r[i]);
      as_stored(this_b[i]);
      const Weights w = weights(i);
      float d0[kN], db[kN];
#pragma unroll
      for (int e = 0; e < kN; e++) {
        const float rh = this_r[i].at(e) * rstd2, bh = this_b[i].at(e) * rstd1, dye = this_dy[i].at(e);
        const float dt = __builtin_fmaf(rstd2, dye * w.pre.at(e) - rh * m1, this_dr[i].at(e));
        d0[e] = p.scale * dt;
        // (without a norm after the block its values, infinite ones too, are no part of its gradient)
        db[e] = rstd1 * (dt * w.gate.at(e) * w.post.at(e) - (p.post ? bh : 0.f) * m2);
        if constexpr (SUMS != kNoSums) {
          sum_pre[i][e] = __builtin_fmaf(dye, rh, sum_pre[i][e]);
          q[i][e] = __builtin_fmaf(dt, bh, q[i][e]);
        }
      }
      const long long at_row = row * p.d + me.column(i);
      if (p.dresidual) store_piece<WHOLE>((T*)p.dresidual + at_row, me.left(i), d0);
      if (p.dblock) store_piece<WHOLE>((T*)p.dblock + at_row, me.left(i), db);
    }
  }
  if constexpr (SUMS != kNoSums) {
    close_gate();
    if (part >= parts.parts) return;
    float* const out = p.partials + part * 2 * p.d;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < kN; e++) {
        if (me.left(i) <= e) continue;
        out[me.column(i) + e] = sum_pre[i][e];
        out[p.d + me.column(i) + e] = SUMS == kGateSums ? sum_post[i % (SUMS == kGateSums ? NV : 1)][e] : q[i][e];
      }
  }
}

// The parts' sums added in their order: 64 columns and 16 waves a workgroup, a wave every
// sixteenth part.  y = 0: of dt bh, which for a gate's parts gives its gradient and its share of
// dpost; there `wpg` waves share a gate (few gates), or a wave takes every sixteenth gate.
// y = 1: of dy rh.
template <class T>
__global__ __launch_bounds__(1024) void norm_sums_kernel(NormGradArgs p, NormParts parts, int wpg) {
  __shared__ float room[16][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = 64 * blockIdx.x + lane;
  const bool in = c < p.d;
  const int at = in ? c : 0;
  // the parts first, first + step ... < last
  auto add = [&](long long first, long long last, long long step, const float* from) {
    float s = 0.f;
#pragma unroll 8
    for (long long i = first; i < last; i += step) s += from[i * 2 * p.d];
    return s;
  };
  if (blockIdx.y == 1) {
    room[wave][lane] = add(wave, parts.parts, 16, p.partials + at);
  } else if (parts.whole) {
    room[wave][lane] = add(wave, parts.parts, 16, p.partials + p.d + at);
  } else {
    const float post = in && p.post ? (float)((const T*)p.post)[c] : 1.f;
    const long long run = parts.parts_per_gate;
    auto gate_of = [&](long long g) { return in && p.gate ? (float)((const T*)p.gate)[g * p.ld_gate + c] : 1.f; };
    float dpost = 0.f;
    if (wpg == 1) {
      for (long long g = wave; g < parts.gates; g += 16) {
        const float q = add(0, run, 1, p.partials + g * run * 2 * p.d + p.d + at);
        if (in && p.dgate) ((T*)p.dgate)[g * p.d + c] = (T)(post * q);
        dpost = __builtin_fmaf(gate_of(g), q, dpost);
      }
    } else {  // (16 / wpg sets of waves, no fewer than there are gates)
      const long long g = wave / wpg;
      room[wave][lane] = g < parts.gates ? add(wave % wpg, run, wpg, p.partials + g * run * 2 * p.d + p.d + at) : 0.f;
      __syncthreads();
      if (wave % wpg == 0 && g < parts.gates) {
        float q = 0.f;
        for (int i = 0; i < wpg; i++) q += room[wave + i][lane];
        if (in && p.dgate) ((T*)p.dgate)[g * p.d + c] = (T)(post * q);
        dpost = gate_of(g) * q;
      }
      __syncthreads();
    }
    room[wave][lane] = dpost;
  }
  __syncthreads();
  T* const out = (T*)(blockIdx.y == 1 ? p.dpre : p.dpost);
  if (wave != 0 || !in || !out) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) s += room[i][lane];
  out[c] = (T)s;
}

namespace {

bool whole16(const void* p, long long ld, int per) { return ((uintptr_t)p & 15) == 0 && ld % per == 0; }

// Pieces of a lane and waves of a row: one piece as long as sixteen waves hold the row
struct NormShape {
  int nv, waves;
};
NormShape norm_shape(int d, int size) {
  const int pieces = (d * size + 15) / 16;
  int waves = 1;
  while (waves < 16 && 64 * waves < pieces) waves *= 2;
  int nv = 1;
  while (64 * waves * nv < pieces) nv *= 2;
  return {nv, waves};
}

template <class T, class F>
void with_shape(int d, F f) {
  const NormShape s = norm_shape(d, sizeof(T));
  using std::integral_constant;
#define SHAPE(NV, W) \
  if (s.nv == NV && s.waves == W) return f(integral_constant<int, NV>{}, integral_constant<int, W>{});
  SHAPE(1, 1)
  SHAPE(1, 2)
  SHAPE(1, 4)
  SHAPE(1, 8)
  SHAPE(1, 16)
  SHAPE(2, 16)
  if constexpr (sizeof(T) == 4) { SHAPE(4, 16) }
#undef SHAPE
}

template <class F>
void with_whole(bool whole, F f) {
  if (whole)
    f(std::true_type{});
  else
    f(std::false_type{});
}

template <class F>
void with_type(NormType type, F f) {
  if (type == kNormFp16) f((half_t)0);
  if (type == kNormBf16) f((bf)0);
  if (type == kNormFp32) f(0.f);
}

constexpr int kPartWaves = 4096;  // waves that the parts of a backward pass make up

}  // namespace

namespace {

bool norm_whole(const NormArgs& a, int size) {
  const int per = 16 / size;
  return a.d % per == 0 && whole16(a.residual, a.ld_residual, per) && whole16(a.block, a.ld_block, per) &&
         whole16(a.gate, a.ld_gate, per) && whole16(a.post, 0, per) && whole16(a.pre, 0, per) &&
         whole16(a.r, 0, per) && whole16(a.y, 0, per);
}
bool norm_whole(const NormGradArgs& a, int size) {
  const int per = 16 / size;
  return a.d % per == 0 && whole16(a.dy, a.ld_dy, per) && whole16(a.dr, a.ld_dr, per) && whole16(a.r, a.ld_r, per) &&
         whole16(a.block, a.ld_block, per) && whole16(a.gate, a.ld_gate, per) && whole16(a.post, 0, per) &&
         whole16(a.pre, 0, per) && whole16(a.dresidual, 0, per) && whole16(a.dblock, 0, per) && whole16(a.dgate, 0, per);
}

}  // namespace

NormParts norm_parts(long long rows, int rows_per_gate, int d, int size) {
  NormParts p = {};
  const long long most = kPartWaves / norm_shape(d, size).waves;
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
    with_whole(norm_whole(a, sizeof(T)), [&](auto whole) {
      with_shape<T>(a.d, [&](auto nv, auto w) {
        constexpr int NV = decltype(nv)::value, W = decltype(w)::value, per_wg = wg_waves(W) / W;
        // as many sets of waves as the chip holds, 32 waves to a compute unit
        const int sets = (int)std::min<long long>(a.rows, (long long)cus * 32 / W);
        hipLaunchKernelGGL((norm_kernel<T, decltype(whole)::value, NV, W>), dim3((sets + per_wg - 1) / per_wg),
                           dim3(64 * wg_waves(W)), 0, stream, a, sets);
      });
    });
  });
}

void launch_norm_grad(const NormGradArgs& a, NormType type, hipStream_t stream) {
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    const NormParts parts = norm_parts(a.rows, a.rows_per_gate, a.d, sizeof(T));
    with_whole(norm_whole(a, sizeof(T)), [&](auto whole) {
      with_shape<T>(a.d, [&](auto nv, auto w) {
        constexpr bool WHOLE = decltype(whole)::value;
        constexpr int NV = decltype(nv)::value, W = decltype(w)::value, per_wg = wg_waves(W) / W;
        const dim3 grid((unsigned)((parts.parts + per_wg - 1) / per_wg)), block(64 * wg_waves(W));
        if (!a.partials)
          hipLaunchKernelGGL((norm_grad_kernel<T, WHOLE, NV, W, kNoSums>), grid, block, 0, stream, a, parts);
        else if (parts.whole)
          hipLaunchKernelGGL((norm_grad_kernel<T, WHOLE, NV, W, kGateSums>), grid, block, 0, stream, a, parts);
        else
          hipLaunchKernelGGL((norm_grad_kernel<T, WHOLE, NV, W, kPartSums>), grid, block, 0, stream, a, parts);
      });
    });
    if (a.partials) {
      int wpg = 16;  // waves that share a gate's parts
      while (wpg > 1 && (long long)(16 / wpg) < parts.gates) wpg /= 2;
      hipLaunchKernelGGL(norm_sums_kernel<T>, dim3((a.d + 63) / 64, a.dpre ? 2 : 1), dim3(1024), 0, stream, a, parts, wpg);
    }
  });
}

}  // namespace w4a16
