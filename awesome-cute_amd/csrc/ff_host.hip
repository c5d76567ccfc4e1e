// C ABI of the feed-forward block's dense parts (include/feedforward_amd.h): checks, the
// choice of kernel, launches.  Nothing here allocates, waits or keeps anything of a call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <mutex>

#include "../../include/feedforward_amd.h"
#include "ff_grads.hpp"
#include "ff_norm.hpp"
#include "ff_products.hpp"

namespace {

using namespace w4a16;

constexpr int kMaxDevices = 16;
thread_local char g_error[256] = "";
thread_local FfTile t_tile = {0, 0};  // feedforward_force_tile
thread_local int t_slices = 0;
thread_local int t_polls = -1;  // feedforward_force_polls

int fail(int code, const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, args);
  va_end(args);
  return code;
}

struct Device {
  int cus = 0;
  bool configured = false;
};
std::mutex g_mu;
Device g_dev[kMaxDevices];

// Runs `launch(cus)` with `dev` current; the kernels' LDS limits are raised by the first call
// on a device.
template <class F>
int on_device(int dev, F launch) {
  if (dev < 0 || dev >= kMaxDevices) return fail(FEEDFORWARD_ERR_RUNTIME, "device index %d out of range", dev);
  int prev = -1;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != dev) e = hipSetDevice(dev);
  if (e != hipSuccess) return fail(FEEDFORWARD_ERR_RUNTIME, "hipSetDevice: %s", hipGetErrorString(e));
  int rc = FEEDFORWARD_OK, cus = 0;
  {
    std::lock_guard<std::mutex> lk(g_mu);
    Device& d = g_dev[dev];
    if (!d.configured) {
      e = hipDeviceGetAttribute(&d.cus, hipDeviceAttributeMultiprocessorCount, dev);
      if (e == hipSuccess) e = configure_product_tiles();
      if (e == hipSuccess) e = configure_product_big_f16();
      if (e == hipSuccess) e = configure_product_big_bf16();
      if (e == hipSuccess) e = configure_product_rows();
      d.configured = e == hipSuccess;
    }
    cus = d.cus;
  }
  if (e == hipSuccess) {
    (void)hipGetLastError();  // an earlier call's error is not this launch's
    launch(cus);
    e = hipGetLastError();
  }
  if (e != hipSuccess) rc = fail(FEEDFORWARD_ERR_RUNTIME, "HIP runtime error: %s", hipGetErrorString(e));
  if (prev != dev) (void)hipSetDevice(prev);
  return rc;
}

// Costs of the tiles in us, as in f16_tiles.hip: a launch, a stage of 64 k-values (dearer the
// fuller the chip), and workgroups beyond one per compute unit.  Fitted to every tile that can
// compute them on 9000 problems, m = 16 ... 8192, widths of 64 to 22016, forward and of the
// backward pass, operands from memory; 5 to 12 % rms (before big tiles took every depth, and before
// one tile's weights were requested as read once).  On 8600 others, with the kernels as they are, the
// choice takes 1.012 of the best tile and slices measured, 1.20 at the 99th percentile and 1.85 at
// worst.  Without any one of the tiles it would be 1.014 to 1.023, without that of 64 x 64 1.116;
// without slices 1.147.  Sixteen slices gain 0.15 % where known, and lose as much by the fit.
struct TileFit {
  FfTile tile;
  double launch, stage, fill, more, more_stage;
};
constexpr TileFit kFits[] = {
    {{64, 64}, 4.26, 0.220, 0.085, 0.66, 0.241}, {{64, 128}, 4.64, 0.340, 0.161, 2.60, 0.452},
    {{96, 128}, 4.70, 0.404, 0.206, 2.68, 0.537}, {{128, 128}, 4.82, 0.459, 0.258, 3.00, 0.625},
    {{96, 256}, 5.28, 0.594, 0.439, 4.03, 0.838}, {{128, 256}, 5.34, 0.748, 0.456, 4.59, 1.004},
    {{160, 256}, 7.68, 0.793, 0.380, 6.47, 1.094}, {{192, 256}, 8.23, 0.911, 0.424, 7.35, 1.256},
    {{224, 256}, 9.14, 1.044, 0.434, 8.56, 1.394}, {{256, 256}, 9.25, 1.104, 0.531, 9.57, 1.483}};
// Tiles of full products (feedforward_linear) alone, beside those above: problems of a few 64 x 64 tiles.
// Fitted to 400 problems of 23 to 4096 rows, widths of 64 to 11585 and depths of 64 to 8192, operands from
// memory, and brought to the others' level by what these cost there.  On 500 more problems, drawn alike, 196 take
// them, and 0.836 of the time (at best 0.60: 200 x 1024 x 2048 9.2 -> 6.1 us; at worst 1.12).
// (Other products' plans, and with them their results' last bits, are as they were.)
constexpr TileFit kSmallFits[] = {{{32, 32}, 4.05, 0.129, 0.031, 1.09, 0.138}, {{32, 64}, 4.18, 0.183, 0.088, 1.17, 0.214}};
// The same of the kernel for few rows (ff_rows.hip) by its blocks of sixteen rows of A, a stage
// being the 64 k-values of one of its four waves: one block of product columns to a workgroup, or
// two.  Fitted to 12000 problems of 1 to 64 rows, widths of 64 to 14336, depths of 64 to 8192,
// weights from memory.  On 22000 others, with the kernels as they are, the choice among these and the
// tiles takes by blocks of rows 1.020, 1.022, 1.017 and 1.012 of the best measured (the better of two
// timings each), 1.18 at the 99th percentile and 1.5 at worst.  Without tiles it takes 1.019, 1.054,
// 1.098 and 1.169; one block alone 1.033, 1.032, 1.028 and 1.021; four blocks, or other depths, gain
// less than 0.003.
constexpr TileFit kFewFits[] = {
    {{16, 16}, 4.36, 0.128, 0.078, 0.0, 0.335},  {{16, 32}, 4.13, 0.264, 0.231, 0.0, 0.594},
    {{32, 16}, 4.17, 0.270, 0.084, 0.0, 0.471},  {{32, 32}, 4.06, 0.381, 0.281, 0.0, 0.822},
    {{48, 16}, 4.12, 0.376, 0.113, 0.09, 0.677}, {{48, 32}, 4.03, 0.518, 0.349, 0.35, 0.956},
    {{64, 16}, 4.00, 0.491, 0.147, 0.24, 0.755}, {{64, 32}, 3.98, 0.648, 0.289, 1.59, 1.293}};
// (the sums of slices written and read again, and the launch that adds them; two slices of a big tile, which
// meet, cost some 10 us of 14 less where C is large, but the choice, and with it results' last bits, is as it was)
constexpr double kSliceLaunch = 2.96, kSliceBytes = 0.327e-6;

constexpr int kMostRows = 0x7ffffe00;  // of a product: rounded up to tiles they are an int

struct ProductPlan {
  FfTile tile;
  int slices;  // 0: no tile computes the product in one launch
  bool few;    // by the kernel for few rows, whose tiles are one of kFewFits
};

// whether a tile of kFits or kSmallFits computes a product
bool tile_takes(const FfTile& t, Layout layout, Finish finish, int m) {
  // (of 32 columns: where the kernel for few rows, whose tiles are named so too, does not compute)
  if (t.rows == 32) return finish == kFull && (t.cols == 64 || (t.cols == 32 && m > kProductRows));
  if (t.cols < 64) return false;  // (one of that kernel's alone)
  return layout != kTurnBoth || t.rows != 96;  // (64, 128 or 256 columns of a turned operand)
}

double fit_cost(const TileFit& f, long long groups, int stages, int cus) {
  const double r = (double)groups / cus;
  const int rounds = (int)((groups + cus - 1) / cus);
  // workgroups beyond one per compute unit: half way between the rounds and their share of one
  const double more = r > 1.0 ? 0.5 * (rounds + r) - 1.0 : 0.0;
  return f.launch + stages * (f.stage + f.fill * (r < 1.0 ? r : 1.0)) + more * (f.more + f.more_stage * stages);
}

// room: bytes for partial sums
ProductPlan choose_plan(int m, int n, int k, Finish finish, Layout layout, int cus, long long room) {
  const bool gated = finish == kGated;
  const int columns = product_columns(n, gated), stages = ceil_div(k, kDnStageK);
  const bool few = layout == kRows && m <= kProductRows;
  const bool forced = t_tile.rows > 0 && ((few && t_tile.cols <= 32) || tile_takes(t_tile, layout, finish, m));
  ProductPlan best = {{64, 64}, 0, false};
  double least = 0.0;
  if (few)
    for (const TileFit& f : kFewFits) {
      if (f.tile.rows != ceil_div(m, 16) * 16 || (forced && f.tile.cols != t_tile.cols)) continue;
      const double cost = fit_cost(f, ceil_div(n, gated ? f.tile.cols / 2 : f.tile.cols), ceil_div(stages, 4), cus);
      if (least == 0.0 || cost < least) {
        best = {f.tile, 1, true};
        least = cost;
      }
    }
  const auto consider = [&](const TileFit& f) {
    if (forced && (f.tile.rows != t_tile.rows || f.tile.cols != t_tile.cols)) return;
    if (!tile_takes(f.tile, layout, finish, m)) return;
    const long long tiles = (long long)ceil_div(m, f.tile.rows) * ceil_div(columns, f.tile.cols);
    for (int slices = 1; slices <= kSlicesMost && slices <= stages; slices++) {
      const double bytes = 4.0 * slices * m * columns;
      if (slices > 1 && (bytes > (double)room || (t_slices == 0 && tiles * slices > 2 * cus))) break;
      if (tiles * slices * tile_threads(f.tile) > kLaunchThreads || (slices > 1 && (long long)m * n / 4 > kLaunchThreads)) break;
      if (t_slices > 0 && slices != t_slices && t_slices <= stages && 4.0 * t_slices * m * columns <= (double)room) continue;
      double cost = fit_cost(f, tiles * slices, ceil_div(stages, slices), cus);
      if (slices > 1) cost += kSliceLaunch + kSliceBytes * bytes;
      if (least == 0.0 || cost < least) {
        best = {f.tile, slices, false};
        least = cost;
      }
    }
  };
  for (const TileFit& f : kFits) consider(f);
  for (const TileFit& f : kSmallFits) consider(f);
  return best;
}
// Two slices of big tiles finish them together: their sums, and behind these the words at which
// they meet.  More, and those of other tiles, are added up by a launch of their own.
struct Meeting {
  int tiles;        // 0: they do not
  long long words;  // bytes ahead of the words
  long long bytes;
};
Meeting meeting(const ProductPlan& p, int m, int columns) {
  const long long tiles = (long long)ceil_div(m, p.tile.rows) * ceil_div(columns, p.tile.cols);
  const long long sums = 2 * tiles * (long long)big_sums(p.tile.rows);
  // (the sums' offsets are ints)
  if (p.few || p.slices != 2 || !big_tile(p.tile) || sums > 0x7fffffffLL) return {0, 0, 0};
  return {(int)tiles, sums, sums + tiles * kWordStride * 8};
}

// a launch's own: products with an odd number do not repeat within 2^61, nor look like data.  (From the
// clock: std::random_device may throw, and the entries are C's.)
unsigned long long next_token() {
  static std::atomic<unsigned long long> launches{
      (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
  unsigned long long token;
  do token = ++launches * 0x9E3779B97F4A7C15ull << 3;
  while (token == 0);
  return token;
}

// A thread's last plans with all the room they want: planning takes the host some 3 us, asked
// for the room and again for the launch, and a model's layers are a few sizes over and over.
struct Planned {
  int m = 0, n = 0, k = 0, cus = 0, form = -1;
  ProductPlan plan = {{0, 0}, 0, false};
  long long bytes = 0;  // of partial sums, and where slices meet in their tiles of the words
};
constexpr int kPlansKept = 16;
thread_local Planned t_plans[kPlansKept];
thread_local int t_oldest = 0;

Planned plan_with_room(int m, int n, int k, Finish finish, Layout layout, int cus) {
  const bool gated = finish == kGated;
  const int form = (int)finish | (int)layout << 2;
  const bool forced = t_tile.rows > 0 || t_slices > 0;
  if (!forced)
    for (const Planned& p : t_plans)
      if (p.m == m && p.n == n && p.k == k && p.cus == cus && p.form == form) return p;
  Planned p;
  p.m = m, p.n = n, p.k = k, p.cus = cus, p.form = form;
  if (m > kMostRows) return p;
  p.plan = choose_plan(m, n, k, finish, layout, cus, 1LL << 40);
  p.bytes = p.plan.slices > 1 ? 4LL * p.plan.slices * m * product_columns(n, gated) : 0;
  p.bytes = std::max(p.bytes, meeting(p.plan, m, product_columns(n, gated)).bytes);
  if (!forced) {
    t_plans[t_oldest] = p;
    t_oldest = (t_oldest + 1) % kPlansKept;
  }
  return p;
}

bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }

constexpr long long kMostDropped = 1LL << 34;  // elements of a call: a launch has fewer than 2^32 threads
constexpr int kWidest = 1 << 21;  // elements from one row to the next

// a matrix of 16-bit elements as the kernels address it: rows start on 16 bytes
int check_matrix(const char* name, const void* p, long long ld, long long width) {
  if (off16(p) || ld % 8 != 0) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows must start on 16 bytes", name);
  if (ld < width) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows of %lld elements lie %lld apart", name, width, ld);
  if (ld > kWidest) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows of more than 4 MiB", name);
  return FEEDFORWARD_OK;
}

int check_sizes(int m, int n, int k, int type) {
  if (m < 0 || n < 0 || k < 0) return fail(FEEDFORWARD_ERR_SHAPE, "negative size (m=%d n=%d k=%d)", m, n, k);
  if (n % 8 != 0) return fail(FEEDFORWARD_ERR_SHAPE, "widths must be multiples of 8 (n = %d)", n);
  if (n > kWidest) return fail(FEEDFORWARD_ERR_SHAPE, "rows of more than 4 MiB (n = %d)", n);
  if (type != FEEDFORWARD_FP16 && type != FEEDFORWARD_BF16)
    return fail(FEEDFORWARD_ERR_SHAPE, "unknown type %d", type);
  return FEEDFORWARD_OK;
}

// the mask's arguments as the kernels take them: nothing below zero, and no seed in memory, where
// nothing is dropped
int drop_args(const feedforward_drop* d, DropArgs* out) {
  *out = {};
  out->factor = 1.f;
  if (!d) return FEEDFORWARD_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return fail(FEEDFORWARD_ERR_SHAPE, "p = %g is no probability", d->p);
  const int below = (int)std::nearbyint(65536.0 * d->p);
  if (below == 0) return FEEDFORWARD_OK;
  if ((uintptr_t)d->seed_at & 7) return fail(FEEDFORWARD_ERR_SHAPE, "the seed must start on 8 bytes");
  out->seed_at = d->seed_at;
  out->seed = (unsigned long long)d->seed;
  out->site = d->site;
  out->below = (unsigned)below;
  out->factor = below == 65536 ? 0.f : (float)(65536.0 / (65536 - below));
  return FEEDFORWARD_OK;
}

Finish finish_of(int gated) { return gated == FEEDFORWARD_FULL ? kFull : gated ? kGated : kPlain; }

bool layout_of(int turned, Layout* layout) {
  *layout = (Layout)turned;
  return turned >= FEEDFORWARD_ROWS && turned <= FEEDFORWARD_TURN_BOTH;
}

int run_product(ProductArgs a, Layout layout, bool bf, void* room, long long room_bytes, int dev, hipStream_t stream) {
  const bool gated = a.finish == kGated;
  const long long columns = product_columns(a.N, gated);
  // (the highest and widest tiles have to be a launch: a plan takes such as are)
  if (a.M > kMostRows || (columns + 255) / 256 * ((a.M + 255) / 256) * 256 > kLaunchThreads)
    return fail(FEEDFORWARD_ERR_SHAPE, "m = %d and n = %d are too many tiles", a.M, a.N);
  // a gated product's rows of either half are addressed from one place
  if (gated && 2LL * a.N * a.ldb * 2 > 0x7fffffffLL)
    return fail(FEEDFORWARD_ERR_SHAPE, "weights of more than 2 GiB (n = %d, rows of %d): split the call", a.N, a.ldb);
  if (!a.A || !a.B || !a.C) return fail(FEEDFORWARD_ERR_SHAPE, "a matrix is missing");
  if (room && off16(room)) return fail(FEEDFORWARD_ERR_SHAPE, "scratch must start on 16 bytes");
  bool fits = true;
  const int rc = on_device(dev, [&](int cus) {
    const Planned planned = plan_with_room(a.M, a.N, a.K, a.finish, layout, cus);
    const long long have = room ? room_bytes : 0;
    const ProductPlan p =
        planned.bytes <= have ? planned.plan : choose_plan(a.M, a.N, a.K, a.finish, layout, cus, have);
    fits = p.slices > 0;
    if (!fits) return;  // (where a tile is forced)
    a.slices = p.slices;
    a.part = p.slices > 1 ? (float*)room : nullptr;
    a.ldpart = (int)columns;
    a.polls = t_polls < 0 ? kFinishPolls : t_polls;
    const Meeting meet = meeting(p, a.M, (int)columns);
    if (meet.tiles > 0 && meet.bytes <= have) {
      a.words = (unsigned long long*)((char*)room + meet.words);
      a.token = next_token();
    }
    if (p.few)
      launch_product_rows(a, p.tile.cols / 16, bf, stream);
    else if (big_tile(p.tile))
      (bf ? launch_product_big_bf16 : launch_product_big_f16)(a, p.tile.rows, layout, stream);
    else
      launch_product_tiles(a, p.tile, layout, bf, stream);
    if (a.part && !a.words) launch_sum_parts(a, bf, stream);
  });
  if (rc == FEEDFORWARD_OK && !fits)
    return fail(FEEDFORWARD_ERR_SHAPE, "m = %d and n = %d are too many tiles", a.M, a.N);
  return rc;
}

int device_cus(int dev) {
  static std::mutex mu;
  static int known[kMaxDevices] = {};
  if (dev < 0 || dev >= kMaxDevices) return 0;
  std::lock_guard<std::mutex> lk(mu);
  if (known[dev] == 0 && hipDeviceGetAttribute(&known[dev], hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    known[dev] = 0;
  return known[dev];
}

int type_bytes(int type) { return type == FEEDFORWARD_FP32 ? 4 : 2; }
NormType norm_type(int type) {
  return type == FEEDFORWARD_FP32 ? kNormFp32 : type == FEEDFORWARD_BF16 ? kNormBf16 : kNormFp16;
}

int check_norm(long long rows, int d, int rows_per_gate, int type) {
  if (rows < 0 || rows > 0x7fffffff || d < 1 || d > kNormMax)
    return fail(FEEDFORWARD_ERR_SHAPE, "%lld rows of %d: rows must hold 1 to %d elements and fit into a C int", rows, d,
                kNormMax);
  if (rows_per_gate < 1 || rows % rows_per_gate != 0)
    return fail(FEEDFORWARD_ERR_SHAPE, "%lld rows are no multiple of the %d of a gate", rows, rows_per_gate);
  if (type != FEEDFORWARD_FP16 && type != FEEDFORWARD_BF16 && type != FEEDFORWARD_FP32)
    return fail(FEEDFORWARD_ERR_SHAPE, "unknown type %d", type);
  return FEEDFORWARD_OK;
}
int check_rows(const char* name, const void* p, long long ld, int d) {
  if (p && ld < d) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows of %d elements lie %lld apart", name, d, ld);
  return FEEDFORWARD_OK;
}

// feedforward_linear and feedforward_linear_train, which differ in the form of the slopes
int run_linear(bool steps, const void* x, const void* w, void* y, const void* bias, const void* residual, void* slopes, int m,
               int n, int k, long long ldx, long long ldw, long long ldy, long long ldr, long long ldslopes,
               int type, int activation, const feedforward_drop* drop, void* room, long long room_bytes,
               int dev, void* stream) {
  int rc = check_sizes(m, n, k, type);
  ProductArgs a = {};
  if (rc == FEEDFORWARD_OK && k % 8 != 0) rc = fail(FEEDFORWARD_ERR_SHAPE, "widths must be multiples of 8 (k = %d)", k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("x", x, ldx, k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("w", w, ldw, k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("y", y, ldy, n);
  if (rc == FEEDFORWARD_OK && bias) rc = check_matrix("bias", bias, n, n);
  if (rc == FEEDFORWARD_OK && residual) rc = check_matrix("residual", residual, ldr, n);
  if (rc == FEEDFORWARD_OK && slopes) rc = check_matrix("slopes", slopes, ldslopes, n);
  if (rc == FEEDFORWARD_OK && activation != kActNone && !act_known(activation))
    rc = fail(FEEDFORWARD_ERR_SHAPE, "unknown activation %d", activation);
  if (rc == FEEDFORWARD_OK && activation == kActNone && slopes)
    rc = fail(FEEDFORWARD_ERR_SHAPE, "slopes belong to an activation");
  if (rc == FEEDFORWARD_OK) rc = drop_args(drop, &a.drop);
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  if (k == 0) return fail(FEEDFORWARD_ERR_SHAPE, "k = 0: an empty sum");
  a.A = x, a.B = w, a.C = y, a.bias = bias, a.residual = residual, a.slopes = (unsigned short*)slopes;
  a.M = m, a.N = n, a.K = k;
  a.lda = (int)ldx, a.ldb = (int)ldw, a.ldc = (int)ldy;
  a.ldr = residual ? (int)ldr : 0, a.ldslopes = slopes ? (int)ldslopes : 0;
  a.slope_steps = steps;
  a.finish = kFull;
  a.act = activation;
  return run_product(a, kRows, type == FEEDFORWARD_BF16, room, room_bytes, dev, (hipStream_t)stream);
}

// of the sums over rows
long long linear_sums_bytes(int m, int n) {
  const int parts = m > 0 && n > 0 ? linear_grad_parts(m, n) : 0;
  return parts > 1 ? 4LL * n * parts : 0;
}

int run_linear_grad(bool steps, const void* dy, const void* slopes, void* dz, void* dbias, int m, int n, long long lddy,
                    long long ldslopes, long long lddz, int type, const feedforward_drop* drop,
                    void* partials, long long partial_bytes, float* factor, int dev, void* stream) {
  int rc = check_sizes(m, n, 0, type);
  LinearGradArgs a = {};
  if (rc == FEEDFORWARD_OK) rc = check_matrix("dy", dy, lddy, n);
  if (rc == FEEDFORWARD_OK && slopes) rc = check_matrix("slopes", slopes, ldslopes, n);
  if (rc == FEEDFORWARD_OK && dz) rc = check_matrix("dz", dz, lddz, n);
  if (rc == FEEDFORWARD_OK) rc = drop_args(drop, &a.drop);
  if (factor) *factor = 1.f;
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  if (!dy || (!dz && !dbias)) return fail(FEEDFORWARD_ERR_SHAPE, "dy, or every output, is missing");
  const long long sums = dbias ? linear_sums_bytes(m, n) : 0;
  if (sums > 0 && (!partials || ((uintptr_t)partials & 3) || partial_bytes < sums))
    return fail(FEEDFORWARD_ERR_SHAPE, "the sums over rows need %lld bytes of scratch", sums);
  a.dy = dy, a.slopes = (const unsigned short*)slopes, a.dz = dz, a.dbias = dbias;
  a.partials = sums > 0 ? (float*)partials : nullptr;
  a.lddy = lddy, a.ldslopes = ldslopes, a.lddz = lddz;
  a.m = m, a.n = n;
  a.slope_steps = steps;
  a.bias_factor = 1.f;
  if (factor) {
    *factor = a.bias_factor = a.drop.factor;
    a.drop.factor = 1.f;
  }
  return on_device(dev, [&](int) { launch_linear_grad(a, type == FEEDFORWARD_BF16, (hipStream_t)stream); });
}

}  // namespace

extern "C" {

int feedforward_product(const void* A, const void* B, void* C, int m, int n, int k, long long lda, long long ldb,
                        long long ldc, int turned, int type, void* room, long long room_bytes, int dev,
                        void* stream) {
  return feedforward_product_scaled(A, B, C, m, n, k, lda, ldb, ldc, turned, type, 1.f, room, room_bytes, dev, stream);
}

int feedforward_product_scaled(const void* A, const void* B, void* C, int m, int n, int k, long long lda, long long ldb,
                               long long ldc, int turned, int type, float scale, void* room, long long room_bytes,
                               int dev, void* stream) {
  int rc = check_sizes(m, n, k, type);
  Layout layout = kRows;
  if (rc == FEEDFORWARD_OK && !layout_of(turned, &layout)) rc = fail(FEEDFORWARD_ERR_SHAPE, "unknown layout %d", turned);
  if (rc == FEEDFORWARD_OK && layout != kTurnBoth && k % 8 != 0)
    rc = fail(FEEDFORWARD_ERR_SHAPE, "widths must be multiples of 8 (k = %d)", k);
  if (rc == FEEDFORWARD_OK && layout == kTurnBoth && m % 8 != 0)
    rc = fail(FEEDFORWARD_ERR_SHAPE, "m = %d must be a multiple of 8 where A is turned over", m);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("A", A, lda, layout == kTurnBoth ? m : k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("B", B, ldb, layout == kRows ? k : n);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("C", C, ldc, n);
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  if (k == 0) return fail(FEEDFORWARD_ERR_SHAPE, "k = 0: an empty sum");
  ProductArgs a = {};
  a.A = A, a.B = B, a.C = C;
  a.M = m, a.N = n, a.K = k;
  a.lda = (int)lda, a.ldb = (int)ldb, a.ldc = (int)ldc;
  a.scale = scale;
  return run_product(a, layout, type == FEEDFORWARD_BF16, room, room_bytes, dev, (hipStream_t)stream);
}

int feedforward_gated(const void* x, const void* w, void* h, float* pre, int m, int n, int k, long long ldx,
                      long long ldw, long long ldh, long long ldpre, int type, int activation, void* room,
                      long long room_bytes, int dev, void* stream) {
  int rc = check_sizes(m, n, k, type);
  if (rc == FEEDFORWARD_OK && k % 8 != 0) rc = fail(FEEDFORWARD_ERR_SHAPE, "widths must be multiples of 8 (k = %d)", k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("x", x, ldx, k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("w", w, ldw, k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("h", h, ldh, n);
  if (rc == FEEDFORWARD_OK && pre) rc = check_matrix("pre", pre, ldpre, (n + 15LL) / 16 * 32);
  if (rc == FEEDFORWARD_OK && !act_known(activation))
    rc = fail(FEEDFORWARD_ERR_SHAPE, "unknown activation %d", activation);
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  if (k == 0) return fail(FEEDFORWARD_ERR_SHAPE, "k = 0: an empty sum");
  ProductArgs a = {};
  a.A = x, a.B = w, a.C = h, a.pre = pre;
  a.M = m, a.N = n, a.K = k;
  a.lda = (int)ldx, a.ldb = (int)ldw, a.ldc = (int)ldh, a.ldpre = (int)ldpre;
  a.finish = kGated;
  a.act = activation;
  return run_product(a, kRows, type == FEEDFORWARD_BF16, room, room_bytes, dev, (hipStream_t)stream);
}

int feedforward_linear(const void* x, const void* w, void* y, const void* bias, const void* residual, void* slopes, int m,
                       int n, int k, long long ldx, long long ldw, long long ldy, long long ldr, long long ldslopes,
                       int type, int activation, const feedforward_drop* drop, void* room, long long room_bytes,
                       int dev, void* stream) {
  return run_linear(true, x, w, y, bias, residual, slopes, m, n, k, ldx, ldw, ldy, ldr, ldslopes, type, activation, drop,
                    room, room_bytes, dev, stream);
}

int feedforward_linear_train(const void* x, const void* w, void* y, const void* bias, const void* residual, void* slopes, int m,
                             int n, int k, long long ldx, long long ldw, long long ldy, long long ldr, long long ldslopes,
                             int type, int activation, const feedforward_drop* drop, void* room, long long room_bytes,
                             int dev, void* stream) {
  return run_linear(false, x, w, y, bias, residual, slopes, m, n, k, ldx, ldw, ldy, ldr, ldslopes, type, activation, drop,
                    room, room_bytes, dev, stream);
}

long long feedforward_linear_grad_bytes(int m, int n) {
  return check_sizes(m, n, 0, FEEDFORWARD_FP16) == FEEDFORWARD_OK ? linear_sums_bytes(m, n) : -1;
}

int feedforward_linear_grad(const void* dy, const void* slopes, void* dz, void* dbias, int m, int n, long long lddy,
                            long long ldslopes, long long lddz, int type, const feedforward_drop* drop,
                            void* partials, long long partial_bytes, int dev, void* stream) {
  return run_linear_grad(true, dy, slopes, dz, dbias, m, n, lddy, ldslopes, lddz, type, drop, partials, partial_bytes,
                         nullptr, dev, stream);
}

int feedforward_linear_backward(const void* dy, const void* slopes, void* dz, void* dbias, int m, int n, long long lddy,
                                long long ldslopes, long long lddz, int type, const feedforward_drop* drop,
                                void* partials, long long partial_bytes, float* factor, int dev, void* stream) {
  return run_linear_grad(false, dy, slopes, dz, dbias, m, n, lddy, ldslopes, lddz, type, drop, partials, partial_bytes,
                         factor, dev, stream);
}

int feedforward_dropout(const void* x, const void* residual, void* y, long long count, int type,
                        const feedforward_drop* drop, int dev, void* stream) {
  if (count < 0 || count > kMostDropped) return fail(FEEDFORWARD_ERR_SHAPE, "%lld elements", count);
  if (type != FEEDFORWARD_FP16 && type != FEEDFORWARD_BF16 && type != FEEDFORWARD_FP32)
    return fail(FEEDFORWARD_ERR_SHAPE, "unknown type %d", type);
  const uintptr_t off = type_bytes(type) - 1;
  if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & off)
    return fail(FEEDFORWARD_ERR_SHAPE, "elements must lie on whole addresses");
  DropoutArgs a = {x, residual, y, count, {}};
  const int rc = drop_args(drop, &a.drop);
  if (rc != FEEDFORWARD_OK || count == 0) return rc;
  if (!x || !y) return fail(FEEDFORWARD_ERR_SHAPE, "a matrix is missing");
  return on_device(dev, [&](int) { launch_dropout(a, type, (hipStream_t)stream); });
}

long long feedforward_product_bytes(int m, int n, int k, int gated, int turned, int dev) {
  Layout layout;
  if (check_sizes(m, n, k, FEEDFORWARD_FP16) != FEEDFORWARD_OK || !layout_of(turned, &layout)) return -1;
  const int cus = device_cus(dev);
  return cus > 0 && m > 0 && n > 0 && k > 0 ? plan_with_room(m, n, k, finish_of(gated), layout, cus).bytes : 0;
}

int feedforward_gated_grad(const void* dh, const float* pre, void* dgu, int m, int n, long long lddh, long long ldpre,
                           long long lddgu, int type, int activation, int dev, void* stream) {
  int rc = check_sizes(m, n, 0, type);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("dh", dh, lddh, n);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("pre", pre, ldpre, (n + 15LL) / 16 * 32);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("dgu", dgu, lddgu, 2LL * n);
  if (rc == FEEDFORWARD_OK && !act_known(activation))
    rc = fail(FEEDFORWARD_ERR_SHAPE, "unknown activation %d", activation);
  if (rc == FEEDFORWARD_OK && (long long)m * (n / 8) > kLaunchThreads - 255)
    rc = fail(FEEDFORWARD_ERR_SHAPE, "m = %d and n = %d are too many", m, n);
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  if (!dh || !pre || !dgu) return fail(FEEDFORWARD_ERR_SHAPE, "a matrix is missing");
  const GatedGradArgs a = {dh, pre, dgu, lddh, ldpre, lddgu, m, n, activation};
  return on_device(dev, [&](int) { launch_gated_grad(a, type == FEEDFORWARD_BF16, (hipStream_t)stream); });
}

int feedforward_norm(const void* residual, long long ld_residual, const void* block, long long ld_block,
                     const void* post, const void* gate, long long ld_gate, int rows_per_gate, const void* pre,
                     float scale, float eps, void* r, void* y, float* stats, long long rows, int d, int type,
                     int dev, void* stream) {
  int rc = check_norm(rows, d, rows_per_gate, type);
  if (rc == FEEDFORWARD_OK) rc = check_rows("residual", residual, ld_residual, d);
  if (rc == FEEDFORWARD_OK) rc = check_rows("block", block, ld_block, d);
  if (rc == FEEDFORWARD_OK) rc = check_rows("gate", rows > rows_per_gate ? gate : nullptr, ld_gate, d);
  if (rc == FEEDFORWARD_OK && !(eps >= 0.f)) rc = fail(FEEDFORWARD_ERR_SHAPE, "eps must not be negative");
  if (rc != FEEDFORWARD_OK || rows == 0) return rc;
  if (!residual || (block ? !r : (post || gate || !pre)) || (pre && !y))
    return fail(FEEDFORWARD_ERR_SHAPE, "a block needs its output r, a norm its output y, and one of them must be there");
  NormArgs a = {};
  a.residual = residual, a.block = block, a.post = post, a.gate = gate, a.pre = pre;
  a.r = block ? r : nullptr, a.y = pre ? y : nullptr, a.stats = stats;
  a.ld_residual = ld_residual, a.ld_block = ld_block, a.ld_gate = ld_gate;
  a.rows = rows, a.rows_per_gate = rows_per_gate, a.d = d;
  a.scale = scale, a.eps = eps;
  return on_device(dev, [&](int cus) { launch_norm(a, norm_type(type), cus, (hipStream_t)stream); });
}

long long feedforward_norm_grad_bytes(long long rows, int d, int rows_per_gate, int type) {
  if (check_norm(rows, d, rows_per_gate, type) != FEEDFORWARD_OK) return -1;
  return (long long)norm_parts(rows, rows_per_gate, d, type_bytes(type)).bytes;
}

int feedforward_norm_grad(const void* dy, long long ld_dy, const void* dr, long long ld_dr, const void* r,
                          long long ld_r, const void* block, long long ld_block, const void* post, const void* gate,
                          long long ld_gate, int rows_per_gate, const void* pre, float scale, const float* stats,
                          void* dresidual, void* dblock, void* dpost, void* dgate, void* dpre, void* partials,
                          long long partial_bytes, long long rows, int d, int type, int dev, void* stream) {
  int rc = check_norm(rows, d, rows_per_gate, type);
  const struct {
    const char* name;
    const void* at;
    long long ld;
  } matrices[] = {{"dy", dy, ld_dy}, {"dr", dr, ld_dr}, {"r", r, ld_r}, {"block", block, ld_block},
                  {"gate", rows > rows_per_gate ? gate : nullptr, ld_gate}};
  for (const auto& m : matrices)
    if (rc == FEEDFORWARD_OK) rc = check_rows(m.name, m.at, m.ld, d);
  if (rc != FEEDFORWARD_OK || rows == 0) return rc;
  if ((pre && (!dy || !r)) || ((pre || post) && !stats) || (!block && (post || gate || dblock || dpost || dgate)) ||
      (!post && dpost) || (!gate && dgate) || (!pre && dpre) || (!pre && !dr))
    return fail(FEEDFORWARD_ERR_SHAPE, "an input that a gradient is made from is missing");
  const bool sums = dpost || dgate || dpre;
  if (sums && (!partials || partial_bytes < feedforward_norm_grad_bytes(rows, d, rows_per_gate, type)))
    return fail(FEEDFORWARD_ERR_SHAPE, "the sums over rows need %lld bytes of scratch",
                feedforward_norm_grad_bytes(rows, d, rows_per_gate, type));
  NormGradArgs a = {};
  a.dy = pre ? dy : nullptr, a.dr = dr, a.r = r, a.block = block, a.post = post, a.gate = gate, a.pre = pre;
  a.stats = stats;
  a.dresidual = dresidual, a.dblock = dblock, a.dpost = dpost, a.dgate = dgate, a.dpre = dpre;
  a.partials = sums ? (float*)partials : nullptr;
  a.ld_dy = ld_dy, a.ld_dr = ld_dr, a.ld_r = ld_r, a.ld_block = ld_block, a.ld_gate = ld_gate;
  a.rows = rows, a.rows_per_gate = rows_per_gate, a.d = d;
  a.scale = block ? scale : 1.f;  // (without a block r is the residual, whatever the scale)
  return on_device(dev, [&](int) { launch_norm_grad(a, norm_type(type), (hipStream_t)stream); });
}

int feedforward_plan(int m, int n, int k, int gated, int turned, int cus, int* out) {
  out[0] = out[1] = out[2] = 0;
  const int rc = check_sizes(m, n, k, FEEDFORWARD_FP16);
  if (rc != FEEDFORWARD_OK || n == 0 || k == 0 || m == 0) return rc;
  Layout layout;
  if (!layout_of(turned, &layout)) return fail(FEEDFORWARD_ERR_SHAPE, "unknown layout %d", turned);
  if (cus < 1) return fail(FEEDFORWARD_ERR_SHAPE, "%d compute units", cus);
  const ProductPlan p = plan_with_room(m, n, k, finish_of(gated), layout, cus).plan;
  if (p.slices == 0) return fail(FEEDFORWARD_ERR_SHAPE, "m = %d and n = %d are too many tiles", m, n);
  out[0] = p.tile.rows;
  out[1] = p.tile.cols;
  out[2] = p.slices;
  return rc;
}

void feedforward_force_tile(int rows, int cols, int slices) {
  t_tile = {0, 0};
  t_slices = slices > kSlicesMost ? kSlicesMost : slices < 0 ? 0 : slices;
  for (const TileFit& f : kFits)
    if (f.tile.rows == rows && f.tile.cols == cols) t_tile = f.tile;
  for (const TileFit& f : kSmallFits)
    if (f.tile.rows == rows && f.tile.cols == cols) t_tile = f.tile;
  for (const TileFit& f : kFewFits)
    if (f.tile.rows == rows && f.tile.cols == cols) t_tile = f.tile;
}

void feedforward_force_polls(int polls) { t_polls = polls < 0 || polls > kFinishPolls ? -1 : polls; }

const char* feedforward_last_error(void) { return g_error; }

}  // extern "C"
