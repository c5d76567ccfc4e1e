// C ABI of the feed-forward block's dense parts (include/feedforward_amd.h): checks, the
// choice of kernel, launches.  Nothing here allocates, waits or keeps anything of a call.
#include <hip/hip_runtime.h>

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
// fuller the chip), and workgroups beyond one per compute unit.
struct TileFit {
  FfTile tile;
  double launch, stage, fill, more, more_stage;
};
constexpr TileFit kFits[] = {
    {{64, 64}, 2.32, 0.191, 0.056, 0.77, 0.179},   {{64, 128}, 3.05, 0.277, 0.088, 2.18, 0.324},
    {{96, 128}, 3.27, 0.359, 0.093, 2.04, 0.436},  {{128, 128}, 3.17, 0.424, 0.095, 2.40, 0.500},
    {{96, 256}, 4.04, 0.531, 0.205, 3.09, 0.828},  {{128, 256}, 4.46, 0.594, 0.294, 4.30, 1.020},
    {{256, 256}, 8.30, 1.186, 0.248, 1.87, 1.92}};

FfTile choose_tile(int m, int columns, int k, int cus) {
  if (t_tile.rows > 0 && (t_tile.rows < 256 || k % kDnStageK == 0)) return t_tile;
  FfTile best = {64, 64};
  double least = 0.0;
  for (const TileFit& f : kFits) {
    if (f.tile.rows == 256 && k % kDnStageK != 0) continue;
    const double tiles = (double)ceil_div(m, f.tile.rows) * ceil_div(columns, f.tile.cols), r = tiles / cus;
    const int stages = ceil_div(k, kDnStageK), rounds = (int)((tiles + cus - 1) / cus);
    // workgroups beyond one per compute unit: half way between the rounds and their share of one
    const double more = r > 1.0 ? 0.5 * (rounds + r) - 1.0 : 0.0;
    const double cost =
        f.launch + stages * (f.stage + f.fill * (r < 1.0 ? r : 1.0)) + more * (f.more + f.more_stage * stages);
    if (least == 0.0 || cost < least) {
      best = f.tile;
      least = cost;
    }
  }
  return best;
}

bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }

// a matrix of 16-bit elements as the kernels address it: rows start on 16 bytes
int check_matrix(const char* name, const void* p, long long ld, long long width) {
  if (off16(p) || ld % 8 != 0) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows must start on 16 bytes", name);
  if (ld < width) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows of %lld elements lie %lld apart", name, width, ld);
  if (ld > (1 << 21)) return fail(FEEDFORWARD_ERR_SHAPE, "%s: rows of more than 4 MiB", name);
  return FEEDFORWARD_OK;
}

int check_sizes(int m, int n, int k, int type) {
  if (m < 0 || n < 0 || k < 0) return fail(FEEDFORWARD_ERR_SHAPE, "negative size (m=%d n=%d k=%d)", m, n, k);
  if (n % 8 != 0 || k % 8 != 0)
    return fail(FEEDFORWARD_ERR_SHAPE, "n = %d and k = %d must be multiples of 8", n, k);
  if (type != FEEDFORWARD_FP16 && type != FEEDFORWARD_BF16)
    return fail(FEEDFORWARD_ERR_SHAPE, "unknown type %d", type);
  return FEEDFORWARD_OK;
}

int run_product(ProductArgs a, bool bf, int dev, hipStream_t stream) {
  const long long columns = a.act == kActNone ? a.N : 2LL * ((a.N + 15) / 16 * 16);
  // (a launch's grid, at the smallest tiles)
  if (columns > 0x3fffffffLL || (columns / 64 + 1) * (a.M / 64 + 1LL) > 0x3fffffffLL)
    return fail(FEEDFORWARD_ERR_SHAPE, "m = %d and n = %d are too many tiles", a.M, a.N);
  // a gated product's rows of either half are addressed from one place
  if (a.act != kActNone && 2LL * a.N * a.ldb * 2 > 0x7fffffffLL)
    return fail(FEEDFORWARD_ERR_SHAPE, "weights of more than 2 GiB (n = %d, rows of %d): split the call", a.N, a.ldb);
  return on_device(dev, [&](int cus) {
    if (a.M <= kProductRows && t_tile.rows <= 0)
      launch_product_rows(a, bf, stream);
    else
      launch_product_tiles(a, choose_tile(a.M, (int)columns, a.K, cus), bf, stream);
  });
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

}  // namespace

extern "C" {

int feedforward_product(const void* A, const void* B, void* C, int m, int n, int k, long long lda, long long ldb,
                        long long ldc, int type, int dev, void* stream) {
  int rc = check_sizes(m, n, k, type);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("A", A, lda, k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("B", B, ldb, k);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("C", C, ldc, n);
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  if (k == 0) return fail(FEEDFORWARD_ERR_SHAPE, "k = 0: an empty sum");
  ProductArgs a = {};
  a.A = A, a.B = B, a.C = C;
  a.M = m, a.N = n, a.K = k;
  a.lda = (int)lda, a.ldb = (int)ldb, a.ldc = (int)ldc;
  return run_product(a, type == FEEDFORWARD_BF16, dev, (hipStream_t)stream);
}

int feedforward_gated(const void* x, const void* w, void* h, float* pre, int m, int n, int k, long long ldx,
                      long long ldw, long long ldh, long long ldpre, int type, int activation, int dev,
                      void* stream) {
  int rc = check_sizes(m, n, k, type);
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
  a.act = activation;
  return run_product(a, type == FEEDFORWARD_BF16, dev, (hipStream_t)stream);
}

int feedforward_gated_grad(const void* dh, const float* pre, void* dgu, void* dgu_t, int m, int n, long long lddh,
                           long long ldpre, long long lddgu, long long lddgu_t, int type, int activation, int dev,
                           void* stream) {
  int rc = check_sizes(m, n, 0, type);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("dh", dh, lddh, n);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("pre", pre, ldpre, (n + 15LL) / 16 * 32);
  if (rc == FEEDFORWARD_OK && dgu) rc = check_matrix("dgu", dgu, lddgu, (2LL * n + 63) / 64 * 64);
  if (rc == FEEDFORWARD_OK && dgu_t) rc = check_matrix("dgu_t", dgu_t, lddgu_t, (m + 63LL) / 64 * 64);
  if (rc == FEEDFORWARD_OK && !act_known(activation))
    rc = fail(FEEDFORWARD_ERR_SHAPE, "unknown activation %d", activation);
  if (rc == FEEDFORWARD_OK && m > 64 * 65535) rc = fail(FEEDFORWARD_ERR_SHAPE, "m = %d: too many rows", m);
  if (rc != FEEDFORWARD_OK || m == 0 || n == 0) return rc;
  const GatedGradArgs a = {dh, pre, dgu, dgu_t, lddh, ldpre, lddgu, lddgu_t, m, n, activation};
  return on_device(dev, [&](int) { launch_gated_grad(a, type == FEEDFORWARD_BF16, (hipStream_t)stream); });
}

int feedforward_transpose(const void* in, void* out, int rows, int cols, long long ld_in, long long ld_out, int dev,
                          void* stream) {
  if (rows < 0 || cols < 0) return fail(FEEDFORWARD_ERR_SHAPE, "negative size (%d x %d)", rows, cols);
  if (cols % 8 != 0) return fail(FEEDFORWARD_ERR_SHAPE, "columns (%d) must be a multiple of 8", cols);
  int rc = check_matrix("in", in, ld_in, cols);
  if (rc == FEEDFORWARD_OK) rc = check_matrix("out", out, ld_out, (rows + 63LL) / 64 * 64);
  if (rc == FEEDFORWARD_OK && rows > 64 * 65535) rc = fail(FEEDFORWARD_ERR_SHAPE, "%d rows: too many", rows);
  if (rc != FEEDFORWARD_OK || rows == 0 || cols == 0) return rc;
  return on_device(dev, [&](int) { launch_transpose(in, ld_in, out, ld_out, rows, cols, (hipStream_t)stream); });
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
  a.scale = scale;
  return on_device(dev, [&](int) { launch_norm_grad(a, norm_type(type), (hipStream_t)stream); });
}

int feedforward_tile(int m, int n, int k, int gated, int cus, int* out) {
  out[0] = out[1] = 0;
  const int rc = check_sizes(m, n, k, FEEDFORWARD_FP16);
  if (rc != FEEDFORWARD_OK || m <= kProductRows || n == 0 || k == 0) return rc;
  const FfTile t = choose_tile(m, gated ? 2 * ((n + 15) / 16 * 16) : n, k, cus);
  out[0] = t.rows;
  out[1] = t.cols;
  return rc;
}

void feedforward_force_tile(int rows, int cols) {
  t_tile = {0, 0};
  for (const TileFit& f : kFits)
    if (f.tile.rows == rows && f.tile.cols == cols) t_tile = f.tile;
}

const char* feedforward_last_error(void) { return g_error; }

}  // extern "C"
