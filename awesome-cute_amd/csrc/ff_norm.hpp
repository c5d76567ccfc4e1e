// The norms around a block: arguments and launches of ff_norm.hip.
#pragma once
#include <hip/hip_runtime.h>

namespace w4a16 {

// rows of d elements; see ff_norm.hip for the formulas.  Null pointers: no block, no norm after
// it, no gate, no norm before the next one.
struct NormArgs {
  const void* residual;
  const void* block;
  const void* post;
  const void* gate;
  const void* pre;
  void* r;      // out: the new residual (null without a block)
  void* y;      // out: its norm (null without `pre`)
  float* stats; // out: both reciprocal lengths of every row, or null
  long long ld_residual, ld_block;  // r and y are contiguous
  long long ld_gate;
  long long rows;
  int rows_per_gate;  // consecutive rows that share a row of `gate`
  int d;
  float scale, eps;
};

struct NormGradArgs {
  const void* dy;     // null without `pre`
  const void* dr;     // null: no gradient of the residual itself
  const void* r;      // the forward pass's residual
  const void* block;
  const void* post;
  const void* gate;
  const void* pre;
  const float* stats;
  void* dresidual;    // outputs, null where not wanted
  void* dblock;
  void* dpost;
  void* dgate;
  void* dpre;
  float* partials;    // norm_parts(...).bytes; null if none of dpost, dgate, dpre is wanted
  long long ld_dy, ld_dr, ld_r, ld_block, ld_gate;
  long long rows;
  int rows_per_gate;
  int d;
  float scale;
};

// How the rows are dealt out to parts, a part a run of rows of which one set of waves keeps the
// sums over rows: `rows_per_part` rows of one gate's, or whole gates' where these are short.
struct NormParts {
  bool whole;         // a part holds whole gates
  long long parts, parts_per_gate, rows_per_part, gates;
  size_t bytes;       // of partial sums: two rows of d floats per part
};
NormParts norm_parts(long long rows, int rows_per_gate, int d, int bytes_per_element);
constexpr int kNormMax = 16384;  // the longest row: sixteen elements to each of a workgroup's 1024 lanes

enum NormType { kNormFp16, kNormBf16, kNormFp32 };
void launch_norm(const NormArgs& a, NormType type, int cus, hipStream_t stream);
void launch_norm_grad(const NormGradArgs& a, NormType type, hipStream_t stream);

}  // namespace w4a16
