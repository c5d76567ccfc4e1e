/* C ABI of the feed-forward half of a decoder block in libmarlin_amd.so (gfx950): gated
 * projections, dense linear layers with what their gradients need, and the norms around
 * the block.  The reference has no counterpart of any of it.
 *
 * Plain pointers and sizes only; every buffer is a caller-owned device pointer, calls are
 * asynchronous on the given HIP stream of device `dev` and allocate nothing (but for
 * feedforward_gated_w4, which shares marlin_gemm's scratch).
 */
#ifndef FEEDFORWARD_AMD_H
#define FEEDFORWARD_AMD_H

#include "marlin_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* activations: g / (1 + exp(-g)), and g/2 (1 + tanh(sqrt(2/pi) (g + 0.044715 g^3))) */
#define FEEDFORWARD_SILU 1
#define FEEDFORWARD_GELU 2

/*
 * A gated projection with 4-bit weights, both products, the activation and the product of
 * the two in one launch: C = act(A G) * (A U), element by element.  No reference counterpart.
 *   A   (prob_m, prob_k) fp16, C (prob_m, prob_n) fp16, overwritten
 *   B   (prob_k/16, 4*prob_n) int32: the packed words of one weight of 2*prob_n columns, in
 *       which columns 16 i + c, c < 8, are columns 8 i + c of G and columns 16 i + 8 + c those
 *       of U; s its scales, permuted as those of marlin_gemm: (prob_k/128, 2*prob_n) or
 *       (1, 2*prob_n) halves, s_rows the number of rows
 *   activation  FEEDFORWARD_SILU or FEEDFORWARD_GELU
 *   workspace   at least prob_n/64*max_par ints, zero on entry and again afterwards
 * prob_n and prob_k are multiples of 128.  Sums, scales per column, activation and product
 * are fp32, the result is rounded once.  Scratch, capture, streams, overlapping calls and
 * operands off 16 bytes: as marlin_gemm of 2*prob_n columns, whose plan it takes.  Returns
 * MARLIN_OK or one of that header's codes, with a message in err (if non-null).
 */
int feedforward_gated_w4(const void *A, const void *B, void *C, const void *s, int prob_m, int prob_n,
                 int prob_k, int s_rows, void *workspace, long long workspace_numel, int activation,
                 int dev, void *stream, int max_par, char *err, int err_len);

#ifdef __cplusplus
}
#endif
#endif
