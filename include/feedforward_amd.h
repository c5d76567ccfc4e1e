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

/* codes of the entries below, text in feedforward_last_error() */
#define FEEDFORWARD_OK 0
#define FEEDFORWARD_ERR_SHAPE 1   /* a size, a stride, an address, a type that no kernel takes */
#define FEEDFORWARD_ERR_RUNTIME 3 /* the HIP runtime reported an error */

/* types of matrices */
#define FEEDFORWARD_FP16 0
#define FEEDFORWARD_BF16 1
#define FEEDFORWARD_FP32 2 /* norms only */

/*
 * Matrices below are row-major in fp16 or bfloat16 (`type`), `ld...` elements from one row to
 * the next; rows start on 16 bytes (addresses, and ld a multiple of 8), are at most 4 MiB
 * apart, and their widths are multiples of 8.  Sums are fp32, results rounded once.  Entries may
 * be called from any thread, on any stream, and captured.
 */

/* how the operands of a product lie: by rows, A m rows of k and B n rows of k; B turned over, k
 * rows of n; or both, A k rows of m (a multiple of 8; k need then be none) */
#define FEEDFORWARD_ROWS 0
#define FEEDFORWARD_TURN_B 1
#define FEEDFORWARD_TURN_BOTH 2

/* C (m x n) = A B^T, the sum over k > 0.  With `room`, device memory of room_bytes on 16 bytes,
 * few tiles over a deep k are computed in slices of it, whose sums are added there in a fixed
 * order; feedforward_product_bytes says what helps (0: nothing does), less or none is correct
 * as well, in another order of the sums. */
int feedforward_product(const void *A, const void *B, void *C, int m, int n, int k, long long lda,
                        long long ldb, long long ldc, int turned, int type, void *room,
                        long long room_bytes, int dev, void *stream);
/* -1 for sizes that are refused */
long long feedforward_product_bytes(int m, int n, int k, int gated, int turned, int dev);

/* h (m x n) = act(x G^T) * (x U^T), element by element, x (m x k), w the n rows of G and behind
 * them the n rows of U.  w holds at most 2 GiB; k > 0.  pre, if not null, keeps both sums for
 * the backward pass: m rows of floats, ldpre >= 32 ceil(n / 16) from one to the next, in which
 * the sums of columns 16 i + c of x G^T are at 32 i + c and those of x U^T 16 further on. */
int feedforward_gated(const void *x, const void *w, void *h, float *pre, int m, int n, int k,
                      long long ldx, long long ldw, long long ldh, long long ldpre, int type,
                      int activation, void *room, long long room_bytes, int dev, void *stream);

/* The gradients of both sums from that of h: rows of [dg | du] (m x 2n). */
int feedforward_gated_grad(const void *dh, const float *pre, void *dgu, int m, int n,
                           long long lddh, long long ldpre, long long lddgu, int type,
                           int activation, int dev, void *stream);

/* out[0..2] = rows and columns of the product's tiles and the slices of k, with room for them, on
 * a device of `cus` compute units (16 or 32 columns: all of up to 64 rows by workgroups of whole
 * columns); no GPU touched */
int feedforward_plan(int m, int n, int k, int gated, int turned, int cus, int *out);
/* such tiles (0 = by cost) and slices (0 = by cost) for every product of the calling thread that
 * they can compute; for tests and tools */
void feedforward_force_tile(int rows, int cols, int slices);

/*
 * The norm after a block, its gate, the residual's scale and the norm before the next block, row
 * by row: p = block rstd(block) post, r = scale residual + gate p, y = r rstd(r) pre, with rstd(v)
 * = 1 / sqrt(mean(v^2) + eps); fp32 inside, r and y rounded once, y from the unrounded r.  Every
 * matrix is of one type (fp32 too), `rows` rows of d <= 16384 elements, `ld...` apart; r and y
 * contiguous.  Null: post (no norm after the block, p = block), gate (1), pre (no norm before
 * the next block, y is not written), block (r = residual whatever the scale, not written; then
 * neither post nor gate).  gate has a row for every rows_per_gate rows.  stats, if not null,
 * (rows x 2) floats: rstd(block) and rstd(r), which the backward pass takes.
 */
int feedforward_norm(const void *residual, long long ld_residual, const void *block,
                     long long ld_block, const void *post, const void *gate, long long ld_gate,
                     int rows_per_gate, const void *pre, float scale, float eps, void *r, void *y,
                     float *stats, long long rows, int d, int type, int dev, void *stream);

/* Its gradients from dy (null without pre) and dr (null: zero), r the forward pass's (without a
 * block the residual, whatever the scale).  Outputs that are null are not computed, and of no
 * rows none is written, dpost and dpre neither; dresidual and dblock (rows x d), dgate (a row
 * per gate), dpost and dpre (d) are contiguous.  The sums over rows go through `partials`, at least feedforward_norm_grad_bytes(...) bytes of device memory, in
 * an order that the sizes alone decide. */
int feedforward_norm_grad(const void *dy, long long ld_dy, const void *dr, long long ld_dr,
                          const void *r, long long ld_r, const void *block, long long ld_block,
                          const void *post, const void *gate, long long ld_gate,
                          int rows_per_gate, const void *pre, float scale, const float *stats,
                          void *dresidual, void *dblock, void *dpost, void *dgate, void *dpre,
                          void *partials, long long partial_bytes, long long rows, int d, int type,
                          int dev, void *stream);
/* -1 for sizes that are refused; no GPU touched */
long long feedforward_norm_grad_bytes(long long rows, int d, int rows_per_gate, int type);

const char *feedforward_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
