/*
 * fusiontrain.h — C ABI of libfusionmoe.so, continued: the training operators
 * around the feed-forward block that fusionmoe.h does not declare (layer norm
 * with its backward pass, orthogonalised updates and the Muon step).
 *
 * The conventions, status codes and dtype codes are those of fusionmoe.h:
 * borrowed device pointers, asynchronous on `stream`, no allocation, no
 * synchronisation, a status instead of an exception.
 */
#ifndef FUSIONTRAIN_H
#define FUSIONTRAIN_H

#include "fusionmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FMOE_LAYER_NORM_MAX_DIM 16384
#define FMOE_MUON_MAX_TENSORS 64
#define FMOE_MUON_MAX_SIDE 65536
#define FMOE_MUON_MAX_ELEMENTS 536870912 /* of a matrix, its sides rounded up to multiples of 64 */
#define FMOE_MUON_MAX_STEPS 64

/* ---------------------------------------------------------------------------
 * Layer norm of the rows of x [T, dim] (dim <= FMOE_LAYER_NORM_MAX_DIM):
 *   mean[t] = sum_c x[t,c] / dim
 *   rstd[t] = 1 / sqrt(sum_c (x[t,c] - mean[t])^2 / dim + eps)
 *   y[t,c]  = ((x[t,c] - mean[t]) * rstd[t]) * weight[c] + bias[c]
 * fp32 arithmetic, the sums over a row in a fixed order; y is rounded once, to
 * y_dtype.  Row t of x starts at x + t * ldx (elements, ldx >= dim unless T <=
 * 1); y is dense.  weight and bias: [dim] of w_dtype, either may be NULL (1, 0).
 * mean and rstd [T] fp32 are kept for the backward pass; both may be NULL.
 * Pointers need the alignment of their element type only.
 * ------------------------------------------------------------------------- */
int fmoe_layer_norm_fwd(const void* x, int x_dtype, int64_t ldx, const void* weight,
                        const void* bias, int w_dtype, int64_t T, int64_t dim, float eps,
                        void* y, int y_dtype, float* mean, float* rstd, void* stream);

/* Workspace of fmoe_layer_norm_bwd when d_weight or d_bias is wanted: two fp32
 * rows of dim for every workgroup of its launch. */
size_t fmoe_layer_norm_bwd_workspace_bytes(int64_t T, int64_t dim);

/* Backward of the layer norm, with g = dy * weight and xh = (x - mean) * rstd:
 *   dx = rstd * (g - sum_c(g) / dim - xh * sum_c(g * xh) / dim) + d_residual
 *   d_weight[c] = sum_t dy[t,c] * xh[t,c],   d_bias[c] = sum_t dy[t,c]
 * x, d_residual ([T, dim] dense, or NULL: the gradient that reaches x past the
 * norm) and dx (dense) have x_dtype, dy dy_dtype, weight, d_weight and d_bias
 * w_dtype.  dx, d_weight and d_bias may each be NULL (not wanted).  The sums
 * over the rows run in a fixed order (no atomics): fp32 per workgroup, then
 * over the workgroups.  No output may overlap an input. */
int fmoe_layer_norm_bwd(const void* dy, int dy_dtype, int64_t lddy, const void* x, int x_dtype,
                        int64_t ldx, const float* mean, const float* rstd, const void* weight,
                        int w_dtype, const void* d_residual, int64_t T, int64_t dim, void* dx,
                        void* d_weight, void* d_bias, void* workspace, size_t workspace_bytes,
                        void* stream);

/* ---------------------------------------------------------------------------
 * Orthogonalised updates by Newton-Schulz products, for up to
 * FMOE_MUON_MAX_TENSORS matrices of one dtype whose sides are the same up to
 * their order (rows[i] x cols[i], row-major and dense; sides up to
 * FMOE_MUON_MAX_SIDE, FMOE_MUON_MAX_ELEMENTS elements).  For each matrix G, with its smaller side first:
 *   X = G / max(|G|_F, eps)
 *   steps times:  A = X X^T,  B = coeffs[1] A + coeffs[2] A^2,  X = coeffs[0] X + B X
 * and dst = X in G's own orientation (dst may be G's storage).  The norm is
 * summed in fp64, the products run on fp16 operands with fp32 sums, X held as
 * fp16 and an fp8 remainder, the result is rounded once, to dtype; for fp32 matrices (and small
 * sides up to 128) every operand is held in 22 bits, and small sides up to 64 with at most
 * 4096 columns run in fp32.  A matrix that holds NaN or
 * infinities gives NaN; a zero matrix gives zeros.  X is stored in steps of 2^-38 at the finest, and a step
 * multiplies what that loses by up to |coeffs[0]|: beside the relative error an element is off by up to
 * about steps |coeffs[0]|^steps 2^-38 (2^-27 for five steps with 3.4445), all the precision that the
 * nearly zero result of a matrix of a norm far below eps has.  Coefficients whose iterates
 * leave the stored range (singular values up to 2.8, |a + b t + c t^2| up to 7.9)
 * return FMOE_ERR_COEFFICIENTS.  Deterministic.
 * workspace: 256-byte aligned, of the size query's bytes (a pair of sides in
 * either order); calls that share one must not overlap.
 * ------------------------------------------------------------------------- */
size_t fmoe_orthogonalize_workspace_bytes(int64_t rows, int64_t cols, int n_tensors, int dtype);
int fmoe_orthogonalize(const void* const* src, void* const* dst, const int64_t* rows,
                       const int64_t* cols, int n_tensors, int dtype, int steps,
                       const double* coeffs, double eps, void* workspace,
                       size_t workspace_bytes, void* stream);

/* FMOE_OK where fmoe_orthogonalize and fmoe_muon_step take this number of steps and these coefficients,
 * the status that they would return otherwise.  Host only. */
int fmoe_newton_schulz_check(int steps, const double* coeffs);

/* Rows of the output tiles (256, 128 or 64) that a launch of n_tensors matrices of these sides takes for
 * its symmetric products (A and A^2), or for its updates of X; 0 where the form of small sides runs, or for
 * sizes that are not taken.  Host only, for tests and profiles. */
int fmoe_newton_schulz_tile(int64_t rows, int64_t cols, int n_tensors, int symmetric);

/* One Muon step of up to FMOE_MUON_MAX_TENSORS matrices (sizes and workspace as
 * fmoe_orthogonalize), in place:
 *   buf = momentum * buf + (1 - momentum) * grad
 *   u   = nesterov ? (1 - momentum) * grad + momentum * buf : buf   (buf before its rounding)
 *   param = decay * param - lr * X(u)
 * with lr = lr_tall for matrices of more rows than columns, lr_wide otherwise
 * (the caller's size adjustment), decay = 1 - learning rate * weight decay.
 * Arithmetic in fp32; buf and param are rounded once, to dtype.  Params, grads
 * and buffers must not overlap. */
int fmoe_muon_step(void* const* params, const void* const* grads, void* const* momentum_bufs,
                   const int64_t* rows, const int64_t* cols, int n_tensors, int dtype,
                   double lr_tall, double lr_wide, double decay, double momentum, int nesterov,
                   int steps, const double* coeffs, double eps, void* workspace,
                   size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FUSIONTRAIN_H */
