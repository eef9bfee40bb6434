/*
 * sgblas-b200: products of language models. Mixture-of-experts products whose
 * groups are ragged, 8-bit products with a scale for each block of 128, the
 * quantisation they need, and the orthogonalisation of an update by
 * Newton-Schulz products. No counterpart in the reference API, whose only
 * product is SGEMM.
 *
 * Matrices are column-major, as everywhere in the library. A row-major tensor
 * [tokens, k] is the same memory as a column-major k x tokens matrix: a token
 * is a column, and its values are contiguous.
 *
 * Every call enqueues on the handle's stream and never synchronizes. Device
 * pointers belong to the current device; outputs must not overlap inputs.
 * Statuses are those of sgblasSgemm; additionally NOT_SUPPORTED when a call
 * has more than SGBLAS_MAX_GROUPS groups, or needs workspace that cannot be
 * provided (it is never allocated inside a stream capture).
 */
#ifndef SGBLAS_SGBLAS_LM_H_
#define SGBLAS_SGBLAS_LM_H_

#include <sgblas/sgblas.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum sgblasDataType_t {
  SGBLAS_TYPE_FP32 = 0,
  SGBLAS_TYPE_BF16 = 1,
  SGBLAS_TYPE_FORCE_INT = 0x7fffffff
} sgblasDataType_t;

#define SGBLAS_MAX_GROUPS 1024

/* Products grouped along n, BF16 inputs: for each group g
 *
 *   C(:, o_g : o_{g+1}) = (*alpha) * op(A_g) * B(:, o_g : o_{g+1}) + (*beta) * C(:, same)
 *
 * op(A_g) is m x k with A_g at a + g * stride_a (elements), B is k x n, C is
 * m x n of type ctype. offsets: DEVICE array of groups + 1 column indices,
 * not decreasing; a group may be empty. Columns outside [o_0, o_groups) are
 * not written; an offset outside [0, n] counts as the nearer end. With
 * transa = T this is the forward product of an expert layer (A_g its weights,
 * k x m), with transa = N the gradient of its tokens.
 *
 * Products are exact, sums are FP32. The tensor core's adder truncates, so
 * at most 512 of k are chained there for an FP32 C, and 4096 for a BF16 C, whose
 * own rounding is far coarser; the chains are added with rounding to nearest,
 * and the result is rounded once to ctype. Scalars as for sgblasSgemm:
 * *beta == 0 writes C without reading it; *alpha == 0 or k == 0 does not read
 * A and B. Any alignment and leading dimension: an operand TMA cannot read (a
 * base not 16-byte aligned, lda, ldb or stride_a not a multiple of 8) is
 * first copied into the handle's workspace. */
sgblasStatus_t sgblasGroupedGemmN(sgblasHandle_t handle, sgblasOperation_t transa, int m, int n,
                                  int k, int groups, const int *offsets, const float *alpha,
                                  const void *a, int lda, long long stride_a, const void *b,
                                  int ldb, const float *beta, void *c, sgblasDataType_t ctype,
                                  int ldc);

/* Products grouped along k, BF16 inputs: for each group g
 *
 *   C_g = (*alpha) * A(:, o_g : o_{g+1}) * B(:, o_g : o_{g+1})^T + (*beta) * C_g
 *
 * A is m x k, B is n x k, C_g is m x n of type ctype at c + g * stride_c
 * (elements). An empty group gives C_g = (*beta) * C_g, which is zero when
 * *beta == 0. This is the weight gradient of an expert layer (A its tokens, B
 * the gradients of its outputs), accumulated where *beta == 1. Columns of A
 * and B outside the groups are never part of a sum, whatever they hold. */
sgblasStatus_t sgblasGroupedGemmK(sgblasHandle_t handle, int m, int n, int k, int groups,
                                  const int *offsets, const float *alpha, const void *a, int lda,
                                  const void *b, int ldb, const float *beta, void *c,
                                  sgblasDataType_t ctype, int ldc, long long stride_c);

/* Quantises `batch` column-major k x n matrices of type xtype to e4m3, with a
 * scale for each block of 128 (along k) by block_n (1 or 128) columns:
 *
 *   scale = max(largest magnitude of the block, 2^-100) / 448
 *   q     = x * (1 / scale), rounded to the nearest e4m3 value
 *
 * The divisions and the product are rounded to nearest in FP32. A NaN or an infinity in a block makes its
 * scale NaN or infinite. scale is a column-major ceil(k/128) x ceil(n/block_n)
 * FP32 matrix. Strides in elements of each array (unused for batch == 1). The
 * values are multiplied by the scale's reciprocal, not divided by the scale, so
 * next to a tie either neighbour may be taken. */
sgblasStatus_t sgblasQuantizeFp8(sgblasHandle_t handle, int k, int n, int batch, int block_n,
                                 const void *x, sgblasDataType_t xtype, int ldx,
                                 long long stride_x, void *q, int ldq, long long stride_q,
                                 float *scale, int ldscale, long long stride_scale);

/* C = A^T * B with e4m3 inputs and a scale for each block of 128 along k:
 *
 *   C(i, j) = sum over blocks b of scale_a(b, i / 128) * scale_b(b, j) *
 *             sum over k in b of A(k, i) * B(k, j)
 *
 * A is k x m (weights, scale_a ceil(k/128) x ceil(m/128)), B is k x n (tokens,
 * scale_b ceil(k/128) x n), C is m x n of type ctype. A block's two scales are
 * multiplied in FP32 first (their product should be in its range), then its sum
 * is scaled and added in FP32. k == 0 writes zeros. */
sgblasStatus_t sgblasGemmFp8(sgblasHandle_t handle, int m, int n, int k, const void *a, int lda,
                             const float *scale_a, int ldsa, const void *b, int ldb,
                             const float *scale_b, int ldsb, void *c, sgblasDataType_t ctype,
                             int ldc);

/* The same grouped along n, as sgblasGroupedGemmN: group g uses A_g at
 * a + g * stride_a and its scales at scale_a + g * stride_sa. */
sgblasStatus_t sgblasGroupedGemmFp8(sgblasHandle_t handle, int m, int n, int k, int groups,
                                    const int *offsets, const void *a, int lda,
                                    long long stride_a, const float *scale_a, int ldsa,
                                    long long stride_sa, const void *b, int ldb,
                                    const float *scale_b, int ldsb, void *c,
                                    sgblasDataType_t ctype, int ldc);

/* Orthogonalises a batch of m x n matrices G (type gtype) by Newton-Schulz
 * products, as an optimiser does with its update:
 *
 *   X = G / (||G||_F + eps)
 *   steps times:  X = c0 X + c1 (X X^T) X + c2 (X X^T)^2 X
 *   O = scale * X                                       (BF16, m x n)
 *
 * (with X^T X on the right where that is the smaller Gram matrix: the same
 * polynomial of the singular values). coefficients: host array {c0, c1, c2}.
 * Iterates are held as pairs of FP16 values (22 bits of values above 2^-16, an
 * absolute 2^-37 of smaller ones) and multiplied on the tensor cores with FP32
 * sums; the last product, whose result is rounded to BF16 at once, takes the
 * first FP16 value of each pair alone (11 bits). O differs from the FP32 iteration
 * by little more than its own rounding (1.70e-3 in norm for BF16's 1.66e-3),
 * unless eps leaves X next to nothing. G may be of any magnitude. Values of X, of the Gram matrix and of the
 * polynomial have to stay below 15.99 in magnitude, as they do for every
 * iteration that keeps singular values near one (|c0| + |c1| + |c2| of up to
 * 12 and singular values of up to 1.2 are safe). 1 <= steps <= 32. */
sgblasStatus_t sgblasOrthogonalize(sgblasHandle_t handle, int m, int n, int batch, int steps,
                                   const float *coefficients, float eps, float scale,
                                   const void *g, sgblasDataType_t gtype, int ldg,
                                   long long stride_g, void *o, int ldo, long long stride_o);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* SGBLAS_SGBLAS_LM_H_ */
