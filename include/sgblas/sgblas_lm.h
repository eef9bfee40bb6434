/*
 * sgblas-b200: products of language models. Mixture-of-experts products whose
 * groups are ragged, 8-bit products with a scale for each block of 128 and 4-bit
 * ones with a power of two for each 32, the quantisation they need, and the orthogonalisation of an update by
 * Newton-Schulz products; around them the norm before a layer, and tokens
 * sorted by expert and back. No counterpart in the reference API, whose only
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
  SGBLAS_TYPE_BYTE = 2,   /* moved as they are: sgblasScatterTokens only */
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

/* Quantises `batch` column-major k x n matrices of type xtype to 4 bits, in the OCP
 * microscaling format MXFP4: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), and for
 * each block of 32 along k a power of two, as a byte (e8m0: 2^(byte - 127)):
 *
 *   byte = max(exponent byte of the block's largest magnitude in FP32 - 2, 0)
 *   q    = the e2m1 value nearest to x * 2^(127 - byte), ties to even, at most 6
 *
 * which is exact but for q's own rounding. A NaN or an infinity in a block makes its
 * byte 255, e8m0's NaN. Two values share a byte of q, the first in its low half;
 * a column is ceil(k/2) bytes (the last half of an odd k is zero) and ldq and stride_q
 * count bytes. scale is a column-major ceil(k/32) x n matrix of bytes. Strides are
 * unused for batch == 1. */
sgblasStatus_t sgblasQuantizeFp4(sgblasHandle_t handle, int k, int n, int batch, const void *x,
                                 sgblasDataType_t xtype, int ldx, long long stride_x, void *q,
                                 int ldq, long long stride_q, void *scale, int ldscale,
                                 long long stride_scale);

/* C = A^T * B with operands as sgblasQuantizeFp4 leaves them:
 *
 *   C(i, j) = sum over blocks b of 32 of k: 2^(sa(b, i) - 127) * 2^(sb(b, j) - 127) *
 *             sum over k in b of A(k, i) * B(k, j)
 *
 * A is k x m (weights, scale_a ceil(k/32) x m), B is k x n (tokens, scale_b ceil(k/32) x
 * n), C is m x n of type ctype; lda and ldb count bytes. Products and scales are
 * exact, sums are FP32, chained in the tensor core over at most 2048 of k for an
 * FP32 C (32 instructions, as in sgblasGroupedGemmN) and 4096 for a BF16 C; a block's two
 * scales together should be in FP32's range. With an odd k, the last half byte of every column has to
 * be zero. k == 0 writes zeros. Any alignment: operands and scales whose base is not
 * 16-byte aligned, or whose leading dimension (or stride) is not a multiple of 16
 * bytes, are first copied into the handle's workspace. */
sgblasStatus_t sgblasGemmFp4(sgblasHandle_t handle, int m, int n, int k, const void *a, int lda,
                             const void *scale_a, int ldsa, const void *b, int ldb,
                             const void *scale_b, int ldsb, void *c, sgblasDataType_t ctype,
                             int ldc);

/* The same grouped along n, as sgblasGroupedGemmFp8: group g uses A_g at a + g *
 * stride_a and its scales at scale_a + g * stride_sa (bytes). */
sgblasStatus_t sgblasGroupedGemmFp4(sgblasHandle_t handle, int m, int n, int k, int groups,
                                    const int *offsets, const void *a, int lda, long long stride_a,
                                    const void *scale_a, int ldsa, long long stride_sa,
                                    const void *b, int ldb, const void *scale_b, int ldsb, void *c,
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

/* Root-mean-square norm of the columns of a k x n matrix, after the residual's
 * addition:
 *
 *   h = x + residual                        rounded to type (residual NULL: h = x)
 *   v = h / sqrt(mean of h^2 + eps) * weight
 *
 * x, residual, weight (k values; NULL: ones), sum and y have type `type`. Written
 * are h to sum (NULL: not), v to y (NULL: not), and v in e4m3 to q (NULL: not),
 * with the scales in `scale`, as sgblasQuantizeFp8 with block_n = 1 writes them;
 * y or q has to be given. Everything between h and the roundings to y and q is
 * FP32: the sum of h^2 over a column has to stay below 2^128 (4096 values of 2^57 do;
 * from there on v is 0), and their mean, where eps is 0, at 2^-126 or above.
 * sum may be x or residual itself (the same address and leading dimension):
 * the residual is then updated in place. */
sgblasStatus_t sgblasRmsNorm(sgblasHandle_t handle, int k, int n, sgblasDataType_t type,
                             const void *x, int ldx, const void *residual, int ldr,
                             const void *weight, float eps, void *sum, int ldsum, void *y, int ldy,
                             void *q, int ldq, float *scale, int ldscale);

/* Its gradients, from dy = d(loss)/dy and h = sum. With s = 1 / sqrt(mean of h^2 +
 * eps), g = weight * dy, for each column:
 *
 *   dx      = dsum + s * (g - h * s^2 * mean of (h * g))
 *   dweight = (*beta) * dweight + sum over the columns of dy * h * s       (FP32)
 *
 * The sums of h^2 and of h * g over a column have to stay below 2^128 in magnitude,
 * and the mean of h^2, where eps is 0, at 2^-126 or above.
 * dx is the gradient of x and of the residual alike; dsum (NULL: zero) that which
 * reaches h past the norm. dweight NULL: not computed, beta unused; *beta == 0
 * writes it without reading. Sums are FP32 in an order that depends on the sizes
 * alone. dx may be dy or dsum itself (the same address and leading dimension).
 * dweight takes workspace: 4 bytes for each value of k and each CTA. */
sgblasStatus_t sgblasRmsNormBackward(sgblasHandle_t handle, int k, int n, sgblasDataType_t type,
                                     const void *dy, int lddy, const void *sum, int ldsum,
                                     const void *weight, float eps, const void *dsum, int lddsum,
                                     void *dx, int lddx, const float *beta, float *dweight);

/* Tokens sorted by group (expert). group is a DEVICE top x n matrix without gaps
 * between its columns (row-major [tokens, top]), the groups that each token goes
 * to; a value outside [0, groups) is none. Written are
 *
 *   offsets   groups + 1 places: where each group begins, as the grouped products
 *             take them; offsets[groups] is the number of choices that have a group
 *   place     top x n: the column of each choice in the sorted order, -1 for none
 *
 * The sort is stable: within a group by token, then by choice. At most 2^30
 * choices. offsets are written for n == 0, too. */
sgblasStatus_t sgblasSortTokens(sgblasHandle_t handle, int n, int top, int groups, const int *group,
                                int *offsets, int *place);

/* Tokens to their places: y(:, place(j, t)) = weights(j, t) * x(:, t), x k x n and y
 * k x rows of type `type`. place and weights (FP32; NULL: ones, and columns are
 * copied) are top x n without gaps. A place outside [0, rows) is none; columns
 * of y that no choice has are left as they were, and no two choices may have the
 * same. SGBLAS_TYPE_BYTE takes k bytes per column (quantised values, scales),
 * without weights. The gradient of sgblasGatherTokens by x. */
sgblasStatus_t sgblasScatterTokens(sgblasHandle_t handle, int k, int n, int top, int rows,
                                   const int *place, const float *weights, const void *x,
                                   sgblasDataType_t type, int ldx, void *y, int ldy);

/* And back: y(:, t) = sum over j of weights(j, t) * x(:, place(j, t)), x k x rows and
 * y k x n. Sums are FP32, in the order of j, rounded once; a choice without a
 * place adds nothing, whatever its weight, and a token without any gets zeros.
 * Choices may share a place; a token has at most 2^30 of them. With weights NULL,
 * the gradient of sgblasScatterTokens without weights. */
sgblasStatus_t sgblasGatherTokens(sgblasHandle_t handle, int k, int n, int top, int rows,
                                  const int *place, const float *weights, const void *x,
                                  sgblasDataType_t type, int ldx, void *y, int ldy);

/* Both gradients of sgblasGatherTokens:
 *
 *   dx(:, place(j, t)) = weights(j, t) * dy(:, t)
 *   dweights(j, t)     = sum over k of dy(k, t) * x(k, place(j, t))       (FP32; 0 for none)
 *
 * dweights NULL: not computed, x unused. No two choices may have the same place;
 * columns of dx that none has are left as they were. At most 2^30 choices of a token. */
sgblasStatus_t sgblasGatherTokensBackward(sgblasHandle_t handle, int k, int n, int top, int rows,
                                          const int *place, const float *weights, const void *dy,
                                          sgblasDataType_t type, int lddy, const void *x, int ldx,
                                          void *dx, int lddx, float *dweights);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* SGBLAS_SGBLAS_LM_H_ */
