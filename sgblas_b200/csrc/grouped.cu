// Entry points of the grouped BF16 products (sgblas_lm.h): argument checks in
// sgblasSgemm's order, then one launch.
#include "product.hpp"

#include <algorithm>

namespace sgblas::detail {
namespace {

namespace t = kern::prod;

}  // namespace
}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasGroupedGemmN(sgblasHandle_t handle, sgblasOperation_t transa,
                                             int m, int n, int k, int groups, const int *offsets,
                                             const float *alpha, const void *a, int lda,
                                             long long stride_a, const void *b, int ldb,
                                             const float *beta, void *c, sgblasDataType_t ctype,
                                             int ldc) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  if ((transa != SGBLAS_OP_N && transa != SGBLAS_OP_T) || m < 0 || n < 0 || k < 0 || groups < 0 ||
      !isType(ctype))
    return SGBLAS_STATUS_INVALID_VALUE;
  const int rows_a = transa == SGBLAS_OP_N ? m : k;
  if (lda < std::max(1, rows_a) || ldb < std::max(1, k) || ldc < std::max(1, m))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || groups == 0) return SGBLAS_STATUS_SUCCESS;
  if (alpha == nullptr || beta == nullptr || offsets == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  const bool product = k > 0 && *alpha != 0.0F;
  if (!product && *beta == 1.0F) return SGBLAS_STATUS_SUCCESS;
  if (c == nullptr || (product && (a == nullptr || b == nullptr)))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (groups > SGBLAS_MAX_GROUPS) return SGBLAS_STATUS_NOT_SUPPORTED;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  t::Params p = {};
  p.offsets = offsets;
  p.groups = groups;
  p.m = m;
  p.n = n;
  p.k = product ? k : 0;
  p.c = c;
  p.c_bf16 = ctype == SGBLAS_TYPE_BF16;
  p.ldc = ldc;
  p.alpha = product ? *alpha : 0.0F;
  p.beta = *beta;
  p.format = t::kFormatBf16;
  NarrowOperand oa, ob;
  oa.ptr = a;
  oa.dim0 = rows_a;
  oa.dim1 = transa == SGBLAS_OP_N ? k : m;
  oa.ld = lda;
  oa.count = groups;
  oa.stride = stride_a;
  ob.ptr = b;
  ob.dim0 = k;
  ob.dim1 = n;
  ob.ld = ldb;
  return launchNarrow(handle, dev, 2, t::Ragged::kN, oa, transa == SGBLAS_OP_N, ob, false, p);
}

extern "C" sgblasStatus_t sgblasGroupedGemmK(sgblasHandle_t handle, int m, int n, int k,
                                             int groups, const int *offsets, const float *alpha,
                                             const void *a, int lda, const void *b, int ldb,
                                             const float *beta, void *c, sgblasDataType_t ctype,
                                             int ldc, long long stride_c) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  if (m < 0 || n < 0 || k < 0 || groups < 0 || !isType(ctype) || lda < std::max(1, m) ||
      ldb < std::max(1, n) || ldc < std::max(1, m))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || groups == 0) return SGBLAS_STATUS_SUCCESS;
  if (alpha == nullptr || beta == nullptr || offsets == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  const bool product = k > 0 && *alpha != 0.0F;
  if (!product && *beta == 1.0F) return SGBLAS_STATUS_SUCCESS;
  if (c == nullptr || (product && (a == nullptr || b == nullptr)))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (groups > SGBLAS_MAX_GROUPS) return SGBLAS_STATUS_NOT_SUPPORTED;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  t::Params p = {};
  p.offsets = offsets;
  p.groups = groups;
  p.m = m;
  p.n = n;
  p.k = product ? k : 0;
  p.c = c;
  p.c_bf16 = ctype == SGBLAS_TYPE_BF16;
  p.ldc = ldc;
  p.stride_c = stride_c;
  p.alpha = product ? *alpha : 0.0F;
  p.beta = *beta;
  p.format = t::kFormatBf16;
  NarrowOperand oa, ob;
  oa.ptr = a;
  oa.dim0 = m;
  oa.dim1 = k;
  oa.ld = lda;
  ob.ptr = b;
  ob.dim0 = n;
  ob.dim1 = k;
  ob.ld = ldb;
  return launchNarrow(handle, dev, 2, t::Ragged::kK, oa, true, ob, true, p);
}
