// Host side of the 16- and 8-bit tensor-core products (product_tile.cuh).
#ifndef SGBLAS_B200_PRODUCT_HPP_
#define SGBLAS_B200_PRODUCT_HPP_

#include "context.hpp"
#include "product_tile.cuh"

#include <sgblas/sgblas_lm.h>

#include <cuda_runtime.h>

#include <cstddef>

namespace sgblas::detail {

// An operand as it lies in memory: `count` matrices of `dim1` rows of `dim0`
// contiguous elements, rows `ld` and matrices `stride` elements apart.
struct NarrowOperand {
  const void *ptr = nullptr;
  int dim0 = 0, dim1 = 0;
  long long ld = 0;
  int count = 1;
  long long stride = 0;
};

// The device a call runs on, checked: SUCCESS, EXECUTION_FAILED or ARCH_MISMATCH.
struct DeviceInfo {
  int device = -1;
  int sms = 0;
  unsigned *err = nullptr;
};
sgblasStatus_t currentDevice(DeviceInfo *info);

// Launches a product of `elem_bytes` operands (1: e4m3, 2: 16-bit). `mn`
// operands are contiguous along m (or n) instead of k. p carries the sizes,
// C, the scalars, scales, offsets and type bits; the maps and tile counts are
// filled in here. An operand that TMA cannot read is copied first.
sgblasStatus_t launchNarrow(sgblasContext *ctx, const DeviceInfo &dev, int elem_bytes,
                            kern::prod::Ragged ragged, NarrowOperand a, bool a_mn,
                            NarrowOperand b, bool b_mn, kern::prod::Params p);

}  // namespace sgblas::detail

#endif  // SGBLAS_B200_PRODUCT_HPP_
