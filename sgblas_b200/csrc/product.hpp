// Host side of the 16- and 8-bit tensor-core products (product_tile.cuh).
#ifndef SGBLAS_B200_PRODUCT_HPP_
#define SGBLAS_B200_PRODUCT_HPP_

#include "context.hpp"
#include "device.hpp"
#include "product_tile.cuh"
#include "sgemm_launch.hpp"

#include <sgblas/sgblas_lm.h>

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstdint>

namespace sgblas::detail {

inline bool isType(sgblasDataType_t type) {
  return type == SGBLAS_TYPE_FP32 || type == SGBLAS_TYPE_BF16;
}

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

// Persistent launch of productKernel<G> over at most `tiles` tiles: a worker
// (a CTA, or a cluster of two) per SM (or two).
template <class G>
sgblasStatus_t launchProductKernel(const DeviceInfo &dev, const kern::prod::Params &p,
                                   long long tiles, cudaStream_t stream) {
  auto kernel = kern::prod::productKernel<G>;
  static std::atomic<uint64_t> configured{0};
  if (!configureKernel(reinterpret_cast<const void *>(kernel), dev.device, G::kSmemBytes,
                       &configured))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  constexpr int kCtas = G::kTwo ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim =
      dim3(static_cast<unsigned>(kCtas * std::min<long long>(tiles, dev.sms / kCtas)));
  cfg.blockDim = dim3(kern::prod::kThreads);
  cfg.dynamicSmemBytes = G::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCtas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = G::kTwo ? 2 : 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, p));
}

// Whether TMA can read the operand as it lies.
bool tmaReadable(const NarrowOperand &o, int elem_bytes);
// Otherwise its copy's size, and the copy: to dst, where `o` then points; with offsets
// only the matrices of groups that have columns.
size_t copyBytes(const NarrowOperand &o, int elem_bytes);
sgblasStatus_t copyOperand(NarrowOperand *o, int elem_bytes, void *dst, int sms, const int *offsets,
                           cudaStream_t stream);
// Tensor map of the operand in boxes of 128 bytes by `rows` (K-major) or 64 rows.
bool encodeOperand(CUtensorMap *map, const NarrowOperand &o, int elem_bytes, bool mn, int rows);
// Whether TMA can write C: addresses and strides of whole 16-byte units (matrices
// `matrix` bytes apart), and such columns too, for it writes a column to the end
// of its last unit: rows beyond C, which are not C's.
bool tmaWritable(const kern::prod::Params &p, int size, long long matrix);

// Launches a product of `elem_bytes` operands (1: e4m3, 2: 16-bit). `mn`
// operands are contiguous along m (or n) instead of k. p carries the sizes,
// C, the scalars, scales, offsets and type bits; the maps and tile counts are
// filled in here. An operand that TMA cannot read is copied first.
sgblasStatus_t launchNarrow(sgblasContext *ctx, const DeviceInfo &dev, int elem_bytes,
                            kern::prod::Ragged ragged, NarrowOperand a, bool a_mn,
                            NarrowOperand b, bool b_mn, kern::prod::Params p);

}  // namespace sgblas::detail

#endif  // SGBLAS_B200_PRODUCT_HPP_
