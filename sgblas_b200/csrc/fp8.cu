// Entry points of the e4m3 products, and the quantisation to e4m3 with a
// scale for each block of 128 (sgblas_lm.h).
#include "product.hpp"

#include "device.hpp"
#include "ptx.cuh"
#include "sgemm_launch.hpp"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>

namespace sgblas::detail {
namespace {

namespace t = kern::prod;

constexpr float kFp8Max = 448.0F;
constexpr unsigned kAmaxFloorBits = 0x0D800000u;   // 2^-100
constexpr int kBlock = 128;
constexpr int kQuantThreads = 256;
constexpr int kQuantBlocks = 64;   // blocks of one CTA (quantizeColumnsKernel), aligned or not

struct QuantParams {
  const void *x;
  unsigned char *q;
  float *scale;
  int k, n, batch, kblocks, ldx, ldq, ldscale;
  long long stride_x, stride_q, stride_scale;
  unsigned blocks;   // of the whole batch
};

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }

// A thread's values of one block of 128, as they lie in memory. Aligned: 16
// consecutive ones, eight threads to a block, read and written as vectors.
// Otherwise a warp to a block, four values per thread 32 apart, so that a
// warp's scalar accesses are contiguous.
template <typename T, bool kVector>
struct Values {
  static constexpr int kPer = kVector ? 16 : 4;
  static constexpr int kLanes = kBlock / kPer;
  static constexpr int kStep = kVector ? 1 : kLanes;   // between a thread's values
  alignas(16) T v[kPer];

  // From `at`, where the block's value of this thread begins; `left` values of
  // the column are there. The rest are zero.
  __device__ __forceinline__ void load(const T *at, int left) {
    if (kVector && left >= kPer) {
#pragma unroll
      for (int j = 0; j < kPer * static_cast<int>(sizeof(T)) / 16; ++j)
        reinterpret_cast<uint4 *>(v)[j] = __ldg(reinterpret_cast<const uint4 *>(at) + j);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        v[j] = j * kStep < left ? at[j * kStep] : static_cast<T>(0.0F);
    }
  }
  // Largest magnitude as the bits of an FP32 value: an integer maximum, which a
  // NaN wins. BF16 values are compared two at a time, as halves of words.
  __device__ __forceinline__ unsigned magnitude() const {
    unsigned m = 0;
    if constexpr (sizeof(T) == 2) {
      const auto *w = reinterpret_cast<const unsigned *>(v);
#pragma unroll
      for (int j = 0; j < kPer / 2; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
      return max(m << 16, m & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      return m;
    }
  }
  __device__ __forceinline__ void store(unsigned char *at, int left, float inverse) const {
    alignas(16) __nv_fp8x2_storage_t q[kPer / 2];
#pragma unroll
    for (int j = 0; j < kPer; j += 2)
      q[j / 2] = __nv_cvt_float2_to_fp8x2(
          make_float2(toFloat(v[j]) * inverse, toFloat(v[j + 1]) * inverse), __NV_SATFINITE,
          __NV_E4M3);
    if (kVector && left >= kPer) {
      *reinterpret_cast<uint4 *>(at) = *reinterpret_cast<const uint4 *>(q);
    } else {
      const auto *bytes = reinterpret_cast<const unsigned char *>(q);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j * kStep < left) at[j * kStep] = bytes[j];
    }
  }
};

__device__ __forceinline__ float scaleOf(unsigned amax_bits) {
  return __fdiv_rn(__uint_as_float(max(amax_bits, kAmaxFloorBits)), kFp8Max);
}

// A scale for each 128 values of one column; kUnroll blocks per thread, whose
// loads are issued together. Memory-bound: one read and one write of each
// value (16384 x 8192 BF16: 65 to 71 us, 5.7 to 6.2 TB/s; by elements, with a
// division each, it took 165).
template <typename T, bool kVector>
__global__ void __launch_bounds__(kQuantThreads) quantizeColumnsKernel(const QuantParams p) {
  using V = Values<T, kVector>;
  constexpr int kUnroll = kVector ? 2 : 8;
  constexpr int kAtOnce = kQuantThreads / V::kLanes;   // blocks
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int part = threadIdx.x % V::kLanes;
  const unsigned first = blockIdx.x * static_cast<unsigned>(kUnroll * kAtOnce) +
                         threadIdx.x / static_cast<unsigned>(V::kLanes);
  V v[kUnroll];
  size_t to[kUnroll];
  float *scale_to[kUnroll];
  int left[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const unsigned block = first + u * kAtOnce;
    const bool in = block < p.blocks;
    const unsigned column = in ? block / static_cast<unsigned>(p.kblocks) : 0;
    const int kb = in ? static_cast<int>(block - column * p.kblocks) : 0;
    const unsigned matrix = p.batch > 1 ? column / static_cast<unsigned>(p.n) : 0;
    const long long col = column - matrix * static_cast<unsigned>(p.n);
    const int k0 = kb * kBlock + part * (kVector ? V::kPer : 1);
    left[u] = in ? min(p.k - k0, kBlock) : 0;
    v[u].load(static_cast<const T *>(p.x) + matrix * p.stride_x + col * p.ldx + k0, left[u]);
    to[u] = static_cast<size_t>(matrix * p.stride_q + col * p.ldq + k0);
    scale_to[u] = in && part == 0 ? p.scale + matrix * p.stride_scale + col * p.ldscale + kb : nullptr;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    unsigned m = v[u].magnitude();
#pragma unroll
    for (int d = V::kLanes / 2; d > 0; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float scale = scaleOf(m);
    v[u].store(p.q + to[u], left[u], __frcp_rn(scale));
    if (scale_to[u] != nullptr) *scale_to[u] = scale;
  }
}

// A scale for each 128 x 128 block: one CTA per block, values in registers.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kQuantThreads) quantizeBlocksKernel(const QuantParams p) {
  using V = Values<T, kVector>;
  constexpr int kAtOnce = kQuantThreads / V::kLanes;   // columns
  constexpr int kPasses = kBlock / kAtOnce;
  __shared__ unsigned warp_max[kQuantThreads / 32];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const unsigned nblocks = static_cast<unsigned>((p.n - 1) / kBlock + 1);
  const unsigned kblocks = static_cast<unsigned>(p.kblocks);
  const int kb = static_cast<int>(blockIdx.x % kblocks);
  const int nb = static_cast<int>(blockIdx.x / kblocks % nblocks);
  const long long matrix = blockIdx.x / kblocks / nblocks;
  const int part = threadIdx.x % V::kLanes;
  const int k0 = kb * kBlock + part * (kVector ? V::kPer : 1);
  const int left_k = min(p.k - k0, kBlock);
  const long long col0 = nb * static_cast<long long>(kBlock) + threadIdx.x / V::kLanes;
  const T *x = static_cast<const T *>(p.x) + matrix * p.stride_x + k0;
  V v[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const long long col = col0 + i * kAtOnce;
    v[i].load(x + col * p.ldx, col < p.n ? left_k : 0);
  }
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) m = max(m, v[i].magnitude());
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / 32; ++w) m = max(m, warp_max[w]);
  const float scale = scaleOf(m);
  const float inverse = __frcp_rn(scale);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const long long col = col0 + i * kAtOnce;
    v[i].store(p.q + matrix * p.stride_q + col * p.ldq + k0, col < p.n ? left_k : 0, inverse);
  }
  if (threadIdx.x == 0)
    p.scale[matrix * p.stride_scale + static_cast<long long>(nb) * p.ldscale + kb] = scale;
}

template <typename T, bool kVector>
cudaError_t launchQuantize(const QuantParams &p, int block_n, unsigned grid, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kQuantThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return block_n == 1 ? cudaLaunchKernelEx(&cfg, quantizeColumnsKernel<T, kVector>, p)
                      : cudaLaunchKernelEx(&cfg, quantizeBlocksKernel<T, kVector>, p);
}

sgblasStatus_t gemmFp8(sgblasHandle_t handle, int m, int n, int k, int groups, const int *offsets,
                       bool grouped, const void *a, int lda, long long stride_a,
                       const float *scale_a, int ldsa, long long stride_sa, const void *b, int ldb,
                       const float *scale_b, int ldsb, void *c, sgblasDataType_t ctype, int ldc) {
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int kblocks = k > 0 ? (k - 1) / kBlock + 1 : 0;
  if (m < 0 || n < 0 || k < 0 || groups < 0 || !isType(ctype) || lda < std::max(1, k) ||
      ldb < std::max(1, k) || ldc < std::max(1, m) || ldsa < std::max(1, kblocks) ||
      ldsb < std::max(1, kblocks))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || groups == 0) return SGBLAS_STATUS_SUCCESS;
  if (c == nullptr || (grouped && offsets == nullptr) ||
      (k > 0 && (a == nullptr || b == nullptr || scale_a == nullptr || scale_b == nullptr)))
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
  p.k = k;
  p.c = c;
  p.c_bf16 = ctype == SGBLAS_TYPE_BF16;
  p.ldc = ldc;
  p.alpha = 1.0F;
  p.scale_a = scale_a;
  p.scale_b = scale_b;
  p.ldsa = ldsa;
  p.ldsb = ldsb;
  p.stride_sa = stride_sa;
  p.format = t::kFormatE4m3;
  NarrowOperand oa, ob;
  oa.ptr = a;
  oa.dim0 = k;
  oa.dim1 = m;
  oa.ld = lda;
  oa.count = groups;
  oa.stride = stride_a;
  ob.ptr = b;
  ob.dim0 = k;
  ob.dim1 = n;
  ob.ld = ldb;
  return launchNarrow(handle, dev, 1, t::Ragged::kN, oa, false, ob, false, p);
}

}  // namespace
}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasQuantizeFp8(sgblasHandle_t handle, int k, int n, int batch,
                                            int block_n, const void *x, sgblasDataType_t xtype,
                                            int ldx, long long stride_x, void *q, int ldq,
                                            long long stride_q, float *scale, int ldscale,
                                            long long stride_scale) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int kblocks = k > 0 ? (k - 1) / kBlock + 1 : 0;
  if (k < 0 || n < 0 || batch < 0 || (block_n != 1 && block_n != kBlock) || !isType(xtype) ||
      ldx < std::max(1, k) || ldq < std::max(1, k) || ldscale < std::max(1, kblocks))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (k == 0 || n == 0 || batch == 0) return SGBLAS_STATUS_SUCCESS;
  if (x == nullptr || q == nullptr || scale == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  QuantParams p = {};
  p.x = x;
  p.q = static_cast<unsigned char *>(q);
  p.scale = scale;
  p.k = k;
  p.n = n;
  p.batch = batch;
  p.kblocks = kblocks;
  p.ldx = ldx;
  p.ldq = ldq;
  p.ldscale = ldscale;
  if (batch > 1) {
    p.stride_x = stride_x;
    p.stride_q = stride_q;
    p.stride_scale = stride_scale;
  }
  const long long nblocks = block_n == 1 ? n : (n - 1) / kBlock + 1;
  const double blocks = static_cast<double>(nblocks) * kblocks * batch;
  if (blocks > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;   // 256 GiB of values
  p.blocks = static_cast<unsigned>(blocks);
  const unsigned grid = block_n == 1 ? (p.blocks + kQuantBlocks - 1) / kQuantBlocks : p.blocks;
  const auto stream = static_cast<cudaStream_t>(handle->stream);
  // Whole vectors where every kPer values start on 16 bytes of x and of q.
  const int xsize = xtype == SGBLAS_TYPE_BF16 ? 2 : 4;
  const bool vector = aligned16(x) && ldx * static_cast<long long>(xsize) % 16 == 0 &&
                      p.stride_x * xsize % 16 == 0 && aligned16(q) && ldq % 16 == 0 &&
                      p.stride_q % 16 == 0;
  if (xtype == SGBLAS_TYPE_BF16)
    return launchStatus(vector ? launchQuantize<__nv_bfloat16, true>(p, block_n, grid, stream)
                               : launchQuantize<__nv_bfloat16, false>(p, block_n, grid, stream));
  return launchStatus(vector ? launchQuantize<float, true>(p, block_n, grid, stream)
                             : launchQuantize<float, false>(p, block_n, grid, stream));
}

extern "C" sgblasStatus_t sgblasGemmFp8(sgblasHandle_t handle, int m, int n, int k, const void *a,
                                        int lda, const float *scale_a, int ldsa, const void *b,
                                        int ldb, const float *scale_b, int ldsb, void *c,
                                        sgblasDataType_t ctype, int ldc) {
  return sgblas::detail::gemmFp8(handle, m, n, k, 1, nullptr, false, a, lda, 0, scale_a, ldsa, 0, b,
                                 ldb, scale_b, ldsb, c, ctype, ldc);
}

extern "C" sgblasStatus_t sgblasGroupedGemmFp8(sgblasHandle_t handle, int m, int n, int k,
                                               int groups, const int *offsets, const void *a,
                                               int lda, long long stride_a, const float *scale_a,
                                               int ldsa, long long stride_sa, const void *b,
                                               int ldb, const float *scale_b, int ldsb, void *c,
                                               sgblasDataType_t ctype, int ldc) {
  return sgblas::detail::gemmFp8(handle, m, n, k, groups, offsets, true, a, lda, stride_a, scale_a,
                                 ldsa, stride_sa, b, ldb, scale_b, ldsb, c, ctype, ldc);
}
