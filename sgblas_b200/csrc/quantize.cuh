// Values to e4m3 (fp8.cu, norm.cu): a block's scale, and the bytes.
#ifndef SGBLAS_B200_QUANTIZE_CUH_
#define SGBLAS_B200_QUANTIZE_CUH_

#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sgblas::kern {

constexpr float kFp8Max = 448.0F;
constexpr unsigned kAmaxFloorBits = 0x0D800000u;   // 2^-100

// The scale of a block whose largest magnitude has these bits (a NaN's are larger
// than any number's).
__device__ __forceinline__ float fp8Scale(unsigned amax_bits) {
  return __fdiv_rn(__uint_as_float(max(amax_bits, kAmaxFloorBits)), kFp8Max);
}

// Pairs of values times `inverse` to bytes kStep apart, `left` of which exist; kStep
// 1: as one word where all do (`at` is then aligned to it).
template <int kPairs, int kStep>
__device__ __forceinline__ void storeFp8(unsigned char *at, const float2 (&f)[kPairs], int left,
                                         float inverse) {
  static_assert(kPairs == 2 || kPairs == 4, "a word or two");
  alignas(8) __nv_fp8x2_storage_t q[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
    q[i] = __nv_cvt_float2_to_fp8x2(__fmul2_rn(f[i], make_float2(inverse, inverse)), __NV_SATFINITE,
                                    __NV_E4M3);
  if (kStep == 1 && left >= 2 * kPairs) {
    if constexpr (kPairs == 4) *reinterpret_cast<uint2 *>(at) = *reinterpret_cast<const uint2 *>(q);
    else *reinterpret_cast<uint32_t *>(at) = *reinterpret_cast<const uint32_t *>(q);
  } else if (kStep > 1) {
    const auto *bytes = reinterpret_cast<const unsigned char *>(q);
#pragma unroll
    for (int j = 0; j < 2 * kPairs; ++j)
      if (j * kStep < left) at[j * kStep] = bytes[j];
  }
}

}  // namespace sgblas::kern

#endif  // SGBLAS_B200_QUANTIZE_CUH_
