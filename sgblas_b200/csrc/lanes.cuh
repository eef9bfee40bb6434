// A column's values spread over threads, for the memory-bound operators: what
// one thread holds of a block of 128 values.
#ifndef SGBLAS_B200_LANES_CUH_
#define SGBLAS_B200_LANES_CUH_

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sgblas::kern {

constexpr int kLaneBlock = 128;

// Columns of whole aligned vectors (kVector): one vector of 16 bytes. Otherwise four
// values 32 apart, so that a warp holds a block and its scalar accesses are
// contiguous.
template <typename T, bool kVector>
struct Lanes {
  static constexpr int kPer = kVector ? 16 / static_cast<int>(sizeof(T)) : 4;
  static constexpr int kThreads = kLaneBlock / kPer;     // of a block
  static constexpr int kStep = kVector ? 1 : kThreads;   // between a thread's values
  alignas(16) T v[kPer];

  // Where thread `slot` of a column's begins: its place in the column.
  static __device__ __forceinline__ int begin(int slot) {
    return kVector ? slot * kPer : slot / kThreads * kLaneBlock + slot % kThreads;
  }
  // From `at`; `left` values of the column are there (whole vectors with kVector),
  // the rest are zero. One predicated load: a branch to a partial form would keep
  // a thread's loads from being issued together.
  __device__ __forceinline__ void load(const T *at, int left) {
    if constexpr (kVector) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (left > 0) w = *reinterpret_cast<const uint4 *>(at);
      *reinterpret_cast<uint4 *>(v) = w;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = j * kStep < left ? at[j * kStep] : T{};
    }
  }
  __device__ __forceinline__ void store(T *at, int left) const {
    if constexpr (kVector) {
      if (left > 0) *reinterpret_cast<uint4 *>(at) = *reinterpret_cast<const uint4 *>(v);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j * kStep < left) at[j * kStep] = v[j];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = T{};
  }
  // Keeps the values as they lie: the compiler would otherwise unpack BF16 ahead of
  // their use, and hold twice the registers across a barrier or a loop.
  __device__ __forceinline__ void hold() {
    if constexpr (sizeof(T) == 2 && kVector) {
      auto *w = reinterpret_cast<uint32_t *>(v);
      asm volatile("" : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]));
    }
  }
  // Two values at a time: packed FP32 arithmetic, and one conversion for both (by
  // single values the norm of 16384 x 4096 took 28 instructions a value, bound by
  // their issue).
  static constexpr int kPairs = kPer / 2;
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 2 && kVector) {
      const uint32_t w = reinterpret_cast<const uint32_t *>(v)[i];
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    } else {
      return make_float2(static_cast<float>(v[2 * i]), static_cast<float>(v[2 * i + 1]));
    }
  }
  __device__ __forceinline__ void setPair(int i, float2 f) {
    if constexpr (sizeof(T) == 2 && kVector) {
      reinterpret_cast<__nv_bfloat162 *>(v)[i] = __float22bfloat162_rn(f);
    } else {
      v[2 * i] = static_cast<T>(f.x);
      v[2 * i + 1] = static_cast<T>(f.y);
    }
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// kWords words from any address of whole values (of 2 or 4 bytes): the aligned vectors
// of 16 bytes that hold them, moved into place. Reads up to 15 bytes beside them, inside
// their first and last vector.
template <int kWords>
__device__ __forceinline__ void loadShifted(const void *at, uint32_t (&w)[kWords]) {
  static_assert(kWords % 4 == 0, "whole vectors");
  const auto address = reinterpret_cast<uintptr_t>(at);
  const auto *from = reinterpret_cast<const uint4 *>(address & ~uintptr_t{15});
  const unsigned shift = static_cast<unsigned>(address & 15);
  uint32_t in[kWords + 4];
#pragma unroll
  for (int j = 0; j <= kWords / 4; ++j) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (j < kWords / 4 || shift != 0) v = __ldg(from + j);
    in[4 * j] = v.x;
    in[4 * j + 1] = v.y;
    in[4 * j + 2] = v.z;
    in[4 * j + 3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < kWords + 2; ++i) in[i] = shift & 8 ? in[i + 2] : in[i];
#pragma unroll
  for (int i = 0; i < kWords + 1; ++i) in[i] = shift & 4 ? in[i + 1] : in[i];
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(in[i], in[i + 1], shift % 4 * 8);
}

}  // namespace sgblas::kern

#endif  // SGBLAS_B200_LANES_CUH_
