// Columns of several operands, copied by cp.async.bulk ahead of the CTA that walks them.
#ifndef SGBLAS_B200_RING_CUH_
#define SGBLAS_B200_RING_CUH_

#include "ptx.cuh"

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace sgblas::kern {

constexpr int kMaxStages = 8;

// Stages in shared memory, each with blockDim.y columns of kRows operands. Registers hold
// a column only while it is worked on, and the copies do not wait for its sums.
template <int kRows>
struct Ring {
  unsigned char *stages;
  uint64_t *full;
  int row_bytes, count;
  const unsigned char *from[kRows];   // NULL: no such operand
  long long ld[kRows];                // bytes

  __device__ __forceinline__ unsigned char *row(int stage, int operand, int y) const {
    return stages + static_cast<size_t>((stage * kRows + operand) * static_cast<int>(blockDim.y) + y) * row_bytes;
  }
  // The columns from `first` on (up to blockDim.y, of n) into a stage, by one warp. Where a
  // lane's `ok` is false, a wait of its own ran out: nothing is copied, and all lanes
  // get false (apart from each other they would not meet at the warp's barrier).
  __device__ __forceinline__ bool fill(int stage, long long first, int n, bool ok) const {
    if (__all_sync(0xffffffffu, ok) == 0) return false;
    const int columns = static_cast<int>(min(static_cast<long long>(blockDim.y), n - first));
    int operands = 0;
#pragma unroll
    for (int o = 0; o < kRows; ++o) operands += from[o] != nullptr;
    const int lane = threadIdx.x % 32;
    if (lane == 0) mbarArriveExpectTx(&full[stage], static_cast<uint32_t>(columns * operands * row_bytes));
    __syncwarp();
    if (lane < columns) {
#pragma unroll
      for (int o = 0; o < kRows; ++o)
        if (from[o] != nullptr)
          bulkLoad(row(stage, o, lane), from[o] + (first + lane) * ld[o], &full[stage],
                   static_cast<uint32_t>(row_bytes));
    }
    return true;
  }
};

// Walks a persistent grid's columns: work(stage, turn, column, in) for blockDim.y of
// them at a time (turn 0 and 1 by turns), which returns after a barrier of the CTA
// that follows its last read of the stage. A thread whose wait ran out polls the copies
// that may still be on their way a few times more, so that they do not outlive the CTA.
constexpr uint32_t kDrainPolls = 1u << 10;
template <int kRows, class Work>
__device__ __forceinline__ void walk(const Ring<kRows> &ring, int n, unsigned *err, Work work) {
  const bool issuer = threadIdx.x < 32 && threadIdx.y == 0;
  const long long first = blockIdx.x * static_cast<long long>(blockDim.y);
  const long long step = gridDim.x * static_cast<long long>(blockDim.y);
  if (issuer) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < ring.count; ++i) mbarInit(&ring.full[i], 1);
      fenceBarrierInit();
    }
    __syncwarp();
    for (int i = 0; i < ring.count; ++i)
      if (first + i * step < n) (void)ring.fill(i, first + i * step, n, true);
  }
  __syncthreads();
  int stage = 0, turn = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (long long c = first; c < n; c += step, turn ^= 1) {
    if (ok) {
      ok = mbarWait(&ring.full[stage], parity, err);
      if (!ok) {
        for (int i = 0, s = stage; i < ring.count && c + i * step < n; ++i) {
          (void)mbarWait(&ring.full[s], s < stage ? parity ^ 1 : parity, nullptr, kDrainPolls);
          if (++s == ring.count) s = 0;
        }
      }
    }
    work(stage, turn, c + threadIdx.y, c + threadIdx.y < n);
    const long long next = c + ring.count * step;
    if (issuer && next < n) {
      fenceProxyAsyncShared();   // the reads above come before the copy
      ok = ring.fill(stage, next, n, ok);
    }
    if (++stage == ring.count) {
      stage = 0;
      parity ^= 1;
    }
  }
}

}  // namespace sgblas::kern

#endif  // SGBLAS_B200_RING_CUH_
