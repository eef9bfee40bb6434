// Device error word and the diagnostics entry point that reads it.
#include "device.hpp"
#include "ptx.cuh"
#include "ring.cuh"

#include <cuda.h>

#include <new>

#include <sgblas/sgblas_ext.h>

namespace sgblas::detail {
namespace {

__device__ unsigned g_device_error;

SymbolCache g_error_word;

struct SymbolEntry {
  void *context;
  void *address;
};

using CtxGetCurrentFn = CUresult (*)(CUcontext *);

// The calling thread's current context, or nullptr (none yet, or the driver
// entry point is unavailable).
void *currentContext() {
  static const CtxGetCurrentFn fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuCtxGetCurrent", &f, 12000, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      return static_cast<CtxGetCurrentFn>(nullptr);
    }
    return reinterpret_cast<CtxGetCurrentFn>(f);
  }();
  CUcontext ctx = nullptr;
  if (fn == nullptr || fn(&ctx) != CUDA_SUCCESS) return nullptr;
  return ctx;
}

}  // namespace

void *symbolAddress(SymbolCache *cache, int device, const void *symbol) {
  if (device < 0 || device >= kMaxDevices) return nullptr;
  const void *context = currentContext();
  const auto *entry =
      static_cast<const SymbolEntry *>(cache->entry[device].load(std::memory_order_acquire));
  if (entry != nullptr && context != nullptr && entry->context == context) return entry->address;
  void *address = nullptr;
  if (cudaGetSymbolAddress(&address, symbol) != cudaSuccess) {   // makes the context current
    (void)cudaGetLastError();
    return nullptr;
  }
  context = currentContext();
  if (context != nullptr) {
    // Published once per (device, context); an entry replaced by a newer
    // one is left allocated (a few bytes per context change), so a reader
    // holding it never sees freed memory.
    auto *fresh = new (std::nothrow) SymbolEntry{const_cast<void *>(context), address};
    if (fresh != nullptr) cache->entry[device].store(fresh, std::memory_order_release);
  }
  return address;
}

unsigned *deviceErrorWord(int device) {
  return static_cast<unsigned *>(symbolAddress(&g_error_word, device, &g_device_error));
}

namespace {

__device__ uint4 g_ring_source = {1, 2, 3, 4};

// Waits on an mbarrier that nothing will ever complete, with a short poll
// limit: the wait must give up, raise the error flag and let the kernel
// return normally. Then a ring's stage is filled by a warp half of whose lanes gave up
// before (nothing may be copied, and all lanes have to know), and by one that did not.
// Reports whether all of it was so.
__global__ void waitTimeoutKernel(unsigned *err, unsigned polls, int *gave_up) {
  __shared__ uint64_t bars[2];
  __shared__ uint4 stage;
  if (threadIdx.x == 0) {
    kern::mbarInit(&bars[0], 1);
    kern::mbarInit(&bars[1], 1);
    kern::fenceBarrierInit();
    stage = make_uint4(0, 0, 0, 0);
  }
  kern::fenceProxyAsyncShared();
  __syncthreads();
  bool right = true;
  if (threadIdx.x == 0) right = !kern::mbarWait(&bars[0], 0, err, polls);
  __syncwarp();
  const kern::Ring<1> ring = {reinterpret_cast<unsigned char *>(&stage), &bars[1], sizeof(uint4), 1,
                              {reinterpret_cast<const unsigned char *>(&g_ring_source)}, {sizeof(uint4)}};
  const bool some = ring.fill(0, 0, 1, threadIdx.x % 2 != 0);
  right = right && !some && stage.x == 0 && !kern::mbarTestWait(&bars[1], 0);
  __syncwarp();
  right = ring.fill(0, 0, 1, true) && right;
  right = kern::mbarWait(&bars[1], 0, err) && right && stage.x == 1 && stage.w == 4;
  const bool all = __all_sync(0xffffffffu, right) != 0;
  if (threadIdx.x == 0) *gave_up = all ? 1 : 0;
}

}  // namespace

}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasSelfTestWaitTimeout(unsigned polls, int *timed_out) {
  if (timed_out == nullptr || polls == 0) return SGBLAS_STATUS_INVALID_VALUE;
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess) {
    (void)cudaGetLastError();
    return SGBLAS_STATUS_EXECUTION_FAILED;
  }
  unsigned *err = sgblas::detail::deviceErrorWord(device);
  if (err == nullptr) return SGBLAS_STATUS_EXECUTION_FAILED;
  int *flag = nullptr;
  if (cudaMallocManaged(&flag, sizeof(int)) != cudaSuccess) {
    (void)cudaGetLastError();
    return SGBLAS_STATUS_ALLOC_FAILED;
  }
  *flag = -1;
  sgblas::detail::waitTimeoutKernel<<<1, 32>>>(err, polls, flag);
  const cudaError_t e = cudaDeviceSynchronize();
  *timed_out = *flag;
  (void)cudaFree(flag);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return SGBLAS_STATUS_EXECUTION_FAILED;
  }
  return SGBLAS_STATUS_SUCCESS;
}

extern "C" sgblasStatus_t sgblasGetDeviceErrors(unsigned *flags, int clear) {
  if (flags == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  if (cudaDeviceSynchronize() != cudaSuccess) {
    (void)cudaGetLastError();
    return SGBLAS_STATUS_EXECUTION_FAILED;
  }
  unsigned value = 0;
  if (cudaMemcpyFromSymbol(&value, sgblas::detail::g_device_error, sizeof(value)) != cudaSuccess) {
    (void)cudaGetLastError();
    return SGBLAS_STATUS_EXECUTION_FAILED;
  }
  *flags = value;
  if (clear != 0) {
    const unsigned zero = 0;
    if (cudaMemcpyToSymbol(sgblas::detail::g_device_error, &zero, sizeof(zero)) != cudaSuccess) {
      (void)cudaGetLastError();
      return SGBLAS_STATUS_EXECUTION_FAILED;
    }
  }
  return SGBLAS_STATUS_SUCCESS;
}
