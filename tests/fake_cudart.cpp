// A stand-in for the CUDA runtime that the host code of the library is linked
// with to be tested without a GPU (tests/fake_cuda.py): one device of compute
// capability 10.0 with 148 SMs, memory that nothing reads, launches that run
// nothing. What the library does is written to a log, a line per call:
//
//   launch <mangled kernel> <grid.x>     record     wait
//   malloc <address> <bytes>             free <address>
//
// fakeFailLaunch(n) makes the n-th launch from now fail, fakeCapture(1) makes
// every stream look captured. Only what the library uses is provided.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {

std::map<const void *, std::string> &kernels() {
  static std::map<const void *, std::string> names;
  return names;
}
std::string &record() {
  static std::string text;
  return text;
}
int fail_launch = 0;
bool captured = false;
uintptr_t next_address = 0x100000000;

void say(const std::string &line) { record() += line + "\n"; }

std::string hex(const void *p) {
  char text[32];
  std::snprintf(text, sizeof(text), "%p", p);
  return text;
}

cudaError_t launch(const void *kernel, dim3 grid) {
  if (fail_launch > 0 && --fail_launch == 0) return cudaErrorLaunchOutOfResources;
  say("launch " + kernels()[kernel] + " " + std::to_string(grid.x));
  return cudaSuccess;
}

cudaError_t allocate(void **p, size_t bytes) {
  *p = reinterpret_cast<void *>(next_address);
  next_address += (bytes + 511) / 512 * 512;
  say("malloc " + hex(*p) + " " + std::to_string(bytes));
  return cudaSuccess;
}
cudaError_t release(void *p) {
  say("free " + hex(p));
  return cudaSuccess;
}

CUresult encodeTiled(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                     const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                     CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                     CUtensorMapFloatOOBfill) {
  return CUDA_SUCCESS;
}
CUresult currentContext(CUcontext *context) {
  *context = reinterpret_cast<CUcontext>(0x10);
  return CUDA_SUCCESS;
}

}  // namespace

extern "C" {

const char *fakeLog() { return record().c_str(); }
const char *fakeKernels() {   // every kernel of the library, a line each
  static std::string text;
  text.clear();
  for (const auto &k : kernels()) text += k.second + "\n";
  return text.c_str();
}
void fakeReset() {
  record().clear();
  fail_launch = 0;
  captured = false;
}
void fakeFailLaunch(int n) { fail_launch = n; }
void fakeCapture(int on) { captured = on != 0; }

void **__cudaRegisterFatBinary(void *) {
  static void *handle;
  return &handle;
}
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *host, char *, const char *name, int, uint3 *,
                            uint3 *, dim3 *, dim3 *, int *) {
  kernels()[host] = name;
}
void __cudaRegisterVar(void **, char *, char *, const char *, int, size_t, int, int) {}
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void *) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3 *grid, dim3 *block, size_t *smem, void *stream) {
  *grid = *block = dim3{1, 1, 1};
  *smem = 0;
  *static_cast<void **>(stream) = nullptr;
  return cudaSuccess;
}

cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *config, const void *kernel, void **) {
  return launch(kernel, config->gridDim);
}
cudaError_t cudaLaunchKernel(const void *kernel, dim3 grid, dim3, void **, size_t, cudaStream_t) {
  return launch(kernel, grid);
}
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int *clusters, const void *,
                                           const cudaLaunchConfig_t *config) {
  *clusters = 148 / static_cast<int>(config->attrs[0].val.clusterDim.x);
  return cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaGetDevice(int *device) {
  *device = 0;
  return cudaSuccess;
}
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int *value, cudaDeviceAttr attribute, int) {
  *value = attribute == cudaDevAttrComputeCapabilityMajor   ? 10
           : attribute == cudaDevAttrComputeCapabilityMinor ? 0
           : attribute == cudaDevAttrMultiProcessorCount    ? 148
                                                            : 1;
  return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() { return cudaSuccess; }
cudaError_t cudaGetDriverEntryPointByVersion(const char *name, void **entry, unsigned,
                                             unsigned long long,
                                             cudaDriverEntryPointQueryResult *found) {
  *entry = std::strcmp(name, "cuTensorMapEncodeTiled") == 0 ? reinterpret_cast<void *>(encodeTiled)
           : std::strcmp(name, "cuCtxGetCurrent") == 0      ? reinterpret_cast<void *>(currentContext)
                                                            : nullptr;
  *found = *entry != nullptr ? cudaDriverEntryPointSuccess : cudaDriverEntryPointSymbolNotFound;
  return cudaSuccess;
}
cudaError_t cudaGetSymbolAddress(void **address, const void *) {
  static unsigned word[1024];
  *address = word;
  return cudaSuccess;
}

cudaError_t cudaMalloc(void **p, size_t bytes) { return allocate(p, bytes); }
cudaError_t cudaMallocAsync(void **p, size_t bytes, cudaStream_t) { return allocate(p, bytes); }
cudaError_t cudaMallocManaged(void **p, size_t bytes, unsigned) { return allocate(p, bytes); }
cudaError_t cudaFree(void *p) { return release(p); }
cudaError_t cudaFreeAsync(void *p, cudaStream_t) { return release(p); }
cudaError_t cudaMemsetAsync(void *, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaMemcpyFromSymbol(void *to, const void *, size_t bytes, size_t, cudaMemcpyKind) {
  std::memset(to, 0, bytes);
  return cudaSuccess;
}
cudaError_t cudaMemcpyToSymbol(const void *, const void *, size_t, size_t, cudaMemcpyKind) {
  return cudaSuccess;
}

cudaError_t cudaEventCreateWithFlags(cudaEvent_t *event, unsigned) {
  *event = reinterpret_cast<cudaEvent_t>(0x20);
  return cudaSuccess;
}
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) {
  say("record");
  return cudaSuccess;
}
cudaError_t cudaStreamWaitEvent(cudaStream_t, cudaEvent_t, unsigned) {
  say("wait");
  return cudaSuccess;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus *status) {
  *status = captured ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}

// The multi-GPU part links against these; no test here calls it.
cudaError_t cudaStreamCreateWithFlags(cudaStream_t *, unsigned) { return cudaErrorNotSupported; }
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaStreamQuery(cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaDeviceEnablePeerAccess(int, unsigned) { return cudaErrorNotSupported; }
cudaError_t cudaHostGetDevicePointer(void **, void *, unsigned) { return cudaErrorNotSupported; }
cudaError_t cudaHostRegister(void *, size_t, unsigned) { return cudaErrorNotSupported; }
cudaError_t cudaHostUnregister(void *) { return cudaErrorNotSupported; }
cudaError_t cudaIpcCloseMemHandle(void *) { return cudaErrorNotSupported; }
cudaError_t cudaIpcGetMemHandle(cudaIpcMemHandle_t *, void *) { return cudaErrorNotSupported; }
cudaError_t cudaIpcOpenMemHandle(void **, cudaIpcMemHandle_t, unsigned) {
  return cudaErrorNotSupported;
}
cudaError_t cudaMemcpy2DAsync(void *, size_t, const void *, size_t, size_t, size_t, cudaMemcpyKind,
                              cudaStream_t) {
  return cudaErrorNotSupported;
}

}  // extern "C"
