// sgblasRmsNorm and sgblasRmsNormBackward (sgblas_lm.h).
//
// Forward, for each column: h = x + r (held in the type), v = h * s * w with
// s = 1 / sqrt(mean h^2 + eps); out goes v, or v in e4m3 with a scale for each
// 128 values. Backward, with g = w dy:
//
//   dx = dsum + s (g - h s^2 mean(h g)),   dw = sum over the columns of dy h s
//
// Both are memory-bound: a column is read once, kept in registers while its
// sums are made, and written once. dw is summed in registers over the columns
// that a CTA walks, then over the CTAs in a second launch, in a fixed order.
#include "device.hpp"
#include "lanes.cuh"
#include "product.hpp"
#include "ptx.cuh"
#include "quantize.cuh"

#include <cuda_bf16.h>

#include <algorithm>

namespace sgblas::detail {
namespace {

using kern::Lanes;
using kern::warpSum;

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxUnits = 4;          // vectors of a column that a thread holds
constexpr int kReduceThreads = 256;
constexpr int kReduceWarps = kReduceThreads / 32;

struct NormParams {
  const void *x, *residual, *weight;
  void *sum, *y;
  unsigned char *q;
  float *scale;
  int k, n;
  float eps;
  int ldx, ldr, ldsum, ldy, ldq, ldscale;
};

struct NormBackwardParams {
  const void *dy, *sum, *weight, *dsum;
  void *dx;
  float *part;        // NULL: no gradient of the weights
  int k, n, part_ld;
  float eps;
  int lddy, ldsum, lddsum, lddx;
};

// The sums of two values over the threads of one column (blockDim.x of them, a
// multiple of 32; blockDim.y columns), the same in every thread, in a fixed order.
__device__ __forceinline__ float2 columnSum(float2 v, float2 *slots) {
  v.x = warpSum(v.x);
  v.y = warpSum(v.y);
  const int warps = static_cast<int>(blockDim.x) / 32;
  if (warps == 1) return v;
  float2 *mine = slots + threadIdx.y * warps;
  if (threadIdx.x % 32 == 0) mine[threadIdx.x / 32] = v;
  __syncthreads();
  float2 s = make_float2(0.0F, 0.0F);
  for (int w = 0; w < warps; ++w) {
    s.x += mine[w].x;
    s.y += mine[w].y;
  }
  __syncthreads();   // the slots are free again
  return s;
}

__device__ __forceinline__ float inverseLength(float squares, int k, float eps) {
  return 1.0F / sqrtf(squares / static_cast<float>(k) + eps);
}

// h = x + r as it is held.
template <typename T, bool kVector>
__device__ __forceinline__ void addResidual(Lanes<T, kVector> *h, const Lanes<T, kVector> &r) {
#pragma unroll
  for (int j = 0; j < Lanes<T, kVector>::kPer; ++j) h->set(j, h->get(j) + r.get(j));
}

// A column per blockDim.x threads, kUnits vectors (or groups of four values) per
// thread; kLong: longer columns than that, read twice.
template <typename T, bool kVector, int kUnits, bool kLong>
__global__ void __launch_bounds__(kMaxThreads) rmsNormKernel(const NormParams p) {
  using L = Lanes<T, kVector>;
  __shared__ float2 slots[kMaxWarps];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const long long col = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
  const bool in = col < p.n;
  const int stride = static_cast<int>(blockDim.x);
  // Slots of the column in whole warps: every thread of a warp takes part in its shuffles.
  const int rounds = ((p.k - 1) / kern::kLaneBlock * L::kThreads + L::kThreads + 31) / 32 * 32;
  const T *x = static_cast<const T *>(p.x) + (in ? col * p.ldx : 0);
  const T *r = p.residual == nullptr
                   ? nullptr
                   : static_cast<const T *>(p.residual) + (in ? col * p.ldr : 0);
  auto left = [&](int slot) { return in ? p.k - L::begin(slot) : 0; };
  auto read = [&](int slot, L *h) {
    const int at = L::begin(slot);
    h->load(x + at, left(slot));
    if (r != nullptr) {
      L v;
      v.load(r + at, left(slot));
      addResidual(h, v);
    }
  };
  L h[kUnits], w[kUnits];
  float squares = 0.0F;
  auto square = [&](const L &v) {
#pragma unroll
    for (int j = 0; j < L::kPer; ++j) squares = fmaf(v.get(j), v.get(j), squares);
  };
  auto readWeight = [&](int slot, L *v) {
    if (p.weight != nullptr)
      v->load(static_cast<const T *>(p.weight) + L::begin(slot), p.k - L::begin(slot));
  };
  if constexpr (kLong) {
    for (int slot = threadIdx.x; slot < rounds; slot += stride) {
      read(slot, &h[0]);
      square(h[0]);
    }
  } else {
    L v[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int slot = threadIdx.x + u * stride;
      h[u].load(x + L::begin(slot), left(slot));
      if (r != nullptr) v[u].load(r + L::begin(slot), left(slot));
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) readWeight(threadIdx.x + u * stride, &w[u]);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (r != nullptr) addResidual(&h[u], v[u]);
      square(h[u]);
    }
  }
  const float s =
      inverseLength(columnSum(make_float2(squares, 0.0F), slots).x, p.k, p.eps);
  auto write = [&](int slot, const L &value, const L &weight) {
    const int at = L::begin(slot), rest = left(slot);
    if (p.sum != nullptr) value.store(static_cast<T *>(p.sum) + (in ? col * p.ldsum : 0) + at, rest);
    float f[L::kPer];
#pragma unroll
    for (int j = 0; j < L::kPer; ++j) {
      f[j] = value.get(j) * s;
      if (p.weight != nullptr) f[j] *= weight.get(j);
    }
    if (p.y != nullptr) {
      L out;
#pragma unroll
      for (int j = 0; j < L::kPer; ++j) out.set(j, f[j]);
      out.store(static_cast<T *>(p.y) + (in ? col * p.ldy : 0) + at, rest);
    }
    if (p.q != nullptr) {
      unsigned m = 0;
#pragma unroll
      for (int j = 0; j < L::kPer; ++j)
        if (j * L::kStep < rest) m = max(m, __float_as_uint(f[j]) & 0x7FFFFFFFu);
#pragma unroll
      for (int d = L::kThreads / 2; d > 0; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float scale = kern::fp8Scale(m);
      kern::storeFp8<L::kPer, L::kStep>(p.q + (in ? col * p.ldq : 0) + at, f, rest, __frcp_rn(scale));
      if (rest > 0 && slot % L::kThreads == 0) p.scale[col * p.ldscale + slot / L::kThreads] = scale;
    }
  };
  if constexpr (kLong) {
    for (int slot = threadIdx.x; slot < rounds; slot += stride) {
      read(slot, &h[0]);
      readWeight(slot, &w[0]);
      write(slot, h[0], w[0]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) write(threadIdx.x + u * stride, h[u], w[u]);
  }
}

// Walks the columns blockIdx.x * blockDim.y + threadIdx.y, ... of a persistent
// grid; a row of partial sums of dw for each of its columns of threads.
template <typename T, bool kVector, int kUnits, bool kLong>
__global__ void __launch_bounds__(kMaxThreads) rmsNormBackwardKernel(const NormBackwardParams p) {
  using L = Lanes<T, kVector>;
  __shared__ float2 slots[kMaxWarps];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int stride = static_cast<int>(blockDim.x);
  const int rounds = ((p.k - 1) / kern::kLaneBlock + 1) * L::kThreads;
  const long long first = blockIdx.x * static_cast<long long>(blockDim.y);
  const long long step = gridDim.x * static_cast<long long>(blockDim.y);
  float *part = p.part == nullptr ? nullptr : p.part + (first + threadIdx.y) * p.part_ld;
  float dw[kLong ? 1 : kUnits][L::kPer];
  L w[kUnits];
  if constexpr (!kLong) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = L::begin(threadIdx.x + u * stride);
      if (p.weight != nullptr) w[u].load(static_cast<const T *>(p.weight) + at, p.k - at);
#pragma unroll
      for (int j = 0; j < L::kPer; ++j) dw[u][j] = 0.0F;
    }
  }
  for (long long c = first; c < p.n; c += step) {
    const long long col = c + threadIdx.y;
    const bool in = col < p.n;
    const T *h0 = static_cast<const T *>(p.sum) + (in ? col * p.ldsum : 0);
    const T *dy0 = static_cast<const T *>(p.dy) + (in ? col * p.lddy : 0);
    const T *ds0 = p.dsum == nullptr ? nullptr
                                     : static_cast<const T *>(p.dsum) + (in ? col * p.lddsum : 0);
    T *dx0 = static_cast<T *>(p.dx) + (in ? col * p.lddx : 0);
    float2 sums = make_float2(0.0F, 0.0F);   // of h^2 and h g
    auto add = [&](const L &h, const L &dy, const L &weight) {
#pragma unroll
      for (int j = 0; j < L::kPer; ++j) {
        const float g = p.weight != nullptr ? dy.get(j) * weight.get(j) : dy.get(j);
        sums.x = fmaf(h.get(j), h.get(j), sums.x);
        sums.y = fmaf(h.get(j), g, sums.y);
      }
    };
    L h[kUnits], dy[kUnits], ds[kUnits];
    if constexpr (kLong) {
      for (int slot = threadIdx.x; slot < rounds; slot += stride) {
        const int at = L::begin(slot), rest = in ? p.k - at : 0;
        h[0].load(h0 + at, rest);
        dy[0].load(dy0 + at, rest);
        if (p.weight != nullptr) w[0].load(static_cast<const T *>(p.weight) + at, p.k - at);
        add(h[0], dy[0], w[0]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int at = L::begin(threadIdx.x + u * stride), rest = in ? p.k - at : 0;
        h[u].load(h0 + at, rest);
        dy[u].load(dy0 + at, rest);
        if (ds0 != nullptr) ds[u].load(ds0 + at, rest);
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) add(h[u], dy[u], w[u]);
    }
    sums = columnSum(sums, slots);
    const float s = inverseLength(sums.x, p.k, p.eps);
    const float along = s * s * (sums.y / static_cast<float>(p.k));
    auto finish = [&](const L &hv, const L &dyv, const L &weight, const L &dsv, int at, int rest,
                      float *acc) {
      L out;
#pragma unroll
      for (int j = 0; j < L::kPer; ++j) {
        const float g = p.weight != nullptr ? dyv.get(j) * weight.get(j) : dyv.get(j);
        float d = s * fmaf(-hv.get(j), along, g);
        if (ds0 != nullptr) d += dsv.get(j);
        out.set(j, d);
        if (in) acc[j] = fmaf(dyv.get(j), hv.get(j) * s, acc[j]);
      }
      out.store(dx0 + at, rest);
    };
    if constexpr (kLong) {
      for (int slot = threadIdx.x; slot < rounds; slot += stride) {
        const int at = L::begin(slot), rest = in ? p.k - at : 0;
        h[0].load(h0 + at, rest);
        dy[0].load(dy0 + at, rest);
        if (p.weight != nullptr) w[0].load(static_cast<const T *>(p.weight) + at, p.k - at);
        if (ds0 != nullptr) ds[0].load(ds0 + at, rest);
#pragma unroll
        for (int j = 0; j < L::kPer; ++j)
          dw[0][j] = part != nullptr && c != first && at + j * L::kStep < p.k ? part[at + j * L::kStep]
                                                                            : 0.0F;
        finish(h[0], dy[0], w[0], ds[0], at, rest, dw[0]);
        if (part != nullptr) {
#pragma unroll
          for (int j = 0; j < L::kPer; ++j)
            if (at + j * L::kStep < p.k) part[at + j * L::kStep] = dw[0][j];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int at = L::begin(threadIdx.x + u * stride);
        finish(h[u], dy[u], w[u], ds[u], at, in ? p.k - at : 0, dw[u]);
      }
    }
  }
  if constexpr (!kLong) {
    if (part != nullptr) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int at = L::begin(threadIdx.x + u * stride);
#pragma unroll
        for (int j = 0; j < L::kPer; ++j)
          if (at + j * L::kStep < p.k) part[at + j * L::kStep] = dw[u][j];
      }
    }
  }
}

// dw = beta dw + the sum of `rows` rows of partial sums, 32 values per CTA, a
// warp per eighth of the rows, in a fixed order.
__global__ void __launch_bounds__(kReduceThreads)
    sumPartsKernel(const float *part, int rows, int part_ld, int k, float beta, float *dw) {
  __shared__ float slots[kReduceWarps][32];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int at = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.0F;
  if (at < k) {
#pragma unroll 8
    for (int r = warp; r < rows; r += kReduceWarps) s += part[static_cast<size_t>(r) * part_ld + at];
  }
  slots[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || at >= k) return;
  s = slots[0][lane];
#pragma unroll
  for (int w = 1; w < kReduceWarps; ++w) s += slots[w][lane];
  if (beta != 0.0F) s = fmaf(beta, dw[at], s);
  dw[at] = s;
}

// How a column is spread over threads.
struct Shape {
  int units;      // 1, 2 or 4; 0: longer than kMaxUnits per thread
  int threads;    // of a column, a multiple of 32
  int columns;    // of a CTA
};
Shape chooseShape(int k, int per, int n, int sms) {
  const int lanes = ((k - 1) / kern::kLaneBlock + 1) * (kern::kLaneBlock / per);
  // Few columns: all of a column's loads at once, on as many threads.
  int units = n <= 2 * sms ? 1 : lanes >= 128 ? 4 : 1;
  while (units < kMaxUnits && lanes > units * kMaxThreads) units *= 2;
  Shape s;
  s.units = lanes > units * kMaxThreads ? 0 : units;
  s.threads = s.units == 0 ? kMaxThreads : ((lanes - 1) / units / 32 + 1) * 32;
  s.columns = std::max(1, 128 / s.threads);
  return s;
}

template <typename P>
sgblasStatus_t launchNorm(void (*kernel)(P), const P &p, dim3 grid, dim3 block, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, p));
}

template <typename T, bool kVector>
sgblasStatus_t launchForward(const NormParams &p, int sms, cudaStream_t stream) {
  const Shape s = chooseShape(p.k, Lanes<T, kVector>::kPer, p.n, sms);
  const dim3 block(static_cast<unsigned>(s.threads), static_cast<unsigned>(s.columns));
  const dim3 grid(static_cast<unsigned>((p.n - 1) / s.columns + 1));
  switch (s.units) {
    case 1: return launchNorm(rmsNormKernel<T, kVector, 1, false>, p, grid, block, stream);
    case 2: return launchNorm(rmsNormKernel<T, kVector, 2, false>, p, grid, block, stream);
    case 4: return launchNorm(rmsNormKernel<T, kVector, 4, false>, p, grid, block, stream);
    default: return launchNorm(rmsNormKernel<T, kVector, 1, true>, p, grid, block, stream);
  }
}

template <typename T, bool kVector>
sgblasStatus_t launchBackward(const NormBackwardParams &p, const Shape &s, int ctas,
                              cudaStream_t stream) {
  const dim3 block(static_cast<unsigned>(s.threads), static_cast<unsigned>(s.columns));
  const dim3 grid(static_cast<unsigned>(ctas));
  switch (s.units) {
    case 1: return launchNorm(rmsNormBackwardKernel<T, kVector, 1, false>, p, grid, block, stream);
    case 2: return launchNorm(rmsNormBackwardKernel<T, kVector, 2, false>, p, grid, block, stream);
    case 4: return launchNorm(rmsNormBackwardKernel<T, kVector, 4, false>, p, grid, block, stream);
    default: return launchNorm(rmsNormBackwardKernel<T, kVector, 1, true>, p, grid, block, stream);
  }
}

// Columns that begin with whole vectors: base and distance multiples of 16 bytes. NULL
// is no matrix.
bool vectorColumns(const void *p, long long ld, int size) {
  return p == nullptr || (aligned16(p) && ld * size % 16 == 0);
}

}  // namespace
}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasRmsNorm(sgblasHandle_t handle, int k, int n, sgblasDataType_t type,
                                        const void *x, int ldx, const void *residual, int ldr,
                                        const void *weight, float eps, void *sum, int ldsum,
                                        void *y, int ldy, void *q, int ldq, float *scale,
                                        int ldscale) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int one = std::max(1, k), blocks = k > 0 ? (k - 1) / sgblas::kern::kLaneBlock + 1 : 1;
  if (k < 0 || n < 0 || !isType(type) || !(eps >= 0.0F) || ldx < one ||
      (residual != nullptr && ldr < one) || (sum != nullptr && ldsum < one) ||
      (y != nullptr && ldy < one) || (q != nullptr && (ldq < one || ldscale < blocks)))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (k == 0 || n == 0) return SGBLAS_STATUS_SUCCESS;
  if (x == nullptr || (y == nullptr && q == nullptr) || (q != nullptr && scale == nullptr))
    return SGBLAS_STATUS_INVALID_VALUE;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  NormParams p = {};
  p.x = x;
  p.residual = residual;
  p.weight = weight;
  p.sum = sum;
  p.y = y;
  p.q = static_cast<unsigned char *>(q);
  p.scale = scale;
  p.k = k;
  p.n = n;
  p.eps = eps;
  p.ldx = ldx;
  p.ldr = ldr;
  p.ldsum = ldsum;
  p.ldy = ldy;
  p.ldq = ldq;
  p.ldscale = ldscale;
  const int size = type == SGBLAS_TYPE_BF16 ? 2 : 4;
  const bool vector = k * static_cast<long long>(size) % 16 == 0 && vectorColumns(x, ldx, size) && vectorColumns(residual, ldr, size) &&
                      vectorColumns(weight, 0, size) && vectorColumns(sum, ldsum, size) &&
                      vectorColumns(y, ldy, size) &&
                      (q == nullptr || (reinterpret_cast<uintptr_t>(q) | static_cast<unsigned>(ldq)) %
                                               static_cast<unsigned>(16 / size) == 0);
  const auto stream = static_cast<cudaStream_t>(handle->stream);
  if (type == SGBLAS_TYPE_BF16)
    return vector ? launchForward<__nv_bfloat16, true>(p, dev.sms, stream)
                  : launchForward<__nv_bfloat16, false>(p, dev.sms, stream);
  return vector ? launchForward<float, true>(p, dev.sms, stream)
                : launchForward<float, false>(p, dev.sms, stream);
}

extern "C" sgblasStatus_t sgblasRmsNormBackward(sgblasHandle_t handle, int k, int n,
                                                sgblasDataType_t type, const void *dy, int lddy,
                                                const void *sum, int ldsum, const void *weight,
                                                float eps, const void *dsum, int lddsum, void *dx,
                                                int lddx, const float *beta, float *dweight) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int one = std::max(1, k);
  if (k < 0 || n < 0 || !isType(type) || !(eps >= 0.0F) || lddy < one || ldsum < one ||
      (dsum != nullptr && lddsum < one) || lddx < one || (dweight != nullptr && beta == nullptr))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (k == 0) return SGBLAS_STATUS_SUCCESS;
  if (n > 0 && (dy == nullptr || sum == nullptr || dx == nullptr)) return SGBLAS_STATUS_INVALID_VALUE;
  if (n == 0 && (dweight == nullptr || *beta == 1.0F)) return SGBLAS_STATUS_SUCCESS;
  DeviceInfo dev;
  sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  NormBackwardParams p = {};
  p.dy = dy;
  p.sum = sum;
  p.weight = weight;
  p.dsum = dsum;
  p.dx = dx;
  p.k = k;
  p.n = n;
  p.eps = eps;
  p.lddy = lddy;
  p.ldsum = ldsum;
  p.lddsum = lddsum;
  p.lddx = lddx;
  const int size = type == SGBLAS_TYPE_BF16 ? 2 : 4;
  const bool vector = k * static_cast<long long>(size) % 16 == 0 && vectorColumns(dy, lddy, size) && vectorColumns(sum, ldsum, size) &&
                      vectorColumns(weight, 0, size) && vectorColumns(dsum, lddsum, size) &&
                      vectorColumns(dx, lddx, size);
  const auto stream = static_cast<cudaStream_t>(handle->stream);
  int rows = 0;
  if (n > 0) {
    const Shape s = chooseShape(k, vector ? 16 / size : 4, n, dev.sms);
    const int threads = s.threads * s.columns;
    const int ctas = std::min((n - 1) / s.columns + 1, dev.sms * std::max(1, 512 / threads));
    rows = ctas * s.columns;
    p.part_ld = (k + 3) / 4 * 4;
    if (dweight != nullptr) {
      const size_t bytes = sizeof(float) * static_cast<size_t>(p.part_ld) * static_cast<size_t>(rows);
      if (!ensureWorkspace(handle, kCounterRegionBytes + bytes, dev.device, stream))
        return SGBLAS_STATUS_NOT_SUPPORTED;
      p.part = reinterpret_cast<float *>(static_cast<unsigned char *>(handle->workspace) +
                                         kCounterRegionBytes);
    }
    if (type == SGBLAS_TYPE_BF16)
      st = vector ? launchBackward<__nv_bfloat16, true>(p, s, ctas, stream)
                  : launchBackward<__nv_bfloat16, false>(p, s, ctas, stream);
    else
      st = vector ? launchBackward<float, true>(p, s, ctas, stream)
                  : launchBackward<float, false>(p, s, ctas, stream);
  }
  if (dweight == nullptr) return st;
  if (st == SGBLAS_STATUS_SUCCESS) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((k - 1) / 32 + 1));
    cfg.blockDim = dim3(kReduceThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    st = launchStatus(cudaLaunchKernelEx(&cfg, sumPartsKernel, static_cast<const float *>(p.part),
                                         rows, p.part_ld, k, *beta, dweight));
  }
  // Failed or not: partial sums may be on their way, and later users wait for them.
  if (n > 0 && !markWorkspaceUse(handle, stream) && st == SGBLAS_STATUS_SUCCESS)
    return SGBLAS_STATUS_EXECUTION_FAILED;
  return st;
}
