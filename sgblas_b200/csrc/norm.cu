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
#include "ring.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

namespace sgblas::detail {
namespace {

using kern::both;
using kern::kMaxStages;
using kern::Lanes;
using kern::Ring;
using kern::walk;

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxUnits = 4;          // vectors of a column that a thread holds
// Of the kernels fed by a ring: threads that have to fit an SM, in CTAs of at most
// streamCta. The backward pass holds four operands and the sums of dw: with 768
// threads, 80 registers each, it spilled (16384 x 4096 BF16 270 us for 92).
constexpr int streamThreads(int units, bool backward) {
  return units == 1 ? 1024 : backward ? 512 : 768;
}
constexpr int streamCta(int units, bool backward) {
  return backward && units > 1 ? kMaxThreads : 256;
}
constexpr int kReduceThreads = 1024;
constexpr int kReduceWarps = kReduceThreads / 32;

struct NormParams {
  const void *x, *residual, *weight;
  void *sum, *y;
  unsigned char *q;
  float *scale;
  int k, n;
  float eps, over_k;   // 1 / k
  int ldx, ldr, ldsum, ldy, ldq, ldscale;
};

struct NormBackwardParams {
  const void *dy, *sum, *weight, *dsum;
  void *dx;
  float *part;        // NULL: no gradient of the weights
  long long part_ld;
  int k, n;
  float eps, over_k;
  int lddy, ldsum, lddsum, lddx;
};

// Room for two values of each warp of a CTA, twice: sums in turn use one and the
// other, so that one barrier each is enough.
struct Slots {
  float2 of[2][kMaxWarps];
};

// The sums of two values over the threads of one column (blockDim.x of them, a
// multiple of 32; blockDim.y columns), the same in every thread, in a fixed order.
// kBarrier: a barrier of the CTA even where a warp has the whole column.
template <bool kBarrier = false>
__device__ __forceinline__ float2 columnSum(float2 v, Slots *slots, int turn) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2)
    v = __fadd2_rn(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d)));
  const int warps = static_cast<int>(blockDim.x) / 32;
  if (warps == 1) {
    if (kBarrier) __syncthreads();
    return v;
  }
  float2 *mine = slots->of[turn] + threadIdx.y * warps;
  if (threadIdx.x % 32 == 0) mine[threadIdx.x / 32] = v;
  __syncthreads();
  float2 s = mine[0];
#pragma unroll 4
  for (int w = 1; w < warps; ++w) s = __fadd2_rn(s, mine[w]);
  return s;
}

// 1 / sqrt of the mean plus eps (rsqrtf: two units in the last place at most).
__device__ __forceinline__ float inverseLength(float squares, float over_k, float eps) {
  return rsqrtf(fmaf(squares, over_k, eps));
}

// h = x + r as it is held.
template <typename T, bool kVector>
__device__ __forceinline__ void addResidual(Lanes<T, kVector> *h, const Lanes<T, kVector> &r) {
#pragma unroll
  for (int i = 0; i < Lanes<T, kVector>::kPairs; ++i) h->setPair(i, __fadd2_rn(h->pair(i), r.pair(i)));
}

// A thread's weights: ones where there are none.
template <typename T, bool kVector>
__device__ __forceinline__ void loadWeight(const void *weight, int k, int slot, Lanes<T, kVector> *w) {
  using L = Lanes<T, kVector>;
  const int at = L::begin(slot);
  if (weight != nullptr) {
    w->load(static_cast<const T *>(weight) + at, k - at);
  } else {
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) w->setPair(i, both(1.0F));
  }
}

// What a thread does with its values of a column, whichever way they came: `rest`
// values of the column are there from the thread's place `at` on.
template <typename T, bool kVector>
struct NormOf {
  using L = Lanes<T, kVector>;
  // In two sums, of the even and the odd values.
  static __device__ __forceinline__ void square(const L &h, float2 *sum) {
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) *sum = __ffma2_rn(h.pair(i), h.pair(i), *sum);
  }
  // Every thread of a block of 128 values calls it (they share the block's scale).
  static __device__ __forceinline__ void write(const NormParams &p, long long col, int slot, int rest,
                                               float s, const L &h, const L &weight) {
    const int at = L::begin(slot);
    if (p.sum != nullptr) h.store(static_cast<T *>(p.sum) + col * p.ldsum + at, rest);
    float2 f[L::kPairs];
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) {
      f[i] = __fmul2_rn(__fmul2_rn(h.pair(i), both(s)), weight.pair(i));
    }
    if (p.y != nullptr) {
      L out;
#pragma unroll
      for (int i = 0; i < L::kPairs; ++i) out.setPair(i, f[i]);
      out.store(static_cast<T *>(p.y) + col * p.ldy + at, rest);
    }
    if (p.q != nullptr) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < L::kPairs; ++i) {
        const unsigned a = __float_as_uint(f[i].x) & 0x7FFFFFFFu, b = __float_as_uint(f[i].y) & 0x7FFFFFFFu;
        // A thread's values are all there or none with kVector.
        if (kVector || 2 * i * L::kStep < rest) m = max(m, a);
        if (kVector || (2 * i + 1) * L::kStep < rest) m = max(m, b);
      }
      if (rest <= 0) m = 0;
#pragma unroll
      for (int d = L::kThreads / 2; d > 0; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float scale = kern::fp8Scale(m);
      kern::storeFp8<L::kPairs, L::kStep>(p.q + col * p.ldq + at, f, rest, __frcp_rn(scale));
      if (rest > 0 && slot % L::kThreads == 0) p.scale[col * p.ldscale + slot / L::kThreads] = scale;
    }
  }
};

template <typename T, bool kVector>
struct NormBackwardOf {
  using L = Lanes<T, kVector>;
  // Adds to the sums of h^2 and of h g, each in two parts.
  static __device__ __forceinline__ void add(const L &h, const L &dy, const L &weight,
                                             float2 *squares, float2 *products) {
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) {
      const float2 v = h.pair(i);
      const float2 g = __fmul2_rn(dy.pair(i), weight.pair(i));
      *squares = __ffma2_rn(v, v, *squares);
      *products = __ffma2_rn(v, g, *products);
    }
  }
  // dx to `dx`, and this column's part of dw. A thread without values adds nothing: 0
  // times an s that is not finite would be a NaN.
  static __device__ __forceinline__ void finish(T *dx, int rest, float2 f,
                                                const L &h, const L &dy, const L &weight, const L &ds,
                                                float2 *dw) {
    L out;
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) {
      const float2 v = h.pair(i), y = dy.pair(i);
      const float2 g = __fmul2_rn(y, weight.pair(i));
      out.setPair(i, __ffma2_rn(__ffma2_rn(v, both(-f.y), g), both(f.x), ds.pair(i)));
      if (rest > 0) dw[i] = __ffma2_rn(y, __fmul2_rn(v, both(f.x)), dw[i]);
    }
    out.store(dx, rest);
  }
};

// s, and s^2 times the mean of h g.
__device__ __forceinline__ float2 backwardFactors(float2 sums, float over_k, float eps) {
  const float s = inverseLength(sums.x, over_k, eps);
  return make_float2(s, s * s * (sums.y * over_k));
}

// ---- few columns, or columns that are not whole vectors ----------------------------

// Many columns of odd places are bound by their accesses of single values, latency and
// issue, not by HBM: 16384 x 4095 BF16 forward 173 us (floor 82), e4m3 190 (72), backward 240
// (82); 8192 x 4095 FP32 106, 99 (67) and 126.

// A column per blockDim.x threads, kUnits vectors (or groups of four values) per
// thread; kLong: longer columns than that, read twice.
template <typename T, bool kVector, int kUnits, bool kLong>
__global__ void __launch_bounds__(kMaxThreads) rmsNormKernel(const NormParams p) {
  using L = Lanes<T, kVector>;
  using N = NormOf<T, kVector>;
  __shared__ Slots slots;
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const long long at = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
  const bool in = at < p.n;
  const long long col = in ? at : 0;
  const int stride = static_cast<int>(blockDim.x);
  // Slots of the column in whole warps: every thread of a warp takes part in its shuffles.
  const int rounds = ((p.k - 1) / kern::kLaneBlock * L::kThreads + L::kThreads + 31) / 32 * 32;
  const T *x = static_cast<const T *>(p.x) + col * p.ldx;
  const T *r = p.residual == nullptr ? nullptr : static_cast<const T *>(p.residual) + col * p.ldr;
  auto left = [&](int slot) { return in ? p.k - L::begin(slot) : 0; };
  float2 squares = make_float2(0.0F, 0.0F);
  if constexpr (kLong) {
    auto read = [&](int slot) {
      L h;
      h.load(x + L::begin(slot), left(slot));
      if (r != nullptr) {
        L v;
        v.load(r + L::begin(slot), left(slot));
        addResidual(&h, v);
      }
      return h;
    };
    for (int slot = threadIdx.x; slot < rounds; slot += stride) N::square(read(slot), &squares);
    const float s = inverseLength(columnSum(make_float2(squares.x + squares.y, 0.0F), &slots, 0).x,
                                  p.over_k, p.eps);
    for (int slot = threadIdx.x; slot < rounds; slot += stride) {
      L w;
      loadWeight(p.weight, p.k, slot, &w);
      N::write(p, col, slot, left(slot), s, read(slot), w);
    }
  } else {
    L h[kUnits], w[kUnits], v[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int slot = threadIdx.x + u * stride;
      h[u].load(x + L::begin(slot), left(slot));
      if (r != nullptr) v[u].load(r + L::begin(slot), left(slot));
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) loadWeight(p.weight, p.k, threadIdx.x + u * stride, &w[u]);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (r != nullptr) addResidual(&h[u], v[u]);
      N::square(h[u], &squares);
    }
    const float s = inverseLength(columnSum(make_float2(squares.x + squares.y, 0.0F), &slots, 0).x,
                                  p.over_k, p.eps);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int slot = threadIdx.x + u * stride;
      N::write(p, col, slot, left(slot), s, h[u], w[u]);
    }
  }
}

// The sums of dw of a CTA's columns of threads (blockDim.y of them) to its row of
// partial sums, in their order: kVector as vectors, whose rows are padded to 32 values.
template <typename T, bool kVector, int kUnits>
__device__ __forceinline__ void storePart(const NormBackwardParams &p,
                                          float2 (&dw)[kUnits][Lanes<T, kVector>::kPairs],
                                          float2 *exchange) {
  using L = Lanes<T, kVector>;
  float *part = p.part + blockIdx.x * p.part_ld;
  const int stride = static_cast<int>(blockDim.x);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int at = L::begin(threadIdx.x + u * stride);
    if (blockDim.y > 1) {
#pragma unroll
      for (int i = 0; i < L::kPairs; ++i) {
        __syncthreads();
        exchange[threadIdx.y * stride + threadIdx.x] = dw[u][i];
        __syncthreads();
        float2 sum = exchange[threadIdx.x];
        for (unsigned y = 1; y < blockDim.y; ++y) sum = __fadd2_rn(sum, exchange[y * stride + threadIdx.x]);
        dw[u][i] = sum;
      }
    }
    if (threadIdx.y != 0) continue;
    if constexpr (kVector) {
      if (at < p.k) {
#pragma unroll
        for (int i = 0; i < L::kPairs; i += 2)
          *reinterpret_cast<float4 *>(part + at + 2 * i) =
              make_float4(dw[u][i].x, dw[u][i].y, dw[u][i + 1].x, dw[u][i + 1].y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < L::kPer; ++j)
        if (at + j * L::kStep < p.k) part[at + j * L::kStep] = j % 2 ? dw[u][j / 2].y : dw[u][j / 2].x;
    }
  }
}

// Walks the columns blockIdx.x * blockDim.y + threadIdx.y, ... of a persistent
// grid, each CTA with a row of partial sums of dw.
template <typename T, bool kVector, int kUnits, bool kLong>
__global__ void __launch_bounds__(kMaxThreads) rmsNormBackwardKernel(const NormBackwardParams p) {
  using L = Lanes<T, kVector>;
  using N = NormBackwardOf<T, kVector>;
  __shared__ Slots slots;
  __shared__ float2 exchange[kMaxThreads];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int stride = static_cast<int>(blockDim.x);
  const int rounds = ((p.k - 1) / kern::kLaneBlock + 1) * L::kThreads;
  const long long first = blockIdx.x * static_cast<long long>(blockDim.y);
  const long long step = gridDim.x * static_cast<long long>(blockDim.y);
  const bool past = p.dsum != nullptr;
  float2 dw[kLong ? 1 : kUnits][L::kPairs];
  L w[kUnits];
  if constexpr (!kLong) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      loadWeight(p.weight, p.k, threadIdx.x + u * stride, &w[u]);
#pragma unroll
      for (int i = 0; i < L::kPairs; ++i) dw[u][i] = make_float2(0.0F, 0.0F);
    }
  }
  int turn = 0;
  for (long long c = first; c < p.n; c += step, turn ^= 1) {
    const bool in = c + threadIdx.y < p.n;
    const long long col = in ? c + threadIdx.y : 0;
    const T *h0 = static_cast<const T *>(p.sum) + col * p.ldsum;
    const T *dy0 = static_cast<const T *>(p.dy) + col * p.lddy;
    const T *ds0 = past ? static_cast<const T *>(p.dsum) + col * p.lddsum : nullptr;
    T *dx0 = static_cast<T *>(p.dx) + col * p.lddx;
    float2 squares = make_float2(0.0F, 0.0F), products = squares;
    L h[kUnits], dy[kUnits], ds[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) ds[u].clear();
    if constexpr (kLong) {
      float *part = p.part == nullptr ? nullptr : p.part + blockIdx.x * p.part_ld;
      auto read = [&](int slot) {
        const int at = L::begin(slot);
        h[0].load(h0 + at, p.k - at);
        dy[0].load(dy0 + at, p.k - at);
        loadWeight(p.weight, p.k, slot, &w[0]);
      };
      for (int slot = threadIdx.x; slot < rounds; slot += stride) {
        read(slot);
        N::add(h[0], dy[0], w[0], &squares, &products);
      }
      const float2 f = backwardFactors(
          columnSum(make_float2(squares.x + squares.y, products.x + products.y), &slots, turn),
          p.over_k, p.eps);
      for (int slot = threadIdx.x; slot < rounds; slot += stride) {
        const int at = L::begin(slot);
        read(slot);
        if (past) ds[0].load(ds0 + at, p.k - at);
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) dw[0][i] = make_float2(0.0F, 0.0F);
        N::finish(dx0 + at, p.k - at, f, h[0], dy[0], w[0], ds[0], dw[0]);
        if (part != nullptr) {
#pragma unroll
          for (int j = 0; j < L::kPer; ++j) {
            const int to = at + j * L::kStep;
            const float v = j % 2 ? dw[0][j / 2].y : dw[0][j / 2].x;
            if (to < p.k) part[to] = c != first ? part[to] + v : v;
          }
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int at = L::begin(threadIdx.x + u * stride), rest = in ? p.k - at : 0;
        h[u].load(h0 + at, rest);
        dy[u].load(dy0 + at, rest);
        if (past) ds[u].load(ds0 + at, rest);
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) N::add(h[u], dy[u], w[u], &squares, &products);
      const float2 f = backwardFactors(
          columnSum(make_float2(squares.x + squares.y, products.x + products.y), &slots, turn),
          p.over_k, p.eps);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int at = L::begin(threadIdx.x + u * stride);
        N::finish(dx0 + at, in ? p.k - at : 0, f, h[u], dy[u], w[u], ds[u], dw[u]);
      }
    }
  }
  if constexpr (!kLong) {
    if (p.part != nullptr) storePart<T, kVector, kUnits>(p, dw, exchange);
  }
}

// ---- many columns of whole vectors: a persistent grid fed by bulk copies -------------

// With loads straight into registers, each column's latency was uncovered (16384 x 4096
// BF16 backward 152 to 192 us, forward 100 to 104). Bound by HBM: that backward 86 to 93
// us (5.8 to 6.2 TB/s), forward 94 (5.7), in e4m3 76 (6.2).
template <typename T, int kUnits>
__global__ void __launch_bounds__(streamCta(kUnits, false), streamThreads(kUnits, false) / streamCta(kUnits, false))
    rmsNormStreamKernel(const NormParams p, int stages, unsigned *err) {
  using L = Lanes<T, true>;
  using N = NormOf<T, true>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Slots slots;
  __shared__ uint64_t full[kMaxStages];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int stride = static_cast<int>(blockDim.x);
  Ring<2> ring = {smem, full, p.k * static_cast<int>(sizeof(T)), stages,
                  {static_cast<const unsigned char *>(p.x), static_cast<const unsigned char *>(p.residual)},
                  {p.ldx * static_cast<long long>(sizeof(T)), p.ldr * static_cast<long long>(sizeof(T))}};
  L w[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) loadWeight(p.weight, p.k, threadIdx.x + u * stride, &w[u]);
  walk(ring, p.n, err, [&](int stage, int turn, long long col, bool in) {
    const T *x = reinterpret_cast<const T *>(ring.row(stage, 0, threadIdx.y));
    const T *r = reinterpret_cast<const T *>(ring.row(stage, 1, threadIdx.y));
    L h[kUnits];
    float2 squares = make_float2(0.0F, 0.0F);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = L::begin(threadIdx.x + u * stride), rest = in ? p.k - at : 0;
      h[u].load(x + at, rest);
      if (p.residual != nullptr) {
        L v;
        v.load(r + at, rest);
        addResidual(&h[u], v);
      }
      N::square(h[u], &squares);
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      h[u].hold();
      w[u].hold();
    }
    const float s = inverseLength(
        columnSum<true>(make_float2(squares.x + squares.y, 0.0F), &slots, turn).x, p.over_k, p.eps);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int slot = threadIdx.x + u * stride;
      N::write(p, in ? col : 0, slot, in ? p.k - L::begin(slot) : 0, s, h[u], w[u]);
    }
  });
}

template <typename T, int kUnits>
__global__ void __launch_bounds__(streamCta(kUnits, true), streamThreads(kUnits, true) / streamCta(kUnits, true))
    rmsNormBackwardStreamKernel(const NormBackwardParams p, int stages, unsigned *err) {
  using L = Lanes<T, true>;
  using N = NormBackwardOf<T, true>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Slots slots;
  __shared__ uint64_t full[kMaxStages];
  __shared__ float2 exchange[kMaxThreads];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int stride = static_cast<int>(blockDim.x);
  constexpr long long kSize = sizeof(T);
  Ring<3> ring = {smem, full, p.k * static_cast<int>(sizeof(T)), stages,
                  {static_cast<const unsigned char *>(p.sum), static_cast<const unsigned char *>(p.dy),
                   static_cast<const unsigned char *>(p.dsum)},
                  {p.ldsum * kSize, p.lddy * kSize, p.lddsum * kSize}};
  // Long columns are read from the ring again for dx: held, they would not fit the registers.
  constexpr bool kAgain = kUnits == 4;
  const bool past = p.dsum != nullptr;
  float2 dw[kUnits][L::kPairs];
  L w[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    loadWeight(p.weight, p.k, threadIdx.x + u * stride, &w[u]);
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) dw[u][i] = make_float2(0.0F, 0.0F);
  }
  walk(ring, p.n, err, [&](int stage, int turn, long long col, bool in) {
    const T *h0 = reinterpret_cast<const T *>(ring.row(stage, 0, threadIdx.y));
    const T *dy0 = reinterpret_cast<const T *>(ring.row(stage, 1, threadIdx.y));
    const T *ds0 = reinterpret_cast<const T *>(ring.row(stage, 2, threadIdx.y));
    L h[kUnits], dy[kUnits], ds[kUnits];
    float2 squares = make_float2(0.0F, 0.0F), products = squares;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = L::begin(threadIdx.x + u * stride), rest = in ? p.k - at : 0;
      h[u].load(h0 + at, rest);
      dy[u].load(dy0 + at, rest);
      if (!kAgain) {
        if (past) ds[u].load(ds0 + at, rest);
        else ds[u].clear();
      }
      N::add(h[u], dy[u], w[u], &squares, &products);
    }
    const float2 f = backwardFactors(
        columnSum<true>(make_float2(squares.x + squares.y, products.x + products.y), &slots, turn), p.over_k, p.eps);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (!kAgain) {
        h[u].hold();
        dy[u].hold();
      }
      w[u].hold();
    }
    T *dx0 = static_cast<T *>(p.dx) + (in ? col * p.lddx : 0);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = L::begin(threadIdx.x + u * stride), rest = in ? p.k - at : 0;
      if (kAgain) {
        h[u].load(h0 + at, rest);
        dy[u].load(dy0 + at, rest);
        if (past) ds[u].load(ds0 + at, rest);
        else ds[u].clear();
      }
      N::finish(dx0 + at, rest, f, h[u], dy[u], w[u], ds[u], dw[u]);
    }
    if (kAgain) __syncthreads();   // the stage has been read
  });
  if (p.part != nullptr) storePart<T, true, kUnits>(p, dw, exchange);
}

// dw = beta dw + the sum of `rows` rows of partial sums, 32 values per CTA, a
// warp per kReduceWarps-th row, in a fixed order. Bound by latency: 296 rows of 4096
// values, which lie in L2, 3 us.
__global__ void __launch_bounds__(kReduceThreads)
    sumPartsKernel(const float *part, int rows, long long part_ld, int k, float beta, float *dw) {
  __shared__ float slots[kReduceWarps][32];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int at = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.0F;
  if (at < k) {
#pragma unroll 8
    for (int r = warp; r < rows; r += kReduceWarps) s += part[r * part_ld + at];
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

constexpr int kForwardRows = 2, kBackwardRows = 3;   // of a stage

// How columns are spread over threads.
struct Shape {
  int units;      // vectors of a thread: 1, 2 or 4; 0: more than kMaxUnits
  int threads;    // of a column, a multiple of 32
  int columns;    // of a CTA at a time
  int stages;     // of the ring; 0: loads straight into registers
  int resident;   // CTAs per SM, of a persistent grid
};
// For columns read `vector`-wise or not, whichever results are asked for. A ring pays
// where a CTA walks several columns. More vectors per thread mean fewer instructions a
// column: forward 16384 x 4096 BF16 94 us with four, 101 with two, without a residual 43
// and 54, with e4m3 results 76 and 83.
Shape chooseShape(int k, int size, bool vector, int n, bool backward, int sms) {
  const int per = vector ? 16 / size : 4;
  const int lanes = ((k - 1) / kern::kLaneBlock + 1) * (kern::kLaneBlock / per);
  const int operands = backward ? kBackwardRows : kForwardRows;
  Shape s = {};
  if (vector && n >= 4 * sms) {
    const int two = backward ? 2 * kMaxThreads : 128;   // lanes for two vectors each
    s.units = lanes <= 32 ? 1 : lanes <= two ? 2 : 4;
    s.threads = ((lanes - 1) / s.units / 32 + 1) * 32;
    s.columns = std::max(1, 256 / s.threads);
    s.resident = std::max(1, streamThreads(s.units, backward) / (s.threads * s.columns));
    const long long stage = static_cast<long long>(operands) * s.columns * k * size;
    s.stages = static_cast<int>(std::min<long long>(kMaxStages, (216 * 1024 / s.resident - 6 * 1024) / stage));
    if (s.threads <= streamCta(s.units, backward) && s.stages >= 2) return s;
  }
  // Few columns: all of a column's loads at once, on as many threads.
  const int most = backward ? 2 : kMaxUnits;
  int units = n <= 2 * sms ? 1 : lanes >= 128 ? 2 : 1;
  while (units < most && lanes > units * kMaxThreads) units *= 2;
  s.units = lanes > units * kMaxThreads ? 0 : units;
  s.threads = s.units == 0 ? kMaxThreads : ((lanes - 1) / units / 32 + 1) * 32;
  s.columns = std::max(1, 128 / s.threads);
  s.resident = std::max(1, 768 / (s.threads * s.columns));
  s.stages = 0;
  return s;
}

int persistentCtas(const Shape &s, int n, int sms) {
  return std::min((n - 1) / s.columns + 1, sms * s.resident);
}

template <typename... Args, typename... Given>
sgblasStatus_t launchNorm(void (*kernel)(Args...), dim3 grid, const Shape &s, size_t smem,
                          cudaStream_t stream, const Given &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(s.threads), static_cast<unsigned>(s.columns));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, static_cast<Args>(args)...));
}

template <typename P>
sgblasStatus_t launchStream(void (*kernel)(P, int, unsigned *), std::atomic<uint64_t> *configured,
                            const DeviceInfo &dev, int operands, int size, const Shape &s,
                            cudaStream_t stream, const P &p) {
  if (!configureKernel(reinterpret_cast<const void *>(kernel), dev.device, 216 * 1024, configured))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  const size_t smem = static_cast<size_t>(s.stages) * operands * s.columns * p.k * size;
  return launchNorm(kernel, dim3(static_cast<unsigned>(persistentCtas(s, p.n, dev.sms))), s, smem, stream, p,
                    s.stages, dev.err);
}

template <typename T, int kUnits>
sgblasStatus_t launchForwardStream(const NormParams &p, const Shape &s, const DeviceInfo &dev,
                                   cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  return launchStream(rmsNormStreamKernel<T, kUnits>, &configured, dev, kForwardRows, sizeof(T), s, stream, p);
}
template <typename T, int kUnits>
sgblasStatus_t launchBackwardStream(const NormBackwardParams &p, const Shape &s, const DeviceInfo &dev,
                                    cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  return launchStream(rmsNormBackwardStreamKernel<T, kUnits>, &configured, dev, kBackwardRows, sizeof(T), s,
                      stream, p);
}

template <typename T, bool kVector>
sgblasStatus_t launchForward(const NormParams &p, const DeviceInfo &dev, cudaStream_t stream) {
  const Shape s = chooseShape(p.k, sizeof(T), kVector, p.n, false, dev.sms);
  if constexpr (kVector) {
    if (s.stages > 0)
      return s.units == 1   ? launchForwardStream<T, 1>(p, s, dev, stream)
             : s.units == 2 ? launchForwardStream<T, 2>(p, s, dev, stream)
                            : launchForwardStream<T, 4>(p, s, dev, stream);
  }
  const dim3 grid(static_cast<unsigned>((p.n - 1) / s.columns + 1));
  switch (s.units) {
    case 1: return launchNorm(rmsNormKernel<T, kVector, 1, false>, grid, s, 0, stream, p);
    case 2: return launchNorm(rmsNormKernel<T, kVector, 2, false>, grid, s, 0, stream, p);
    case 4: return launchNorm(rmsNormKernel<T, kVector, 4, false>, grid, s, 0, stream, p);
    default: return launchNorm(rmsNormKernel<T, kVector, 1, true>, grid, s, 0, stream, p);
  }
}

template <typename T, bool kVector>
sgblasStatus_t launchBackward(const NormBackwardParams &p, const Shape &s, const DeviceInfo &dev,
                              cudaStream_t stream) {
  if constexpr (kVector) {
    if (s.stages > 0)
      return s.units == 1   ? launchBackwardStream<T, 1>(p, s, dev, stream)
             : s.units == 2 ? launchBackwardStream<T, 2>(p, s, dev, stream)
                            : launchBackwardStream<T, 4>(p, s, dev, stream);
  }
  const dim3 grid(static_cast<unsigned>(persistentCtas(s, p.n, dev.sms)));
  switch (s.units) {
    case 1: return launchNorm(rmsNormBackwardKernel<T, kVector, 1, false>, grid, s, 0, stream, p);
    case 2: return launchNorm(rmsNormBackwardKernel<T, kVector, 2, false>, grid, s, 0, stream, p);
    default: return launchNorm(rmsNormBackwardKernel<T, kVector, 1, true>, grid, s, 0, stream, p);
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
  p.over_k = 1.0F / static_cast<float>(k);
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
    return vector ? launchForward<__nv_bfloat16, true>(p, dev, stream)
                  : launchForward<__nv_bfloat16, false>(p, dev, stream);
  return vector ? launchForward<float, true>(p, dev, stream)
                : launchForward<float, false>(p, dev, stream);
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
  p.over_k = 1.0F / static_cast<float>(k);
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
    const Shape s = chooseShape(k, size, vector, n, true, dev.sms);
    rows = persistentCtas(s, n, dev.sms);
    p.part_ld = (k + 31LL) / 32 * 32;
    if (dweight != nullptr) {
      const size_t bytes = sizeof(float) * static_cast<size_t>(p.part_ld) * static_cast<size_t>(rows);
      if (!ensureWorkspace(handle, kCounterRegionBytes + bytes, dev.device, stream))
        return SGBLAS_STATUS_NOT_SUPPORTED;
      p.part = reinterpret_cast<float *>(static_cast<unsigned char *>(handle->workspace) +
                                         kCounterRegionBytes);
    }
    if (type == SGBLAS_TYPE_BF16)
      st = vector ? launchBackward<__nv_bfloat16, true>(p, s, dev, stream)
                  : launchBackward<__nv_bfloat16, false>(p, s, dev, stream);
    else
      st = vector ? launchBackward<float, true>(p, s, dev, stream)
                  : launchBackward<float, false>(p, s, dev, stream);
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
