// sgblasOrthogonalize (sgblas_lm.h): Newton-Schulz steps on pairs of fp16
// matrices.
//
// With X scaled to Frobenius norm 1, one step is X <- (c0 I + c1 A + c2 A A) X,
// A the smaller Gram matrix of X. Three products: A (symmetric, half its
// tiles), P = c0 I + c1 A + c2 A A (symmetric, half its tiles, the polynomial
// in the epilogue) and P X. The iteration multiplies small singular values by
// |c0| per step (3.4^5 = 485 for the usual five steps), and an error in X with
// them, so single bf16 or fp16 iterates cost digits; pairs hi + lo of fp16
// keep 22 bits for three products of the tensor core. (With single fp16
// iterates in every step, emulated: 2e-3 to 2.6e-2 off, by the spectrum; with the
// last product's operands alone rounded to 11 bits, 2e-4 to 8e-4, under BF16's
// own 1.7e-3.)
//
// Where it pays, two steps share a Gram product and an update (pairsSteps).
//
// Measured: 4096 x 2048 FP32, five steps, 690 us (790 with every step apart),
// where the three-fold products take 345 us of the tensor core's time at its full
// clock (the pipe is busy 48 to 64 % of a product's cycles: one or two tiles per
// worker leave the first loads and the last stores uncovered). 8 x 256 x 512 BF16,
// 87 us: 17 launches, each a chain of latencies (the first slice 1.4 us,
// the stream 2 to 4, the stores 1).
//
// X stays in G's orientation. m >= n: A = X^T X (both operands contiguous
// along k), X P (X contiguous along m). m < n: A = X X^T (both contiguous along
// m and n), P X (both contiguous along k; P is symmetric).
#include "product.hpp"

#include "device.hpp"
#include "sgemm_launch.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <utility>

namespace sgblas::detail {
namespace {

namespace t = kern::prod;

constexpr int kNormThreads = 256;
constexpr int kMaxPartials = 1024;   // partial sums of squares per matrix

struct NormParams {
  const void *g;
  int m, n, ldg;
  long long stride_g;
  int partials;        // per matrix
  double *sums;        // [batch][partials]
  float eps;
  __half *hi, *lo;     // written by splitKernel
  int ldx;
  long long stride_x;
};

// Values of one column a thread reads at once: 16 bytes where G is aligned.
template <typename T, bool kVector>
struct Run {
  static constexpr int kCount = kVector ? 16 / static_cast<int>(sizeof(T)) : 1;
  alignas(16) T v[kCount];
  // From row `row` of a column of `rows`; zeros past its end.
  __device__ __forceinline__ void load(const T *column, int row, int rows) {
    if (kVector && row + kCount <= rows) {
      *reinterpret_cast<uint4 *>(v) = __ldg(reinterpret_cast<const uint4 *>(column + row));
    } else {
#pragma unroll
      for (int j = 0; j < kCount; ++j) v[j] = row + j < rows ? column[row + j] : static_cast<T>(0.0F);
    }
  }
};

// Sum over the block, the same in every thread; the order is fixed.
__device__ __forceinline__ double blockSum(double v) {
  __shared__ double part[kNormThreads / 32];
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kNormThreads / 32; ++w) s += part[w];
  return s;
}

// sums[matrix][i] = sum of squares of the columns i, i + partials, ... In 64 bits:
// the squares of FP32 values leave FP32's range above 2^64 and below 2^-64, and
// G may be of any magnitude. Memory-bound, as is splitKernel.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kNormThreads) squaresKernel(const NormParams p) {
  using R = Run<T, kVector>;
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  double s = 0.0;
  for (int col = blockIdx.x; col < p.n; col += p.partials) {
    const T *column = static_cast<const T *>(p.g) + blockIdx.y * p.stride_g +
                      static_cast<long long>(col) * p.ldg;
#pragma unroll 4
    for (int row = threadIdx.x * R::kCount; row < p.m; row += kNormThreads * R::kCount) {
      R r;
      r.load(column, row, p.m);
#pragma unroll
      for (int j = 0; j < R::kCount; ++j) {
        const double v = static_cast<float>(r.v[j]);
        s = fma(v, v, s);
      }
    }
  }
  s = blockSum(s);
  if (threadIdx.x == 0) p.sums[static_cast<size_t>(blockIdx.y) * p.partials + blockIdx.x] = s;
}

// X = G / (norm + eps) as pairs. The factor can leave FP32's range too, so where
// it is beyond 2^-100 .. 2^100 a power of two of it is applied first: exactly, but
// for values so far below the norm that a pair holds nothing of them.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kNormThreads) splitKernel(const NormParams p) {
  using R = Run<T, kVector>;
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const double *sums = p.sums + static_cast<size_t>(blockIdx.y) * p.partials;
  double part = 0.0;
  for (int i = threadIdx.x; i < p.partials; i += kNormThreads) part += sums[i];
  const double whole = t::kPairScale / (sqrt(blockSum(part)) + p.eps);
  const float power = whole > 0x1p100 ? 0x1p80F : whole < 0x1p-100 ? 0x1p-80F : 1.0F;
  const float factor = static_cast<float>(whole / power);
  for (int col = blockIdx.x; col < p.n; col += gridDim.x) {
    const T *column = static_cast<const T *>(p.g) + blockIdx.y * p.stride_g +
                      static_cast<long long>(col) * p.ldg;
    const size_t to = blockIdx.y * static_cast<size_t>(p.stride_x) +
                      static_cast<size_t>(col) * p.ldx;
#pragma unroll 2
    for (int row = threadIdx.x * R::kCount; row < p.m; row += kNormThreads * R::kCount) {
      R r;
      r.load(column, row, p.m);
      // Columns of X are padded to 64 rows: whole vectors may be written.
      alignas(16) __half hi[R::kCount], lo[R::kCount];
#pragma unroll
      for (int j = 0; j < R::kCount; ++j)
        t::splitPair(static_cast<float>(r.v[j]) * power * factor, &hi[j], &lo[j]);
      if constexpr (R::kCount == 8) {
        *reinterpret_cast<uint4 *>(p.hi + to + row) = *reinterpret_cast<const uint4 *>(hi);
        *reinterpret_cast<uint4 *>(p.lo + to + row) = *reinterpret_cast<const uint4 *>(lo);
      } else if constexpr (R::kCount == 4) {
        *reinterpret_cast<uint2 *>(p.hi + to + row) = *reinterpret_cast<const uint2 *>(hi);
        *reinterpret_cast<uint2 *>(p.lo + to + row) = *reinterpret_cast<const uint2 *>(lo);
      } else {
        p.hi[to + row] = hi[0];
        p.lo[to + row] = lo[0];
      }
    }
  }
}

// One pair matrix of the workspace: `batch` matrices of dim0 x dim1.
struct PairMatrix {
  __half *hi = nullptr, *lo = nullptr;
  int dim0 = 0, dim1 = 0;
  long long ld = 0, stride = 0;
};

bool encodePair(CUtensorMap *hi, CUtensorMap *lo, const PairMatrix &x, int batch, bool mn,
                int rows) {
  const unsigned long long s1 = x.ld * 2ULL, s2 = x.stride * 2ULL;
  const unsigned box1 = mn ? 64u : static_cast<unsigned>(rows);
  return encodeTyped3d(hi, CU_TENSOR_MAP_DATA_TYPE_UINT16, x.hi, x.dim0, x.dim1, batch, s1, s2, 64,
                       box1, CU_TENSOR_MAP_SWIZZLE_128B) &&
         encodeTyped3d(lo, CU_TENSOR_MAP_DATA_TYPE_UINT16, x.lo, x.dim0, x.dim1, batch, s1, s2, 64,
                       box1, CU_TENSOR_MAP_SWIZZLE_128B);
}

cudaError_t launchWith(const void *kernel, dim3 grid, int threads, int smem, cudaStream_t stream,
                       void **args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, kernel, args);
}

// Tiles of one matrix.
template <class G>
long long pairTiles(int m, int n) {
  const int tm = (m + G::kTileM - 1) / G::kTileM, tn = (n + G::kBN - 1) / G::kBN;
  return G::kSymmetric ? t::symmetricTiles<G>(tm, tn) : static_cast<long long>(tm) * tn;
}

// p.m x p.n product of depth p.k over the batch; the epilogue is p.pair.out.
template <class G>
sgblasStatus_t launchPairTyped(const DeviceInfo &dev, int batch, const PairMatrix &a,
                               const PairMatrix &b, t::Params &p, cudaStream_t stream) {
  if (!encodePair(&p.tma_a, &p.pair.tma_a_lo, a, batch, G::kAMN, t::kBM) ||
      !encodePair(&p.tma_b, &p.pair.tma_b_lo, b, batch, G::kBMN, G::kBRows))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  p.groups = batch;
  p.format = t::kFormatFp16;
  p.chunk_iters = 4;   // 256 of k: 48 instructions
  p.err = dev.err;
  p.tiles_m = (p.m + G::kTileM - 1) / G::kTileM;
  p.tiles_n = (p.n + G::kBN - 1) / G::kBN;
  const long long tiles = batch * pairTiles<G>(p.m, p.n);
  if (tiles > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;
  return launchProductKernel<G>(dev, p, tiles, stream);
}

// Clocks of a product on tiles G, less what all kinds share: whole waves, each
// of the longer of a tile's slices and its epilogue, which overlap the next tile's.
// `slice` is what 64 of k take; 16 columns of a warp take 1500 in the epilogue.
template <class G>
long long pairClocks(const DeviceInfo &dev, int batch, const t::Params &p, int slice) {
  const long long workers = G::kTwo ? dev.sms / 2 : dev.sms;
  const long long waves = (batch * pairTiles<G>(p.m, p.n) + workers - 1) / workers;
  const long long stream = (p.k + 63LL) / 64 * slice / (p.pair.planes == 1 ? 3 : 1);
  const long long epilogue = 1500 * (G::kBN / 32);
  return stream + (waves - 1) * std::max(stream, epilogue) + epilogue;
}

// The tiles that take the fewest clocks: pairs of CTAs on 256 x 256 (a symmetric
// product's are 128 wide, for 2048 x 2048 has 72 of them for 74 pairs, and 36
// square ones), single CTAs on 128 x 128, 64 or 32 (B contiguous along n comes in
// boxes of 64). Wide tiles load less per product, narrow ones fill the last wave
// and have short epilogues. The clocks of a slice are fitted to 23 shapes run with
// each kind of tile alone (64 x 64 to 2304 x 1536, batches of 1 to 16; the times
// come out within 6 %); they are those of the loads more than of the
// instructions (1536, 768, 768, 448 and 356). Against the widest tiles that about
// every worker had one of, five steps: 16 x 640 x 320 262 -> 198 us, 4 x 1024 x
// 1024 380 -> 324, 1300 x 1300 278 -> 227, 15 x 512 x 384 213 -> 191, 1024 x 1024
// and 64 x 64 the same; at worst 4 x 512 x 640 136 -> 138. Tiles of 32 for those
// of 64, 8 x 256 x 512: 107 and 93.
template <bool kAMN, bool kBMN, bool kSymmetric>
sgblasStatus_t launchPairProduct(const DeviceInfo &dev, int batch, const PairMatrix &a,
                                 const PairMatrix &b, const t::Params &product,
                                 cudaStream_t stream) {
  constexpr auto kB = t::Ragged::kBatch;
  t::Params p = product;
  constexpr int kWide = kSymmetric ? 128 : 256;
  using Two = t::Cfg<2, kB, kWide, kAMN, kBMN, true, true, 2, kSymmetric>;
  using One = t::Cfg<2, kB, 128, kAMN, kBMN, false, true, 2, kSymmetric>;
  using Half = t::Cfg<2, kB, 64, kAMN, kBMN, false, true, 2, kSymmetric>;
  const long long two = pairClocks<Two>(dev, batch, p, kSymmetric ? 1180 : 1870),
                  one = pairClocks<One>(dev, batch, p, 1300),
                  half = pairClocks<Half>(dev, batch, p, 880);
  long long least = std::min({two, one, half});
  if constexpr (!kBMN) {
    using Quarter = t::Cfg<2, kB, 32, kAMN, kBMN, false, true, 2, kSymmetric>;
    if (pairClocks<Quarter>(dev, batch, p, 690) <= least)
      return launchPairTyped<Quarter>(dev, batch, a, b, p, stream);
  }
  if (half == least) return launchPairTyped<Half>(dev, batch, a, b, p, stream);
  if (one == least) return launchPairTyped<One>(dev, batch, a, b, p, stream);
  return launchPairTyped<Two>(dev, batch, a, b, p, stream);
}

// The sums of squares, then the scaled pairs.
template <typename T, bool kVector>
sgblasStatus_t launchNorm(NormParams q, int batch, cudaStream_t stream) {
  void *args[] = {&q};
  const dim3 grid(static_cast<unsigned>(q.partials), static_cast<unsigned>(batch));
  const cudaError_t e = launchWith(reinterpret_cast<const void *>(squaresKernel<T, kVector>), grid,
                                   kNormThreads, 0, stream, args);
  if (e != cudaSuccess) return launchStatus(e);
  return launchStatus(launchWith(reinterpret_cast<const void *>(splitKernel<T, kVector>), grid,
                                 kNormThreads, 0, stream, args));
}

// Whether two steps share one Gram matrix and one update of X:
//
//   A, P = P(A), A' = P A P, P' = P(A'), X <- X (P P')
//
// All are polynomials of A, so symmetric and at half their tiles: five
// s x s products for one more Gram product and update of X, 3 l s^2 + 5 s^3
// multiplications for 6 l s^2 + 2 s^3.
//
// An error d in A is one of P P' too, through its derivative (212 at a zero
// singular value for the usual coefficients): 2^-22 of the largest entry stays
// below 6e-5 there. Over all five steps that derivative is 1.5e7: hence two at a
// time. The product has to fit the pairs' range (15.99), as c0^2 = 11.9 does.
//
// It has one launch more (7 for 6), which much saved work, or a Gram product of
// few and long tiles (7 ns per row), must repay. Five steps, apart and paired:
// 4096 x 2048 792 and 690 us, 4 x 1024 x 4096 842 and 644, 1024 x 2560 242 and
// 213, 2000 x 600 203 and 175, 128 x 2048 (2) 100 and 88, 64 x 1024 68 and 64; at
// the rule's edges 1536 x 2304 378 and 377, 384 x 1536 108 and 109, 128 x 768 68
// and 68; kept apart: 4 x 512 x 1024 147 and 151, 256 x 1024 87 and 89, 16 x 64 x
// 512 61 and 63 (but also 16 x 128 x 640, 99 and 89).
bool pairsSteps(int l, int s, int batch, const float *c) {
  const double saved = 9.0 * batch * (l - s) * s * s;   // operations, three products each
  const bool pays = saved >= 1e10 || (l >= 2.5 * s && saved >= 1.5e9) || (l >= 768 && l >= 5.0 * s);
  if (!pays) return false;
  for (int i = 0; i <= 48; ++i) {   // squared singular values of 0 to 1.5
    const float a = static_cast<float>(i) / 32.0F, p = c[0] + a * (c[1] + a * c[2]),
                b = a * p * p;
    if (!(std::fabs(p * (c[0] + b * (c[1] + b * c[2]))) < 15.0F)) return false;
  }
  return true;
}

constexpr size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace
}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasOrthogonalize(sgblasHandle_t handle, int m, int n, int batch,
                                              int steps, const float *coefficients, float eps,
                                              float scale, const void *g, sgblasDataType_t gtype,
                                              int ldg, long long stride_g, void *o, int ldo,
                                              long long stride_o) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  if (m < 0 || n < 0 || batch < 0 || steps < 1 || steps > 32 || !isType(gtype) ||
      ldg < std::max(1, m) || ldo < std::max(1, m))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || batch == 0) return SGBLAS_STATUS_SUCCESS;
  if (coefficients == nullptr || g == nullptr || o == nullptr || !(eps >= 0.0F))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (batch > 65535) return SGBLAS_STATUS_NOT_SUPPORTED;   // grid y
  DeviceInfo dev;
  sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  const auto stream = static_cast<cudaStream_t>(handle->stream);

  // Workspace: partial sums; X twice (an update cannot overwrite what it
  // reads), A and P, each a pair.
  const bool tall = m >= n;
  const int s = std::min(m, n), l = std::max(m, n);
  const long long ldx = (m + 63LL) / 64 * 64, lds = (s + 63LL) / 64 * 64;
  // About eight blocks per SM over the batch.
  const int partials = std::min({n, kMaxPartials, std::max(1, 8 * dev.sms / batch)});
  const size_t sum_bytes = align256(static_cast<size_t>(batch) * partials * sizeof(double));
  const size_t x_bytes = static_cast<size_t>(ldx) * n * batch * sizeof(__half);   // 128-byte units
  const size_t s_bytes = static_cast<size_t>(lds) * s * batch * sizeof(__half);
  const bool paired = steps > 2 && pairsSteps(l, s, batch, coefficients);
  const size_t s_matrices = paired ? 6 : 4;
  if (!ensureWorkspace(handle, kCounterRegionBytes + sum_bytes + 4 * x_bytes + s_matrices * s_bytes,
                       dev.device, stream))
    return SGBLAS_STATUS_NOT_SUPPORTED;
  auto *base = static_cast<unsigned char *>(handle->workspace) + kCounterRegionBytes;
  auto *sums = reinterpret_cast<double *>(base);
  base += sum_bytes;
  auto take = [&](int dim0, int dim1, long long ld, size_t bytes) {
    PairMatrix x;
    x.hi = reinterpret_cast<__half *>(base);
    x.lo = reinterpret_cast<__half *>(base + bytes);
    base += 2 * bytes;
    x.dim0 = dim0;
    x.dim1 = dim1;
    x.ld = ld;
    x.stride = ld * dim1;
    return x;
  };
  PairMatrix x = take(m, n, ldx, x_bytes), next = take(m, n, ldx, x_bytes);
  PairMatrix gram = take(s, s, lds, s_bytes), poly = take(s, s, lds, s_bytes);
  const PairMatrix other = paired ? take(s, s, lds, s_bytes) : PairMatrix{};

  NormParams q = {};
  q.g = g;
  q.m = m;
  q.n = n;
  q.ldg = ldg;
  q.stride_g = batch > 1 ? stride_g : 0;
  q.partials = partials;
  q.sums = sums;
  q.eps = eps;
  q.hi = x.hi;
  q.lo = x.lo;
  q.ldx = static_cast<int>(ldx);
  q.stride_x = x.stride;
  const int gsize = gtype == SGBLAS_TYPE_BF16 ? 2 : 4;
  const bool vector = aligned16(g) && static_cast<long long>(ldg) * gsize % 16 == 0 &&
                      q.stride_g * gsize % 16 == 0;
  if (gtype == SGBLAS_TYPE_BF16)
    st = vector ? launchNorm<__nv_bfloat16, true>(q, batch, stream)
                : launchNorm<__nv_bfloat16, false>(q, batch, stream);
  else
    st = vector ? launchNorm<float, true>(q, batch, stream)
                : launchNorm<float, false>(q, batch, stream);
  // A symmetric s x s product of matrices that commute, if all went well so far.
  auto square = [&](const PairMatrix &a, const PairMatrix &b, const PairMatrix &out,
                    t::PairOut what) {
    if (st != SGBLAS_STATUS_SUCCESS) return;
    t::Params p = {};
    p.pair.planes = 2;
    p.m = p.n = p.k = s;
    p.ldc = static_cast<int>(lds);
    p.stride_c = out.stride;
    p.pair.out = what;
    p.pair.hi = out.hi;
    p.pair.lo = out.lo;
    if (what == t::PairOut::kPoly) {
      p.pair.prev_hi = a.hi;
      p.pair.prev_lo = a.lo;
      p.pair.c0 = coefficients[0];
      p.pair.c1 = coefficients[1];
      p.pair.c2 = coefficients[2];
    }
    st = launchPairProduct<false, false, true>(dev, batch, a, b, p, stream);
  };
  for (int step = 0; step < steps && st == SGBLAS_STATUS_SUCCESS; ++step) {
    t::Params p = {};
    p.pair.planes = 2;
    // A = X^T X or X X^T.
    p.m = p.n = s;
    p.k = l;
    p.ldc = static_cast<int>(lds);
    p.stride_c = gram.stride;
    p.pair.out = t::PairOut::kSum;
    p.pair.hi = gram.hi;
    p.pair.lo = gram.lo;
    st = tall ? launchPairProduct<false, false, true>(dev, batch, x, x, p, stream)
              : launchPairProduct<true, true, true>(dev, batch, x, x, p, stream);
    square(gram, gram, poly, t::PairOut::kPoly);
    PairMatrix by = poly;
    if (paired && step + 2 < steps) {
      // The next step's A = P A P and P, and the two polynomials' product.
      square(poly, gram, other, t::PairOut::kSum);
      square(other, poly, gram, t::PairOut::kSum);
      square(gram, gram, other, t::PairOut::kPoly);
      square(poly, other, gram, t::PairOut::kSum);
      by = gram;
      ++step;
    }
    // X P or P X; the last one is the result.
    p.m = m;
    p.n = n;
    p.k = s;
    if (step == steps - 1) {
      // Rounded to BF16 at once: the hi parts' 11 bits add a tenth to that
      // rounding's error, and take a third of the instructions.
      p.pair.planes = 1;
      p.pair.out = t::PairOut::kFinal;
      p.c = o;
      p.c_bf16 = 1;
      p.ldc = ldo;
      p.stride_c = batch > 1 ? stride_o : 0;
      p.alpha = scale / (t::kPairScale * t::kPairScale);
    } else {
      p.pair.hi = next.hi;
      p.pair.lo = next.lo;
      p.ldc = static_cast<int>(ldx);
      p.stride_c = next.stride;
    }
    if (st != SGBLAS_STATUS_SUCCESS) break;
    st = tall ? launchPairProduct<true, false, false>(dev, batch, x, by, p, stream)
              : launchPairProduct<false, false, false>(dev, batch, by, x, p, stream);
    std::swap(x, next);
  }
  if (!markWorkspaceUse(handle, stream) && st == SGBLAS_STATUS_SUCCESS)
    return SGBLAS_STATUS_EXECUTION_FAILED;
  return st;
}
