// 4-bit products with a power of two for each 32 of k (MXFP4), and the
// quantisation to that form (sgblas_lm.h).
#include "product_fp4.cuh"

#include "device.hpp"
#include "lanes.cuh"
#include "product.hpp"
#include "ptx.cuh"
#include "sgemm_launch.hpp"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

namespace sgblas::detail {
namespace {

namespace t = kern::prod;

constexpr int kBlock = 32;
constexpr int kQuantThreads = 256;
constexpr int kUnroll = 2;   // blocks of a thread

struct QuantParams {
  const void *x;
  unsigned char *q, *scale;
  int k, n, batch, kblocks, ldx, ldq, ldscale;
  long long stride_x, stride_q, stride_scale;
  unsigned blocks;   // of the whole batch
  bool q_words;      // 16 values start on 8 bytes of q
};

// The scale byte of a block whose largest magnitude has these bits: its exponent
// less 2, that of the largest e2m1 value (4 <= 6 < 8), so that magnitudes from 6 to 8
// times the power of two are cut to 6; 255 (NaN) where a value is none or infinite.
__device__ __forceinline__ unsigned scaleByte(unsigned amax_bits) {
  const unsigned exponent = amax_bits >> 23;
  return exponent == 255 ? 255u : max(exponent, 2u) - 2u;
}
// 2^(127 - byte), exact: byte is 0 to 252 for numbers.
__device__ __forceinline__ float inverseOf(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// Eight values to e2m1, the first in the lowest half byte: rounded to nearest, ties to
// even, at most 6.
__device__ __forceinline__ uint32_t eightOf(const float2 (&f)[4]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(f[0].x), "f"(f[0].y), "f"(f[1].x), "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x),
        "f"(f[3].y));
  return w;
}

// Two threads to a block of 32, 16 consecutive values each, kUnroll blocks per
// thread whose loads are issued together. Memory-bound (16384 x 8192 BF16 51 to 53 us, 6.4
// to 6.6 TB/s). kAligned: 16 values start on 16 bytes of x; otherwise they are read as
// vectors all the same, and moved into place: 8192 x 4095 20 us in a row, 23 from HBM, for
// a floor of 13 (by single values 195), bound by neither HBM nor issue (61 % of the slots)
// alone.
template <typename T, bool kAligned>
__global__ void __launch_bounds__(kQuantThreads) quantizeFp4Kernel(const QuantParams p) {
  constexpr int kPer = 16, kVectors = kPer * static_cast<int>(sizeof(T)) / 16;
  constexpr int kAtOnce = kQuantThreads / 2;
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int part = threadIdx.x % 2;
  const unsigned first = blockIdx.x * static_cast<unsigned>(kUnroll * kAtOnce) + threadIdx.x / 2;
  alignas(16) uint32_t v[kUnroll][4 * kVectors];
  int left[kUnroll];
  unsigned char *q_to[kUnroll], *scale_to[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const unsigned block = first + u * kAtOnce;
    const bool in = block < p.blocks;
    const unsigned column = in ? block / static_cast<unsigned>(p.kblocks) : 0;
    const int kb = in ? static_cast<int>(block - column * p.kblocks) : 0;
    const unsigned matrix = p.batch > 1 ? column / static_cast<unsigned>(p.n) : 0;
    const long long col = column - matrix * static_cast<unsigned>(p.n);
    const int k0 = kb * kBlock + part * kPer;
    left[u] = in ? p.k - k0 : 0;
    const T *x = static_cast<const T *>(p.x) + matrix * p.stride_x + col * p.ldx + k0;
    if (left[u] >= kPer) {
      if constexpr (kAligned) {
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
          reinterpret_cast<uint4 *>(v[u])[j] = __ldg(reinterpret_cast<const uint4 *>(x) + j);
      } else {
        kern::loadShifted(x, v[u]);
      }
    } else {
      alignas(4) T some[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) some[j] = j < left[u] ? x[j] : static_cast<T>(0.0F);
#pragma unroll
      for (int j = 0; j < 4 * kVectors; ++j) v[u][j] = reinterpret_cast<const uint32_t *>(some)[j];
    }
    q_to[u] = p.q + matrix * p.stride_q + col * p.ldq + k0 / 2;
    scale_to[u] = in && part == 0 ? p.scale + matrix * p.stride_scale + col * p.ldscale + kb : nullptr;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t(&w)[4 * kVectors] = v[u];
    float2 f[kPer / 2];
    unsigned m = 0;
    if constexpr (sizeof(T) == 2) {
      // BF16 values compare as halves of words.
#pragma unroll
      for (int j = 0; j < kPer / 2; ++j) {
        m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
        f[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
      }
      m = max(m << 16, m & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int j = 0; j < kPer / 2; ++j) {
        m = max(m, max(w[2 * j] & 0x7FFFFFFFu, w[2 * j + 1] & 0x7FFFFFFFu));
        f[j] = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
      }
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const unsigned byte = scaleByte(m);
    const float inverse = inverseOf(byte);
    uint32_t q[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float2 scaled[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) scaled[j] = __fmul2_rn(f[half * 4 + j], make_float2(inverse, inverse));
      q[half] = eightOf(scaled);
    }
    if (left[u] >= kPer && p.q_words) {
      *reinterpret_cast<uint2 *>(q_to[u]) = make_uint2(q[0], q[1]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer / 2; ++j)
        if (2 * j < left[u]) q_to[u][j] = static_cast<unsigned char>(q[j / 4] >> (j % 4 * 8));
    }
    if (scale_to[u] != nullptr) *scale_to[u] = static_cast<unsigned char>(byte);
  }
}

sgblasStatus_t launchQuantize(void (*kernel)(QuantParams), const QuantParams &p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.blocks - 1) / (kUnroll * kQuantThreads / 2) + 1);
  cfg.blockDim = dim3(kQuantThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, p));
}

// ---- products --------------------------------------------------------------------

constexpr int kPairWidth = 192;
using PairCfg = t::Fp4Cfg<kPairWidth, true, false>;   // or true: the same tiles

// Lays out the scales in the workspace at `at` and sets the maps.
sgblasStatus_t layScales(const DeviceInfo &dev, t::Fp4Params &f, unsigned char *at, cudaStream_t stream) {
  t::Params &p = f.p;
  const t::LaidSize size = t::laidSize<PairCfg>(p);
  f.laid_a = at;
  f.laid_b = at + size.a;
  f.laid_tiles = static_cast<int>(size.tiles);
  p.tiles_m = (p.m - 1) / PairCfg::kTileM + 1;
  auto encode = [](CUtensorMap *map, const void *from, long long bytes, int rows) {
    return encodeTyped3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, from, t::kScaleRowBytes, bytes / t::kScaleRowBytes, 1,
                         t::kScaleRowBytes, bytes, t::kScaleRowBytes, rows, CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  if (!encode(&f.tma_sa, f.laid_a, size.a, t::kScaleRowsA) || !encode(&f.tma_sb, f.laid_b, size.b, t::kScaleRowsB))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  constexpr long long kWarps = t::kLayThreads / 32;
  const long long items = (size.a + size.b) / (4 * t::kScaleBlock) + 1;   // four blocks each, about
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>((items - 1) / kWarps + 1, 8LL * dev.sms)));
  cfg.blockDim = dim3(t::kLayThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, t::layScalesKernel<PairCfg>, f));
}

template <class G>
sgblasStatus_t launchTile(const DeviceInfo &dev, const NarrowOperand &a, const NarrowOperand &b,
                          t::Fp4Params &f, cudaStream_t stream) {
  t::Params &p = f.p;
  if (p.k > 0 && (!encodeOperand(&p.tma_a, a, 1, false, t::kBM) ||
                  !encodeOperand(&p.tma_b, b, 1, false, G::kBRows)))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  p.tiles_m = (p.m - 1) / G::kTileM + 1;
  const long long tiles = static_cast<long long>(p.tiles_m) *
                          (p.n / G::kBN + std::min<long long>(p.groups, p.n));
  if (tiles > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;
  constexpr int kSize = G::kFp32 ? 4 : 2;
  const long long column = static_cast<long long>(p.ldc) * kSize;
  p.c_tma = tmaWritable(p, kSize, column * p.n);
  if (p.c_tma &&
      !encodeTyped3d(&p.tma_c,
                     G::kFp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                     p.c, p.m, p.n, 1, column, column * p.n, G::kFp32 ? 32 : 64, t::kOutCols,
                     G::kFp32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  auto kernel = t::fp4TileKernel<G>;
  static std::atomic<uint64_t> configured{0};
  if (!configureKernel(reinterpret_cast<const void *>(kernel), dev.device, G::kSmemBytes, &configured))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  constexpr int kCtas = G::kTwo ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(kCtas * std::min<long long>(tiles, dev.sms / kCtas)));
  cfg.blockDim = dim3(t::kThreads);
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
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, f));
}

// Clusters of `split` CTAs per 128 x kBN tile, chosen as launchThin (product.cu) does.
template <class G>
sgblasStatus_t launchThin(const DeviceInfo &dev, const NarrowOperand &a, const NarrowOperand &b,
                          t::Fp4Params &f, cudaStream_t stream) {
  t::Params &p = f.p;
  if (p.k > 0 && (!encodeOperand(&p.tma_a, a, 1, false, t::kBM) ||
                  !encodeOperand(&p.tma_b, b, 1, false, t::kThinBox)))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  p.tiles_m = (p.m - 1) / t::kBM + 1;
  const long long most =
      static_cast<long long>(p.tiles_m) * (p.n / G::kBN + std::min<long long>(p.groups, p.n));
  if (most > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;
  const long long tiles = static_cast<long long>(p.tiles_m) *
                          std::max<long long>(std::min(p.groups, p.n), p.n / G::kBN);
  auto kernel = t::fp4ThinKernel<G>;
  static std::atomic<uint64_t> configured{0};
  if (!configureKernel(reinterpret_cast<const void *>(kernel), dev.device, G::kSmemBytes, &configured))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(t::kThinThreads);
  cfg.dynamicSmemBytes = G::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  static std::atomic<int> resident[kMaxDevices][4];   // clusters of 2^i CTAs
  const int iters = (p.k + t::kRowBytes - 1) / t::kRowBytes;
  int split = 1, grid = 0;
  double best = 1e30;
  for (int i = 0, s = 1; s <= t::kMaxSplit; ++i, s *= 2) {
    if (s > 1 && iters < 2 * s) break;
    int clusters = s == 1 ? dev.sms : resident[dev.device][i].load(std::memory_order_relaxed);
    if (clusters == 0) {
      attr[0].val.clusterDim.x = static_cast<unsigned>(s);
      cfg.gridDim = dim3(static_cast<unsigned>(s));
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        clusters = 0;
      }
      if (clusters <= 0) clusters = -1;
      resident[dev.device][i].store(clusters, std::memory_order_relaxed);
    }
    if (clusters < 0) break;
    if (s > 1 && tiles > clusters && iters < 32 * s) continue;
    const double run = static_cast<double>((tiles + clusters - 1) / clusters) / s;
    if (run < 0.97 * best) {
      best = run;
      split = s;
      grid = static_cast<int>(std::min<long long>(most, clusters));
    }
  }
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  cfg.gridDim = dim3(static_cast<unsigned>(split * grid));
  cfg.attrs = split > 1 ? attr : attr + 1;   // without a split there is no cluster to launch
  cfg.numAttrs = split > 1 ? 2 : 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, f, split));
}

// Width (columns of tokens) of the tiles: 16 or 32 for the thin kernel, 128 for single
// CTAs, 192 for pairs. The host knows the number of tokens, not how they fall to the
// groups: a group is taken to end in half a tile.
//
// Thin tiles, whose k several CTAs may share, pay while a group has few tokens (4 x
// 4096 x 4096, 8 tokens each: 11.0 us in 16 columns, 16.8 in 128; 16: 10.4 and 8.2), those
// of 32 columns where groups of more than 16 are to be expected (384 tokens unevenly over
// 32 x 2048 x 2048, with their quantisation: 16.3 us in 16 columns, 15.4 in 32, 17.6 in
// 128). A wave of single tiles takes 0.40 us a slice of k and no less than 2.2, of pairs
// 0.44 and 3.1, with 3 us for the scales' blocks (32 x 2048 x 2048, 512 tokens each:
// singles 48.7 us, pairs 44.8; 2048: 181 and 145; 16 x 1024 x 2048, 2048: 46 and 41).
//
// Against the best of the four widths the rule loses 2.6 % in the geometric mean over 153
// shapes with even groups, 1.4 % over 85 with uneven ones, more than 10 % in 11 and 5 of
// them. It errs towards pairs where a wave or two of them stand against full waves of single
// tiles (4 x 4096 x 4096, 96 tokens each: pairs taken, 14.3 us, singles 9.2; 256: 19.3 and
// 14.3; 32 x 2048 x 2048, 256: 32.0 and 27.2), and towards thin tiles where m and k are
// small (1 x 1024 x 1024, 12 tokens: 5.5 in 32 columns, 4.2 in 128): its least times are
// those of long waves, and below 14 tokens it looks at the mean alone.
int chooseWidth(const DeviceInfo &dev, const t::Params &p) {
  const int active = std::min(p.groups, p.n);
  const double mean = static_cast<double>(p.n) / std::max(p.groups, 1);
  if (mean <= 6) return 16;
  if (mean <= 14) return 32;
  auto waves = [&](int rows, int width, int workers) {
    const double columns = p.groups == 1
                               ? static_cast<double>((p.n - 1) / width + 1)
                               : std::max<double>(active, static_cast<double>(p.n) / width + 0.5 * active);
    return std::ceil(columns * ((p.m - 1) / rows + 1) / workers);
  };
  const int iters = (p.k - 1) / t::kRowBytes + 1;   // slices of k
  const double single = waves(t::kBM, 128, dev.sms) * std::max(0.40 * iters, 2.2);
  const double pair = waves(2 * t::kBM, kPairWidth, dev.sms / 2) * std::max(0.44 * iters, 3.1) + 3.0;
  return pair < single ? kPairWidth : 128;
}

sgblasStatus_t launchFp4(const DeviceInfo &dev, int width, const NarrowOperand &a, const NarrowOperand &b,
                         t::Fp4Params &f, cudaStream_t stream) {
  const bool fp32 = !f.p.c_bf16;
  switch (width) {
    case 16: return launchThin<t::Fp4ThinCfg<16>>(dev, a, b, f, stream);
    case 32: return launchThin<t::Fp4ThinCfg<32>>(dev, a, b, f, stream);
    case 128:
      return fp32 ? launchTile<t::Fp4Cfg<128, false, true>>(dev, a, b, f, stream)
                  : launchTile<t::Fp4Cfg<128, false, false>>(dev, a, b, f, stream);
    default:
      return fp32 ? launchTile<t::Fp4Cfg<kPairWidth, true, true>>(dev, a, b, f, stream)
                  : launchTile<PairCfg>(dev, a, b, f, stream);
  }
}

sgblasStatus_t gemmFp4(sgblasHandle_t handle, int m, int n, int k, int groups, const int *offsets,
                       bool grouped, const void *a, int lda, long long stride_a, const void *scale_a,
                       int ldsa, long long stride_sa, const void *b, int ldb, const void *scale_b,
                       int ldsb, void *c, sgblasDataType_t ctype, int ldc) {
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int bytes = k > 0 ? (k - 1) / 2 + 1 : 0, blocks = k > 0 ? (k - 1) / kBlock + 1 : 0;
  if (m < 0 || n < 0 || k < 0 || groups < 0 || !isType(ctype) || lda < std::max(1, bytes) ||
      ldb < std::max(1, bytes) || ldc < std::max(1, m) || ldsa < std::max(1, blocks) ||
      ldsb < std::max(1, blocks))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || groups == 0) return SGBLAS_STATUS_SUCCESS;
  if (c == nullptr || (grouped && offsets == nullptr) ||
      (k > 0 && (a == nullptr || b == nullptr || scale_a == nullptr || scale_b == nullptr)))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (groups > SGBLAS_MAX_GROUPS) return SGBLAS_STATUS_NOT_SUPPORTED;
  DeviceInfo dev;
  sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  t::Fp4Params f = {};
  t::Params &p = f.p;
  p.offsets = offsets;
  p.groups = groups;
  p.m = m;
  p.n = n;
  p.k = bytes;
  p.c = c;
  p.c_bf16 = ctype == SGBLAS_TYPE_BF16;
  p.ldc = ldc;
  p.alpha = 1.0F;
  p.err = dev.err;
  // Chains of 32 instructions, 2048 of k, for an FP32 result, as the BF16 products have
  // (launchNarrow), and of 4096 of k for a BF16 one (in chains of 512 an FP32 result of
  // 8192 x 8192 x 4096 took 136 us).
  p.chunk_iters = p.c_bf16 ? 16 : 8;
  // Operands, then their scales, whose rows the kernels read 16 bytes at a time.
  NarrowOperand op[4];
  const void *ptr[4] = {a, b, scale_a, scale_b};
  const int row[4] = {bytes, bytes, blocks, blocks};
  const int ld[4] = {lda, ldb, ldsa, ldsb};
  for (int i = 0; i < 4; ++i) {
    op[i].ptr = ptr[i];
    op[i].dim0 = row[i];
    op[i].dim1 = i % 2 == 0 ? m : n;
    op[i].ld = ld[i];
    op[i].count = i % 2 == 0 ? groups : 1;
    op[i].stride = i == 0 ? stride_a : i == 2 ? stride_sa : 0;
  }
  const auto stream = static_cast<cudaStream_t>(handle->stream);
  bool used_workspace = false;
  int width = chooseWidth(dev, p);
  unsigned char *laid = nullptr;
  if (k > 0) {
    size_t size[4], all = 0;
    for (int i = 0; i < 4; ++i) {
      size[i] = tmaReadable(op[i], 1) ? 0 : copyBytes(op[i], 1);
      all += size[i];
    }
    const t::LaidSize extra = t::laidSize<PairCfg>(p);
    if (width == kPairWidth) {
      // Without a workspace for the scales, single CTAs, which stage them.
      if (std::max(extra.a, extra.b) / t::kScaleRowBytes <= INT_MAX &&
          ensureWorkspace(handle, kCounterRegionBytes + all + static_cast<size_t>(extra.a + extra.b),
                          dev.device, stream)) {
        used_workspace = true;
        laid = static_cast<unsigned char *>(handle->workspace) + kCounterRegionBytes + all;
      } else {
        width = 128;
      }
    }
    if (all > 0) {
      if (!used_workspace && !ensureWorkspace(handle, kCounterRegionBytes + all, dev.device, stream))
        return SGBLAS_STATUS_NOT_SUPPORTED;
      used_workspace = true;
      auto *to = static_cast<unsigned char *>(handle->workspace) + kCounterRegionBytes;
      for (int i = 0; i < 4 && st == SGBLAS_STATUS_SUCCESS; ++i) {
        if (size[i] == 0) continue;
        st = copyOperand(&op[i], 1, to, dev.sms, i % 2 == 0 ? offsets : nullptr, stream);
        to += size[i];
      }
    }
  }
  f.scale_a = static_cast<const unsigned char *>(op[2].ptr);   // of the copies, where there are any
  f.scale_b = static_cast<const unsigned char *>(op[3].ptr);
  f.ldsa = static_cast<int>(op[2].ld);
  f.ldsb = static_cast<int>(op[3].ld);
  f.stride_sa = op[2].count == 1 ? 0 : op[2].stride;
  f.blocks = blocks;
  if (st == SGBLAS_STATUS_SUCCESS && laid != nullptr) st = layScales(dev, f, laid, stream);
  if (st == SGBLAS_STATUS_SUCCESS) st = launchFp4(dev, width, op[0], op[1], f, stream);
  // Failed or not: a copy may be on its way, and later users wait for it.
  if (used_workspace && !markWorkspaceUse(handle, stream) && st == SGBLAS_STATUS_SUCCESS)
    return SGBLAS_STATUS_EXECUTION_FAILED;
  return st;
}

}  // namespace
}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasQuantizeFp4(sgblasHandle_t handle, int k, int n, int batch,
                                            const void *x, sgblasDataType_t xtype, int ldx,
                                            long long stride_x, void *q, int ldq, long long stride_q,
                                            void *scale, int ldscale, long long stride_scale) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int bytes = k > 0 ? (k - 1) / 2 + 1 : 0, kblocks = k > 0 ? (k - 1) / kBlock + 1 : 0;
  if (k < 0 || n < 0 || batch < 0 || !isType(xtype) || ldx < std::max(1, k) ||
      ldq < std::max(1, bytes) || ldscale < std::max(1, kblocks))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (k == 0 || n == 0 || batch == 0) return SGBLAS_STATUS_SUCCESS;
  if (x == nullptr || q == nullptr || scale == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  const double blocks = static_cast<double>(n) * kblocks * batch;
  if (blocks > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;   // 64 Gi values
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  QuantParams p = {};
  p.x = x;
  p.q = static_cast<unsigned char *>(q);
  p.scale = static_cast<unsigned char *>(scale);
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
  p.blocks = static_cast<unsigned>(blocks);
  const auto stream = static_cast<cudaStream_t>(handle->stream);
  const int size = xtype == SGBLAS_TYPE_BF16 ? 2 : 4;
  const bool aligned = aligned16(x) && ldx * static_cast<long long>(size) % 16 == 0 && p.stride_x * size % 16 == 0;
  p.q_words = reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0 && p.stride_q % 8 == 0;
  if (xtype == SGBLAS_TYPE_BF16)
    return launchQuantize(aligned ? quantizeFp4Kernel<__nv_bfloat16, true> : quantizeFp4Kernel<__nv_bfloat16, false>,
                          p, stream);
  return launchQuantize(aligned ? quantizeFp4Kernel<float, true> : quantizeFp4Kernel<float, false>, p, stream);
}

extern "C" sgblasStatus_t sgblasGemmFp4(sgblasHandle_t handle, int m, int n, int k, const void *a,
                                        int lda, const void *scale_a, int ldsa, const void *b, int ldb,
                                        const void *scale_b, int ldsb, void *c, sgblasDataType_t ctype,
                                        int ldc) {
  return sgblas::detail::gemmFp4(handle, m, n, k, 1, nullptr, false, a, lda, 0, scale_a, ldsa, 0, b, ldb,
                                 scale_b, ldsb, c, ctype, ldc);
}

extern "C" sgblasStatus_t sgblasGroupedGemmFp4(sgblasHandle_t handle, int m, int n, int k, int groups,
                                               const int *offsets, const void *a, int lda,
                                               long long stride_a, const void *scale_a, int ldsa,
                                               long long stride_sa, const void *b, int ldb,
                                               const void *scale_b, int ldsb, void *c,
                                               sgblasDataType_t ctype, int ldc) {
  return sgblas::detail::gemmFp4(handle, m, n, k, groups, offsets, true, a, lda, stride_a, scale_a, ldsa,
                                 stride_sa, b, ldb, scale_b, ldsb, c, ctype, ldc);
}
