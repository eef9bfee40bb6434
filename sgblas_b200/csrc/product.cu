// Launch of the 16- and 8-bit tensor-core products: operand copies, tensor
// maps, tile width, persistent grid.
#include "product.hpp"

#include "device.hpp"
#include "product_thin.cuh"
#include "sgemm_launch.hpp"

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

namespace sgblas::detail {

namespace t = kern::prod;

sgblasStatus_t currentDevice(DeviceInfo *info) {
  if (cudaGetDevice(&info->device) != cudaSuccess) {
    (void)cudaGetLastError();
    return SGBLAS_STATUS_EXECUTION_FAILED;
  }
  const int arch = isSm100(info->device);
  if (arch < 0) return SGBLAS_STATUS_EXECUTION_FAILED;
  if (arch == 0) return SGBLAS_STATUS_ARCH_MISMATCH;
  info->err = deviceErrorWord(info->device);
  info->sms = smCount(info->device);
  return info->err == nullptr || info->sms <= 0 ? SGBLAS_STATUS_EXECUTION_FAILED
                                                : SGBLAS_STATUS_SUCCESS;
}

namespace {

// Copies rows of `bytes` bytes, at any address, to rows a multiple of 16 bytes
// apart, so that TMA can read them: a warp per row, kCopyWords loads per lane
// in flight, aligned words of the source, each joined with its neighbour's
// first bytes. Bytes of the last word beyond the row are not read by TMA. Words
// are read whole, so up to three bytes beside a row are, inside the row's first
// and last aligned word. With offsets, matrices of groups without columns are
// left out (nothing reads their copies): 1 token of 9 x 2368 x 1177, 24.5 -> 8.5 us
// with the product. Memory-bound.
constexpr int kCopyWords = 8;
__global__ void __launch_bounds__(256) copyRowsKernel(const unsigned char *__restrict__ src,
                                                      long long bytes, long long rows_per_matrix,
                                                      long long ld, long long stride,
                                                      unsigned char *__restrict__ dst, long long ldp,
                                                      long long rows,
                                                      const int *__restrict__ offsets) {
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int lane = threadIdx.x % 32;
  const int words = static_cast<int>((bytes + 3) / 4);
  for (long long row = blockIdx.x * 8LL + threadIdx.x / 32; row < rows; row += gridDim.x * 8LL) {
    const long long matrix = rows_per_matrix == rows ? 0 : row / rows_per_matrix;
    if (offsets != nullptr && __ldg(offsets + matrix + 1) <= __ldg(offsets + matrix)) continue;
    const auto from = reinterpret_cast<uintptr_t>(src) +
                      static_cast<uintptr_t>(matrix * stride + (row - matrix * rows_per_matrix) * ld);
    const auto *aligned = reinterpret_cast<const uint32_t *>(from & ~uintptr_t{3});
    const unsigned shift = static_cast<unsigned>(from & 3) * 8;
    const int last = static_cast<int>((static_cast<long long>(from & 3) + bytes - 1) / 4);
    auto *to = reinterpret_cast<uint32_t *>(dst + row * ldp);
    for (int word0 = lane; word0 - lane < words; word0 += 32 * kCopyWords) {
      uint32_t v[kCopyWords], edge = 0;
#pragma unroll
      for (int u = 0; u < kCopyWords; ++u)
        v[u] = word0 + u * 32 <= last ? __ldg(aligned + word0 + u * 32) : 0;
      // After the last lane's word comes the first lane's next one, and after
      // its last word the one that follows this run.
      if (lane == 0 && word0 + kCopyWords * 32 <= last) edge = __ldg(aligned + word0 + kCopyWords * 32);
#pragma unroll
      for (int u = 0; u < kCopyWords; ++u) {
        const uint32_t mine = lane == 0 ? (u + 1 < kCopyWords ? v[u + 1 < kCopyWords ? u + 1 : u] : edge) : v[u];
        const uint32_t next = __shfl_sync(0xffffffffu, mine, (lane + 1) % 32);
        if (word0 + u * 32 < words) to[word0 + u * 32] = __funnelshift_r(v[u], next, shift);
      }
    }
  }
}

}  // namespace

bool tmaReadable(const NarrowOperand &o, int elem_bytes) {
  return aligned16(o.ptr) && o.ld * elem_bytes % 16 == 0 &&
         (o.count == 1 || (o.stride * elem_bytes % 16 == 0 && o.stride > 0));
}

static long long copyLd(const NarrowOperand &o, int elem_bytes) {
  const int unit = 128 / elem_bytes;   // whole 128-byte lines
  return (o.dim0 + unit - 1LL) / unit * unit;
}

size_t copyBytes(const NarrowOperand &o, int elem_bytes) {
  return static_cast<size_t>(copyLd(o, elem_bytes)) * elem_bytes * o.dim1 * o.count;
}

sgblasStatus_t copyOperand(NarrowOperand *o, int elem_bytes, void *dst, int sms,
                           const int *offsets, cudaStream_t stream) {
  const long long ldp = copyLd(*o, elem_bytes);
  const long long rows = static_cast<long long>(o->dim1) * o->count;
  const long long bytes = static_cast<long long>(o->dim0) * elem_bytes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>((rows + 7) / 8, 8LL * sms)));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(
      &cfg, copyRowsKernel, static_cast<const unsigned char *>(o->ptr), bytes,
      static_cast<long long>(o->dim1), o->ld * elem_bytes, o->stride * elem_bytes,
      static_cast<unsigned char *>(dst), ldp * elem_bytes, rows, offsets);
  o->ptr = dst;
  o->ld = ldp;
  o->stride = ldp * o->dim1;
  return launchStatus(e);
}

bool encodeOperand(CUtensorMap *map, const NarrowOperand &o, int elem_bytes, bool mn, int rows) {
  const auto type = elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const unsigned long long stride1 = static_cast<unsigned long long>(o.ld) * elem_bytes;
  const unsigned long long stride2 =
      o.count == 1 ? stride1 * o.dim1 : static_cast<unsigned long long>(o.stride) * elem_bytes;
  if (stride1 >= (1ULL << 40) || stride2 >= (1ULL << 40)) return false;
  const unsigned box0 = static_cast<unsigned>(t::kRowBytes / elem_bytes);
  return encodeTyped3d(map, type, o.ptr, o.dim0, o.dim1, o.count, stride1, stride2, box0,
                       mn ? 64u : static_cast<unsigned>(rows), CU_TENSOR_MAP_SWIZZLE_128B);
}

bool tmaWritable(const t::Params &p, int size, long long matrix) {
  const long long column = static_cast<long long>(p.ldc) * size;
  return aligned16(p.c) && column % 16 == 0 && static_cast<long long>(p.m) * size % 16 == 0 &&
         matrix > 0 && matrix % 16 == 0 && matrix < (1LL << 40);
}

namespace {

template <class G>
sgblasStatus_t launchTyped(const DeviceInfo &dev, const NarrowOperand &a, const NarrowOperand &b,
                           t::Params &p, cudaStream_t stream) {
  if (p.k > 0 && (!encodeOperand(&p.tma_a, a, G::kElemBytes, G::kAMN, t::kBM) ||
                  !encodeOperand(&p.tma_b, b, G::kElemBytes, G::kBMN, G::kBRows)))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  p.tiles_m = (p.m + G::kTileM - 1) / G::kTileM;
  p.tiles_n = (p.n + G::kBN - 1) / G::kBN;
  // Tiles, or for ragged columns a bound on them: each group adds at most
  // one partial tile.
  const long long tiles =
      G::kRagged == t::Ragged::kN
          ? static_cast<long long>(p.tiles_m) * (p.n / G::kBN + std::min<long long>(p.groups, p.n))
          : static_cast<long long>(p.tiles_m) * p.tiles_n * p.groups;
  if (tiles > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;
  constexpr unsigned kSize = G::kFp32 ? 4 : 2;
  const int matrices = G::kRagged == t::Ragged::kN ? 1 : p.groups;
  const unsigned long long column = static_cast<unsigned long long>(p.ldc) * kSize;
  const long long matrix = matrices == 1 ? static_cast<long long>(column * p.n)
                                         : p.stride_c * static_cast<long long>(kSize);
  p.c_tma = p.beta == 0.0F && (p.c_bf16 != 0) == (kSize == 2) && tmaWritable(p, kSize, matrix);
  if (p.c_tma &&
      !encodeTyped3d(&p.tma_c,
                     G::kFp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                     p.c, p.m, p.n, matrices, column, static_cast<unsigned long long>(matrix),
                     G::kFp32 ? 32 : 64, t::kOutCols,
                     G::kFp32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  return launchProductKernel<G>(dev, p, tiles, stream);
}

// The thin kernel: clusters of `split` CTAs per 128 x kBN tile.
template <class G>
sgblasStatus_t launchThin(const DeviceInfo &dev, const NarrowOperand &a, const NarrowOperand &b,
                          t::Params &p, cudaStream_t stream) {
  if (p.k > 0 && (!encodeOperand(&p.tma_a, a, G::kElemBytes, G::kAMN, t::kBM) ||
                  !encodeOperand(&p.tma_b, b, G::kElemBytes, false, t::kThinBox)))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  p.tiles_m = (p.m + t::kBM - 1) / t::kBM;
  const long long most =
      static_cast<long long>(p.tiles_m) * (p.n / G::kBN + std::min<long long>(p.groups, p.n));
  if (most > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;
  // About as many as there will be: every group has a tile, few have two.
  const long long tiles = static_cast<long long>(p.tiles_m) *
                          std::max<long long>(std::min(p.groups, p.n), p.n / G::kBN);
  auto kernel = t::thinProductKernel<G>;
  static std::atomic<uint64_t> configured{0};
  if (!configureKernel(reinterpret_cast<const void *>(kernel), dev.device, G::kSmemBytes,
                       &configured))
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
  // The split with the shortest run: waves of tiles over the clusters that
  // fit the GPU at once, each 1 / split of a tile long. A CTA keeps at least
  // four slices of k, and 32 where clusters take several tiles in turn and
  // the hand-overs add up (measured: 32 experts of 2048 x 2048 e4m3, 16 slices,
  // 28.1 us whole and 29.8 in halves; of 2048 x 4096 bf16, 64 slices, 86.2 us
  // whole and 80.1 in halves; 4096 x 4096 e4m3, one token, 11.3 us whole and
  // 6.7 in quarters).
  static std::atomic<int> resident[kMaxDevices][4];   // clusters of 2^i CTAs
  const int iters = (p.k + G::kBK - 1) / G::kBK;
  int split = 1, grid = 0;
  double best = 1e30;
  for (int i = 0, s = 1; s <= t::kMaxSplit; ++i, s *= 2) {
    if (s > 1 && iters < 4 * s) break;
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
  // Without a split there is no cluster to launch.
  cfg.attrs = split > 1 ? attr : attr + 1;
  cfg.numAttrs = split > 1 ? 2 : 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, p, split));
}

// e4m3 products with the tokens on the rows of the tile.
sgblasStatus_t launchRows(const DeviceInfo &dev, const NarrowOperand &a, const NarrowOperand &b,
                          t::Params &p, cudaStream_t stream) {
  using G = t::Cfg<1, t::Ragged::kM, 256, false, false, true>;
  if (p.k > 0 && (!encodeOperand(&p.tma_a, b, 1, false, t::kBM) ||
                  !encodeOperand(&p.tma_b, a, 1, false, G::kBRows)))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  p.tiles_n = (p.m + G::kBN - 1) / G::kBN;
  const long long tiles = static_cast<long long>(p.tiles_n) *
                          (p.n / G::kTileM + std::min<long long>(p.groups, p.n));
  if (tiles > INT_MAX) return SGBLAS_STATUS_NOT_SUPPORTED;
  const long long column = static_cast<long long>(p.ldc) * 2;
  p.c_tma = p.c_bf16 && tmaWritable(p, 2, column * p.n);
  if (p.c_tma && !encodeTyped3d(&p.tma_c, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.c, p.m, p.n, 1, column,
                                column * p.n, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B))
    return SGBLAS_STATUS_EXECUTION_FAILED;
  return launchProductKernel<G>(dev, p, tiles, stream);
}

// Width (columns of tokens) of the tiles of a product ragged along n: 16, 32
// or 64 for the thin kernel, 128 for single CTAs, 256 for pairs. The host
// knows the number of tokens, not how they fall to the groups: a group is
// taken to end in half a tile.
//
// Thin tiles, whose k several CTAs may share, pay while a group has few tokens
// (8 x 2048 x 2048 BF16, 2 tokens each: 13.3 us against 19.0 in 128 columns; 12:
// 14.8 and 14.4; 32 x 2048 x 2048 e4m3, 12: 28.4 and 29.5; tiles of 16 up to 6,
// which is not always best: 32 x 512 x 1024, 6 tokens, 12.0 us and 8.3 in a wider
// one), longer where 128-wide tiles would leave half the SMs idle over
// a long k (2 x 4096 x 4096, 12 tokens: 16.3 and 18.1; 48: 18.7 and 19.0), and
// longest where they would leave three quarters (4096 x 4096 e4m3, 48 tokens:
// 10.0 and 13.1; 160: 22.6 and 15.3).
//
// Of the wide ones, pairs have the faster clock per product, single CTAs the
// finer waves: a wave of 256-wide pair tiles takes about 1.35 times one of
// 128-wide tiles (e4m3: 1.45) for four times the work of a worker (8 x 2048 x
// 2048 BF16, 160 tokens each: pairs 18.9 us in one wave, singles 21.5 in two;
// 2 x 1024 x 1024, 700 tokens: pairs 10.0 us, singles 7.4, both in one wave).
int chooseWidth(const DeviceInfo &dev, const t::Params &p, int elem_bytes) {
  const int active = std::min(p.groups, p.n);
  const double mean = static_cast<double>(p.n) / std::max(p.groups, 1);
  auto tiles = [&](int rows, int width) {
    const double columns = p.groups == 1
                               ? static_cast<double>((p.n - 1) / width + 1)
                               : std::max<double>(active, static_cast<double>(p.n) / width + 0.5 * active);
    return columns * ((p.m - 1) / rows + 1);
  };
  const int iters = (p.k * elem_bytes - 1) / t::kRowBytes + 1;   // slices of k
  const double single = tiles(t::kBM, 128);
  if (mean <= 6) return 16;
  const bool thin = mean <= 12 || (mean <= 16 && 2 * single <= dev.sms && iters >= 32) ||
                    (mean <= 64 && 4 * single <= dev.sms && iters >= 16);
  if (thin) return mean <= 16 ? 32 : 64;
  const double waves = std::ceil(single / dev.sms);
  const double pair_waves = std::ceil(tiles(2 * t::kBM, 256) / (dev.sms / 2));
  return pair_waves * (elem_bytes == 1 ? 1.45 : 1.35) < waves ? 256 : 128;
}

template <int kElemBytes, bool kAMN>
sgblasStatus_t launchRaggedN(const DeviceInfo &dev, const NarrowOperand &a, const NarrowOperand &b,
                             t::Params &p, cudaStream_t stream) {
  constexpr auto kN = t::Ragged::kN;
  const bool plain = p.c_bf16 && p.beta == 0.0F;   // else rows of FP32 sums
  switch (chooseWidth(dev, p, kElemBytes)) {
    case 16: return launchThin<t::ThinCfg<kElemBytes, 16, kAMN>>(dev, a, b, p, stream);
    case 32: return launchThin<t::ThinCfg<kElemBytes, 32, kAMN>>(dev, a, b, p, stream);
    case 64: return launchThin<t::ThinCfg<kElemBytes, 64, kAMN>>(dev, a, b, p, stream);
    case 128:
      if (plain)
        return launchTyped<t::Cfg<kElemBytes, kN, 128, kAMN, false, false, false>>(dev, a, b, p,
                                                                                   stream);
      return launchTyped<t::Cfg<kElemBytes, kN, 128, kAMN, false, false, true>>(dev, a, b, p,
                                                                                stream);
    default:
      if constexpr (kElemBytes == 1) {
        return launchRows(dev, a, b, p, stream);
      } else {
        if (plain)
          return launchTyped<t::Cfg<2, kN, 256, kAMN, false, true, false>>(dev, a, b, p, stream);
        return launchTyped<t::Cfg<2, kN, 256, kAMN, false, true, true>>(dev, a, b, p, stream);
      }
  }
}

sgblasStatus_t launchKind(const DeviceInfo &dev, int elem_bytes, t::Ragged ragged,
                          const NarrowOperand &a, bool a_mn, const NarrowOperand &b, bool b_mn,
                          t::Params &p, cudaStream_t stream) {
  if (ragged == t::Ragged::kN && elem_bytes == 2 && a_mn && !b_mn)
    return launchRaggedN<2, true>(dev, a, b, p, stream);
  if (ragged == t::Ragged::kN && elem_bytes == 2 && !a_mn && !b_mn)
    return launchRaggedN<2, false>(dev, a, b, p, stream);
  if (ragged == t::Ragged::kN && elem_bytes == 1 && !a_mn && !b_mn)
    return launchRaggedN<1, false>(dev, a, b, p, stream);
  if (ragged == t::Ragged::kK && elem_bytes == 2 && a_mn && b_mn)
    return p.c_bf16 && p.beta == 0.0F
               ? launchTyped<t::Cfg<2, t::Ragged::kK, 256, true, true, true, false>>(dev, a, b, p, stream)
               : launchTyped<t::Cfg<2, t::Ragged::kK, 256, true, true, true, true>>(dev, a, b, p, stream);
  return SGBLAS_STATUS_INTERNAL_ERROR;
}

}  // namespace

sgblasStatus_t launchNarrow(sgblasContext *ctx, const DeviceInfo &dev, int elem_bytes,
                            t::Ragged ragged, NarrowOperand a, bool a_mn, NarrowOperand b,
                            bool b_mn, t::Params p) {
  const auto stream = static_cast<cudaStream_t>(ctx->stream);
  p.err = dev.err;
  // Chains of one block of 128 (e4m3), of 512 of k, or, for a BF16 result of BF16
  // operands, of 4096: its own rounding is up to 2^-8, a chain of 4096 positive
  // products comes out 8e-6 too small (6e-5 at most: 256 instructions, 2^-22
  // each). The whole of k in one chain, which may be an expert's tokens, would
  // not do: sums of 2^17 came out 8e-4 too small, of 2^20 6.6e-3 (2e-5 in chains
  // of 4096, at the same speed: 2048 x 2048 x 16384 96 us).
  p.chunk_iters = elem_bytes == 1 ? 1 : p.c_bf16 ? 64 : 8;
  sgblasStatus_t st = SGBLAS_STATUS_SUCCESS;
  bool used_workspace = false;
  if (p.k > 0) {
    const bool copy_a = !tmaReadable(a, elem_bytes), copy_b = !tmaReadable(b, elem_bytes);
    const size_t bytes_a = copy_a ? copyBytes(a, elem_bytes) : 0;
    const size_t bytes_b = copy_b ? copyBytes(b, elem_bytes) : 0;
    if (copy_a || copy_b) {
      if (!ensureWorkspace(ctx, kCounterRegionBytes + bytes_a + bytes_b, dev.device, stream))
        return SGBLAS_STATUS_NOT_SUPPORTED;
      used_workspace = true;
      auto *base = static_cast<unsigned char *>(ctx->workspace) + kCounterRegionBytes;
      const int *reached = ragged == t::Ragged::kN ? p.offsets : nullptr;
      if (copy_a) st = copyOperand(&a, elem_bytes, base, dev.sms, reached, stream);
      if (copy_b && st == SGBLAS_STATUS_SUCCESS)
        st = copyOperand(&b, elem_bytes, base + bytes_a, dev.sms, nullptr, stream);
    }
  }
  if (st == SGBLAS_STATUS_SUCCESS)
    st = launchKind(dev, elem_bytes, ragged, a, a_mn, b, b_mn, p, stream);
  // Failed or not: a copy may be on its way, and later users wait for it.
  if (used_workspace && !markWorkspaceUse(ctx, stream) && st == SGBLAS_STATUS_SUCCESS)
    return SGBLAS_STATUS_EXECUTION_FAILED;
  return st;
}

}  // namespace sgblas::detail
