// Tokens to their experts and back (sgblas_lm.h): sgblasSortTokens,
// sgblasScatterTokens, sgblasGatherTokens, sgblasGatherTokensBackward.
//
// A token t has `top` choices; choice j goes to column place(j, t) of the sorted
// matrix, or nowhere (a place outside [0, rows)). Moving columns is
// memory-bound: each is read and written once, in vectors of 16 bytes, and a
// token's column is read once for all of its choices.
#include "device.hpp"
#include "lanes.cuh"
#include "product.hpp"
#include "ptx.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

namespace sgblas::detail {
namespace {

using kern::both;
using kern::Lanes;

// ---- the sort ------------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortMaxCluster = 16;      // 8 where the device has no room for 16 (clusterLimit)
constexpr int kSortCtaWarps = 8;
constexpr int kSortWarpEntries = 64;   // of a warp, before another warp (CTA) joins

constexpr int kSortBatch = 8;          // entries of a lane whose loads are issued together
constexpr int kSortMaxEntries = 1 << 30;
constexpr int kMaxTop = 1 << 30;       // kBatch choices past the last are counted in 32 bits, too

struct SortParams {
  const int *group;
  int *offsets, *place;
  int entries, groups;
};

// Exclusive sum over the CTA's threads, and the total; `slots` a word per warp.
__device__ __forceinline__ int blockScan(int v, int *slots, int *total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  int scan = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += o;
  }
  if (lane == 31) slots[warp] = scan;
  __syncthreads();
  int before = 0, sum = 0;
  for (int w = 0; w < warps; ++w) {
    if (w == warp) before = sum;
    sum += slots[w];
  }
  __syncthreads();
  *total = sum;
  return before + scan - v;
}

// A stable counting sort by group: one cluster, whose warps hold consecutive
// ranges of the entries. Each warp walks its range, 32 entries at a time: lanes of one
// group find each other by a ballot for each bit of the group's number, and an entry's
// place within the warp's part of its group is that group's count so far plus the
// lanes before. The counts are summed over a CTA's warps, over the cluster's CTAs
// (through distributed shared memory) and over the groups, and each entry adds where
// its warp's part of its group begins. Bound by latencies: the loads', the counts'
// and the cluster's (65536 entries, 64 groups: 7.0 us, in clusters of 8 CTAs 10.1; 524288
// entries 25 and 51; with 8, __match_any_sync and a second walk 65536 took 22.5).
template <int kBits>   // of a group's number, p.groups (none) among them
__global__ void __launch_bounds__(kSortThreads) sortTokensKernel(const SortParams p, int ctas) {
  extern __shared__ int counts[];   // [warps][groups], the CTA's sums, where its groups begin
  __shared__ int slots[kSortThreads / 32];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int rank = static_cast<int>(blockIdx.x);
  int *mine = counts + warp * p.groups;
  int *sums = counts + warps * p.groups, *starts = sums + p.groups;
  // 2^30 entries at most, and 2^9 warps of 32 of them more.
  const int parts = ctas * warps;
  const int per = ((p.entries + parts - 1) / parts + 31) / 32 * 32;
  const int begin = min(per * (rank * warps + warp), p.entries), end = min(begin + per, p.entries);
  const bool once = per <= 32 * kSortBatch;   // the range fits the registers
  for (int g = lane; g < p.groups; g += 32) mine[g] = 0;
  __syncwarp();
  int group[kSortBatch], local[kSortBatch];   // of entries i0 + 32 b + lane; the group p.groups is none
  auto readGroups = [&](int i0) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      const int i = i0 + b * 32 + lane;
      const int g = i < end ? __ldg(p.group + i) : -1;
      group[b] = static_cast<unsigned>(g) < static_cast<unsigned>(p.groups) ? g : p.groups;
    }
  };
  for (int i0 = begin; i0 < end; i0 += 32 * kSortBatch) {
    readGroups(i0);
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      if (i0 + b * 32 >= end) break;
      const int g = group[b];
      unsigned same = 0xffffffffu;
#pragma unroll
      for (int bit = 0; bit < kBits; ++bit) {
        const int unset = (g >> bit & 1) - 1;   // all ones where the bit is zero
        same &= __ballot_sync(0xffffffffu, unset == 0) ^ static_cast<unsigned>(unset);
      }
      const bool live = g < p.groups;
      const int before = live ? mine[g] : 0;
      __syncwarp();
      if (live && __ffs(same) - 1 == lane) mine[g] = before + __popc(same);
      __syncwarp();
      local[b] = before + __popc(same & ((1u << lane) - 1));
      const int i = i0 + b * 32 + lane;
      if (!once && i < end) p.place[i] = local[b];
    }
  }
  __syncthreads();
  for (int g = threadIdx.x; g < p.groups; g += blockDim.x) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < warps; ++w) {
      const int c = counts[w * p.groups + g];
      counts[w * p.groups + g] = sum;
      sum += c;
    }
    sums[g] = sum;
  }
  if (ctas > 1) kern::clusterSync();
  else __syncthreads();
  int carry = 0;   // entries of the groups so far
  for (int g0 = 0; g0 < p.groups; g0 += blockDim.x) {
    const int g = g0 + threadIdx.x;
    int total = 0, before = 0;
    if (g < p.groups) {
      // All CTAs' sums at once: one latency of the cluster's, not one each.
      int there[kSortMaxCluster];
#pragma unroll
      for (int c = 0; c < kSortMaxCluster; ++c) {
        there[c] = 0;
        if (ctas == 1 && c == 0) there[c] = sums[g];
        if (ctas > 1 && c < ctas) there[c] = kern::ldCluster(kern::clusterAddr(kern::smemAddr(sums + g), c));
      }
#pragma unroll
      for (int c = 0; c < kSortMaxCluster; ++c) {
        if (c < rank) before += there[c];
        total += there[c];
      }
    }
    int all;
    const int at = carry + blockScan(total, slots, &all);
    if (g < p.groups) {
      if (rank == 0) p.offsets[g] = at;
      starts[g] = at + before;
    }
    carry += all;
  }
  if (rank == 0 && threadIdx.x == 0) p.offsets[p.groups] = carry;
  __syncthreads();
  // No CTA leaves while another reads its sums; this one has them, in `starts`.
  if (ctas > 1) kern::clusterArriveRelaxed();
  for (int i0 = begin; i0 < end; i0 += 32 * kSortBatch) {
    if (!once) {
      readGroups(i0);
#pragma unroll
      for (int b = 0; b < kSortBatch; ++b)
        if (i0 + b * 32 + lane < end) local[b] = p.place[i0 + b * 32 + lane];
    }
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      const int i = i0 + b * 32 + lane, g = group[b];
      if (i < end) p.place[i] = g < p.groups ? starts[g] + mine[g] + local[b] : -1;
    }
  }
  if (ctas > 1) kern::clusterWait();
}

// The largest cluster that the kernel can have on the device: 16 CTAs are allowed to
// kernels that ask for them, not promised (a part of a GPU may have no 16 SMs together).
int clusterLimit(const void *kernel, int device, int smem, std::atomic<int> *known) {
  int limit = known[device].load(std::memory_order_relaxed);
  if (limit > 0) return limit;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kSortMaxCluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSortMaxCluster);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    clusters = 0;
  }
  limit = clusters > 0 ? kSortMaxCluster : kSortMaxCluster / 2;
  known[device].store(limit, std::memory_order_relaxed);
  return limit;
}

// ---- moving columns ------------------------------------------------------------

// A CTA's threads. With sums over choices more and smaller CTAs have columns on their way
// while others wait for places or shuffle: 8192 tokens with 8 choices, 2048 values, on 256,
// 128 and 64 threads combined in 51, 47 and 46 us, their gradients in 94, 86 and 90;
// sorted and scattered in 57.5 and 58.7. 16 tokens' gradients 2.6, 2.9.
constexpr int kScatterThreads = 256;
constexpr int kGatherThreads = 128;
constexpr int kBatch = 4;   // choices whose columns are on their way at once (sumFour)

struct MoveParams {
  const int *place;
  const float *weight;    // NULL: ones
  const void *x, *dy;
  void *y;
  float *dweight;
  int k, n, top, rows;
  int ldx, lddy, ldy;
  int slots;              // threads that a column keeps busy, rounded to whole blocks
};

__device__ __forceinline__ bool placed(const MoveParams &p, int at) { return at >= 0 && at < p.rows; }

template <typename T>
constexpr bool kNumber = sizeof(T) > 1;   // bytes move as they are

// y(:, place(j, t)) = weight(j, t) x(:, t). Bound by its stores: 8192 tokens with 8
// choices, 2048 BF16 values, 48 us (293 MB, 6.1 TB/s).
template <typename T, bool kVector>
__global__ void __launch_bounds__(kScatterThreads) scatterTokensKernel(const MoveParams p) {
  using L = Lanes<T, kVector>;
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const long long t = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
  if (t >= p.n) return;
  const int *place = p.place + t * p.top;
  for (int slot = blockIdx.y * blockDim.x + threadIdx.x; slot < p.slots; slot += gridDim.y * blockDim.x) {
    const int at = L::begin(slot), left = p.k - at;
    if (left <= 0) continue;
    L v;
    v.load(static_cast<const T *>(p.x) + t * p.ldx + at, left);
    for (int j = 0; j < p.top; ++j) {
      const int to = __ldg(place + j);
      if (!placed(p, to)) continue;
      T *y = static_cast<T *>(p.y) + static_cast<long long>(to) * p.ldy + at;
      if constexpr (kNumber<T>) {
        if (p.weight != nullptr) {
          const float w = __ldg(p.weight + t * p.top + j);
          L out;
#pragma unroll
          for (int i = 0; i < L::kPairs; ++i) out.setPair(i, __fmul2_rn(both(w), v.pair(i)));
          out.store(y, left);
          continue;
        }
      }
      v.store(y, left);
    }
  }
}

// y(:, t) = sum over j of weight(j, t) x(:, place(j, t)), in the order of j. Bound by its
// loads, kBatch columns of a token at a time: the same tokens 47 us (6.2 TB/s).
template <typename T, bool kVector>
__global__ void __launch_bounds__(kGatherThreads) gatherTokensKernel(const MoveParams p) {
  using L = Lanes<T, kVector>;
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const long long t = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
  if (t >= p.n) return;
  const int *place = p.place + t * p.top;
  const float *weight = p.weight == nullptr ? nullptr : p.weight + t * p.top;
  for (int slot = blockIdx.y * blockDim.x + threadIdx.x; slot < p.slots; slot += gridDim.y * blockDim.x) {
    const int at = L::begin(slot), left = p.k - at;
    if (left <= 0) continue;
    float2 sum[L::kPairs];
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) sum[i] = make_float2(0.0F, 0.0F);
    for (int j0 = 0; j0 < p.top; j0 += kBatch) {
      L v[kBatch];
      float w[kBatch];
      bool live[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int from = j0 + b < p.top ? __ldg(place + j0 + b) : -1;
        live[b] = placed(p, from);
        w[b] = live[b] && weight != nullptr ? __ldg(weight + j0 + b) : 1.0F;
        if (live[b]) v[b].load(static_cast<const T *>(p.x) + static_cast<long long>(from) * p.ldx + at, left);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (!live[b]) continue;
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) sum[i] = __ffma2_rn(both(w[b]), v[b].pair(i), sum[i]);
      }
    }
    L out;
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) out.setPair(i, sum[i]);
    out.store(static_cast<T *>(p.y) + t * p.ldy + at, left);
  }
}

// The sums over a warp of four values; lanes 8 b to 8 b + 7 get the b-th.
__device__ __forceinline__ float sumFour(const float (&v)[4], int lane) {
  const bool upper = (lane & 16) != 0, odd = (lane & 8) != 0;
  float a = upper ? v[2] : v[0], b = upper ? v[3] : v[1];
  a += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], 16);
  b += __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], 16);
  float s = odd ? b : a;
  s += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
  for (int d = 4; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
  return s;
}

// y(:, place(j, t)) = weight(j, t) dy(:, t) and, with dweight,
// dweight(j, t) = sum over k of dy(k, t) x(k, place(j, t)); a CTA's row of
// blockDim.x threads per token, so that dy is read once for kBatch choices and dweight
// needs no second pass. Bound by HBM: the same tokens 86 to 89 us (6.4 TB/s); 3001 tokens with
// 3 choices, 1537 values on odd addresses, by accesses of one value: 19 us (3.3 TB/s), 12.5
// where L2 has them; 8192 with 8, 2047 values, 133 (scattered 68, gathered 71).
template <typename T, bool kVector>
__global__ void __launch_bounds__(kGatherThreads, 8) gatherTokensBackwardKernel(const MoveParams p) {
  using L = Lanes<T, kVector>;
  __shared__ float partial[kGatherThreads / 32][kBatch];
  kern::gridDependencyWait();
  kern::allowDependentLaunch();
  const long long t = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
  const bool in = t < p.n;
  const int warps = blockDim.x / 32, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int j0 = 0; j0 < p.top; j0 += kBatch) {
    int to[kBatch];
    float w[kBatch];
    float2 dots[kBatch];   // sums of the even and the odd values
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      to[b] = in && j0 + b < p.top ? __ldg(p.place + t * p.top + j0 + b) : -1;
      if (!placed(p, to[b])) to[b] = -1;
      w[b] = to[b] >= 0 && p.weight != nullptr ? __ldg(p.weight + t * p.top + j0 + b) : 1.0F;
      dots[b] = make_float2(0.0F, 0.0F);
    }
    for (int slot = threadIdx.x; slot < p.slots; slot += blockDim.x) {
      const int at = L::begin(slot), left = p.k - at;
      if (!in || left <= 0) continue;
      L dy, x[kBatch];
      dy.load(static_cast<const T *>(p.dy) + t * p.lddy + at, left);
      if (p.dweight != nullptr) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (to[b] >= 0)
            x[b].load(static_cast<const T *>(p.x) + static_cast<long long>(to[b]) * p.ldx + at, left);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (to[b] < 0) continue;
        L out;
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) out.setPair(i, __fmul2_rn(both(w[b]), dy.pair(i)));
        out.store(static_cast<T *>(p.y) + static_cast<long long>(to[b]) * p.ldy + at, left);
        if (p.dweight != nullptr) {
#pragma unroll
          for (int i = 0; i < L::kPairs; ++i) dots[b] = __ffma2_rn(dy.pair(i), x[b].pair(i), dots[b]);
        }
      }
    }
    if (p.dweight == nullptr) continue;
    float dot[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) dot[b] = dots[b].x + dots[b].y;
    const float sum = sumFour(dot, lane);   // of choice lane / 8
    if (warps > 1) {   // one token
      if (lane % 8 == 0) partial[warp][lane / 8] = sum;
      __syncthreads();
      if (threadIdx.x < kBatch) {
        float s = 0.0F;
        for (int v = 0; v < warps; ++v) s += partial[v][threadIdx.x];
        if (j0 + static_cast<int>(threadIdx.x) < p.top) p.dweight[t * p.top + j0 + threadIdx.x] = s;
      }
      __syncthreads();
    } else if (in && lane % 8 == 0 && j0 + lane / 8 < p.top) {
      p.dweight[t * p.top + j0 + lane / 8] = sum;
    }
  }
}

template <typename P, typename... Rest>
sgblasStatus_t launchTokens(void (*kernel)(P, Rest...), dim3 grid, dim3 block, cudaStream_t stream,
                            const P &p) {
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

enum class Move { kScatter, kGather, kBackward };

template <typename T, bool kVector>
sgblasStatus_t launchMove(Move move, MoveParams p, int sms, cudaStream_t stream) {
  using L = Lanes<T, kVector>;
  p.slots = ((p.k - 1) / kern::kLaneBlock + 1) * L::kThreads;
  const bool whole = move == Move::kBackward;   // a token's threads share its sums
  // Threads in whole warps, as busy in their last turn as in the others.
  const int limit = move == Move::kScatter ? kScatterThreads : kGatherThreads;
  const int turns = (p.slots - 1) / limit + 1;
  const int threads = ((p.slots - 1) / turns / 32 + 1) * 32;
  const int tokens = whole && threads > 32 ? 1 : limit / threads;
  const dim3 block(static_cast<unsigned>(threads), static_cast<unsigned>(tokens));
  const int across = (p.n - 1) / tokens + 1;
  // Long columns of few tokens are cut, so that every SM has some.
  const int cuts = whole ? 1 : std::max(1, std::min((p.slots - 1) / threads + 1, 2 * sms / across));
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(cuts));
  if constexpr (!kNumber<T>) {
    return launchTokens(scatterTokensKernel<T, kVector>, grid, block, stream, p);
  } else {
    switch (move) {
      case Move::kScatter: return launchTokens(scatterTokensKernel<T, kVector>, grid, block, stream, p);
      case Move::kGather: return launchTokens(gatherTokensKernel<T, kVector>, grid, block, stream, p);
      default: return launchTokens(gatherTokensBackwardKernel<T, kVector>, grid, block, stream, p);
    }
  }
}

sgblasStatus_t launchMoveTyped(Move move, const MoveParams &p, sgblasDataType_t type, int sms,
                               cudaStream_t stream) {
  const int size = type == SGBLAS_TYPE_FP32 ? 4 : type == SGBLAS_TYPE_BF16 ? 2 : 1;
  auto whole = [&](const void *at, long long ld) {
    return at == nullptr || (aligned16(at) && ld * size % 16 == 0);
  };
  const bool vector = p.k * static_cast<long long>(size) % 16 == 0 && whole(p.x, p.ldx) && whole(p.dy, p.lddy) && whole(p.y, p.ldy);
  if (type == SGBLAS_TYPE_FP32)
    return vector ? launchMove<float, true>(move, p, sms, stream)
                  : launchMove<float, false>(move, p, sms, stream);
  if (type == SGBLAS_TYPE_BF16)
    return vector ? launchMove<__nv_bfloat16, true>(move, p, sms, stream)
                  : launchMove<__nv_bfloat16, false>(move, p, sms, stream);
  return vector ? launchMove<unsigned char, true>(move, p, sms, stream)
                : launchMove<unsigned char, false>(move, p, sms, stream);
}

}  // namespace
}  // namespace sgblas::detail

extern "C" sgblasStatus_t sgblasSortTokens(sgblasHandle_t handle, int n, int top, int groups,
                                           const int *group, int *offsets, int *place) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  if (n < 0 || top < 0 || groups < 0 || offsets == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  const long long entries = static_cast<long long>(n) * top;
  if (entries > 0 && (group == nullptr || place == nullptr)) return SGBLAS_STATUS_INVALID_VALUE;
  if (groups > SGBLAS_MAX_GROUPS || entries > kSortMaxEntries) return SGBLAS_STATUS_NOT_SUPPORTED;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  constexpr int kMost = (kSortThreads / 32 + 2) * SGBLAS_MAX_GROUPS * 4;
  static_assert(SGBLAS_MAX_GROUPS < 1 << 11, "a group's bits");
  static std::atomic<uint64_t> configured[2];
  static std::atomic<int> known[2][kMaxDevices];
  auto *kernel = groups < 256 ? sortTokensKernel<8> : sortTokensKernel<11>;
  const auto *entry = reinterpret_cast<const void *>(kernel);
  const int which = groups < 256 ? 0 : 1;
  if (!configureKernel(entry, dev.device, kMost, &configured[which])) return SGBLAS_STATUS_EXECUTION_FAILED;
  const int most = clusterLimit(entry, dev.device, kMost, known[which]);
  SortParams p = {};
  p.group = group;
  p.offsets = offsets;
  p.place = place;
  p.entries = static_cast<int>(entries);
  p.groups = groups;
  // Spread over SMs first: kSortCtaWarps warps in each CTA, then more CTAs, up to a
  // cluster's, then more warps.
  const long long wanted = std::max(1LL, (entries + kSortWarpEntries - 1) / kSortWarpEntries);
  int ctas = 1;
  while (ctas < most && static_cast<long long>(ctas) * kSortCtaWarps < wanted) ctas *= 2;
  const int warps = static_cast<int>(std::min<long long>(kSortThreads / 32, std::max((wanted - 1) / ctas + 1, 4LL)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(32 * warps));
  cfg.dynamicSmemBytes = sizeof(int) * static_cast<size_t>(warps + 2) * std::max(groups, 1);
  cfg.stream = static_cast<cudaStream_t>(handle->stream);
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return launchStatus(cudaLaunchKernelEx(&cfg, kernel, p, ctas));
}

extern "C" sgblasStatus_t sgblasScatterTokens(sgblasHandle_t handle, int k, int n, int top, int rows,
                                              const int *place, const float *weights, const void *x,
                                              sgblasDataType_t type, int ldx, void *y, int ldy) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const bool bytes = type == SGBLAS_TYPE_BYTE;
  if (k < 0 || n < 0 || top < 0 || rows < 0 || !(bytes || isType(type)) ||
      (bytes && weights != nullptr) || ldx < std::max(1, k) || ldy < std::max(1, k))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (k == 0 || n == 0 || top == 0 || rows == 0) return SGBLAS_STATUS_SUCCESS;
  if (place == nullptr || x == nullptr || y == nullptr) return SGBLAS_STATUS_INVALID_VALUE;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  MoveParams p = {};
  p.place = place;
  p.weight = weights;
  p.x = x;
  p.y = y;
  p.k = k;
  p.n = n;
  p.top = top;
  p.rows = rows;
  p.ldx = ldx;
  p.ldy = ldy;
  return launchMoveTyped(Move::kScatter, p, type, dev.sms, static_cast<cudaStream_t>(handle->stream));
}

extern "C" sgblasStatus_t sgblasGatherTokens(sgblasHandle_t handle, int k, int n, int top, int rows,
                                             const int *place, const float *weights, const void *x,
                                             sgblasDataType_t type, int ldx, void *y, int ldy) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  if (k < 0 || n < 0 || top < 0 || rows < 0 || !isType(type) || ldx < std::max(1, k) ||
      ldy < std::max(1, k))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (k == 0 || n == 0) return SGBLAS_STATUS_SUCCESS;
  if (y == nullptr || (top > 0 && place == nullptr) || (top > 0 && rows > 0 && x == nullptr))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (top > kMaxTop) return SGBLAS_STATUS_NOT_SUPPORTED;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  MoveParams p = {};
  p.place = place;
  p.weight = weights;
  p.x = x;
  p.y = y;
  p.k = k;
  p.n = n;
  p.top = top;
  p.rows = rows;
  p.ldx = ldx;
  p.ldy = ldy;
  return launchMoveTyped(Move::kGather, p, type, dev.sms, static_cast<cudaStream_t>(handle->stream));
}

extern "C" sgblasStatus_t sgblasGatherTokensBackward(sgblasHandle_t handle, int k, int n, int top,
                                                     int rows, const int *place,
                                                     const float *weights, const void *dy,
                                                     sgblasDataType_t type, int lddy, const void *x,
                                                     int ldx, void *dx, int lddx, float *dweights) {
  using namespace sgblas::detail;
  if (handle == nullptr) return SGBLAS_STATUS_NOT_INITIALIZED;
  const int one = std::max(1, k);
  if (k < 0 || n < 0 || top < 0 || rows < 0 || !isType(type) || lddy < one || lddx < one ||
      (dweights != nullptr && ldx < one))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (n == 0 || top == 0 || (k == 0 && dweights == nullptr)) return SGBLAS_STATUS_SUCCESS;
  if (place == nullptr || (rows > 0 && (dy == nullptr || dx == nullptr)) ||
      (rows > 0 && dweights != nullptr && x == nullptr))
    return SGBLAS_STATUS_INVALID_VALUE;
  if (rows == 0 && dweights == nullptr) return SGBLAS_STATUS_SUCCESS;
  if (top > kMaxTop) return SGBLAS_STATUS_NOT_SUPPORTED;
  DeviceInfo dev;
  const sgblasStatus_t st = currentDevice(&dev);
  if (st != SGBLAS_STATUS_SUCCESS) return st;
  MoveParams p = {};
  p.place = place;
  p.weight = weights;
  p.dy = dy;
  p.x = dweights == nullptr ? nullptr : x;
  p.y = dx;
  p.dweight = dweights;
  p.k = rows > 0 ? k : 0;   // without rows dy, x and dx may be NULL: only zeros are written
  p.n = n;
  p.top = top;
  p.rows = rows;
  p.lddy = lddy;
  p.ldx = ldx;
  p.ldy = lddx;
  return launchMoveTyped(Move::kBackward, p, type, dev.sms, static_cast<cudaStream_t>(handle->stream));
}
