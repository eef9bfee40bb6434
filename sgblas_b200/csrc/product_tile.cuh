// Tensor-core products with 16- and 8-bit operands (bf16, pairs of fp16,
// e4m3): C = op(A) * op(B) per group or matrix, FP32 sums.
//
// One persistent CTA per SM walks 128 x N tiles of C: rows (m) on the 128
// TMEM lanes, columns (n; tokens, where the groups are ragged along n) on the
// instruction's N. A ragged group's last tile costs what it holds: N is set
// per tile in steps of 16. Warp roles (12 warps):
//   warp 0      TMA producer: 128-byte wide k slices of A and B into a ring;
//   warp 1      MMA issuer: tcgen05.mma into one of two TMEM accumulators;
//   warp 2      allocates and frees TMEM;
//   warps 4-11  epilogue: two warps per TMEM lane quarter, half the columns
//               each, keep the tile's sums in registers.
//
// Sums. The tensor core's FP32 adder truncates: the relative error of a chain
// grows with its length (measured 3e-7 after 32 instructions, 3e-6 after 512).
// So the k range is cut into chunks of kChunkIters slices; the issuer
// alternates between the two accumulators, and the epilogue adds each chunk
// to the registers with rounding to nearest. For e4m3 the chunk is one block
// of 128, and the same addition applies the block's scales.
//
// Operands are K-major (k contiguous) or, 16-bit only, MN-major (m or n
// contiguous); both are staged as TMA writes them and described to the tensor
// core accordingly.
#ifndef SGBLAS_B200_PRODUCT_TILE_CUH_
#define SGBLAS_B200_PRODUCT_TILE_CUH_

#include "ptx.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace sgblas::kern::prod {

constexpr int kBM = 128;            // tile rows: TMEM lanes
constexpr int kRowBytes = 128;      // one 128-byte swizzle row
constexpr int kAccums = 2;
constexpr int kThreads = 384;
constexpr int kEpilogueWarp0 = 4;
constexpr int kEpilogueThreads = 256;
constexpr int kMaxGroups = 1024;
constexpr int kScaleBatch = 8;      // blocks of 128 whose scales are staged at once

// Which index the groups divide: n (columns of B and C), k (columns of A and
// B), or none (a strided batch).
enum class Ragged { kN, kK, kBatch };

// kPlanes 2: every operand is a pair of fp16 matrices, hi + lo, and a product
// is hi hi + hi lo + lo hi. kSymmetric: C is symmetric; only tiles on and
// below the diagonal are computed, and stored twice.
template <int kElemBytes, Ragged kRagged, int kBN_, bool kAMN, bool kBMN, int kPlanes,
          bool kSymmetric>
struct Cfg {
  static constexpr bool kBytes = kElemBytes == 1;
  static constexpr int kBN = kBN_;
  static constexpr int kBK = kRowBytes / kElemBytes;   // 64 or 128
  static constexpr int kMmaK = 32 / kElemBytes;        // 16 or 32
  static constexpr int kChunkIters = kBytes ? 1 : kPlanes == 2 ? 4 : 8;   // 128, 256 or 512 of k
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBBytes = kBN * kRowBytes;
  static constexpr int kStageBytes = kPlanes * (kABytes + kBBytes);
  static constexpr int kScaleBytes = kBytes ? 2 * kScaleBatch * kBN * 4 : 0;
  static constexpr int kFit = (208 * 1024 - kScaleBytes) / kStageBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kTmemColumns = kAccums * kBN < 32 ? 32 : kAccums * kBN;
  static constexpr int kBarrierBytes = 8 * (2 * kStages + 2 * kAccums);
  static constexpr int kSmemBytes = kStages * kStageBytes + kScaleBytes + kBarrierBytes + 1024;
  static_assert(kBN == 32 || kBN == 64 || kBN == 128 || kBN == 256, "tile width");
  static_assert(!kSymmetric || kBN == kBM, "square tiles");
  static_assert(!kBytes || (!kAMN && !kBMN), "8-bit operands are K-major");
  static_assert(kSmemBytes <= 218 * 1024, "shared memory per CTA, beside the group table");
};

// What the epilogue of a pair product writes (values v of the sum):
//   kGram    hi + lo of v * 2^-12
//   kPoly    hi + lo of c2 v 2^-12 + c1 A + c0 2^12 I, A the pair at prev
//   kUpdate  hi + lo of v * 2^-12
//   kFinal   bf16 of v * 2^-24 * alpha
// Pairs hold 2^12 times their value: fp16 then keeps 22 bits of every value
// above 2^-16 and an absolute 2^-37 below, and reaches 15.99.
enum class PairOut { kGram, kPoly, kUpdate, kFinal };
constexpr float kPairScale = 4096.0F;

struct PairParams {
  CUtensorMap tma_a_lo, tma_b_lo;
  PairOut out;
  __half *hi, *lo;                   // written
  const __half *prev_hi, *prev_lo;   // kPoly reads
  float c0, c1, c2;
};

struct Params {
  CUtensorMap tma_a, tma_b;   // 3-D: (contiguous, strided, matrix)
  const int *offsets;         // groups + 1 device offsets; NULL: one group of everything
  int groups;                 // or matrices of the batch
  int m, n, k;                // n (Ragged::kN) and k (Ragged::kK) are totals
  int tiles_m, tiles_n;       // tiles_n: Ragged::kK and kBatch
  void *c;
  int c_bf16;
  int ldc;
  long long stride_c;         // Ragged::kK and kBatch
  float alpha, beta;
  const float *scale_a, *scale_b;   // e4m3: per (128 of k, 128 of m) and (128 of k, column)
  int ldsa, ldsb;
  long long stride_sa;
  unsigned format;            // the instruction descriptor's type bits
  unsigned *err;
  PairParams pair;
};

// Type bits of the instruction descriptor (A and B alike).
constexpr unsigned kFormatBf16 = (1u << 7) | (1u << 10);
constexpr unsigned kFormatFp16 = 0;
constexpr unsigned kFormatE4m3 = 0;

// Shared-memory matrix descriptor, 128-byte swizzle. K-major: rows of 128
// bytes, 8-row groups 1024 bytes apart (SBO). MN-major: 128-byte rows of 64
// consecutive m (or n) per k, 8-row (k) groups 1024 bytes apart (SBO), 64-wide
// chunks of m one 64-row box apart (LBO).
template <bool kMN>
__device__ __forceinline__ uint64_t smemDesc(uint32_t addr) {
  constexpr uint32_t lbo = kMN ? 64 * kRowBytes : 16;
  constexpr uint32_t sbo = 1024;
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16;
  d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFF) << 32;
  d |= static_cast<uint64_t>(1) << 46;   // version
  d |= static_cast<uint64_t>(2) << 61;   // SWIZZLE_128B
  return d;
}

template <bool kAMN, bool kBMN>
__device__ __forceinline__ uint32_t instrDesc(unsigned format, int n) {
  return (1u << 4) | format | (static_cast<uint32_t>(kAMN) << 15) |
         (static_cast<uint32_t>(kBMN) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kBM >> 4) << 24);
}

// The groups as one CTA sees them: offsets clamped to [0, total], and for
// groups ragged along n the running count of column tiles.
struct GroupTable {
  int offset[kMaxGroups + 1];
  int first[kMaxGroups + 1];
};

// One tile: its matrix, origin, valid columns, and k range.
struct Tile {
  int group, m0, n0, cols, k0, klen;
};

template <Ragged kRagged, int kBN, bool kSymmetric>
__device__ __forceinline__ int tileCount(const Params &p, const GroupTable &t) {
  if constexpr (kSymmetric) return p.tiles_m * (p.tiles_m + 1) / 2 * p.groups;
  if constexpr (kRagged == Ragged::kN) return p.tiles_m * t.first[p.groups];
  return p.tiles_m * p.tiles_n * p.groups;
}

template <Ragged kRagged, int kBN, bool kSymmetric>
__device__ __forceinline__ Tile tileAt(const Params &p, const GroupTable &t, int index) {
  Tile r;
  if constexpr (kSymmetric) {
    const int per = p.tiles_m * (p.tiles_m + 1) / 2;
    r.group = index / per;
    const int i = index - r.group * per;
    // Row of a triangle: the largest tm with tm (tm + 1) / 2 <= i.
    int tm = static_cast<int>((sqrtf(8.0F * static_cast<float>(i) + 1.0F) - 1.0F) * 0.5F);
    while (tm * (tm + 1) / 2 > i) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= i) ++tm;
    r.m0 = tm * kBM;
    r.n0 = (i - tm * (tm + 1) / 2) * kBN;
    r.cols = min(kBN, p.n - r.n0);
    r.k0 = 0;
    r.klen = p.k;
  } else if constexpr (kRagged == Ragged::kN) {
    const int nt = index / p.tiles_m;
    r.m0 = (index - nt * p.tiles_m) * kBM;
    int lo = 0, hi = p.groups;   // the last group whose first tile is <= nt
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (t.first[mid] <= nt) lo = mid;
      else hi = mid;
    }
    r.group = lo;
    r.n0 = t.offset[lo] + (nt - t.first[lo]) * kBN;
    r.cols = min(kBN, t.offset[lo + 1] - r.n0);
    r.k0 = 0;
    r.klen = p.k;
  } else {
    const int per = p.tiles_m * p.tiles_n;
    r.group = index / per;
    const int i = index - r.group * per;
    const int tn = i / p.tiles_m;
    r.m0 = (i - tn * p.tiles_m) * kBM;
    r.n0 = tn * kBN;
    r.cols = min(kBN, p.n - r.n0);
    r.k0 = 0;
    r.klen = p.k;
    if constexpr (kRagged == Ragged::kK) {
      r.k0 = t.offset[r.group];
      r.klen = max(0, t.offset[r.group + 1] - r.k0);
    }
  }
  return r;
}

// Fills the table (all threads; ends with a barrier).
template <Ragged kRagged, int kBN>
__device__ __forceinline__ void readGroups(const Params &p, GroupTable *t) {
  if constexpr (kRagged == Ragged::kBatch) return;
  const int total = kRagged == Ragged::kN ? p.n : p.k;
  if (p.offsets == nullptr) {
    if (threadIdx.x == 0) {
      t->offset[0] = 0;
      t->offset[1] = total;
    }
  } else {
    for (int g = threadIdx.x; g <= p.groups; g += kThreads)
      t->offset[g] = min(max(p.offsets[g], 0), total);
  }
  __syncthreads();
  if constexpr (kRagged == Ragged::kN) {
    if (threadIdx.x < 32) {
      int sum = 0;
      for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + static_cast<int>(threadIdx.x);
        int v = 0;
        if (g < p.groups) v = (max(0, t->offset[g + 1] - t->offset[g]) + kBN - 1) / kBN;
        int scan = v;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int o = __shfl_up_sync(0xffffffffu, scan, d);
          if (static_cast<int>(threadIdx.x) >= d) scan += o;
        }
        if (g < p.groups) t->first[g] = sum + scan - v;
        sum += __shfl_sync(0xffffffffu, scan, 31);
      }
      if (threadIdx.x == 0) t->first[p.groups] = sum;
    }
    __syncthreads();
  }
}

// Zeroes the 128-byte rows [row0, row1) of each 64-row box of an MN-major
// operand (all lanes of one warp).
template <int kBoxes>
__device__ __forceinline__ void zeroRows(unsigned char *operand, int row0, int row1, int lane) {
  const int chunks = (row1 - row0) * (kRowBytes / 16);
  for (int box = 0; box < kBoxes; ++box) {
    unsigned char *base = operand + box * 64 * kRowBytes + row0 * kRowBytes;
    for (int i = lane; i < chunks; i += 32)
      *reinterpret_cast<uint4 *>(base + i * 16) = make_uint4(0, 0, 0, 0);
  }
}

// hi + lo = v to 22 bits.
__device__ __forceinline__ void splitPair(float v, __half *hi, __half *lo) {
  *hi = __float2half_rn(v);
  *lo = __float2half_rn(v - __half2float(*hi));
}

// Epilogue of a pair product: this thread's row, kHalf columns from col_begin.
template <int kHalf, bool kSymmetric>
__device__ __forceinline__ void storePair(const Params &p, const Tile &t, int row, int col_begin,
                                          const float (&acc)[kHalf]) {
  if (row >= p.m) return;
  const size_t matrix = static_cast<size_t>(t.group) * static_cast<size_t>(p.stride_c);
  const bool mirror = kSymmetric && t.m0 != t.n0;
#pragma unroll
  for (int j0 = 0; j0 < kHalf; j0 += 8) {
    if (col_begin + j0 >= t.cols) break;
    alignas(16) __half hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = t.n0 + col_begin + j0 + j;
      const bool in = col_begin + j0 + j < t.cols;
      const size_t at = matrix + static_cast<size_t>(col) * p.ldc + row;
      if (p.pair.out == PairOut::kFinal) {
        if (in)
          static_cast<__nv_bfloat16 *>(p.c)[at] =
              __float2bfloat16(acc[j0 + j] * (1.0F / (kPairScale * kPairScale)) * p.alpha);
        continue;
      }
      float v = acc[j0 + j] * (1.0F / kPairScale);
      if (p.pair.out == PairOut::kPoly) {
        v *= p.pair.c2;
        if (in)
          v = fmaf(p.pair.c1, __half2float(p.pair.prev_hi[at]) + __half2float(p.pair.prev_lo[at]),
                   v);
        if (col == row) v = fmaf(p.pair.c0, kPairScale, v);
      }
      splitPair(v, &hi[j], &lo[j]);
      if (in) {
        p.pair.hi[at] = hi[j];
        p.pair.lo[at] = lo[j];
      }
    }
    // The mirrored tile: rows are padded to 64 elements, so a vector may
    // reach past n into the padding, which nothing reads.
    if (mirror) {
      const size_t at = matrix + static_cast<size_t>(row) * p.ldc + t.n0 + col_begin + j0;
      *reinterpret_cast<uint4 *>(p.pair.hi + at) = *reinterpret_cast<const uint4 *>(hi);
      *reinterpret_cast<uint4 *>(p.pair.lo + at) = *reinterpret_cast<const uint4 *>(lo);
    }
  }
}

template <int kElemBytes, Ragged kRagged, int kBN, bool kAMN, bool kBMN, int kPlanes = 1,
          bool kSymmetric = false>
__global__ void __launch_bounds__(kThreads, 1) productKernel(const __grid_constant__ Params p) {
  using G = Cfg<kElemBytes, kRagged, kBN, kAMN, kBMN, kPlanes, kSymmetric>;
  constexpr int kStages = G::kStages;
  constexpr int kStageBytes = G::kStageBytes;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ GroupTable table;
  unsigned char *smem = smem_raw + ((1024 - (smemAddr(smem_raw) & 1023)) & 1023);
  float *scales = reinterpret_cast<float *>(smem + kStages * kStageBytes);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStages * kStageBytes + G::kScaleBytes);
  uint64_t *empty = full + kStages;
  uint64_t *acc_full = empty + kStages;
  uint64_t *acc_empty = acc_full + kAccums;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    if (p.k > 0) {
      prefetchTensorMap(&p.tma_a);
      prefetchTensorMap(&p.tma_b);
    }
    for (int s = 0; s < kStages; ++s) {
      mbarInit(&full[s], 1);
      mbarInit(&empty[s], 1);
    }
    for (int b = 0; b < kAccums; ++b) {
      mbarInit(&acc_full[b], 1);
      mbarInit(&acc_empty[b], kEpilogueThreads);
    }
    fenceBarrierInit();
  }
  if (warp == 2) {
    tmemAlloc(&tmem_base_slot, G::kTmemColumns);
    tmemRelinquish();
  }
  gridDependencyWait();
  readGroups<kRagged, kBN>(p, &table);
  tcgenFenceBefore();
  __syncthreads();
  tcgenFenceAfter();
  allowDependentLaunch();
  const uint32_t tmem_base = tmem_base_slot;
  const int tiles = tileCount<kRagged, kBN, kSymmetric>(p, table);

  bool ok = true;
  auto wait = [&](uint64_t *bar, int parity) {
    if (ok) ok = mbarWait(bar, static_cast<uint32_t>(parity), p.err);
  };

  if (warp < kEpilogueWarp0) {
    regDealloc<56>();
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer ----------------
      int s = 0, parity = 1;   // the first pass over the ring waits for nothing
      for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
        const Tile t = tileAt<kRagged, kBN, kSymmetric>(p, table, i);
        const int za = kRagged == Ragged::kK ? 0 : t.group;
        const int zb = kRagged == Ragged::kBatch ? t.group : 0;
        for (int kk = 0; kk < t.klen; kk += G::kBK) {
          wait(&empty[s], parity);
          const int k0 = t.k0 + kk;
          mbarArriveExpectTx(&full[s], kStageBytes);
#pragma unroll
          for (int plane = 0; plane < kPlanes; ++plane) {
            unsigned char *sa = smem + s * kStageBytes + plane * G::kABytes;
            unsigned char *sb = smem + s * kStageBytes + kPlanes * G::kABytes + plane * G::kBBytes;
            const CUtensorMap *map_a = plane == 0 ? &p.tma_a : &p.pair.tma_a_lo;
            const CUtensorMap *map_b = plane == 0 ? &p.tma_b : &p.pair.tma_b_lo;
            if constexpr (kAMN) {
              for (int j = 0; j < kBM / 64; ++j)
                tmaLoad3d(sa + j * 64 * kRowBytes, map_a, &full[s], t.m0 + 64 * j, k0, za);
            } else {
              tmaLoad3d(sa, map_a, &full[s], k0, t.m0, za);
            }
            if constexpr (kBMN) {
              for (int j = 0; j < kBN / 64; ++j)
                tmaLoad3d(sb + j * 64 * kRowBytes, map_b, &full[s], t.n0 + 64 * j, k0, zb);
            } else {
              tmaLoad3d(sb, map_b, &full[s], k0, t.n0, zb);
            }
          }
          if (++s == kStages) {
            s = 0;
            parity ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      int s = 0, parity = 0;
      int b = 0, acc_parity = 1;
      for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
        const Tile t = tileAt<kRagged, kBN, kSymmetric>(p, table, i);
        const uint32_t idesc = instrDesc<kAMN, kBMN>(p.format, (t.cols + 15) / 16 * 16);
        const int iters = (t.klen + G::kBK - 1) / G::kBK;
        for (int kb = 0; kb < iters; ++kb) {
          const bool first = kb % G::kChunkIters == 0;
          const bool last = kb % G::kChunkIters == G::kChunkIters - 1 || kb == iters - 1;
          if (first) wait(&acc_empty[b], acc_parity);
          wait(&full[s], parity);
          unsigned char *stage = smem + s * kStageBytes;
          int steps = G::kBK / G::kMmaK;
          if constexpr (kRagged == Ragged::kK) {
            // The group's last slice: rows of k beyond it belong to the next
            // group. Both operands' rows up to the next multiple of 16 are
            // zeroed (zero times a NaN is a NaN), the rest is not multiplied.
            const int rows = t.klen - kb * G::kBK;
            if (rows < G::kBK) {
              steps = (rows + G::kMmaK - 1) / G::kMmaK;
              zeroRows<kBM / 64>(stage, rows, steps * G::kMmaK, lane);
              zeroRows<kBN / 64>(stage + G::kABytes, rows, steps * G::kMmaK, lane);
              fenceProxyAsyncShared();
              __syncwarp();
            }
          }
          if (lane == 0) {
            tcgenFenceAfter();
            const uint32_t sa = smemAddr(stage);
            const uint32_t sb = sa + kPlanes * G::kABytes;
            const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(b * kBN);
            for (int j = 0; j < steps; ++j) {
              // K-major: the next instruction's k are 32 bytes further along
              // each row; MN-major: 16 rows of 128 bytes further.
              const uint32_t a0 = sa + (kAMN ? j * 16u * kRowBytes : j * 32u);
              const uint32_t b0 = sb + (kBMN ? j * 16u * kRowBytes : j * 32u);
              mmaNarrow<G::kBytes>(d_tmem, smemDesc<kAMN>(a0), smemDesc<kBMN>(b0), idesc,
                                   !first || j > 0);
              if constexpr (kPlanes == 2) {
                mmaNarrow<false>(d_tmem, smemDesc<kAMN>(a0), smemDesc<kBMN>(b0 + G::kBBytes), idesc,
                                 true);
                mmaNarrow<false>(d_tmem, smemDesc<kAMN>(a0 + G::kABytes), smemDesc<kBMN>(b0), idesc,
                                 true);
              }
            }
            mmaCommit(&empty[s]);
            if (last) mmaCommit(&acc_full[b]);
          }
          __syncwarp();
          if (last) {
            b ^= 1;
            if (b == 0) acc_parity ^= 1;
          }
          if (++s == kStages) {
            s = 0;
            parity ^= 1;
          }
        }
      }
    }
  } else {
    // ---------------- epilogue ----------------
    regAlloc<224>();
    constexpr int kHalf = kBN / 2;                     // columns of this warp
    constexpr int kLoad = kHalf < 32 ? kHalf : 32;     // columns of one TMEM load
    const int quarter = warp % 4;
    const int col_begin = (warp - kEpilogueWarp0) / 4 * kHalf;
    const int row_in_tile = quarter * 32 + lane;
    const int etid = threadIdx.x - 32 * kEpilogueWarp0;
    int b = 0, acc_parity = 0;
    int scale_batches = 0;
    for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
      const Tile t = tileAt<kRagged, kBN, kSymmetric>(p, table, i);
      const int row = t.m0 + row_in_tile;
      const int iters = (t.klen + G::kBK - 1) / G::kBK;
      const int chunks = (iters + G::kChunkIters - 1) / G::kChunkIters;
      float acc[kHalf];
#pragma unroll
      for (int j = 0; j < kHalf; ++j) acc[j] = 0.0F;
      for (int ch = 0; ch < chunks; ++ch) {
        const float *sc = nullptr;
        if constexpr (G::kBytes) {
          // Scales of the next kScaleBatch blocks: scale_a * scale_b per
          // (block, column), staged by one thread per column.
          if (ch % kScaleBatch == 0) {
            float *dst = scales + (scale_batches & 1) * kScaleBatch * kBN;
            if (etid < kBN) {
              const bool in = etid < t.cols;
              const float *sb = p.scale_b + static_cast<size_t>(in ? t.n0 + etid : 0) * p.ldsb;
              const float *sa = p.scale_a + t.group * p.stride_sa +
                                static_cast<size_t>(t.m0 / 128) * p.ldsa;
              float v[kScaleBatch];
#pragma unroll
              for (int q = 0; q < kScaleBatch; ++q) {
                const bool live = in && ch + q < chunks;
                v[q] = live ? sb[ch + q] * sa[ch + q] : 0.0F;
              }
#pragma unroll
              for (int q = 0; q < kScaleBatch; ++q) dst[q * kBN + etid] = v[q];
            }
            namedBarrier<1, kEpilogueThreads>();
            ++scale_batches;
          }
          sc = scales + ((scale_batches - 1) & 1) * kScaleBatch * kBN +
               (ch % kScaleBatch) * kBN + col_begin;
        }
        wait(&acc_full[b], acc_parity);
        tcgenFenceAfter();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                               static_cast<uint32_t>(b * kBN + col_begin);
#pragma unroll
        for (int c = 0; c < kHalf; c += kLoad) {
          if (col_begin + c >= t.cols) break;
          uint32_t v[32];
          if constexpr (kLoad == 32) tmemLoad32(taddr + c, v);
          else tmemLoad16(taddr + c, v);
          if constexpr (G::kBytes) {
#pragma unroll
            for (int j = 0; j < kLoad; j += 4) {
              const float4 s4 = *reinterpret_cast<const float4 *>(sc + c + j);
              acc[c + j] = fmaf(__uint_as_float(v[j]), s4.x, acc[c + j]);
              acc[c + j + 1] = fmaf(__uint_as_float(v[j + 1]), s4.y, acc[c + j + 1]);
              acc[c + j + 2] = fmaf(__uint_as_float(v[j + 2]), s4.z, acc[c + j + 2]);
              acc[c + j + 3] = fmaf(__uint_as_float(v[j + 3]), s4.w, acc[c + j + 3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < kLoad; ++j) acc[c + j] += __uint_as_float(v[j]);
          }
        }
        tcgenFenceBefore();
        mbarArrive(&acc_empty[b]);
        b ^= 1;
        if (b == 0) acc_parity ^= 1;
      }
      if constexpr (kPlanes == 2) {
        storePair<kHalf, kSymmetric>(p, t, row, col_begin, acc);
        continue;
      }
      // C = alpha * acc + beta * C; a warp writes 32 consecutive rows of a column.
      if (row < p.m) {
        const long long matrix = kRagged == Ragged::kN ? 0 : t.group * p.stride_c;
#pragma unroll
        for (int j = 0; j < kHalf; ++j) {
          const int col = col_begin + j;
          if (col < t.cols) {
            const size_t at = static_cast<size_t>(matrix) +
                              static_cast<size_t>(t.n0 + col) * p.ldc + row;
            float v = p.alpha * acc[j];
            if (p.c_bf16) {
              __nv_bfloat16 *c = static_cast<__nv_bfloat16 *>(p.c) + at;
              if (p.beta != 0.0F) v = fmaf(p.beta, __bfloat162float(*c), v);
              *c = __float2bfloat16(v);
            } else {
              float *c = static_cast<float *>(p.c) + at;
              if (p.beta != 0.0F) v = fmaf(p.beta, *c, v);
              *c = v;
            }
          }
        }
      }
    }
  }

  tcgenFenceBefore();
  __syncthreads();
  if (warp == 2) {
    tcgenFenceAfter();
    tmemDealloc(tmem_base, G::kTmemColumns);
  }
}

}  // namespace sgblas::kern::prod

#endif  // SGBLAS_B200_PRODUCT_TILE_CUH_
