// Tensor-core products with 16- and 8-bit operands (bf16, pairs of fp16,
// e4m3): C = op(A) * op(B) per group or matrix, FP32 sums.
//
// One persistent CTA per SM walks 128 x N tiles of C, or a pair of CTAs
// (cta_group::2) 256 x 256 ones: rows (m) on the TMEM lanes, columns (n;
// tokens, where the groups are ragged along n) on the instruction's N. A
// ragged group's last tile costs what it holds: N is set per tile in steps of
// 16 (32 for a pair). Warp roles (12 warps):
//   warp 0      TMA producer: 128-byte wide k slices of A and B into a ring;
//   warp 1      MMA issuer: tcgen05.mma into one of two TMEM accumulators;
//   warp 2      allocates and frees TMEM;
//   warps 4-11  epilogue: two warps per TMEM lane quarter, half the columns
//               each, keep the tile's sums in registers and write them out
//               through shared memory.
// In a pair, CTA r loads and holds rows [128 r, 128 r + 128) of the tile and
// half of its columns' operand; the even CTA issues for both. A k slice then
// costs each SM 32 KiB of operands instead of 48 for the same work, which
// is what a single CTA's 128 x 256 tile is bound by (96 bytes per clock at
// the tensor core's rate).
//
// Sums. The tensor core's FP32 adder truncates: the relative error of a chain
// grows with its length (measured 3e-7 after 32 instructions, 3e-6 after 512).
// So the k range is cut into chunks (128 to 512 of k; 4096 for a BF16 result of
// BF16 operands, whose own rounding is a hundred times such a chain's). The issuer
// alternates between the two accumulators, and the epilogue adds each chunk to
// the registers with rounding to nearest. For e4m3 the chunk is one block of
// 128, and the same addition applies the block's scales.
//
// What bounds it, measured. Large BF16 products: the tensor core and the power
// limit (16384 x 4096 x 4096 over 16 uneven experts: the pipe is busy 84 % of the
// cycles, SM clocks fall to 1.1 to 1.4 GHz; 395 to 421 us in replays back to
// back, 486 to 524 as calls on changing inputs, 1.05 to 1.4 PFLOP/s). Large e4m3 products: the power limit and the epilogue, which scales
// every block of 128 in registers (860 clocks a chunk where the tensor core
// takes 512; 8192 x 8192 x 4096 228 to 236 us in replays, 275 to 283 as calls,
// 1.94 to 2.4 PFLOP/s). Weight gradients of few tokens: writing C. Results with a
// beta: reading C (updateColumns). An elected lane of a warp that the
// compiler knows to be uniform issues the instructions in 40 clocks each, a
// lane picked by a test in 57 and, between the waits of this loop, over 100
// (forward 16384: 547 -> 448 us).
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
constexpr int kEpilogueWarps = 8;
constexpr int kEpilogueThreads = 32 * kEpilogueWarps;
constexpr int kOutCols = 16;         // columns in one of a warp's two staging buffers
constexpr int kPairCols = 16;        // columns a warp of a pair product stages
constexpr int kMaxGroups = 1024;
constexpr int kScaleBatch = 8;      // blocks of 128 whose scales are staged at once

// Which index the groups divide: n (columns of B and C), k (columns of A and
// B), or none (a strided batch). kM is kN with the operands' places exchanged
// (e4m3 only): tokens on the TMEM lanes, so that a thread's row has one scale
// per block instead of one per column, and C's contiguous rows of features
// lie along a thread's registers.
enum class Ragged { kN, kK, kBatch, kM };

// kPlanes 2: every operand is a pair of fp16 matrices, hi + lo, and a product
// is hi hi + hi lo + lo hi. kSymmetric: C is symmetric; only tiles that reach
// the diagonal or lie below it are computed, those below are stored twice.
// kTwo: a pair of CTAs. kFp32: C is FP32 or BF16 with a beta, or a pair's
// sums are staged, and a thread holds a row of the tile: a warp's store is then
// 32 contiguous rows, whatever C's alignment.
template <int kElemBytes_, Ragged kRagged_, int kBN_, bool kAMN_, bool kBMN_, bool kTwo_,
          bool kFp32_ = false, int kPlanes_ = 1, bool kSymmetric_ = false>
struct Cfg {
  static constexpr int kElemBytes = kElemBytes_;
  static constexpr Ragged kRagged = kRagged_;
  static constexpr int kBN = kBN_;                     // columns of the tile
  static constexpr bool kAMN = kAMN_, kBMN = kBMN_;
  static constexpr bool kTwo = kTwo_;
  static constexpr bool kFp32 = kFp32_;
  static constexpr int kPlanes = kPlanes_;
  static constexpr bool kSymmetric = kSymmetric_;
  static constexpr bool kBytes = kElemBytes == 1;
  static constexpr int kTileM = kTwo ? 2 * kBM : kBM;  // rows of the tile
  static constexpr int kBRows = kTwo ? kBN / 2 : kBN;  // columns whose operand this CTA loads
  static constexpr int kNStep = kTwo ? 32 : 16;        // granularity of the instruction's N
  static constexpr int kBK = kRowBytes / kElemBytes;   // 64 or 128
  static constexpr int kMmaK = 32 / kElemBytes;        // 16 or 32
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBBytes = kBRows * kRowBytes;
  static constexpr int kStageBytes = kPlanes * (kABytes + kBBytes);
  static constexpr bool kRows = kRagged == Ragged::kM;
  // Scales of the tile's columns, then the weights' one.
  static constexpr bool kStaged = kBytes && !kRows;
  static constexpr int kScalePitch = kBN + 4;
  static constexpr int kScaleBytes = kStaged ? 2 * kScaleBatch * kScalePitch * 4 : 0;
  // Staging of a warp: 32 rows by 128 columns of BF16, the FP32 sums of
  // kPairCols columns, or two buffers of kOutCols columns.
  static constexpr int kOutWarp = kRows          ? 32 * kBN
                                  : kPlanes == 2 ? kPairCols * 32 * 4
                                                 : 2 * kOutCols * 32 * (kFp32 ? 4 : 2);
  static constexpr int kOutBytes = kEpilogueWarps * kOutWarp;
  static constexpr int kFit = (217 * 1024 - kScaleBytes - kOutBytes) / kStageBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  // Narrow pairs: one instruction multiplies A's hi by B's hi and lo, which lie
  // one after the other, into columns of their own (tiles of 32: 48 + 41 clocks
  // for three of 41).
  static constexpr bool kJoined = kPlanes == 2 && !kTwo && kBN <= 64;
  static constexpr int kAccColumns = kJoined ? 2 * kBN : kBN;
  static constexpr int kTmemColumns = kAccums * kAccColumns;
  static constexpr int kBarrierBytes = 8 * (3 * kStages + 2 * kAccums);
  static constexpr int kSmemBytes =
      kStages * kStageBytes + kScaleBytes + kOutBytes + kBarrierBytes + 1024;
  static_assert((kBN == 32 && kPlanes == 2) || kBN == 64 || kBN == 128 || kBN == 256, "tile width");
  static_assert(!kSymmetric || kTileM % kBN == 0, "tiles end at the diagonal");
  static_assert(!kBytes || (!kAMN && !kBMN), "8-bit operands are K-major");
  static_assert(!kRows || (kBytes && kBN == 256), "rows of tokens: e4m3, two blocks of weights");
  static_assert(kPlanes == 1 || kFp32, "pairs leave from FP32 sums");
  static_assert(!kStaged || !kTwo, "a CTA's tile has one block of weights");
  static_assert(!kBMN || kBRows % 64 == 0, "whole boxes");
  static_assert(kStages >= 2 && kSmemBytes <= 218 * 1024 + 512, "shared memory beside the table");
};

// What the epilogue of a pair product writes (values v of the sum):
//   kSum     hi + lo of v * 2^-12
//   kPoly    hi + lo of c2 v 2^-12 + c1 A + c0 2^12 I, A the pair at prev
//   kFinal   bf16 of v * alpha
// Pairs hold 2^12 times their value: fp16 then keeps 22 bits of every value
// above 2^-16 and an absolute 2^-37 below, and reaches 15.99.
enum class PairOut { kSum, kPoly, kFinal };
constexpr float kPairScale = 4096.0F;

struct PairParams {
  CUtensorMap tma_a_lo, tma_b_lo;
  PairOut out;
  __half *hi, *lo;                   // written
  const __half *prev_hi, *prev_lo;   // kPoly reads
  float c0, c1, c2;
  int planes;   // 2, or 1 to multiply the hi parts alone
};

struct Params {
  CUtensorMap tma_a, tma_b;   // 3-D: (contiguous, strided, matrix)
  const int *offsets;         // groups + 1 device offsets; NULL: one group of everything
  int groups;                 // or matrices of the batch
  int m, n, k;                // n (Ragged::kN) and k (Ragged::kK) are totals
  int tiles_m, tiles_n;       // tiles_n: Ragged::kK and kBatch
  void *c;
  int c_bf16;
  CUtensorMap tma_c;          // where c_tma: C in boxes of 64 rows (FP32: 32) and 16 columns (kM: 32)
  int c_tma;                  // TMA can write C (tmaWritable), and beta is 0
  int ldc;
  long long stride_c;         // Ragged::kK and kBatch
  float alpha, beta;
  const float *scale_a, *scale_b;   // e4m3: per (128 of k, 128 of m) and (128 of k, column)
  int ldsa, ldsb;
  long long stride_sa;
  int chunk_iters;            // k slices of one chain
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

template <class G>
__device__ __forceinline__ uint32_t instrDesc(unsigned format, int n) {
  return (1u << 4) | format | (static_cast<uint32_t>(G::kAMN) << 15) |
         (static_cast<uint32_t>(G::kBMN) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(G::kTileM >> 4) << 24);
}

// The groups as one CTA sees them: offsets clamped to [0, total], and for
// groups ragged along n the running count of column tiles.
struct GroupTable {
  int offset[kMaxGroups + 1];
  int first[kMaxGroups + 1];
};

// One tile: its matrix, origin, valid columns (and rows, Ragged::kM), k range.
struct Tile {
  int group, m0, n0, cols, k0, klen, rows;
};

// Tiles of one symmetric matrix: kWays times (tm + 1) in the row of tiles tm,
// less those past the last column.
template <class G>
__host__ __device__ __forceinline__ int symmetricTiles(int tiles_m, int tiles_n) {
  constexpr int kWays = G::kTileM / G::kBN;
  const int past = kWays * tiles_m - tiles_n;
  return kWays * (tiles_m * (tiles_m + 1) / 2) - (past > 0 ? past : 0);
}

template <class G>
__device__ __forceinline__ int tileCount(const Params &p, const GroupTable &t) {
  if constexpr (G::kSymmetric) return symmetricTiles<G>(p.tiles_m, p.tiles_n) * p.groups;
  if constexpr (G::kRagged == Ragged::kN) return p.tiles_m * t.first[p.groups];
  if constexpr (G::kRagged == Ragged::kM) return p.tiles_n * t.first[p.groups];
  return p.tiles_m * p.tiles_n * p.groups;
}

template <class G>
__host__ __device__ __forceinline__ Tile tileAt(const Params &p, const GroupTable &t, int index) {
  Tile r;
  if constexpr (G::kSymmetric) {
    constexpr int kWays = G::kTileM / G::kBN;
    const int per = symmetricTiles<G>(p.tiles_m, p.tiles_n);
    r.group = index / per;
    const int i = index - r.group * per;
    // The row of tiles: the largest tm with kWays tm (tm + 1) / 2 <= i.
    int tm = static_cast<int>((sqrtf(8.0F / kWays * static_cast<float>(i) + 1.0F) - 1.0F) * 0.5F);
    while (kWays * (tm * (tm + 1) / 2) > i) --tm;
    while (kWays * ((tm + 1) * (tm + 2) / 2) <= i) ++tm;
    r.m0 = tm * G::kTileM;
    r.n0 = (i - kWays * (tm * (tm + 1) / 2)) * G::kBN;
    r.cols = min(G::kBN, p.n - r.n0);
    r.k0 = 0;
    r.klen = p.k;
  } else if constexpr (G::kRagged == Ragged::kN || G::kRagged == Ragged::kM) {
    // Tiles of weights vary fastest: the tiles at work at one time share tokens.
    const int fixed = G::kRagged == Ragged::kN ? p.tiles_m : p.tiles_n;
    const int nt = index / fixed;
    const int at = index - nt * fixed;
    int lo = 0, hi = p.groups;   // the last group whose first tile is <= nt
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (t.first[mid] <= nt) lo = mid;
      else hi = mid;
    }
    r.group = lo;
    r.k0 = 0;
    r.klen = p.k;
    if constexpr (G::kRagged == Ragged::kN) {
      r.m0 = at * G::kTileM;
      r.n0 = t.offset[lo] + (nt - t.first[lo]) * G::kBN;
      r.cols = min(G::kBN, t.offset[lo + 1] - r.n0);
    } else {
      r.m0 = t.offset[lo] + (nt - t.first[lo]) * G::kTileM;
      r.rows = t.offset[lo + 1] - r.m0;
      r.n0 = at * G::kBN;
      r.cols = min(G::kBN, p.m - r.n0);
    }
  } else {
    const int per = p.tiles_m * p.tiles_n;
    r.group = index / per;
    const int i = index - r.group * per;
    const int tn = i / p.tiles_m;
    r.m0 = (i - tn * p.tiles_m) * G::kTileM;
    r.n0 = tn * G::kBN;
    r.cols = min(G::kBN, p.n - r.n0);
    r.k0 = 0;
    r.klen = p.k;
    if constexpr (G::kRagged == Ragged::kK) {
      r.k0 = t.offset[r.group];
      r.klen = max(0, t.offset[r.group + 1] - r.k0);
    }
  }
  return r;
}

// Fills the table (one warp; a barrier of the CTA must follow).
template <class G>
__device__ __forceinline__ void readGroups(const Params &p, GroupTable *t, int lane) {
  if constexpr (G::kRagged == Ragged::kBatch) return;
  const int total = G::kRagged == Ragged::kK ? p.k : p.n;
  constexpr int kTokens = G::kRagged == Ragged::kM ? G::kTileM : G::kBN;   // of a tile
  if (p.offsets == nullptr) {   // one group
    if (lane == 0) {
      t->offset[0] = 0;
      t->offset[1] = total;
      t->first[0] = 0;
      t->first[1] = (total + kTokens - 1) / kTokens;
    }
    return;
  }
  int sum = 0;   // column tiles of the groups so far
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    const int begin = min(max(p.offsets[min(g, p.groups)], 0), total);
    const int end = min(max(p.offsets[min(g + 1, p.groups)], 0), total);
    const int v = (max(0, end - begin) + kTokens - 1) / kTokens;
    int scan = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += o;
    }
    if (g < p.groups) {
      t->offset[g] = begin;
      t->first[g] = sum + scan - v;
    }
    if (g == p.groups - 1) t->offset[p.groups] = end;
    sum += __shfl_sync(0xffffffffu, scan, 31);
  }
  if (lane == 0) t->first[p.groups] = sum;
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

// ---- a chunk's sums from TMEM, added to the registers -----------------------
// In each the next load is in flight while one is added. Columns past the
// tile's width hold what an earlier tile left; they are not written.

// acc[j] += row of kCols columns, a row per lane, times one scale.
template <int kCols>
__device__ __forceinline__ void addScaledRow(uint32_t taddr, float2 (&acc)[kCols / 2], float2 scale) {
  uint32_t v[2][16];
  tmemLoadAsync16(taddr, v[0]);
#pragma unroll
  for (int c = 0; c < kCols; c += 16) {
    uint32_t(&now)[16] = v[c / 16 % 2];
    tmemWait16(now);
    if (c + 16 < kCols) tmemLoadAsync16(taddr + c + 16, v[(c / 16 + 1) % 2]);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      float2 &a = acc[(c + j) / 2];
      a = __ffma2_rn(make_float2(__uint_as_float(now[j]), __uint_as_float(now[j + 1])), scale, a);
    }
  }
}

// The same, each column times its own scale (kScaled) or none.
template <int kCols, bool kScaled>
__device__ __forceinline__ void addRows(uint32_t taddr, float2 (&acc)[kCols / 2],
                                        const float *scales, float weight) {
  uint32_t v[2][16];
  tmemLoadAsync16(taddr, v[0]);
#pragma unroll
  for (int c = 0; c < kCols; c += 16) {
    uint32_t(&now)[16] = v[c / 16 % 2];
    tmemWait16(now);
    if (c + 16 < kCols) tmemLoadAsync16(taddr + c + 16, v[(c / 16 + 1) % 2]);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 x = make_float2(__uint_as_float(now[j]), __uint_as_float(now[j + 1]));
      float2 &a = acc[(c + j) / 2];
      if constexpr (kScaled) {
        const float2 s = *reinterpret_cast<const float2 *>(scales + c + j);
        a = __ffma2_rn(x, make_float2(s.x * weight, s.y * weight), a);
      } else {
        a = __fadd2_rn(a, x);
      }
    }
  }
}

// The same into fragments: acc[4 * i + r] holds columns 8 i + 2 (t % 4) + {0, 1}
// of row 8 r + t / 4 for lane t.
template <int kCols, bool kScaled>
__device__ __forceinline__ void addFragments(uint32_t taddr, float2 (&acc)[kCols / 2],
                                             const float *scales, float weight, int lane) {
  constexpr uint32_t kLower = 16u << 16;   // the quarter's lanes 16-31
  uint32_t v[2][32];                       // rows 0-15 of 32 columns, then rows 16-31
  tmemFragments(taddr, v[0], 0);
  tmemFragments(taddr + kLower, v[0], 16);
#pragma unroll
  for (int c = 0; c < kCols; c += 32) {
    uint32_t(&now)[32] = v[c / 32 % 2];
    uint32_t(&next)[32] = v[(c / 32 + 1) % 2];
    tmemWait32(now);
    if (c + 32 < kCols) {
      tmemFragments(taddr + c + 32, next, 0);
      tmemFragments(taddr + kLower + c + 32, next, 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 scale = make_float2(0.0F, 0.0F);
      if constexpr (kScaled) {
        const float2 s = *reinterpret_cast<const float2 *>(scales + c + i * 8 + lane % 4 * 2);
        scale = make_float2(s.x * weight, s.y * weight);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = r / 2 * 16 + i * 4 + r % 2 * 2;
        const float2 x = make_float2(__uint_as_float(now[at]), __uint_as_float(now[at + 1]));
        float2 &a = acc[(c / 8 + i) * 4 + r];
        if constexpr (kScaled) a = __ffma2_rn(x, scale, a);
        else a = __fadd2_rn(a, x);
      }
    }
  }
}

// ---- from registers to C -----------------------------------------------------

// Where a warp's share of a tile goes: its first element in C, that element's
// row, column and matrix, and how many rows and columns of it exist. Columns
// past the tile's last are another group's (kN) unless `clip` says that C ends
// there.
struct Place {
  size_t at;
  int row, col, matrix, rows, cols;
  bool clip, vector;
};

// 16-bit results (fragments) pass through shared memory, 16 columns at a time in two
// buffers that two warps share: stmatrix transposes each 8 x 8 block, so that a
// column's 64 rows (128 bytes) lie together. TMA takes them from there while
// the next columns are staged (a group's last columns, and a C that TMA cannot
// write, leave by copyOut). Within a tile the buffers take turns, so one store may
// still be reading, the other buffer's; a tile begins with the first buffer,
// whichever the last one ended with, so it waits for both (counting the turns
// over all tiles instead: 30 gradients of 2048 x 2048 of four tokens 79.1 us against
// 77.5 in BF16, 83.4 and 83.6 in FP32). TMA stores about one row of a box per four clocks,
// whatever its length: 64-byte rows of single warps left at 4.7 TB/s. The
// 16-byte pieces of a column are exchanged by the column, as the 128-byte
// swizzle has them, which spreads eight columns over all banks.
__device__ __forceinline__ uint32_t outSlot(int col, int piece) {
  return static_cast<uint32_t>(col * 128 + ((piece ^ (col % 8)) * 16));
}

// Block i of the columns (8 of them), the upper or lower 32 rows, into the
// staging buffer.
__device__ __forceinline__ void stageBlock(unsigned char *out, int block, int lower, int lane,
                                           const uint32_t (&w)[4]) {
  storeMatrixTrans4(smemAddr(out) + outSlot(block * 8 + lane % 8, lower * 4 + lane / 8), w[0], w[1],
                    w[2], w[3]);
}

// Waits, in the thread that issues a warp's stores, until the columns last staged
// in the next buffer have left.
__device__ __forceinline__ void waitStaging(bool tile_begins) {
  if (tile_begins) bulkWaitRead<0>();
  else bulkWaitRead<1>();
}

// A warp's rows of the staged columns (`cols` of them exist) to c: vectors of
// eight rows where the address allows, else a row per lane, eight columns at a
// time (24 gradients of 1000 x 1537 68.8 -> 63.4 us against a rolled loop; 28.7 at
// 1536 by TMA).
__device__ __forceinline__ void copyOut(const unsigned char *out, int lower, uint16_t *c,
                                        long long ldc, int cols, int rows, int lane, bool vector) {
  if (vector && rows >= 32) {
#pragma unroll
    for (int i = 0; i < kOutCols / 8; ++i) {
      const int col = i * 8 + lane / 4;
      if (col < cols)
        *reinterpret_cast<uint4 *>(c + col * ldc + lane % 4 * 8) =
            *reinterpret_cast<const uint4 *>(out + outSlot(col, lower * 4 + lane % 4));
    }
  } else if (lane < rows) {
    c += lane;
#pragma unroll
    for (int col0 = 0; col0 < kOutCols; col0 += 8) {
      uint16_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = *reinterpret_cast<const uint16_t *>(
            out + outSlot(col0 + j, lower * 4 + lane / 8) + lane % 8 * 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (col0 + j < cols) *c = v[j];
        c += ldc;
      }
    }
  }
}

// The two warps that share staging buffers (`pair` 0 to 3).
__device__ __forceinline__ void pairBarrier(int pair) {
  asm volatile("bar.sync %0, 64;" ::"r"(2 + pair) : "memory");
}

__device__ __forceinline__ uint32_t packBf16(float2 v) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// C = alpha * acc in BF16 (beta is 0 here: its reads of C, even unused, would
// double the code that every tile runs through). Both warps of a pair call
// it; one of them may have no rows.
template <int kBlocks>
__device__ __forceinline__ void storeBf16(const Params &p, const Place &to,
                                          const float2 (&acc)[kBlocks * 4], unsigned char *out,
                                          int pair, int lower, int lane) {
  static_assert(kBlocks % 2 == 0, "whole buffers");
  uint16_t *c = static_cast<uint16_t *>(p.c) + to.at;
  const bool issues = lower == 0 && lane == 0;
#pragma unroll
  for (int i0 = 0; i0 < kBlocks; i0 += 2) {
    if (i0 * 8 >= to.cols) break;
    unsigned char *buffer = out + i0 / 2 % 2 * (kOutCols * 128);
    if (issues) waitStaging(i0 == 0);
    pairBarrier(pair);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float2 v = acc[(i0 + i) * 4 + r];
        w[r] = packBf16(make_float2(v.x * p.alpha, v.y * p.alpha));
      }
      stageBlock(buffer, i, lower, lane, w);
    }
    if (p.c_tma && (to.clip || i0 * 8 + kOutCols <= to.cols)) {
      fenceProxyAsyncShared();
      pairBarrier(pair);
      if (issues) tmaStore3d(&p.tma_c, buffer, to.row, to.col + i0 * 8, to.matrix);
    } else {
      __syncwarp();
      copyOut(buffer, lower, c, p.ldc, to.cols - i0 * 8, to.rows, lane, to.vector);
    }
    if (issues) bulkCommit();
    c += static_cast<long long>(kOutCols) * p.ldc;
  }
}

// C = alpha * acc + beta * C from rows (kFp32): FP32, or BF16 with beta, whose
// columns' rows are read and written 32 at a time. Each column is read after the
// one before is written, so a warp's columns take a memory latency each: weight
// gradients of 16384 tokens, 16 x 2048 x 4096 in FP32, 249 us without beta and
// 1780 with it, of 3001 tokens, 24 x 1000 x 1537, 60 and 575.
template <typename T>
__device__ __forceinline__ void updateColumns(const Params &p, T *c, int cols, const float *sums,
                                              int lane) {
#pragma unroll 4
  for (int j = 0; j < cols; ++j) {
    float v = p.alpha * sums[j * 32 + lane];
    if (p.beta != 0.0F) v = fmaf(p.beta, static_cast<float>(*c), v);
    *c = static_cast<T>(v);
    c += p.ldc;
  }
}

// A kFp32 warp's share: acc holds one row's columns, in pairs. FP32 without
// beta leaves 16 columns at a time, by TMA from two buffers (a column's 32 rows
// are 128 bytes there) or, where TMA cannot write them, a column per store.
// The rest passes through a loop that is not unrolled over the columns.
template <int kCols>
__device__ __forceinline__ void storeFp32(const Params &p, const Place &to,
                                          const float2 (&acc)[kCols / 2], unsigned char *out,
                                          int lane) {
  auto sum = [&](int j) { return j % 2 ? acc[j / 2].y : acc[j / 2].x; };
  float *buffers = reinterpret_cast<float *>(out);
  if (p.beta == 0.0F && !p.c_bf16) {
    float *c = static_cast<float *>(p.c) + to.at + lane;
#pragma unroll
    for (int j0 = 0; j0 < kCols; j0 += kOutCols) {
      if (j0 >= to.cols) break;
      float *buffer = buffers + j0 / kOutCols % 2 * (kOutCols * 32);
      if (p.c_tma) {
        if (lane == 0) waitStaging(j0 == 0);
        __syncwarp();
      }
      if (p.c_tma && (to.clip || j0 + kOutCols <= to.cols)) {
#pragma unroll
        for (int j = 0; j < kOutCols; ++j) buffer[j * 32 + lane] = p.alpha * sum(j0 + j);
        fenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) tmaStore3d(&p.tma_c, buffer, to.row, to.col + j0, to.matrix);
      } else if (lane < to.rows) {
#pragma unroll
        for (int j = 0; j < kOutCols; ++j)
          if (j0 + j < to.cols) c[static_cast<long long>(j) * p.ldc] = p.alpha * sum(j0 + j);
      }
      if (p.c_tma && lane == 0) bulkCommit();
      c += static_cast<long long>(kOutCols) * p.ldc;
    }
    return;
  }
#pragma unroll 1
  for (int j0 = 0; j0 < min(to.cols, kCols); j0 += kOutCols) {
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kCols; k += kOutCols) {
      if (k != j0) continue;
#pragma unroll
      for (int j = 0; j < kOutCols; ++j) buffers[j * 32 + lane] = sum(k + j);
    }
    if (lane < to.rows) {
      const size_t at = to.at + static_cast<size_t>(j0) * p.ldc + lane;
      const int cols = min(to.cols - j0, kOutCols);
      if (p.c_bf16) updateColumns(p, static_cast<__nv_bfloat16 *>(p.c) + at, cols, buffers, lane);
      else updateColumns(p, static_cast<float *>(p.c) + at, cols, buffers, lane);
    }
  }
  __syncwarp();
}

// A pair product's result (PairOut) leaves kPairCols columns at a time: FP32
// sums to shared memory, then flushPair, in a loop that is not unrolled over
// the warp's columns (unrolled, it ran from a cold instruction cache: 11 to
// 14 us of a 2048 x 2048 symmetric product's 45).

// Word of (column, row) in a warp's staging block: groups of four rows are
// rotated by the column, so that a row's columns, a column's rows and the
// eight-row vectors of eight columns all spread over the banks.
__device__ __forceinline__ int pairSlot(int col, int row) {
  return col * 32 + ((row / 4 + col + col / 8) % 8) * 4 + row % 4;
}

// A's hi and lo at the places that a lane of flushPair writes, for the polynomial.
struct PairColumns {
  uint4 v[kPairCols / 8][2];
};
__device__ __forceinline__ void readPair(const Params &p, size_t matrix, int row0, int col0,
                                         int cols, int lane, PairColumns *prev) {
#pragma unroll
  for (int pass = 0; pass < kPairCols / 8; ++pass) {
    const int col = pass * 8 + lane / 4, row = lane % 4 * 8;
    const size_t at = matrix + static_cast<size_t>(col0 + col) * p.ldc + row0 + row;
    prev->v[pass][0] = prev->v[pass][1] = make_uint4(0, 0, 0, 0);
    if (col < cols && row < p.m - row0) {
      prev->v[pass][0] = *reinterpret_cast<const uint4 *>(p.pair.prev_hi + at);
      prev->v[pass][1] = *reinterpret_cast<const uint4 *>(p.pair.prev_lo + at);
    }
  }
}

// Writes the staged columns (`cols` of them exist) at row0, col0 of the
// matrix: hi and lo of each value in vectors of eight rows, and (mirror) of
// eight columns across the diagonal. The polynomial reads A the same way. Rows
// of the pair matrices are padded to 64 elements, so vectors may reach past
// the last row or column into padding that nothing reads.
__device__ __forceinline__ void flushPair(const Params &p, size_t matrix, bool mirror, int row0,
                                          int col0, int cols, const PairColumns &prev,
                                          uint32_t *out, int lane, bool vector) {
  const int rows = p.m - row0;
  __syncwarp();
#pragma unroll
  for (int pass = 0; pass < kPairCols / 8; ++pass) {
    const int col = pass * 8 + lane / 4, row = lane % 4 * 8;
    const bool live = col < cols && row < rows;
    uint4 *slot[2] = {reinterpret_cast<uint4 *>(out + pairSlot(col, row)),
                      reinterpret_cast<uint4 *>(out + pairSlot(col, row + 4))};
    const size_t at = matrix + static_cast<size_t>(col0 + col) * p.ldc + row0 + row;
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 w = *slot[h];
      v[4 * h] = __uint_as_float(w.x);
      v[4 * h + 1] = __uint_as_float(w.y);
      v[4 * h + 2] = __uint_as_float(w.z);
      v[4 * h + 3] = __uint_as_float(w.w);
    }
    if (p.pair.out == PairOut::kFinal) {
      __nv_bfloat16 *c = static_cast<__nv_bfloat16 *>(p.c) + at;
      alignas(16) __nv_bfloat16 r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = __float2bfloat16(v[j] * p.alpha);
      if (live && vector && row + 8 <= rows) {
        *reinterpret_cast<uint4 *>(c) = *reinterpret_cast<const uint4 *>(r);
      } else if (live) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (row + j < rows) c[j] = r[j];
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= 1.0F / kPairScale;
    if (p.pair.out == PairOut::kPoly) {
      const __half *ph = reinterpret_cast<const __half *>(&prev.v[pass][0]);
      const __half *pl = reinterpret_cast<const __half *>(&prev.v[pass][1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = fmaf(p.pair.c1, __half2float(ph[j]) + __half2float(pl[j]), v[j] * p.pair.c2);
        if (row0 + row + j == col0 + col) v[j] = fmaf(p.pair.c0, kPairScale, v[j]);
      }
    }
    alignas(16) __half hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) splitPair(v[j], &hi[j], &lo[j]);
    const uint4 h = *reinterpret_cast<const uint4 *>(hi), l = *reinterpret_cast<const uint4 *>(lo);
    if (live) {
      *reinterpret_cast<uint4 *>(p.pair.hi + at) = h;
      *reinterpret_cast<uint4 *>(p.pair.lo + at) = l;
    }
    if (mirror) {   // the pairs take the sums' places
      *slot[0] = make_uint4(__byte_perm(h.x, l.x, 0x5410), __byte_perm(h.x, l.x, 0x7632),
                            __byte_perm(h.y, l.y, 0x5410), __byte_perm(h.y, l.y, 0x7632));
      *slot[1] = make_uint4(__byte_perm(h.z, l.z, 0x5410), __byte_perm(h.z, l.z, 0x7632),
                            __byte_perm(h.w, l.w, 0x5410), __byte_perm(h.w, l.w, 0x7632));
    }
  }
  __syncwarp();
  if (!mirror) return;
#pragma unroll
  for (int pass = 0; pass < kPairCols / 8; ++pass) {
    const int row = pass * 16 + lane / 2, col = lane % 2 * 8;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = out[pairSlot(col + j, row)];
    if (row >= rows || col >= cols) continue;
    const size_t at = matrix + static_cast<size_t>(row0 + row) * p.ldc + col0 + col;
    *reinterpret_cast<uint4 *>(p.pair.hi + at) =
        make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410),
                   __byte_perm(w[4], w[5], 0x5410), __byte_perm(w[6], w[7], 0x5410));
    *reinterpret_cast<uint4 *>(p.pair.lo + at) =
        make_uint4(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632),
                   __byte_perm(w[4], w[5], 0x7632), __byte_perm(w[6], w[7], 0x7632));
  }
  __syncwarp();
}

// Four scales, of which `live` exist (zeros for the others).
__device__ __forceinline__ float4 loadScales(const float *s, int live, bool aligned) {
  if (aligned && live >= 4) return __ldg(reinterpret_cast<const float4 *>(s));
  return make_float4(__ldg(s), live > 1 ? __ldg(s + 1) : 0.0F, live > 2 ? __ldg(s + 2) : 0.0F,
                     live > 3 ? __ldg(s + 3) : 0.0F);
}

// A warp's 32 tokens (`live` of them in the group) by kCols features from
// `feature0` (`cols` of them exist), a token per thread, through shared
// memory. A whole tile of BF16 leaves by TMA (which cuts it at C's last
// feature); one that ends a group, or another C, row by row.
template <int kCols>
__device__ __forceinline__ void storeTokens(const Params &p, int token0, int live, int feature0,
                                            int cols, const float2 (&acc)[kCols / 2],
                                            unsigned char *out, int lane) {
  if (lane == 0) bulkWaitRead<0>();   // the tile before has left
  __syncwarp();
  const size_t at = static_cast<size_t>(token0) * p.ldc + feature0;
  if (p.c_bf16) {
#pragma unroll
    for (int j = 0; j < kCols / 8; ++j) {
      // Eight features, in the box of 64 that holds them: 128-byte rows, 16-byte
      // pieces exchanged by the row as the map's swizzle has them.
      uint4 w;
      w.x = packBf16(acc[4 * j]);
      w.y = packBf16(acc[4 * j + 1]);
      w.z = packBf16(acc[4 * j + 2]);
      w.w = packBf16(acc[4 * j + 3]);
      *reinterpret_cast<uint4 *>(out + j / 8 * 4096 + lane * 128 + ((j % 8) ^ (lane % 8)) * 16) = w;
    }
    if (p.c_tma && live >= 32) {
      fenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int j = 0; j < kCols / 64; ++j)
          if (j * 64 < cols) tmaStore3d(&p.tma_c, out + j * 4096, feature0 + j * 64, token0, 0);
        bulkCommit();
      }
      return;
    }
    __syncwarp();
    __nv_bfloat16 *c = static_cast<__nv_bfloat16 *>(p.c) + at;
    const int f = 2 * lane;   // two features of each box
#pragma unroll 2
    for (int r = 0; r < min(live, 32); ++r) {
      const bool pairs = reinterpret_cast<uintptr_t>(c) % 4 == 0;
#pragma unroll
      for (int j = 0; j < kCols / 64; ++j) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(
            out + j * 4096 + r * 128 + ((lane / 4) ^ (r % 8)) * 16 + lane % 4 * 4);
        const int first = j * 64 + f;
        if (pairs && first + 1 < cols) {
          *reinterpret_cast<uint32_t *>(c + first) = w;
        } else {
          const auto *h = reinterpret_cast<const __nv_bfloat16 *>(&w);
          if (first < cols) c[first] = h[0];
          if (first + 1 < cols) c[first + 1] = h[1];
        }
      }
      c += p.ldc;
    }
    __syncwarp();
    return;
  }
  // FP32: 64 features at a time, 256-byte rows with their pieces exchanged by the row.
#pragma unroll
  for (int f0 = 0; f0 < kCols; f0 += 64) {
    if (f0 >= cols) break;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      *reinterpret_cast<float4 *>(out + lane * 256 + (j ^ (lane % 16)) * 16) =
          make_float4(acc[f0 / 2 + 2 * j].x, acc[f0 / 2 + 2 * j].y, acc[f0 / 2 + 2 * j + 1].x,
                      acc[f0 / 2 + 2 * j + 1].y);
    __syncwarp();
    float *c = static_cast<float *>(p.c) + at + f0 + lane;
#pragma unroll 2
    for (int r = 0; r < min(live, 32); ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (f0 + h * 32 + lane < cols)
          c[h * 32] = *reinterpret_cast<const float *>(
              out + r * 256 + ((lane / 4 + h * 8) ^ (r % 16)) * 16 + lane % 4 * 4);
      c += p.ldc;
    }
    __syncwarp();
  }
}

// The MMA of either form, and its completion signal to this CTA or both.
template <class G>
__device__ __forceinline__ void issueMma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                         bool accumulate) {
  if constexpr (G::kTwo) mmaNarrowPair<G::kBytes>(d_tmem, a, b, idesc, accumulate);
  else mmaNarrow<G::kBytes>(d_tmem, a, b, idesc, accumulate);
}
template <class G>
__device__ __forceinline__ void commitMma(uint64_t *bar) {
  if constexpr (G::kTwo) mmaCommitBoth(bar);
  else mmaCommit(bar);
}
// A box of operand `map` into this CTA's shared memory, counted on `bar` of
// this CTA, or (kShared, a pair) of the even CTA.
template <class G, bool kShared>
__device__ __forceinline__ void loadBox(unsigned char *dst, const CUtensorMap *map, uint64_t *bar,
                                        int x, int y, int z) {
  if constexpr (kShared) tmaLoad3dPair(dst, map, clusterAddr(smemAddr(bar), 0), x, y, z);
  else tmaLoad3d(dst, map, bar, x, y, z);
}
template <class G, bool kShared>
__device__ __forceinline__ void loadStage(const Params &p, unsigned char *stage, uint64_t *bar,
                                          int m0, int n0, int k0, int za, int zb) {
#pragma unroll
  for (int plane = 0; plane < G::kPlanes; ++plane) {
    if (G::kPlanes == 2 && plane == p.pair.planes) break;
    unsigned char *sa = stage + plane * G::kABytes;
    unsigned char *sb = stage + G::kPlanes * G::kABytes + plane * G::kBBytes;
    const CUtensorMap *map_a = plane == 0 ? &p.tma_a : &p.pair.tma_a_lo;
    const CUtensorMap *map_b = plane == 0 ? &p.tma_b : &p.pair.tma_b_lo;
    if constexpr (G::kAMN) {
      for (int j = 0; j < kBM / 64; ++j)
        loadBox<G, kShared>(sa + j * 64 * kRowBytes, map_a, bar, m0 + 64 * j, k0, za);
    } else {
      loadBox<G, kShared>(sa, map_a, bar, k0, m0, za);
    }
    if constexpr (G::kBMN) {
      for (int j = 0; j < G::kBRows / 64; ++j)
        loadBox<G, kShared>(sb + j * 64 * kRowBytes, map_b, bar, n0 + 64 * j, k0, zb);
    } else {
      loadBox<G, kShared>(sb, map_b, bar, k0, n0, zb);
    }
  }
}

// mbarriers (all waits bounded; in a pair the even CTA's, except where noted):
//   full[s]       stage s loaded: TMA bytes of both CTAs
//   empty[s]      the MMAs reading stage s completed (each CTA its own)
//   acc_full[b]   accumulator b holds a chunk (each CTA its own)
//   acc_empty[b]  every epilogue warp has read accumulator b
//   tail[s]       a pair's odd CTA has cut off the last slice of a group, in stage s
// A wait that gives up (after seconds: what was on its way before it has arrived)
// makes its role go on without waiting, but the producer copy nothing more.
// Otherwise the producer stays until its last copies have landed and been read, so
// no CTA ends, and frees its TMEM, with a copy or an MMA of its own on the way.
// A slice that ends a group ragged along k holds rows of the next group. The
// issuer's warp zeroes them in both operands (zero times a NaN is a NaN) up to
// the next multiple of 16, and multiplies no further. In a pair the odd CTA
// does the same for its half: such a slice is counted on its own full[s], and
// tail[s] tells the even CTA.
template <class G>
__global__ void __launch_bounds__(kThreads, 1) productKernel(const __grid_constant__ Params p) {
  constexpr int kBN = G::kBN;
  constexpr int kStages = G::kStages;
  constexpr int kStageBytes = G::kStageBytes;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ GroupTable table;
  unsigned char *smem = smem_raw + ((1024 - (smemAddr(smem_raw) & 1023)) & 1023);
  float *scales = reinterpret_cast<float *>(smem + kStages * kStageBytes + G::kOutBytes);
  unsigned char *out_smem = smem + kStages * kStageBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(out_smem + G::kOutBytes + G::kScaleBytes);
  uint64_t *empty = full + kStages;
  uint64_t *acc_full = empty + kStages;
  uint64_t *acc_empty = acc_full + kAccums;
  uint64_t *tail = acc_empty + kAccums;

  const int warp = uniformWarp(), lane = threadIdx.x % 32;
  // A worker is a CTA, or a pair: its position among them, and this CTA's in it.
  const int rank = G::kTwo ? static_cast<int>(blockIdx.x & 1) : 0;
  const int worker = G::kTwo ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int workers = G::kTwo ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  if (threadIdx.x == 0) {
    if (p.k > 0) {
      prefetchTensorMap(&p.tma_a);
      prefetchTensorMap(&p.tma_b);
      if constexpr (G::kPlanes == 2) {
        prefetchTensorMap(&p.pair.tma_a_lo);
        prefetchTensorMap(&p.pair.tma_b_lo);
      }
    }
    if (p.c_tma) prefetchTensorMap(&p.tma_c);
    for (int s = 0; s < kStages; ++s) {
      mbarInit(&full[s], 1);
      mbarInit(&empty[s], 1);
      mbarInit(&tail[s], 1);
    }
    for (int b = 0; b < kAccums; ++b) {
      mbarInit(&acc_full[b], 1);
      mbarInit(&acc_empty[b], (G::kTwo ? 2 : 1) * kEpilogueWarps);
    }
    fenceBarrierInit();
  }
  if (warp == 2) {
    if constexpr (G::kTwo) {
      tmemAllocPair(&tmem_base_slot, G::kTmemColumns);
      tmemRelinquishPair();
    } else {
      tmemAlloc(&tmem_base_slot, G::kTmemColumns);
      tmemRelinquish();
    }
  }
  tcgenFenceBefore();
  __syncthreads();
  if constexpr (G::kTwo) clusterSync();   // both CTAs' barriers and TMEM exist
  tcgenFenceAfter();
  allowDependentLaunch();
  gridDependencyWait();
  if constexpr (G::kRagged != Ragged::kBatch) {
    if (warp == 0) readGroups<G>(p, &table, lane);
    __syncthreads();
  }
  const uint32_t tmem_base = tmem_base_slot;
  const int tiles = tileCount<G>(p, table);

  bool ok = true;
  auto wait = [&](uint64_t *bar, int parity) {
    if (ok) ok = mbarWait(bar, static_cast<uint32_t>(parity), p.err);
  };
  // The instruction's N for a tile's valid columns.
  auto widthOf = [](int cols) { return (cols + G::kNStep - 1) / G::kNStep * G::kNStep; };

  if (warp < kEpilogueWarp0) {
    regDealloc<72>();
    if (warp == 0 && electOne()) {
      // ---------------- TMA producer ----------------
      int s = 0, parity = 1;   // the first pass over the ring waits for nothing
      for (int i = worker; i < tiles; i += workers) {
        const Tile t = tileAt<G>(p, table, i);
        const int za = G::kRagged == Ragged::kN || G::kRagged == Ragged::kBatch ? t.group : 0;
        const int zb = G::kRagged == Ragged::kM || G::kRagged == Ragged::kBatch ? t.group : 0;
        const int m0 = t.m0 + rank * kBM;
        const int n0 = t.n0 + (G::kTwo ? rank * (widthOf(t.cols) / 2) : 0);
        for (int kk = 0; kk < t.klen; kk += G::kBK) {
          wait(&empty[s], parity);
          if (!ok) continue;
          unsigned char *stage = smem + s * kStageBytes;
          const bool cut = G::kRagged == Ragged::kK && t.klen - kk < G::kBK;
          const uint32_t bytes =
              G::kPlanes == 2 && p.pair.planes == 1 ? kStageBytes / 2 : kStageBytes;
          if (!G::kTwo || cut) {
            mbarArriveExpectTx(&full[s], bytes);
            loadStage<G, false>(p, stage, &full[s], m0, n0, t.k0 + kk, za, zb);
          } else {
            if (rank == 0) mbarArriveExpectTx(&full[s], 2 * bytes);
            loadStage<G, G::kTwo>(p, stage, &full[s], m0, n0, t.k0 + kk, za, zb);
          }
          if (++s == kStages) {
            s = 0;
            parity ^= 1;
          }
        }
      }
      // In a pair the even CTA counts both CTAs' copies, and its signals to the odd
      // one have landed, too. (Small code: unrolled, it took 0.1 us of each launch of
      // a small Newton-Schulz iteration; 8 x 256 x 512 89.0 -> 89.6 us with it.)
#pragma unroll 1
      for (int j = 0; j < kStages; ++j) {
        if (rank == 0) wait(&full[s], parity);
        wait(&empty[s], parity);
        if (++s == kStages) {
          s = 0;
          parity ^= 1;
        }
      }
    } else if (warp == 1 && rank == 0) {
      // ---------------- MMA issuer ----------------
      const bool leader = electOne();
      int s = 0, parity = 0;
      int b = 0, acc_parity = 1;
      unsigned tails = 0;   // bit s: parity of the next cut slice in stage s
      const uint64_t desc_a = smemDesc<G::kAMN>(smemAddr(smem));
      const uint64_t desc_b = smemDesc<G::kBMN>(smemAddr(smem) + G::kPlanes * G::kABytes);
      for (int i = worker; i < tiles; i += workers) {
        const Tile t = tileAt<G>(p, table, i);
        const uint32_t idesc = instrDesc<G>(p.format, widthOf(t.cols));
        const uint32_t idesc_hi =
            G::kJoined && p.pair.planes == 2 ? instrDesc<G>(p.format, 2 * kBN) : idesc;
        const int iters = (t.klen + G::kBK - 1) / G::kBK;
        int in_chunk = 0;
        for (int kb = 0; kb < iters; ++kb) {
          const bool first = in_chunk == 0;
          const bool last = ++in_chunk == p.chunk_iters || kb == iters - 1;
          if (last) in_chunk = 0;
          if (first) wait(&acc_empty[b], acc_parity);
          wait(&full[s], parity);
          int steps = G::kBK / G::kMmaK;
          if constexpr (G::kRagged == Ragged::kK) {
            const int rows = t.klen - kb * G::kBK;
            if (rows < G::kBK) {
              unsigned char *stage = smem + s * kStageBytes;
              steps = (rows + G::kMmaK - 1) / G::kMmaK;
              zeroRows<kBM / 64>(stage, rows, steps * G::kMmaK, lane);
              zeroRows<G::kBRows / 64>(stage + G::kABytes, rows, steps * G::kMmaK, lane);
              fenceProxyAsyncShared();
              __syncwarp();
              if constexpr (G::kTwo) {
                if (ok) ok = mbarWaitCluster(&tail[s], (tails >> s) & 1, p.err);
                tails ^= 1u << s;
              }
            }
          }
          if (leader) {
            tcgenFenceAfter();
            const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(b * G::kAccColumns);
            // Descriptors count 16 bytes. K-major: the next instruction's k
            // are 32 bytes further along each row; MN-major: 16 rows of 128
            // bytes further.
            constexpr uint64_t kNextA = (G::kAMN ? 16 * kRowBytes : 32) / 16;
            constexpr uint64_t kNextB = (G::kBMN ? 16 * kRowBytes : 32) / 16;
            uint64_t ad = desc_a + static_cast<uint64_t>(s) * (kStageBytes / 16);
            uint64_t bd = desc_b + static_cast<uint64_t>(s) * (kStageBytes / 16);
#pragma unroll
            for (int j = 0; j < G::kBK / G::kMmaK; ++j) {
              if (j < steps) {
                issueMma<G>(d_tmem, ad, bd, idesc_hi, !first || j > 0);
                if (G::kPlanes == 2 && p.pair.planes == 2) {
                  if constexpr (!G::kJoined)
                    issueMma<G>(d_tmem, ad, bd + G::kBBytes / 16, idesc, true);
                  issueMma<G>(d_tmem, ad + G::kABytes / 16, bd, idesc, true);
                }
              }
              ad += kNextA;
              bd += kNextB;
            }
            commitMma<G>(&empty[s]);
            if (last) commitMma<G>(&acc_full[b]);
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
    } else if (warp == 1 && G::kRagged == Ragged::kK) {
      // ---------------- the odd CTA's cut slices ----------------
      int s = 0;
      unsigned seen = 0;   // bit s: parity of the next cut slice in stage s
      for (int i = worker; i < tiles; i += workers) {
        const Tile t = tileAt<G>(p, table, i);
        const int iters = (t.klen + G::kBK - 1) / G::kBK;
        if (iters == 0) continue;
        const int at = (s + iters - 1) % kStages;
        s = (s + iters) % kStages;
        const int rows = t.klen - (iters - 1) * G::kBK;
        if (rows == G::kBK) continue;
        wait(&full[at], (seen >> at) & 1);
        seen ^= 1u << at;
        unsigned char *stage = smem + at * kStageBytes;
        const int end = (rows + G::kMmaK - 1) / G::kMmaK * G::kMmaK;
        zeroRows<kBM / 64>(stage, rows, end, lane);
        zeroRows<G::kBRows / 64>(stage + G::kABytes, rows, end, lane);
        fenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) mbarArriveCluster(clusterAddr(smemAddr(&tail[at]), 0));
      }
    }
  } else {
    // ---------------- epilogue ----------------
    regAlloc<216>();
    constexpr int kHalf = kBN / 2;                     // columns of this warp
    constexpr int kBlocks = kHalf / 8;
    const int quarter = warp % 4;
    const int col_begin = (warp - kEpilogueWarp0) / 4 * kHalf;
    const int etid = threadIdx.x - 32 * kEpilogueWarp0;
    // Warps that hold neighbouring rows of the same columns share staging.
    const int lower = quarter % 2, pair = (warp - kEpilogueWarp0) / 2;
    unsigned char *out = out_smem + (warp - kEpilogueWarp0) * G::kOutWarp;
    // Vectors of eight 16-bit rows: columns aligned to 16 bytes.
    const bool vector = reinterpret_cast<uintptr_t>(p.c) % 16 == 0 && p.ldc % 8 == 0 &&
                        p.stride_c % 8 == 0;
    int b = 0, acc_parity = 0;
    // Scales of kScaleBatch blocks (zeros where there are none), copied into
    // one of two buffers while the other is in use.
    int batches = 0;
    auto fetchScales = [&](const Tile &t, int ch) {
      float *dst = scales + (batches & 1) * kScaleBatch * G::kScalePitch;
      const int live = (t.klen + G::kBK - 1) / G::kBK - ch;
      const int c = etid % kBN;
      const bool in = c < t.cols;
      const float *sb = p.scale_b + static_cast<size_t>(in ? t.n0 + c : 0) * p.ldsb + ch;
      for (int q = etid / kBN; q < kScaleBatch; q += kEpilogueThreads / kBN) {
        const bool there = in && q < live;
        cpAsync4(dst + q * G::kScalePitch + c, there ? sb + q : p.scale_b, there ? 4 : 0);
      }
      if (etid < kScaleBatch) {
        const float *sa = p.scale_a + t.group * p.stride_sa +
                          static_cast<size_t>(t.m0 / 128) * p.ldsa + ch + etid;
        const bool there = etid < live;
        cpAsync4(dst + etid * G::kScalePitch + kBN, there ? sa : p.scale_a, there ? 4 : 0);
      }
      cpAsyncCommit();
      ++batches;
    };
    // The scales of block ch of tile i, the tile of this call's loop.
    auto scalesOf = [&](const Tile &t, int i, int ch, int chunks) {
      if (ch % kScaleBatch == 0) {
        cpAsyncWait<0>();
        namedBarrier<1, kEpilogueThreads>();   // here for all; the other buffer is free
        if (ch + kScaleBatch < chunks) fetchScales(t, ch + kScaleBatch);
        else if (i + workers < tiles) fetchScales(tileAt<G>(p, table, i + workers), 0);
        else ++batches;
      }
      return scales + ((batches & 1) * kScaleBatch + ch % kScaleBatch) * G::kScalePitch;
    };
    if constexpr (G::kStaged) {
      if (worker < tiles) fetchScales(tileAt<G>(p, table, worker), 0);
    }
    if constexpr (G::kRows) {
      // A row of the tile, one token, per thread. Its scales, four blocks at
      // a time: those at work, and the next ones on their way.
      const int row = quarter * 32 + lane;
      const uint32_t acc_empty_even = clusterAddr(smemAddr(acc_empty), 0);
      const bool aligned = reinterpret_cast<uintptr_t>(p.scale_a) % 16 == 0 &&
                           reinterpret_cast<uintptr_t>(p.scale_b) % 16 == 0 && p.ldsa % 4 == 0 &&
                           p.ldsb % 4 == 0 && p.stride_sa % 4 == 0;
      // Where a tile's scales begin; NULL for a thread without a token.
      const float *sb_at = nullptr, *sa_at = nullptr;
      auto locate = [&](const Tile &t) {
        const int block = (t.n0 + col_begin) / 128;
        const bool in = rank * kBM + row < t.rows && block * 128 < p.m;
        sb_at = in ? p.scale_b + static_cast<size_t>(t.m0 + rank * kBM + row) * p.ldsb : nullptr;
        sa_at = p.scale_a + t.group * p.stride_sa + static_cast<size_t>(block) * p.ldsa;
      };
      float4 sb = make_float4(0.0F, 0.0F, 0.0F, 0.0F), sa = sb;
      auto fetch = [&](int ch, int live) {
        if (sb_at != nullptr && live > 0) {
          sb = loadScales(sb_at + ch, live, aligned);
          sa = loadScales(sa_at + ch, live, aligned);
        }
      };
      const int chunks = (p.k + G::kBK - 1) / G::kBK;
      if (worker < tiles) {
        locate(tileAt<G>(p, table, worker));
        fetch(0, chunks);
      }
      for (int i = worker; i < tiles; i += workers) {
        const Tile t = tileAt<G>(p, table, i);
        float2 acc[kHalf / 2];
#pragma unroll
        for (int j = 0; j < kHalf / 2; ++j) acc[j] = make_float2(0.0F, 0.0F);
#pragma unroll 1
        for (int ch = 0; ch < chunks; ch += 4) {
          const float scale[4] = {sb.x * sa.x, sb.y * sa.y, sb.z * sa.z, sb.w * sa.w};
          if (ch + 4 < chunks) {
            fetch(ch + 4, chunks - ch - 4);
          } else if (i + workers < tiles) {
            locate(tileAt<G>(p, table, i + workers));
            fetch(0, chunks);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (ch + q >= chunks) break;
            const float2 s = make_float2(scale[q], scale[q]);
            wait(&acc_full[b], acc_parity);
            tcgenFenceAfter();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                                   static_cast<uint32_t>(b * kBN + col_begin);
            addScaledRow<kHalf>(taddr, acc, s);
            tcgenFenceBefore();
            __syncwarp();
            if (lane == 0) mbarArriveClusterRelaxed(acc_empty_even + b * 8);
            b ^= 1;
            if (b == 0) acc_parity ^= 1;
          }
        }
        const int token0 = t.m0 + rank * kBM + quarter * 32;
        const int live = t.rows - rank * kBM - quarter * 32;
        const int cols = t.cols - col_begin;
        if (live > 0 && cols > 0)
          storeTokens<kHalf>(p, token0, live, t.n0 + col_begin, cols, acc, out, lane);
      }
    } else
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      const int m0 = t.m0 + rank * kBM;
      const int iters = (t.klen + G::kBK - 1) / G::kBK;
      const int chunks = iters > 0 ? (iters - 1) / p.chunk_iters + 1 : 0;
      // The polynomial's A, while the products are made (wider tiles have no
      // registers for it): 16 x 100 x 200 65 -> 63 us, 512 x 512 90 -> 88.
      constexpr bool kEarly = G::kPlanes == 2 && kHalf == kPairCols;
      [[maybe_unused]] PairColumns prev;
      if constexpr (kEarly) {
        if (p.pair.out == PairOut::kPoly)
          readPair(p, static_cast<size_t>(t.group * p.stride_c), m0 + quarter * 32,
                   t.n0 + col_begin, t.cols - col_begin, lane, &prev);
      }
      float2 acc[kBlocks * 4];
#pragma unroll
      for (int j = 0; j < kBlocks * 4; ++j) acc[j] = make_float2(0.0F, 0.0F);
      for (int ch = 0; ch < chunks; ++ch) {
        const float *sc = nullptr;
        if constexpr (G::kBytes) sc = scalesOf(t, i, ch, chunks);
        wait(&acc_full[b], acc_parity);
        tcgenFenceAfter();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                               static_cast<uint32_t>(b * G::kAccColumns + col_begin);
        float weight = 0.0F;
        if constexpr (G::kStaged) {
          weight = sc[kBN];
          sc += col_begin;
        }
        if constexpr (G::kJoined) {
          if (p.pair.planes == 2) addRows<kHalf, false>(taddr + kBN, acc, nullptr, 0.0F);
        }
        if constexpr (G::kFp32) addRows<kHalf, G::kStaged>(taddr, acc, sc, weight);
        else addFragments<kHalf, G::kStaged>(taddr, acc, sc, weight, lane);
        tcgenFenceBefore();
        __syncwarp();
        if (lane == 0) {
          if constexpr (G::kTwo) mbarArriveClusterRelaxed(clusterAddr(smemAddr(&acc_empty[b]), 0));
          else mbarArrive(&acc_empty[b]);
        }
        b ^= 1;
        if (b == 0) acc_parity ^= 1;
      }
      const size_t matrix =
          G::kRagged == Ragged::kN ? 0 : static_cast<size_t>(t.group * p.stride_c);
      const int row0 = m0 + quarter * 32;
      const int col0 = t.n0 + col_begin, cols = t.cols - col_begin;
      constexpr bool kShared = G::kPlanes == 1 && !G::kFp32;
      if (row0 - (kShared ? lower * 32 : 0) < p.m && cols > 0) {
        if constexpr (G::kPlanes == 2) {
          uint32_t *words = reinterpret_cast<uint32_t *>(out);
          const bool mirror = G::kSymmetric && t.n0 + kBN <= t.m0;
#pragma unroll 1
          for (int c = 0; c < min(cols, kHalf); c += kPairCols) {
#pragma unroll
            for (int k = 0; k < kHalf; k += kPairCols) {
              if (k != c) continue;
#pragma unroll
              for (int j = 0; j < kPairCols; ++j)
                words[pairSlot(j, lane)] =
                    __float_as_uint(j % 2 ? acc[(k + j) / 2].y : acc[(k + j) / 2].x);
            }
            if constexpr (!kEarly) {
              if (p.pair.out == PairOut::kPoly)
                readPair(p, matrix, row0, col0 + c, cols - c, lane, &prev);
            }
            flushPair(p, matrix, mirror, row0, col0 + c, cols - c, prev, words, lane, vector);
          }
        } else {
          Place to;
          to.at = matrix + static_cast<size_t>(col0) * p.ldc + row0;
          to.row = row0;
          to.col = col0;
          to.matrix = G::kRagged == Ragged::kN ? 0 : t.group;
          to.rows = p.m - row0;
          to.cols = cols;
          to.clip = G::kRagged != Ragged::kN;
          to.vector = vector;
          if constexpr (G::kFp32) storeFp32<kHalf>(p, to, acc, out, lane);
          else storeBf16<kBlocks>(p, to, acc, out - lower * G::kOutWarp, pair, lower, lane);
        }
      }
    }
    if (lane == 0) bulkWait();   // every store has been made
  }

  tcgenFenceBefore();
  __syncthreads();
  if constexpr (G::kTwo) clusterSync();   // neither CTA leaves while the pair still works
  if (warp == 2) {
    tcgenFenceAfter();
    if constexpr (G::kTwo) tmemDeallocPair(tmem_base, G::kTmemColumns);
    else tmemDealloc(tmem_base, G::kTmemColumns);
  }
}

}  // namespace sgblas::kern::prod

#endif  // SGBLAS_B200_PRODUCT_TILE_CUH_
