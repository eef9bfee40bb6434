// Products of 4-bit operands (e2m1 values, a power of two for each 32 of k, as
// the OCP microscaling format MXFP4 has them): C = A^T B per group, FP32 sums.
//
// The tiles, roles and ragged groups are those of product_tile.cuh (many tokens)
// and product_thin.cuh (few); operands are rows of bytes, two values each, and a
// k slice of 128 bytes is 256 of k. What differs is the scales: the tensor core
// applies them itself (kind::mxf4), from tensor memory, where each instruction (64
// of k) takes two for every row of A and of B.
//
// Scales' way. In global memory they lie as bytes, contiguous along k, a row per
// column of A or B; tcgen05.cp takes them to TMEM in 512-byte blocks: 32 rows (lanes)
// of four words, word i the four scales of row lane + 32 i for 128 of k. The issuer copies
// a slice's blocks before its four instructions. Single CTAs stage them as they go: two
// warps in turn copy 16 of a row at once (a chunk: two slices) into shared memory by
// cp.async, each lane the rows lane + 32 i, a chunk or more ahead, and then write the
// slices' blocks. (Gathering them directly from global memory into the blocks would
// take a 4-byte access per row and 128 of k, twice what the L1 cache can look up.) A
// pair's tensor cores leave no time for that: each row's 16 bytes cost shared memory
// a clock of their own, in every tile again (8192 x 8192 x 4096 121 us, 99 without). For
// pairs layScalesKernel writes all blocks once, into the workspace, and TMA loads them.
// A stage of the ring holds a slice of A, of B and of the blocks; its TMEM columns
// are the stage's, too, so one barrier frees all of it.
#ifndef SGBLAS_B200_PRODUCT_FP4_CUH_
#define SGBLAS_B200_PRODUCT_FP4_CUH_

#include "product_thin.cuh"
#include "product_tile.cuh"

namespace sgblas::kern::prod {

constexpr int kScaleBlock = 512;     // bytes: four scales of each of 128 rows
constexpr int kScaleWarp0 = 2, kScaleWarps = 2;
constexpr int kRawChunks = 2;        // chunks of 16 scales per row: one at work, the next on its way
constexpr int kScaleRowBytes = 256;  // of the laid-out scales
constexpr int kScaleRowsA = 2 * kScaleBlock / kScaleRowBytes;
constexpr int kScaleRowsB = 2 * kScaleRowsA;

struct Fp4Params {
  Params p;                          // k in bytes
  const unsigned char *scale_a, *scale_b;
  int ldsa, ldsb, blocks;            // blocks of 32 along k
  long long stride_sa;
  // Pairs: the scales' blocks, and the maps they are read by: rows of 256 bytes, a slice's
  // kScaleRowsA of each 128 rows of a matrix of A, and kScaleRowsB of each tile's columns.
  unsigned char *laid_a, *laid_b;
  int laid_tiles;                    // tiles of columns that laid_b has room for
  CUtensorMap tma_sa, tma_sb;
};

// Shared layout of both forms: kBN columns of the tile, all of whose scales each
// CTA has.
template <int kBN_, bool kTwo_, bool kThin_>
struct Fp4Shape {
  static constexpr Ragged kRagged = Ragged::kN;
  static constexpr int kElemBytes = 1;
  static constexpr int kBN = kBN_;
  static constexpr bool kTwo = kTwo_, kSymmetric = false;
  static constexpr int kTileM = kTwo ? 2 * kBM : kBM;
  static constexpr int kBRows = kTwo ? kBN / 2 : kBN;
  static constexpr int kNStep = kTwo ? 32 : 16;
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBBytes = kBRows * kRowBytes;
  static constexpr int kBBlocks = (kBN + 127) / 128;   // of scales of B, per 128 of k
  static constexpr int kScaleBytes = 2 * (1 + kBBlocks) * kScaleBlock;
  static constexpr int kScaleColumns = kScaleBytes / 128;   // of TMEM
  static constexpr int kStageBytes = kABytes + kBBytes + kScaleBytes;
  static constexpr int kRawRows = kBM + kBN;
  static constexpr int kRawBytes = kTwo ? 0 : kScaleWarps * kRawChunks * kRawRows * 16;
  static constexpr int kAccums = kThin_ ? 8 : 2;
  static constexpr int kScaleColumn0 = kAccums * kBN;
  static constexpr int kFitColumns = (512 - kScaleColumn0) / kScaleColumns;
  static constexpr int kTmemColumns = 512;
  static_assert(kBN % 16 == 0 && kBN <= 256, "the instruction's N");
  static_assert(!kTwo || (kBN % 32 == 0 && kBBlocks == 2), "halves of whole swizzle groups, kScaleRowsB");
};

template <int kBN_, bool kTwo_, bool kFp32_>
struct Fp4Cfg : Fp4Shape<kBN_, kTwo_, false> {
  using S = Fp4Shape<kBN_, kTwo_, false>;
  static constexpr bool kFp32 = kFp32_;
  static constexpr int kOutWarp = 2 * kOutCols * 32 * (kFp32 ? 4 : 2);
  static constexpr int kOutBytes = kEpilogueWarps * kOutWarp;
  static constexpr int kFit = (217 * 1024 - kOutBytes - S::kRawBytes) / S::kStageBytes;
  static constexpr int kLess = kFit < S::kFitColumns ? kFit : S::kFitColumns;
  static constexpr int kStages = kLess > 8 ? 8 : kLess;
  static constexpr int kBarrierBytes = 8 * (2 * kStages + 2 * S::kAccums);
  static constexpr int kSmemBytes =
      kStages * S::kStageBytes + kOutBytes + S::kRawBytes + kBarrierBytes + 1024;
  static_assert(kStages >= 3 && kSmemBytes <= 218 * 1024 + 512, "shared memory beside the table");
  static_assert(S::kBN / 2 % 32 == 0, "an epilogue warp's columns");
};

template <int kBN_>
struct Fp4ThinCfg : Fp4Shape<kBN_, false, true> {
  using S = Fp4Shape<kBN_, false, true>;
  static constexpr int kPartPitch = S::kBN + 4;
  static constexpr int kPartBytes = kPartPitch * kBM * 4;
  static constexpr int kFit = (kThinSmem - kPartBytes - S::kRawBytes) / S::kStageBytes;
  static constexpr int kStages = kFit < S::kFitColumns ? kFit : S::kFitColumns;
  static constexpr int kBarrierBytes = 8 * (2 * kStages + 2 * S::kAccums + 2);
  static constexpr int kSmemBytes =
      kStages * S::kStageBytes + kPartBytes + S::kRawBytes + kBarrierBytes + 1024;
  static_assert(S::kBN == 16 || S::kBN == 32, "tile width");
  static_assert(kSmemBytes <= 218 * 1024, "shared memory beside the table");
};

// Instruction descriptor: e2m1 operands, e8m0 scales; `half` of a word of four
// scales (bits 4-5 and 29-30: the first byte's number).
template <class G>
__device__ __forceinline__ uint32_t fp4InstrDesc(int n, int half) {
  return (static_cast<uint32_t>(2 * half) << 4) | (1u << 7) | (1u << 10) |
         (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(G::kTileM >> 4) << 24) | (static_cast<uint32_t>(2 * half) << 29);
}

// Descriptor of a block of scales: 16-byte rows without swizzle, groups of eight
// rows 128 bytes apart.
__device__ __forceinline__ uint64_t scaleDesc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(8) << 16) |
         (static_cast<uint64_t>(8) << 32) | (static_cast<uint64_t>(1) << 46);
}

// The role of the scales' warps: the scales of every slice [kb0, kb1) of this worker's
// tiles into the ring's stages. Warp `part` of kScaleWarps takes every kScaleWarps-th
// chunk, with its own raw buffers; `ready(s)` announces stage s.
template <class G, int kStages, class Wait, class Ready>
__device__ __forceinline__ void stageScales(const Fp4Params &f, const GroupTable &table, int tiles,
                                            int worker, int workers, int kb0, int kb1,
                                            unsigned char *ring, unsigned char *raw, int part,
                                            int lane, Wait wait, Ready ready) {
  const Params &p = f.p;
  const int chunk0 = kb0 / 2, chunk1 = (kb1 + 1) / 2;
  if (kb0 >= kb1) return;
  raw += part * (kRawChunks * G::kRawRows * 16);
  // The chunk fetched next, ahead of the one at work: chunks are numbered over all
  // of this worker's tiles, and every kScaleWarps-th is this warp's.
  int fetch_tile = worker, fetch_chunk = chunk0, fetched = 0;
  auto skip = [&](int chunks) {
    fetch_chunk += chunks;
    while (fetch_chunk >= chunk1) {
      fetch_chunk -= chunk1 - chunk0;
      fetch_tile += workers;
    }
  };
  auto fetch = [&]() {
    if (fetch_tile < tiles) {
      const Tile t = tileAt<G>(p, table, fetch_tile);
      const int m0 = t.m0;
      const unsigned char *a = f.scale_a + t.group * f.stride_sa +
                               static_cast<long long>(m0 + lane) * f.ldsa + fetch_chunk * 16;
      const unsigned char *b =
          f.scale_b + static_cast<long long>(t.n0 + lane) * f.ldsb + fetch_chunk * 16;
      unsigned char *to = raw + (fetched % kRawChunks) * (G::kRawRows * 16) + lane * 16;
      const uint32_t bytes = static_cast<uint32_t>(min(16, f.blocks - fetch_chunk * 16));
#pragma unroll
      for (int i = 0; i < kBM / 32; ++i) {
        const bool in = lane + 32 * i < p.m - m0;
        cpAsync16Cg(to + i * 512, in ? a + static_cast<long long>(32 * i) * f.ldsa : f.scale_a, in ? bytes : 0);
      }
#pragma unroll
      for (int i = 0; i < (G::kBN + 31) / 32; ++i) {
        if (G::kBN % 32 != 0 && lane >= G::kBN) break;
        const bool in = lane + 32 * i < t.cols;
        cpAsync16Cg(to + (kBM / 32 + i) * 512, in ? b + static_cast<long long>(32 * i) * f.ldsb : f.scale_b,
                    in ? bytes : 0);
      }
      skip(kScaleWarps);
    }
    cpAsyncCommit();
    ++fetched;
  };
  skip(part);
#pragma unroll 1
  for (int i = 0; i < kRawChunks - 1; ++i) fetch();
  int s = 0, parity = 1, turn = 0, done = 0;
  for (int i = worker; i < tiles; i += workers) {
#pragma unroll 1
    for (int c = chunk0; c < chunk1; ++c) {
      const int first = max(2 * c, kb0), slices = min(2 * c + 2, kb1) - first;
      const bool mine = turn == part;
      if (++turn == kScaleWarps) turn = 0;
      int s2 = s + 1, parity2 = parity;   // of a second slice
      if (s2 == kStages) {
        s2 = 0;
        parity2 ^= 1;
      }
      if (mine) {
        fetch();   // into the chunk that this lane read last
        cpAsyncWait<kRawChunks - 1>();
        const unsigned char *from = raw + (done % kRawChunks) * (G::kRawRows * 16) + lane * 16;
        ++done;
        wait(s, parity);
        if (slices > 1) wait(s2, parity2);
        unsigned char *blocks = ring + G::kABytes + G::kBBytes + lane * 16;
        // The chunk's first or second half goes to stage s, its second to s2 where
        // both are there.
        unsigned char *to = blocks + s * G::kStageBytes, *to2 = blocks + s2 * G::kStageBytes;
        const bool upper = first % 2 != 0;
        // Blocks of a stage: A's of the first and second 128 of k, then B's likewise.
#pragma unroll
        for (int b = 0; b < 1 + G::kBBlocks; ++b) {
          uint4 w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row0 = (b * 4 + r) * 32;   // of the raw rows
            w[r] = make_uint4(0, 0, 0, 0);
            if (row0 < G::kRawRows && (row0 + 32 <= G::kRawRows || lane < G::kRawRows - row0))
              w[r] = *reinterpret_cast<const uint4 *>(from + row0 * 16);
          }
          const int at = (b == 0 ? 0 : 1 + b) * kScaleBlock;
          const int next = at + (b == 0 ? 1 : G::kBBlocks) * kScaleBlock;
          const uint4 low[2] = {make_uint4(w[0].x, w[1].x, w[2].x, w[3].x),
                                make_uint4(w[0].y, w[1].y, w[2].y, w[3].y)};
          const uint4 high[2] = {make_uint4(w[0].z, w[1].z, w[2].z, w[3].z),
                                 make_uint4(w[0].w, w[1].w, w[2].w, w[3].w)};
          *reinterpret_cast<uint4 *>(to + at) = upper ? high[0] : low[0];
          *reinterpret_cast<uint4 *>(to + next) = upper ? high[1] : low[1];
          if (slices > 1) {
            *reinterpret_cast<uint4 *>(to2 + at) = high[0];
            *reinterpret_cast<uint4 *>(to2 + next) = high[1];
          }
        }
        fenceProxyAsyncShared();
        __syncwarp();
        ready(s);
        if (slices > 1) ready(s2);
      }
      s = s2;
      parity = parity2;
      if (slices > 1 && ++s == kStages) {
        s = 0;
        parity ^= 1;
      }
    }
  }
  cpAsyncWait<0>();
}

// One slice: its scales to TMEM, then its instructions (one thread).
template <class G>
__device__ __forceinline__ void issueSlice(uint32_t tmem_base, uint32_t d_tmem, uint32_t stage_addr,
                                           uint64_t desc_a, uint64_t desc_b, int s, int n,
                                           bool accumulate) {
  const uint32_t sf = tmem_base + G::kScaleColumn0 + static_cast<uint32_t>(s * G::kScaleColumns);
  const uint64_t from =
      scaleDesc(stage_addr + static_cast<uint32_t>(s * G::kStageBytes + G::kABytes + G::kBBytes));
#pragma unroll
  for (int b = 0; b < 2 * (1 + G::kBBlocks); ++b)
    tmemCopyScales<G::kTwo>(sf + 4 * b, from + b * (kScaleBlock / 16));
  uint64_t ad = desc_a + static_cast<uint64_t>(s) * (G::kStageBytes / 16);
  uint64_t bd = desc_b + static_cast<uint64_t>(s) * (G::kStageBytes / 16);
  const uint32_t idesc[2] = {fp4InstrDesc<G>(n, 0), fp4InstrDesc<G>(n, 1)};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mmaFp4<G::kTwo>(d_tmem, ad, bd, idesc[j % 2], sf + j / 2 * 4, sf + 8 + j / 2 * (4 * G::kBBlocks),
                    accumulate || j > 0);
    ad += 2;   // 32 bytes
    bd += 2;
  }
}

// Blocks of 128 rows of a matrix of A.
__host__ __device__ __forceinline__ int scaleBlocksA(int m) { return (m + kBM - 1) / kBM; }

// Room for the laid-out scales of pairs of width G::kBN: those of A, then those of B, in
// bytes. Groups whose offsets do not decrease have no more tiles than that.
struct LaidSize {
  long long a, b, tiles;
};
template <class G>
__host__ __device__ __forceinline__ LaidSize laidSize(const Params &p) {
  const long long iters = (p.k + kRowBytes - 1) / kRowBytes;
  LaidSize s;
  s.tiles = p.n / G::kBN + (p.groups < p.n ? p.groups : p.n);
  s.a = static_cast<long long>(p.groups) * scaleBlocksA(p.m) * iters * kScaleRowsA * kScaleRowBytes;
  s.b = s.tiles * iters * kScaleRowsB * kScaleRowBytes;
  return s;
}

// The scales' blocks in items: a chunk (16 scales) of 128 rows of A, or of half a tile's
// columns. Offsets that decrease, which the host cannot see, give more tiles than it has
// counted: blocks past its room are left out.
__host__ __device__ __forceinline__ long long laidItemsA(const Params &p) {
  const int iters = (p.k + kRowBytes - 1) / kRowBytes;
  return static_cast<long long>(p.groups) * scaleBlocksA(p.m) * ((iters + 1) / 2);
}
template <class G>
__host__ __device__ __forceinline__ long long laidItems(const Fp4Params &f, const GroupTable &table) {
  const int iters = (f.p.k + kRowBytes - 1) / kRowBytes;
  const int tiles = table.first[f.p.groups] < f.laid_tiles ? table.first[f.p.groups] : f.laid_tiles;
  return laidItemsA(f.p) + static_cast<long long>(tiles) * G::kBBlocks * ((iters + 1) / 2);
}

struct LaidItem {
  const unsigned char *from;
  unsigned char *to;           // of the chunk's first slice
  int rows, ld, chunk;         // no rows: nothing to lay out
  int slice, next;             // bytes of a slice, and from its first 128 of k to its second
};
template <class G>
__host__ __device__ __forceinline__ LaidItem laidItem(const Fp4Params &f, const GroupTable &table, long long i) {
  const Params &p = f.p;
  const int iters = (p.k + kRowBytes - 1) / kRowBytes, chunks = (iters + 1) / 2;
  const int blocks_a = scaleBlocksA(p.m);
  const long long items_a = laidItemsA(p);
  const bool is_a = i < items_a;
  const long long at = is_a ? i : i - items_a;
  const int block = static_cast<int>(at / chunks);
  LaidItem r;
  r.chunk = static_cast<int>(at % chunks);
  if (is_a) {
    const int group = block / blocks_a, row0 = (block - group * blocks_a) * kBM;
    r.from = f.scale_a + group * f.stride_sa + static_cast<long long>(row0) * f.ldsa;
    r.rows = table.offset[group + 1] <= table.offset[group] ? 0 : p.m - row0;
    r.ld = f.ldsa;
    r.slice = kScaleRowsA * kScaleRowBytes;
    r.next = kScaleBlock;
    r.to = f.laid_a + (static_cast<long long>(block) * iters + 2 * r.chunk) * r.slice;
  } else {
    const int tile = block / G::kBBlocks, half = block - tile * G::kBBlocks;
    const Tile t = tileAt<G>(p, table, tile * p.tiles_m);
    r.from = f.scale_b + static_cast<long long>(t.n0 + half * kBM) * f.ldsb;
    r.rows = t.cols - half * kBM;
    r.ld = f.ldsb;
    r.slice = kScaleRowsB * kScaleRowBytes;
    r.next = G::kBBlocks * kScaleBlock;
    r.to = f.laid_b + (static_cast<long long>(tile) * iters + 2 * r.chunk) * r.slice + half * kScaleBlock;
  }
  return r;
}

// Writes the scales' blocks of pairs of width G::kBN (1 MB of each operand's for 8192 x
// 8192 x 4096: 4 us): a warp per item, of groups that have columns.
constexpr int kLayThreads = 256;
template <class G>
__global__ void __launch_bounds__(kLayThreads) layScalesKernel(const __grid_constant__ Fp4Params f) {
  const Params &p = f.p;
  __shared__ GroupTable table;
  gridDependencyWait();
  allowDependentLaunch();
  const int lane = threadIdx.x % 32;
  if (threadIdx.x < 32) readGroups<G>(p, &table, lane);
  __syncthreads();
  const int iters = (p.k + kRowBytes - 1) / kRowBytes;
  const long long items = laidItems<G>(f, table);
  const long long step = gridDim.x * static_cast<long long>(kLayThreads / 32);
  for (long long i = blockIdx.x * (kLayThreads / 32LL) + threadIdx.x / 32; i < items; i += step) {
    const LaidItem it = laidItem<G>(f, table, i);
    if (i < laidItemsA(p) && it.rows <= 0) continue;
    const int bytes = min(16, f.blocks - it.chunk * 16);
    uint4 w[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      w[r] = make_uint4(0, 0, 0, 0);
      const unsigned char *row = it.from + static_cast<long long>(lane + 32 * r) * it.ld + it.chunk * 16;
      if (lane + 32 * r >= it.rows) continue;
      if (bytes == 16) {
        w[r] = __ldg(reinterpret_cast<const uint4 *>(row));
      } else {
        uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 15; ++j)
          if (j < bytes) v[j / 4] |= static_cast<uint32_t>(row[j]) << (j % 4 * 8);
        w[r] = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
    uint4 *out = reinterpret_cast<uint4 *>(it.to) + lane;
    out[0] = make_uint4(w[0].x, w[1].x, w[2].x, w[3].x);
    out[it.next / 16] = make_uint4(w[0].y, w[1].y, w[2].y, w[3].y);
    if (2 * it.chunk + 1 < iters) {
      out += it.slice / 16;
      out[0] = make_uint4(w[0].z, w[1].z, w[2].z, w[3].z);
      out[it.next / 16] = make_uint4(w[0].w, w[1].w, w[2].w, w[3].w);
    }
  }
}

// Many tokens: as productKernel. 8192 x 8192 x 4096 in pairs, BF16 out: 108 us with the
// scales' blocks, 5.1 PFLOP/s; the tensor pipe is busy 76 % of the cycles, shared memory
// (operands and scales in, operands out) the rest. FP32 out 130 us: its epilogue. Pairs
// are 192 wide: two accumulators of 256 columns would leave the scales no TMEM.
//   full[s]   stage s has its operands and scales: TMA's bytes (of both CTAs of a pair),
//             and a single CTA's scales' warps
template <class G>
__global__ void __launch_bounds__(kThreads, 1) fp4TileKernel(const __grid_constant__ Fp4Params f) {
  constexpr int kBN = G::kBN;
  constexpr int kStages = G::kStages;
  constexpr int kStageBytes = G::kStageBytes;
  const Params &p = f.p;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ GroupTable table;
  unsigned char *smem = smem_raw + ((1024 - (smemAddr(smem_raw) & 1023)) & 1023);
  unsigned char *out_smem = smem + kStages * kStageBytes;
  unsigned char *raw = out_smem + G::kOutBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(raw + G::kRawBytes);
  uint64_t *empty = full + kStages;
  uint64_t *acc_full = empty + kStages;
  uint64_t *acc_empty = acc_full + kAccums;

  const int warp = uniformWarp(), lane = threadIdx.x % 32;
  const int rank = G::kTwo ? static_cast<int>(blockIdx.x & 1) : 0;
  const int worker = G::kTwo ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int workers = G::kTwo ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  if (threadIdx.x == 0) {
    if (p.k > 0) {
      prefetchTensorMap(&p.tma_a);
      prefetchTensorMap(&p.tma_b);
    }
    if (p.c_tma) prefetchTensorMap(&p.tma_c);
    if (G::kTwo && p.k > 0) {
      prefetchTensorMap(&f.tma_sa);
      prefetchTensorMap(&f.tma_sb);
    }
    for (int s = 0; s < kStages; ++s) {
      mbarInit(&full[s], G::kTwo ? 1 : 2);
      mbarInit(&empty[s], 1);
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
  if (warp == 0) readGroups<G>(p, &table, lane);
  __syncthreads();
  const uint32_t tmem_base = tmem_base_slot;
  const int tiles = tileCount<G>(p, table);
  const int iters = (p.k + kRowBytes - 1) / kRowBytes;

  bool ok = true;
  auto wait = [&](uint64_t *bar, int parity) {
    if (ok) ok = mbarWait(bar, static_cast<uint32_t>(parity), p.err);
  };
  auto widthOf = [](int cols) { return (cols + G::kNStep - 1) / G::kNStep * G::kNStep; };

  if (warp < kEpilogueWarp0) {
    regDealloc<72>();
    if (warp == 0 && electOne()) {
      // ---------------- TMA producer ----------------
      int s = 0, parity = 1;
      for (int i = worker; i < tiles; i += workers) {
        const Tile t = tileAt<G>(p, table, i);
        const int m0 = t.m0 + rank * kBM;
        const int n0 = t.n0 + (G::kTwo ? rank * (widthOf(t.cols) / 2) : 0);
        // A pair's: where the laid-out scales of this tile begin, in slices. Rows past
        // the matrix's last block are the next one's, or zeros; they reach no row of C.
        const int scale_a = (t.group * scaleBlocksA(p.m) + m0 / kBM) * iters;
        const int scale_b = i / p.tiles_m * iters;
        for (int kb = 0; kb < iters; ++kb) {
          wait(&empty[s], parity);
          if (!ok) continue;
          unsigned char *stage = smem + s * kStageBytes;
          if constexpr (G::kTwo) {
            if (rank == 0) mbarArriveExpectTx(&full[s], 2 * kStageBytes);
            const uint32_t bar = clusterAddr(smemAddr(&full[s]), 0);
            tmaLoad3dPair(stage, &p.tma_a, bar, kb * kRowBytes, m0, t.group);
            tmaLoad3dPair(stage + G::kABytes, &p.tma_b, bar, kb * kRowBytes, n0, 0);
            unsigned char *scales = stage + G::kABytes + G::kBBytes;
            tmaLoad3dPair(scales, &f.tma_sa, bar, 0, (scale_a + kb) * kScaleRowsA, 0);
            tmaLoad3dPair(scales + 2 * kScaleBlock, &f.tma_sb, bar, 0, (scale_b + kb) * kScaleRowsB, 0);
          } else {
            mbarArriveExpectTx(&full[s], G::kABytes + G::kBBytes);
            tmaLoad3d(stage, &p.tma_a, &full[s], kb * kRowBytes, m0, t.group);
            tmaLoad3d(stage + G::kABytes, &p.tma_b, &full[s], kb * kRowBytes, n0, 0);
          }
          if (++s == kStages) {
            s = 0;
            parity ^= 1;
          }
        }
      }
      // The last copies have landed and been read (productKernel).
#pragma unroll 1
      for (int j = 0; j < kStages; ++j) {
        if (rank == 0) wait(&full[s], parity);
        wait(&empty[s], parity);
        if (++s == kStages) {
          s = 0;
          parity ^= 1;
        }
      }
    } else if (!G::kTwo && warp >= kScaleWarp0) {
      // ---------------- scales ----------------
      if constexpr (!G::kTwo)
        stageScales<G, kStages>(
            f, table, tiles, worker, workers, 0, iters, smem, raw, warp - kScaleWarp0, lane,
            [&](int s, int parity) { wait(&empty[s], parity); },
            [&](int s) {
              if (lane == 0) mbarArrive(&full[s]);
            });
    } else if (warp == 1 && rank == 0) {
      // ---------------- MMA issuer ----------------
      const bool leader = electOne();
      int s = 0, parity = 0;
      int b = 0, acc_parity = 1;
      const uint64_t desc_a = smemDesc<false>(smemAddr(smem));
      const uint64_t desc_b = smemDesc<false>(smemAddr(smem) + G::kABytes);
      for (int i = worker; i < tiles; i += workers) {
        const Tile t = tileAt<G>(p, table, i);
        const int n = widthOf(t.cols);
        int in_chunk = 0;
        for (int kb = 0; kb < iters; ++kb) {
          const bool first = in_chunk == 0;
          const bool last = ++in_chunk == p.chunk_iters || kb == iters - 1;
          if (last) in_chunk = 0;
          if (first) wait(&acc_empty[b], acc_parity);
          wait(&full[s], parity);
          if (leader) {
            tcgenFenceAfter();
            issueSlice<G>(tmem_base, tmem_base + static_cast<uint32_t>(b * kBN), smemAddr(smem), desc_a,
                          desc_b, s, n, !first);
            if constexpr (G::kTwo) {
              mmaCommitBoth(&empty[s]);
              if (last) mmaCommitBoth(&acc_full[b]);
            } else {
              mmaCommit(&empty[s]);
              if (last) mmaCommit(&acc_full[b]);
            }
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
    regAlloc<216>();
    constexpr int kHalf = kBN / 2;
    constexpr int kBlocks = kHalf / 8;
    const int quarter = warp % 4;
    const int col_begin = (warp - kEpilogueWarp0) / 4 * kHalf;
    const int lower = quarter % 2, pair = (warp - kEpilogueWarp0) / 2;
    unsigned char *out = out_smem + (warp - kEpilogueWarp0) * G::kOutWarp;
    const bool vector = reinterpret_cast<uintptr_t>(p.c) % 16 == 0 && p.ldc % 8 == 0;
    const int chunks = iters > 0 ? (iters - 1) / p.chunk_iters + 1 : 0;
    int b = 0, acc_parity = 0;
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      float2 acc[kBlocks * 4];
#pragma unroll
      for (int j = 0; j < kBlocks * 4; ++j) acc[j] = make_float2(0.0F, 0.0F);
      for (int ch = 0; ch < chunks; ++ch) {
        wait(&acc_full[b], acc_parity);
        tcgenFenceAfter();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                               static_cast<uint32_t>(b * kBN + col_begin);
        if constexpr (G::kFp32) addRows<kHalf, false>(taddr, acc, nullptr, 0.0F);
        else addFragments<kHalf, false>(taddr, acc, nullptr, 0.0F, lane);
        tcgenFenceBefore();
        __syncwarp();
        if (lane == 0) {
          if constexpr (G::kTwo) mbarArriveClusterRelaxed(clusterAddr(smemAddr(&acc_empty[b]), 0));
          else mbarArrive(&acc_empty[b]);
        }
        b ^= 1;
        if (b == 0) acc_parity ^= 1;
      }
      const int row0 = t.m0 + rank * kBM + quarter * 32;
      const int cols = t.cols - col_begin;
      if (row0 - (G::kFp32 ? 0 : lower * 32) < p.m && cols > 0) {
        Place to;
        to.row = row0;
        to.col = t.n0 + col_begin;
        to.at = static_cast<size_t>(to.col) * p.ldc + row0;
        to.matrix = 0;
        to.rows = p.m - row0;
        to.cols = cols;
        to.clip = false;
        to.vector = vector;
        if constexpr (G::kFp32) storeFp32<kHalf>(p, to, acc, out, lane);
        else storeBf16<kBlocks>(p, to, acc, out - lower * G::kOutWarp, pair, lower, lane);
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

// Few tokens: as thinProductKernel, clusters of `split` CTAs that share k. Bound by HBM
// and by latencies at both ends: 384 tokens unevenly over 32 experts of 2048 x 2048 (71
// MB) 15.4 us, one token of 4096 x 4096 6.1.
template <class G>
__global__ void __launch_bounds__(kThinThreads, 1)
    fp4ThinKernel(const __grid_constant__ Fp4Params f, int split) {
  constexpr int kBN = G::kBN;
  constexpr int kStages = G::kStages;
  constexpr int kStageBytes = G::kStageBytes;
  constexpr int kPitch = G::kPartPitch;
  const Params &p = f.p;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ GroupTable table;
  unsigned char *smem = smem_raw + ((1024 - (smemAddr(smem_raw) & 1023)) & 1023);
  float *part = reinterpret_cast<float *>(smem + kStages * kStageBytes);
  unsigned char *raw = smem + kStages * kStageBytes + G::kPartBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(raw + G::kRawBytes);
  uint64_t *empty = full + kStages;
  uint64_t *acc_full = empty + kStages;
  uint64_t *acc_empty = acc_full + G::kAccums;
  uint64_t *part_full = acc_empty + G::kAccums;
  uint64_t *part_free = part_full + 1;

  const int warp = uniformWarp(), lane = threadIdx.x % 32;
  const int rank = static_cast<int>(blockIdx.x) % split;
  const int worker = static_cast<int>(blockIdx.x) / split;
  const int workers = static_cast<int>(gridDim.x) / split;
  if (threadIdx.x == 0) {
    if (p.k > 0) {
      prefetchTensorMap(&p.tma_a);
      prefetchTensorMap(&p.tma_b);
    }
    for (int s = 0; s < kStages; ++s) {
      mbarInit(&full[s], 2);
      mbarInit(&empty[s], 1);
    }
    for (int b = 0; b < G::kAccums; ++b) {
      mbarInit(&acc_full[b], 1);
      mbarInit(&acc_empty[b], kThinEpilogue / 32);
    }
    mbarInit(part_full, 1);
    mbarInit(part_free, static_cast<uint32_t>(split));
    fenceBarrierInit();
  }
  if (warp == 2) {
    tmemAlloc(&tmem_base_slot, G::kTmemColumns);
    tmemRelinquish();
  }
  tcgenFenceBefore();
  __syncthreads();
  if (split > 1) clusterSync();   // the cluster's barriers exist
  tcgenFenceAfter();
  allowDependentLaunch();
  gridDependencyWait();
  if (warp == 0) readGroups<G>(p, &table, lane);
  __syncthreads();
  const uint32_t tmem_base = tmem_base_slot;
  const int tiles = tileCount<G>(p, table);
  // This CTA's slices of k.
  const int iters = (p.k + kRowBytes - 1) / kRowBytes;
  const int kb0 = static_cast<int>(static_cast<long long>(iters) * rank / split);
  const int kb1 = static_cast<int>(static_cast<long long>(iters) * (rank + 1) / split);
  const int mine = kb1 - kb0;

  bool ok = true;
  auto wait = [&](uint64_t *bar, int parity) {
    if (ok) ok = mbarWait(bar, static_cast<uint32_t>(parity), p.err);
  };

  if (warp == 0 && electOne()) {
    // ---------------- TMA producer ----------------
    int s = 0, parity = 1;
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      const int boxes = (t.cols + kThinBox - 1) / kThinBox;
      for (int kb = kb0; kb < kb1; ++kb) {
        wait(&empty[s], parity);
        if (!ok) continue;
        unsigned char *sa = smem + s * kStageBytes;
        mbarArriveExpectTx(&full[s], G::kABytes + static_cast<uint32_t>(boxes * kThinBox * kRowBytes));
        tmaLoad3d(sa, &p.tma_a, &full[s], kb * kRowBytes, t.m0, t.group);
        for (int j = 0; j < boxes; ++j)
          tmaLoad3d(sa + G::kABytes + j * kThinBox * kRowBytes, &p.tma_b, &full[s], kb * kRowBytes,
                    t.n0 + j * kThinBox, 0);
        if (++s == kStages) {
          s = 0;
          parity ^= 1;
        }
      }
    }
    // The last copies have landed and been read (productKernel).
#pragma unroll 1
    for (int j = 0; j < kStages; ++j) {
      wait(&full[s], parity);
      wait(&empty[s], parity);
      if (++s == kStages) {
        s = 0;
        parity ^= 1;
      }
    }
  } else if (warp == kScaleWarp0 || warp == kScaleWarp0 + 1) {
    // ---------------- scales ----------------
    stageScales<G, kStages>(
        f, table, tiles, worker, workers, kb0, kb1, smem, raw, warp - kScaleWarp0, lane,
        [&](int s, int parity) { wait(&empty[s], parity); },
        [&](int s) {
          if (lane == 0) mbarArrive(&full[s]);
        });
  } else if (warp == 1 && electOne()) {
    // ---------------- MMA issuer ----------------
    int s = 0, parity = 0;
    int b = 0, acc_parity = 1;
    const uint64_t desc_a = smemDesc<false>(smemAddr(smem));
    const uint64_t desc_b = smemDesc<false>(smemAddr(smem) + G::kABytes);
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      const int n = (t.cols + 15) / 16 * 16;
      int in_chunk = 0;
      for (int j = 0; j < mine; ++j) {
        const bool first = in_chunk == 0;
        const bool last = ++in_chunk == p.chunk_iters || j == mine - 1;
        if (last) in_chunk = 0;
        if (first) wait(&acc_empty[b], acc_parity);
        wait(&full[s], parity);
        tcgenFenceAfter();
        issueSlice<G>(tmem_base, tmem_base + static_cast<uint32_t>(b * kBN), smemAddr(smem), desc_a, desc_b,
                      s, n, !first);
        mmaCommit(&empty[s]);
        if (last) {
          mmaCommit(&acc_full[b]);
          if (++b == G::kAccums) {
            b = 0;
            acc_parity ^= 1;
          }
        }
        if (++s == kStages) {
          s = 0;
          parity ^= 1;
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------- epilogue ----------------
    const int quarter = warp % 4;
    const int row = quarter * 32 + lane;
    const int etid = threadIdx.x % kThinEpilogue;
    const int chunks = mine > 0 ? (mine - 1) / p.chunk_iters + 1 : 0;
    int b = 0, acc_parity = 0;
    int part_parity = 0;
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      float acc[kBN];
#pragma unroll
      for (int j = 0; j < kBN; ++j) acc[j] = 0.0F;
      for (int ch = 0; ch < chunks; ++ch) {
        wait(&acc_full[b], acc_parity);
        tcgenFenceAfter();
        const uint32_t taddr =
            tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(b * kBN);
        constexpr int kLoad = kBN < 32 ? kBN : 32;
#pragma unroll
        for (int c = 0; c < kBN; c += kLoad) {
          if (c < t.cols) {
            uint32_t v[kLoad];
            if constexpr (kLoad == 16) tmemLoad16(taddr + c, v);
            else tmemLoad32(taddr + c, v);
#pragma unroll
            for (int j = 0; j < kLoad; ++j) acc[c + j] += __uint_as_float(v[j]);
          }
        }
        tcgenFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArrive(&acc_empty[b]);
        if (++b == G::kAccums) {
          b = 0;
          acc_parity ^= 1;
        }
      }
      if (split == 1) {
        if (t.m0 + row < p.m) {
          const size_t at = static_cast<size_t>(t.n0) * p.ldc + t.m0 + row;
          if (p.c_bf16) storeRow<kBN>(p, static_cast<__nv_bfloat16 *>(p.c) + at, t.cols, acc);
          else storeRow<kBN>(p, static_cast<float *>(p.c) + at, t.cols, acc);
        }
        continue;
      }
      // Each row's sums to the CTA that writes the row (thinProductKernel).
      if (ok) ok = mbarWaitCluster(part_free, part_parity ^ 1, p.err);
      const int rows = kBM / split;
      const int owner = row / rows;
      const int width = (t.cols + 3) / 4 * 4;
      if (etid == 0) mbarArriveExpectTx(part_full, static_cast<uint32_t>(kBM * width * 4));
      const uint32_t to = clusterAddr(
          smemAddr(part) + static_cast<uint32_t>((rank * rows + row - owner * rows) * kPitch) * 4,
          static_cast<uint32_t>(owner));
      const uint32_t bar = clusterAddr(smemAddr(part_full), static_cast<uint32_t>(owner));
#pragma unroll
      for (int j = 0; j < kBN; j += 4)
        if (j < t.cols)
          storeAsyncCluster4(to + static_cast<uint32_t>(j) * 4, bar, acc[j], acc[j + 1], acc[j + 2],
                             acc[j + 3]);
      if (ok) ok = mbarWaitCluster(part_full, part_parity, p.err);
      for (int e = etid; e < rows * t.cols; e += kThinEpilogue) {
        const int col = e / rows, r = e - col * rows;
        float v[kMaxSplit];
#pragma unroll
        for (int q = 0; q < kMaxSplit; ++q)
          v[q] = q < split ? part[(q * rows + r) * kPitch + col] : 0.0F;
        float sum = v[0];
#pragma unroll
        for (int q = 1; q < kMaxSplit; ++q) sum += v[q];
        const int to_row = t.m0 + rank * rows + r;
        if (to_row < p.m) {
          const size_t at = static_cast<size_t>(t.n0 + col) * p.ldc + to_row;
          if (p.c_bf16) storeScaled(p, static_cast<__nv_bfloat16 *>(p.c) + at, sum);
          else storeScaled(p, static_cast<float *>(p.c) + at, sum);
        }
      }
      namedBarrier<1, kThinEpilogue>();
      if (etid < split)
        mbarArriveCluster(clusterAddr(smemAddr(part_free), static_cast<uint32_t>(etid)));
      part_parity ^= 1;
    }
  }

  tcgenFenceBefore();
  __syncthreads();
  if (split > 1) clusterSync();   // no CTA leaves while another reads its part
  if (warp == 2) {
    tcgenFenceAfter();
    tmemDealloc(tmem_base, G::kTmemColumns);
  }
}

}  // namespace sgblas::kern::prod

#endif  // SGBLAS_B200_PRODUCT_FP4_CUH_
