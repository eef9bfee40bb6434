// Products whose groups hold few columns (tokens being decoded): each CTA
// streams its share of the weights once, so what counts is that every SM
// streams all the time.
//
// C(:, group) is cut into 128-row by kBN-column tiles as in product_tile.cuh;
// a tile is computed by a cluster of `split` CTAs, each over its share of the
// k slices. The partial tiles meet in distributed shared memory: each CTA
// receives 128 / split rows from the others (asynchronous stores counted on a
// barrier: no release has to wait for them), adds them in rank order and
// writes them. There is no workspace, no atomic, and no order that varies.
// Splitting k gives SMs to a call with few tiles, and evens out the last wave
// of one with many.
//
// Memory-bound where the weights come from HBM: 32 experts of 2048 x 4096
// BF16 (537 MB), 192 tokens, 80 to 84 us, 6.4 to 6.7 TB/s; of 2048 x 2048 e4m3
// (134 MB), 384 tokens, 28 us, 4.8 TB/s (3.5 waves of tiles in four). The
// smallest calls are a chain of latencies (8 tokens, 8 experts of 1024 x 1024:
// 5.5 us, of which the offsets 0.6, the first slice 1.0, the stream 2.2, the
// hand-over and C 1.5).
//
// Warp roles (8 warps): warp 0 TMA producer, warp 1 MMA issuer, warp 2 TMEM,
// warps 4-7 epilogue (a row of the tile per thread). Chunks of k and e4m3
// scales as in product_tile.cuh; there are more accumulators, so that the
// issuer runs ahead while a tile is handed over.
#ifndef SGBLAS_B200_PRODUCT_THIN_CUH_
#define SGBLAS_B200_PRODUCT_THIN_CUH_

#include "product_tile.cuh"

namespace sgblas::kern::prod {

constexpr int kThinThreads = 256;
constexpr int kThinEpilogue = 128;  // epilogue threads
constexpr int kThinScales = 16;     // blocks of 128 whose scales are staged at once
constexpr int kMaxSplit = 8;
constexpr int kThinSmem = 200 * 1024;
constexpr int kThinBox = 8;         // columns of one box of B: a tile loads only what it holds

template <int kElemBytes_, int kBN_, bool kAMN_>
struct ThinCfg {
  static constexpr int kElemBytes = kElemBytes_;
  static constexpr Ragged kRagged = Ragged::kN;
  static constexpr int kBN = kBN_;
  static constexpr bool kAMN = kAMN_, kBMN = false;
  static constexpr bool kTwo = false, kSymmetric = false;
  static constexpr bool kBytes = kElemBytes == 1;
  static constexpr int kTileM = kBM;
  static constexpr int kBK = kRowBytes / kElemBytes;
  static constexpr int kMmaK = 32 / kElemBytes;
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBBytes = kBN * kRowBytes;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kPartPitch = kBN + 4;             // floats per row
  static constexpr int kPartBytes = kPartPitch * kBM * 4;   // 128 / split rows of each CTA's tile
  static constexpr int kThinAccums = 8;
  static constexpr int kScalePitch = kBN + 4;   // scale_b of each column, then scale_a
  static constexpr int kScaleBytes = kBytes ? 2 * kThinScales * kScalePitch * 4 : 0;
  static constexpr int kStages = (kThinSmem - kPartBytes - kScaleBytes) / kStageBytes;
  static constexpr int kTmemColumns = kThinAccums * kBN;
  static constexpr int kBarrierBytes = 8 * (2 * kStages + 2 * kThinAccums + 2);
  static constexpr int kSmemBytes =
      kStages * kStageBytes + kPartBytes + kScaleBytes + kBarrierBytes + 1024;
  static_assert(kBN == 16 || kBN == 32 || kBN == 64, "tile width");
  static_assert(kSmemBytes <= 218 * 1024, "shared memory beside the table");
};

// *c = alpha * v + beta * *c.
template <typename T>
__device__ __forceinline__ void storeScaled(const Params &p, T *c, float v) {
  v *= p.alpha;
  if (p.beta != 0.0F) v = fmaf(p.beta, static_cast<float>(*c), v);
  *c = static_cast<T>(v);
}
// One row of a tile: `cols` elements ldc apart.
template <int kBN, typename T>
__device__ __forceinline__ void storeRow(const Params &p, T *c, int cols, const float (&v)[kBN]) {
#pragma unroll
  for (int j = 0; j < kBN; ++j) {
    if (j < cols) storeScaled(p, c, v[j]);
    c += p.ldc;
  }
}

template <class G>
__global__ void __launch_bounds__(kThinThreads, 1)
    thinProductKernel(const __grid_constant__ Params p, int split) {
  constexpr int kBN = G::kBN;
  constexpr int kStages = G::kStages;
  constexpr int kStageBytes = G::kStageBytes;
  constexpr int kPitch = G::kPartPitch;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ GroupTable table;
  unsigned char *smem = smem_raw + ((1024 - (smemAddr(smem_raw) & 1023)) & 1023);
  float *part = reinterpret_cast<float *>(smem + kStages * kStageBytes);
  float *scales =
      reinterpret_cast<float *>(smem + kStages * kStageBytes + G::kPartBytes);
  uint64_t *full = reinterpret_cast<uint64_t *>(reinterpret_cast<unsigned char *>(scales) +
                                                G::kScaleBytes);
  uint64_t *empty = full + kStages;
  uint64_t *acc_full = empty + kStages;
  uint64_t *acc_empty = acc_full + G::kThinAccums;
  uint64_t *part_full = acc_empty + G::kThinAccums;   // every CTA's sums of this one's rows are here
  uint64_t *part_free = part_full + 1;                // every CTA has read this one's

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
      mbarInit(&full[s], 1);
      mbarInit(&empty[s], 1);
    }
    for (int b = 0; b < G::kThinAccums; ++b) {
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
  const int iters = (p.k + G::kBK - 1) / G::kBK;
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
        if constexpr (G::kAMN) {
          for (int j = 0; j < kBM / 64; ++j)
            tmaLoad3d(sa + j * 64 * kRowBytes, &p.tma_a, &full[s], t.m0 + 64 * j, kb * G::kBK,
                      t.group);
        } else {
          tmaLoad3d(sa, &p.tma_a, &full[s], kb * G::kBK, t.m0, t.group);
        }
        for (int j = 0; j < boxes; ++j)
          tmaLoad3d(sa + G::kABytes + j * kThinBox * kRowBytes, &p.tma_b, &full[s], kb * G::kBK,
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
  } else if (warp == 1 && electOne()) {
    // ---------------- MMA issuer ----------------
    int s = 0, parity = 0;
    int b = 0, acc_parity = 1;
    const uint64_t desc_a = smemDesc<G::kAMN>(smemAddr(smem));
    const uint64_t desc_b = smemDesc<false>(smemAddr(smem) + G::kABytes);
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      const uint32_t idesc = instrDesc<G>(p.format, (t.cols + 15) / 16 * 16);
      int in_chunk = 0;
      for (int j = 0; j < mine; ++j) {
        const bool first = in_chunk == 0;
        const bool last = ++in_chunk == p.chunk_iters || j == mine - 1;
        if (last) in_chunk = 0;
        if (first) wait(&acc_empty[b], acc_parity);
        wait(&full[s], parity);
        tcgenFenceAfter();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(b * kBN);
        constexpr uint64_t kNextA = (G::kAMN ? 16 * kRowBytes : 32) / 16;
        uint64_t ad = desc_a + static_cast<uint64_t>(s) * (kStageBytes / 16);
        uint64_t bd = desc_b + static_cast<uint64_t>(s) * (kStageBytes / 16);
#pragma unroll
        for (int q = 0; q < G::kBK / G::kMmaK; ++q) {
          mmaNarrow<G::kBytes>(d_tmem, ad, bd, idesc, !first || q > 0);
          ad += kNextA;
          bd += 2;
        }
        mmaCommit(&empty[s]);
        if (last) {
          mmaCommit(&acc_full[b]);
          if (++b == G::kThinAccums) {
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
    int batches = 0;   // scale batches staged so far
    // Fetches the scales of up to kThinScales blocks from this CTA's block j
    // of tile t into the next buffer; zeros where there are none.
    auto fetchScales = [&](const Tile &t, int j) {
      float *dst = scales + (batches & 1) * kThinScales * G::kScalePitch;
      const int live = mine - j;
      const int c = etid % kBN;
      const bool in = c < t.cols;
      const float *sb = p.scale_b + static_cast<size_t>(in ? t.n0 + c : 0) * p.ldsb + kb0 + j;
      for (int q = etid / kBN; q < kThinScales; q += kThinEpilogue / kBN) {
        const bool there = in && q < live;
        cpAsync4(dst + q * G::kScalePitch + c, there ? sb + q : p.scale_b, there ? 4 : 0);
      }
      if (etid < kThinScales) {
        const float *sa = p.scale_a + t.group * p.stride_sa +
                          static_cast<size_t>(t.m0 / 128) * p.ldsa + kb0 + j + etid;
        const bool there = etid < live;
        cpAsync4(dst + etid * G::kScalePitch + kBN, there ? sa : p.scale_a, there ? 4 : 0);
      }
      cpAsyncCommit();
      ++batches;
    };
    if constexpr (G::kBytes) {
      if (worker < tiles && mine > 0) fetchScales(tileAt<G>(p, table, worker), 0);
    }
    for (int i = worker; i < tiles; i += workers) {
      const Tile t = tileAt<G>(p, table, i);
      float acc[kBN];
#pragma unroll
      for (int j = 0; j < kBN; ++j) acc[j] = 0.0F;
      const float *batch = nullptr;
      for (int ch = 0; ch < chunks; ++ch) {
        const float *sc = nullptr;
        if constexpr (G::kBytes) {
          if (ch % kThinScales == 0) {
            batch = scales + ((batches - 1) & 1) * kThinScales * G::kScalePitch;
            cpAsyncWait<0>();
            namedBarrier<1, kThinEpilogue>();   // staged by all; the other buffer is free
            if (ch + kThinScales < chunks) fetchScales(t, ch + kThinScales);
            else if (i + workers < tiles) fetchScales(tileAt<G>(p, table, i + workers), 0);
          }
          sc = batch + ch % kThinScales * G::kScalePitch;
        }
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
            float block_scale = 0.0F;
            if constexpr (G::kBytes) block_scale = sc[kBN];
#pragma unroll
            for (int j = 0; j < kLoad; j += 4) {
              if constexpr (G::kBytes) {
                const float4 s4 = *reinterpret_cast<const float4 *>(sc + c + j);
                acc[c + j] = fmaf(__uint_as_float(v[j]), s4.x * block_scale, acc[c + j]);
                acc[c + j + 1] = fmaf(__uint_as_float(v[j + 1]), s4.y * block_scale, acc[c + j + 1]);
                acc[c + j + 2] = fmaf(__uint_as_float(v[j + 2]), s4.z * block_scale, acc[c + j + 2]);
                acc[c + j + 3] = fmaf(__uint_as_float(v[j + 3]), s4.w * block_scale, acc[c + j + 3]);
              } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[c + j + q] += __uint_as_float(v[j + q]);
              }
            }
          }
        }
        tcgenFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArrive(&acc_empty[b]);
        if (++b == G::kThinAccums) {
          b = 0;
          acc_parity ^= 1;
        }
      }
      if (split == 1) {
        // A warp writes 32 rows of a column.
        if (t.m0 + row < p.m) {
          const size_t at = static_cast<size_t>(t.n0) * p.ldc + t.m0 + row;
          if (p.c_bf16) storeRow<kBN>(p, static_cast<__nv_bfloat16 *>(p.c) + at, t.cols, acc);
          else storeRow<kBN>(p, static_cast<float *>(p.c) + at, t.cols, acc);
        }
        continue;
      }
      // Each row's sums to the CTA that writes the row: into the block of its
      // shared memory that is this CTA's.
      if (ok) ok = mbarWaitCluster(part_free, part_parity ^ 1, p.err);   // of the tile before
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
          storeAsyncCluster4(to + static_cast<uint32_t>(j) * 4, bar, acc[j], acc[j + 1],
                             acc[j + 2], acc[j + 3]);
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

#endif  // SGBLAS_B200_PRODUCT_THIN_CUH_
