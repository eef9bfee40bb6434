// The places where layScalesKernel (csrc/product_fp4.cuh) writes a pair product's scale
// blocks, on the host: inside the workspace's room whatever the offsets hold, and each
// block of a group that has columns once where they do not decrease. Run by
// tests/test_laid_scales.py.
#include "product_fp4.cuh"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <memory>
#include <vector>

using namespace sgblas::kern::prod;
using G = Fp4Cfg<192, true, false>;

// As readGroups fills it.
void fill(const Params &p, const std::vector<int> &offsets, GroupTable *t) {
  int sum = 0;
  for (int g = 0; g < p.groups; ++g) {
    const int begin = std::min(std::max(offsets[g], 0), p.n), end = std::min(std::max(offsets[g + 1], 0), p.n);
    t->offset[g] = begin;
    t->first[g] = sum;
    sum += (std::max(0, end - begin) + G::kBN - 1) / G::kBN;
    t->offset[g + 1] = end;
  }
  t->first[p.groups] = sum;
}

// 0: right; otherwise what is not.
int check(int m, int n, int k, const std::vector<int> &offsets, bool sorted) {
  auto f = std::make_unique<Fp4Params>();
  auto table = std::make_unique<GroupTable>();
  Params &p = f->p;
  p.m = m;
  p.n = n;
  p.k = (k + 1) / 2;
  p.groups = static_cast<int>(offsets.size()) - 1;
  p.tiles_m = (m - 1) / G::kTileM + 1;
  f->blocks = (k + 31) / 32;
  f->ldsa = f->ldsb = f->blocks;
  f->stride_sa = static_cast<long long>(m) * f->ldsa;
  fill(p, offsets, table.get());
  const LaidSize size = laidSize<G>(p);
  f->laid_tiles = static_cast<int>(size.tiles);
  std::vector<unsigned char> room(size.a + size.b), scale_a(f->stride_sa * p.groups), scale_b(static_cast<long long>(n) * f->ldsb);
  f->laid_a = room.data();
  f->laid_b = room.data() + size.a;
  f->scale_a = scale_a.data();
  f->scale_b = scale_b.data();
  const int iters = (p.k + kRowBytes - 1) / kRowBytes;
  const long long items = laidItems<G>(*f, *table), items_a = laidItemsA(p);
  for (long long i = 0; i < items; ++i) {
    const LaidItem it = laidItem<G>(*f, *table, i);
    if (i < items_a && it.rows <= 0) continue;
    const unsigned char *low = i < items_a ? f->laid_a : f->laid_b, *high = low + (i < items_a ? size.a : size.b);
    for (int s = 0; s < (2 * it.chunk + 1 < iters ? 2 : 1); ++s) {
      for (int half = 0; half < 2; ++half) {
        unsigned char *to = it.to + s * it.slice + half * it.next;
        if (to < low || to + kScaleBlock > high) return 1;
        for (int b = 0; b < kScaleBlock; ++b) ++to[b];
      }
    }
    const int rows = std::min(it.rows, kBM), bytes = std::min(16, f->blocks - it.chunk * 16);
    if (rows > 0) {
      const unsigned char *first = it.from + it.chunk * 16, *last = first + static_cast<long long>(rows - 1) * it.ld + bytes;
      const std::vector<unsigned char> &source = i < items_a ? scale_a : scale_b;
      if (bytes < 1 || first < source.data() || last > source.data() + source.size()) return 2;
    }
  }
  if (!sorted) return 0;
  for (int g = 0; g < p.groups; ++g) {
    const long long per = size.a / p.groups;
    for (long long b = 0; b < per; ++b)
      if (room[g * per + b] != (table->offset[g + 1] > table->offset[g] ? 1 : 0)) return 3;
  }
  const long long used = static_cast<long long>(table->first[p.groups]) * iters * kScaleRowsB * kScaleRowBytes;
  for (long long b = 0; b < size.b; ++b)
    if (room[size.a + b] != (b < used ? 1 : 0)) return 4;
  return 0;
}

int main() {
  std::srand(1);
  int cases = 0;
  for (const int n : {1, 191, 192, 193, 1000, 5000}) {
    for (const int groups : {1, 2, 3, 64, 1024}) {
      for (const int k : {1, 256, 257, 512, 513, 2120}) {
        const int m = groups > 3 ? 300 : 700;
        std::vector<int> sorted(groups + 1), swinging(groups + 1), wild(groups + 1), back(groups + 1);
        for (int g = 0; g <= groups; ++g) {
          sorted[g] = std::rand() % (n + 1);
          swinging[g] = g % 2 == 0 ? 0 : n;
          wild[g] = std::rand() - RAND_MAX / 2;
          back[g] = n - g;
        }
        std::sort(sorted.begin(), sorted.end());
        const std::vector<int> *all[] = {&sorted, &swinging, &wild, &back};
        for (const auto *offsets : all) {
          const int wrong = check(m, n, k, *offsets, offsets == &sorted);
          if (wrong != 0) {
            std::printf("n %d groups %d k %d: %d\n", n, groups, k, wrong);
            return 1;
          }
          ++cases;
        }
      }
    }
  }
  std::printf("%d\n", cases);
  return 0;
}
