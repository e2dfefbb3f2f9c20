// How a product of few rows is laid out (few_rows_kernel.cuh): host arithmetic
// alone, so that it can be gone over without a GPU.
#pragma once
#include <cstdint>

namespace mlpk {

constexpr int kFewMostRows = 256;    // of a tile: the instruction's N
constexpr int kFewMaxStages = 8;
constexpr int kFewWBytes = 128 * 64 * 2;  // a stage's weights
constexpr int kFewMaxRanks = 8;      // the portable cluster size

struct FewPlan {
  int nt = 0;      // rows of a tile
  int stages = 0;  // depth of the ring
  int ranks = 0;   // CTAs that share a tile's reduction
  int tiles = 0, row_tiles = 0;
};

// Bytes of dynamic shared memory: the ring (which the fp32 tile reuses), barriers.
inline int few_smem(int nt, int stages) {
  const int ring = stages * (kFewWBytes + nt * 128), tile = nt * 128 * 4;
  return 1024 + (ring > tile ? ring : tile) + 8 * (2 * kFewMaxStages + 1) + 32;
}

// tile_cols: weight columns of a tile; nk: blocks of 64 of the reduction.
inline FewPlan few_plan(int64_t rows, int cols, int nk, int tile_cols, int sm_count) {
  FewPlan p;
  p.nt = 16;
  while (p.nt < rows && p.nt < kFewMostRows) p.nt *= 2;
  // Two CTAs an SM for the narrowest tiles, one for the others: a wide tile meets
  // in more shared memory than it is worth to share it further (128 x 4096 x 4096
  // bf16: 8 ranks 15.6 us, 4 ranks 11.4).
  const int each_sm = p.nt <= 32 ? 2 : 1;
  p.stages = kFewMaxStages;
  while (p.stages > 2 && few_smem(p.nt, p.stages) > (each_sm == 2 ? 113 * 1024 : 226 * 1024)) --p.stages;
  p.tiles = (cols + tile_cols - 1) / tile_cols;
  p.row_tiles = static_cast<int>((rows + p.nt - 1) / p.nt);
  // As many shares as fill the SMs in one go, 4 blocks in each at least.
  p.ranks = 1;
  while (p.ranks < kFewMaxRanks && static_cast<int64_t>(p.tiles) * p.row_tiles * p.ranks * 2 <= each_sm * sm_count &&
         nk >= p.ranks * 2 * 4)
    p.ranks *= 2;
  return p;
}

}  // namespace mlpk
