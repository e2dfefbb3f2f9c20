// How a product of few rows is laid out (few_rows_kernel.cuh): host arithmetic
// alone, so that it can be gone over without a GPU.
#pragma once
#include <cstdint>
#include <initializer_list>

namespace mlpk {

constexpr int kFewMostRows = 256;    // of a tile: the instruction's N
constexpr int kFewMaxStages = 8;
constexpr int kFewWBytes = 128 * 64 * 2;  // a stage's weights
constexpr int kFewMaxRanks = 8;      // the portable cluster size

struct FewPlan {
  int nt = 0;      // rows of a tile, a multiple of 16 up to 256
  int stages = 0;  // depth of the ring
  int ranks = 0;   // CTAs that share a tile's reduction
  int each_sm = 0; // CTAs that an SM is to hold
  int tiles = 0, row_tiles = 0;
  double us = 0.0;  // about what it takes, where the weights are in L2
};

// Bytes of dynamic shared memory: the ring (which the fp32 tile reuses), barriers.
inline int few_smem(int nt, int stages) {
  const int ring = stages * (kFewWBytes + nt * 128), tile = nt * 128 * 4;
  return 1024 + (ring > tile ? ring : tile) + 8 * (2 * kFewMaxStages + 1) + 32;
}

// tile_cols: weight columns of a tile; nk: blocks of 64 of the reduction.
inline FewPlan few_plan(int64_t rows, int cols, int nk, int tile_cols, int sm_count) {
  FewPlan p;
  // As few tiles of rows as their most allows, alike, of a multiple of 16.
  p.row_tiles = static_cast<int>((rows + kFewMostRows - 1) / kFewMostRows);
  p.nt = static_cast<int>((rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles)) * 16;
  p.tiles = (cols + tile_cols - 1) / tile_cols;
  // Shares of a tile's reduction: as many as fill the SMs in one go with `each`
  // CTAs, 4 blocks in each at least, 2 where that is few CTAs (64 x 256 x 256 fp16: 4
  // shares of one tile's 4 blocks 6.2 us, 2 shares 6.0, one 6.7).  A cluster has its
  // SMs from one part of the chip, so larger ones leave some out: a ninth of them, or
  // a fifth with clusters of 8 that have an SM a CTA (15 of them on 148 SMs); beyond
  // that, and with clusters of 7, or of 3 with an SM a CTA, they ended in two goes (8
  // x 5120 x 5120 bf16: 7 shares 15.1 us, 4 shares 10.6; 64 x 2048 x 5120: 3 shares
  // 17.2, 2 shares 10.1).
  const int64_t tiles = static_cast<int64_t>(p.tiles) * p.row_tiles;
  const auto shares = [&](int each) {
    for (int n : {8, 4, 3, 2}) {
      const int left_out = n == 2 ? 8 : n == 8 && each == 1 ? 10 : 9;  // in eighths
      if ((n != 3 || each == 2) && tiles * n * left_out <= static_cast<int64_t>(each) * sm_count * 8 && nk >= (tiles * n <= 64 ? 2 : 4) * n)
        return n;
    }
    return 1;
  };
  // One CTA an SM with a deep ring, which also leaves room for the next kernel's
  // CTAs to begin, where two would not have more of the SMs at work (weights from
  // memory: 1 x 4096 x 4096 bf16 10.5 us with two of 8 shares, 9.8 with one of 4; 1 x
  // 14336 x 4096, gated, 39.5 and 37.4; 128 x 4096 x 4096 15.6 and 11.4, where the
  // shares meet in more shared memory than it is worth.  But 48 x 4096 x 14336, gated,
  // 224 tiles: two an SM 39.5, one 45.0; 64 x 4096 x 11008, 86 tiles: three shares
  // 17.1, one 21.1).
  const int64_t one = tiles * shares(1), two = tiles * shares(2);
  const bool fuller = 20 * two > 23 * 2 * (one < sm_count ? one : sm_count) || one > sm_count;
  p.each_sm = p.nt <= 128 && fuller ? 2 : 1;
  p.ranks = shares(p.each_sm);
  p.stages = kFewMaxStages;
  while (p.stages > 2 && few_smem(p.nt, p.stages) > (p.each_sm == 2 ? 113 * 1024 : 226 * 1024)) --p.stages;
  // Shares of the blocks at 115 GB/s an SM and the tile's way through shared memory
  // at 45 GB/s (its own and the others'; longer where 8 meet: 1500 x 2048
  // x 256 bf16 15.1 us), for each CTA that an SM has.
  const int64_t ctas = tiles * p.ranks, room = static_cast<int64_t>(p.each_sm) * sm_count;
  const double turns = ctas <= sm_count ? 1.0
                       : ctas <= room   ? static_cast<double>(ctas) / sm_count
                                        : static_cast<double>((ctas + room - 1) / room * p.each_sm);
  const double block = (kFewWBytes + 128.0 * p.nt) / 115e3, meet = 512.0 * p.nt * (p.ranks == 8 ? 3.0 : 2.0 - 1.0 / p.ranks) / 45e3;
  p.us = 3.5 + turns * ((nk + p.ranks - 1) / p.ranks * block + 1.0 + meet);
  return p;
}

}  // namespace mlpk
