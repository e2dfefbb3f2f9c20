// How a product in tiles of 256 rows is laid out over the pairs of CTAs
// (product_kernel.cuh): host arithmetic alone, so that it can be gone over without
// a GPU.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define MLPK_HOST_DEVICE __host__ __device__
#else
#define MLPK_HOST_DEVICE
#endif

namespace mlpk {

struct ProductPlan {
  int cols = 256;     // columns of a tile, of both matrices together for the gate
  int64_t full = 0;   // tiles computed whole, the first ones
  int64_t tail = 0;   // tiles that `splits` items share, the last ones
  int splits = 1;     // shares of a tail tile's reduction; 1: it is computed whole too
  double us = 0.0;    // about what it takes
  int64_t items() const { return full + tail * splits; }
  // fp32 values that the shares leave in the workspace.
  int64_t partials() const { return splits > 1 ? tail * splits * 256 * cols : 0; }
};

// rows, cols: of each output; out_cols: columns of an output that a tile of 256 has;
// nk: blocks of 64 of the reduction; may_split, may_narrow, may_any: whether the
// product's epilogue allows shares, tiles of 128 columns, tiles of 160 to 224.
//
// The tiles go over the pairs in turns; a turn takes nk blocks' time: 0.3 us each at
// 256 columns, less for narrower tiles, but not in their proportion (their rows are
// loaded for fewer products).  Narrower ones pay where they fill the last turn
// better (a linear layer, bf16, us: 2000 x 5120 x 1280 in 40 tiles of 256 columns
// 33.4, in 64 of 160 26.3; 3000 x 2048 x 5120 in 240 of 256 55.9, in 276 of 224 52.4;
// 8192 x 1024 x 4096 in 512 of 256 58, in 1024 of 128 85).  What is left behind the
// last full turn of tiles of 256 or 128 columns may be shared out over all pairs in
// shares of the reduction: ceil(tail splits / pairs) turns of nk / splits blocks,
// the traffic of the shares (0.5 us a megabyte, written and read) and a second
// kernel (4 us); dw of 20011 x 1024 x 2816: 136 whole, 119 so.  A kernel's beginning
// and end are 5 us.
//
// The estimate compares tiles of one product; it has no term for the epilogue.  One
// that keeps z, adds a residual and evaluates an activation beside a short reduction
// takes longer than it says (5003 x 1000 x 2056 fp16, bias, gelu, residual, z kept:
// 32 us, the estimate 18).
inline ProductPlan product_plan(int64_t rows, int cols, int outputs, int out_cols, int nk, int pairs, bool may_split,
                                bool may_narrow, bool may_any) {
  ProductPlan best;
  for (int wide = 256; wide >= 128; wide -= 32) {
    if (wide == 128 ? !may_narrow : wide < 256 && !may_any) continue;
    const int each = wide * out_cols / 256;
    const int64_t tiles = (rows + 255) / 256 * ((cols + each - 1) / each) * outputs;
    const double block_us = wide == 128 ? 0.21 : 0.3 * (512 + wide) / 768.0;
    const int64_t left = tiles % pairs;
    const double full_us = 5.0 + static_cast<double>(tiles / pairs) * nk * block_us;
    const int most = may_split && left && wide % 128 == 0 ? (nk / 4 < 32 ? nk / 4 : 32) : 1;
    for (int splits = 1; splits <= (most > 1 ? most : 1); ++splits) {
      ProductPlan p;
      p.cols = wide;
      p.splits = splits;
      p.tail = splits > 1 ? left : 0;
      p.full = tiles - p.tail;
      double us = full_us;
      if (left) us += static_cast<double>((left * splits + pairs - 1) / pairs) * ((nk + splits - 1) / splits) * block_us;
      if (splits > 1) us += 4.0 + 0.5 * 4e-6 * static_cast<double>(p.partials());
      p.us = us;
      if (best.us == 0.0 || us < best.us) best = p;
    }
  }
  return best;
}

// The t-th tile: row tiles in groups of `group`, over all column tiles of all
// outputs.
struct TileAt {
  int m, n, output;
};
MLPK_HOST_DEVICE inline TileAt product_tile(int t, int tiles_m, int tiles_n, int outputs, int group) {
  const int wide = tiles_n * outputs;
  TileAt at;
  const int first = t / (group * wide) * group;
  const int high = tiles_m - first < group ? tiles_m - first : group;
  t -= first * wide;
  at.m = first + t % high;
  const int n = t / high;
  at.output = n / tiles_n;
  at.n = n - at.output * tiles_n;
  return at;
}

// Where the share of an item's value in `row` (of 256) and the 4 columns from
// `col` (a multiple of 4) lies among the item's values, in units of 4: each
// epilogue warp has runs of 32 rows x 32 columns, the 8 units of a row turned
// around by the row (as its shared memory has them, against bank conflicts).
// Epilogue warp w has the rows from 32 ((w + 2) % 4) on of its CTA's 128, and every
// fourth run of columns from the (w / 4)-th on.
MLPK_HOST_DEVICE inline int share_unit(int row, int col, int tile_cols) {
  const int chunks = tile_cols / 128;
  const int rank = row / 128, quarter = row % 128 / 32, lane = row % 32;
  const int warp = col / 32 % 4 * 4 + (quarter + 2) % 4, chunk = col / 128;
  return ((rank * 16 + warp) * chunks + chunk) * 256 + lane * 8 + ((col % 32 / 4) ^ (lane % 8));
}

}  // namespace mlpk
