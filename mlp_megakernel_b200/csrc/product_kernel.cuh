// The matrix products of the feed-forward operators on tensor cores, with what
// stands behind each product in its epilogue:
//
//   kEpiPlain     D = A B                                     (dx, dW)
//   kEpiLinear    z = A B + bias; out = act(z) + residual; z kept for the backward
//   kEpiGated     g = A Bg, u = A Bu; h = act(g) u; g and u kept for the backward
//   kEpiGatedBwd  dh = A B; dg = dh u act'(g), du = dh act(g), h = act(g) u again
//
// A tile of D is 256 rows x TN columns (kEpiPlain, and kEpiLinear without 8-bit
// values: any multiple of 32 up to TN) of a pair of CTAs (pair.cuh), reduced in
// blocks of 64 through a ring of TMA loads; operands are fp16 or bf16 in either
// order (K contiguous, or the row / column index), chosen at run time by the
// descriptors alone.  Roles of a CTA: warp 0 loads, warp 1 of the leader issues
// the tcgen05 instructions, warps 2..17 are the epilogue (thread = row; four warps
// share the 32 rows of a TMEM lane quarter and have a quarter of the runs of 32
// columns each: an epilogue is a chain of waits, and eight warps left the gate's
// backward at twice the time of its products).  Two accumulators of TN columns, so
// the epilogue of a tile runs beside the products of the next.  The kernel is
// persistent: tiles are taken in groups of `group` row tiles over all column tiles,
// so that the pairs at work share rows and columns in L2.  The tiles behind the
// last full turn of the pairs may be shared out (kEpiPlain, and kEpiLinear that
// keeps nothing): an item is then a share of a tile's reduction, whose fp32 values
// go to a workspace, and tail_sum_kernel adds them in order and runs the epilogue.
// All tiles' first shares come first: the pairs at work then read one part of the
// operands (2816 x 20011 x 1024: 309 MB from memory tile by tile, 177 so).
//
// Everything between the operands and the stored values is fp32: accumulators,
// bias, activation, residual.  What is kept for the backward is rounded once, to
// the operands' type (as a 16-bit activation is anywhere else in training; a finite
// value beyond the type's largest becomes that, vec.cuh's kept_pair) or to 8 bits
// with a scale for each row and 128 columns (act.cuh).
#pragma once
#include "act.cuh"
#include "layout.cuh"
#include "pair.cuh"
#include "product_epi.cuh"
#include "product_plan.cuh"

namespace mlpk {

enum Keep : int { kKeepNone = 0, kKeep16 = 1, kKeep8 = 2 };

constexpr int kPairRows = 256;      // rows of a pair's tile
constexpr int kBlockK = 64;         // reduction of a stage: one 128-byte row of 16-bit values
constexpr int kKeepGroup = 128;     // columns that share a scale
constexpr int kEpiWarps = 16;
constexpr int kProductThreads = 32 * (2 + kEpiWarps);

struct alignas(64) ProductArgs {
  CUtensorMap a[2], b[2];  // [1]: the second reduction range (nk0 < nk), or the gate's partner / second output's B
  CUtensorMap out[2];      // plain: D (two of them with `outputs` 2); linear: out; gated: h; backward: dg, du
  CUtensorMap keep[2];     // linear: z; gated: g, u; backward: h
  CUtensorMap in[2];       // backward: g, u (16 bits)
  int rows, cols;          // of each output
  int nk0, nk;             // blocks of the first reduction range, and of both
  int tile_cols, b_bytes;  // columns of a tile (at most TN), bytes of a CTA's loads of B in a stage
  int tiles_m, tiles_n, outputs, group;
  int full, splits, items; // tiles computed whole, shares of each of the others, and both together
  int a_mn, b_mn;          // the operand's contiguous index is the row / column, not the reduction
  int out_a;               // with two outputs: A differs, not B
  uint32_t idesc;
  int act, keep_kind, bias32;
  const void* bias;
  const void* residual;
  uint8_t* q[2];           // 8-bit values, rows of q_pitch bytes
  float* scale[2];         // [rows][scale_pitch]
  int64_t q_pitch;
  int scale_pitch;
  float* partials;         // of the shares, each as share_unit says
  int* status;
};

template <int EPI, int TN>
struct ProductCfg {
  static constexpr int A_BYTES = 128 * kBlockK * 2;
  static constexpr int B_BYTES = TN / 2 * kBlockK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int OUT_COLS = EPI == kEpiGated ? TN / 2 : TN;  // columns of an output that a tile has
  static constexpr int PART = OUT_COLS / 4;  // columns of an epilogue warp
  // A warp's unit of TMA traffic: 32 rows of at most 32 columns, in two buffers
  // in turn.
  static constexpr int CHUNK = PART < 32 ? PART : 32;
  static constexpr int PITCH = CHUNK * 2;
  static constexpr int TILE = 32 * PITCH;
  static constexpr int BUFS = 2;
  static constexpr int OFF_EPI = 0;
  static constexpr int EPI_BYTES = kEpiWarps * BUFS * TILE;
  static constexpr int STAGES_FIT = (227 * 1024 - 2048 - EPI_BYTES) / STAGE;
  static constexpr int STAGES = STAGES_FIT < 8 ? STAGES_FIT : 8;
  static constexpr int OFF_STAGE = EPI_BYTES;
  static constexpr int OFF_BAR = OFF_STAGE + STAGES * STAGE;
  static constexpr int NUM_BARS = 2 * STAGES + 5 + kEpiWarps;
  static constexpr int OFF_MISC = OFF_BAR + 8 * NUM_BARS;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
  static constexpr int CHUNKS = PART / CHUNK;
  static_assert(EPI_BYTES % 1024 == 0 && STAGE % 1024 == 0 && SMEM <= 227 * 1024, "shared memory");
  static_assert(STAGES >= 3 && (TN == 128 || TN == 256), "tile");
};

// The tile and the blocks of the t-th item.
struct ItemAt {
  TileAt tile;
  int k0, k1, share;  // share: below 0 for a whole tile
};
__device__ __forceinline__ ItemAt product_item(const ProductArgs& p, int t) {
  ItemAt it;
  it.share = t - p.full;
  int tile = t;
  it.k0 = 0;
  it.k1 = p.nk;
  if (it.share >= 0) {
    const int tail = (p.items - p.full) / p.splits, s = it.share / tail;
    tile = p.full + it.share - s * tail;
    it.k0 = static_cast<int>(static_cast<int64_t>(s) * p.nk / p.splits);
    it.k1 = static_cast<int>(static_cast<int64_t>(s + 1) * p.nk / p.splits);
  }
  it.tile = product_tile(tile, p.tiles_m, p.tiles_n, p.outputs, p.group);
  return it;
}

// Shared memory to consecutive global memory (16-byte units).
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld_wait_x32(taddr, r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 values of a row to 8 bits (q is 32-byte aligned).
__device__ __forceinline__ void store_fp8x32(uint8_t* q, const float (&v)[32], float inv) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t lo = to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv));
    const uint32_t hi = to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv));
    w[i] = lo | hi << 16;
  }
  reinterpret_cast<uint4*>(q)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(q)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
// 16 of a row's 8-bit values (4 words of them) as fp32.
__device__ __forceinline__ void widen_fp8x16(const uint32_t* w, float scale, float (&v)[16]) {
  Raw<uint16_t, 8> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[2 * i] = static_cast<uint16_t>(w[i]), r.v[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
  float2 f[8];
  unpack_fp8<16>(r, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[2 * i] = f[i].x * scale, v[2 * i + 1] = f[i].y * scale;
}

// v += bias[col ..]; a vector of 8 columns is inside the tensor or outside.
template <class T>
__device__ __forceinline__ void add_bias(const ProductArgs& p, int col, float (&v)[32]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (col + 8 * k >= p.cols) break;
    float b[8];
    if (p.bias32) {
      const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + col + 8 * k);
      const float4 x = __ldg(f), y = __ldg(f + 1);
      b[0] = x.x, b[1] = x.y, b[2] = x.z, b[3] = x.w, b[4] = y.x, b[5] = y.y, b[6] = y.z, b[7] = y.w;
    } else {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.bias) + col + 8 * k));
      unpack<T, 8>(*reinterpret_cast<const Raw<T, 8>*>(&x), b);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[8 * k + e] += b[e];
  }
}

// 32 values of a row, 16 bits each, from `at` on: those of `cols` columns (a
// multiple of 8), zeros beyond.  A thread takes its own row: whole sectors of 32
// bytes where the rows are aligned to them.
template <class T>
__device__ __forceinline__ void row_load32(const void* in, int64_t at, int cols, uint32_t (&p)[16]) {
  const T* src = static_cast<const T*>(in) + at;
  if (cols >= 32 && reinterpret_cast<uintptr_t>(src) % 32 == 0) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(p[8 * k]), "=r"(p[8 * k + 1]), "=r"(p[8 * k + 2]), "=r"(p[8 * k + 3]), "=r"(p[8 * k + 4]),
                     "=r"(p[8 * k + 5]), "=r"(p[8 * k + 6]), "=r"(p[8 * k + 7])
                   : "l"(src + 16 * k)
                   : "memory");
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (8 * k < cols) v = *reinterpret_cast<const uint4*>(src + 8 * k);
    p[4 * k] = v.x, p[4 * k + 1] = v.y, p[4 * k + 2] = v.z, p[4 * k + 3] = v.w;
  }
}
// Pairs of the type as fp32.
template <class T>
__device__ __forceinline__ float2 widen(uint32_t p) {
  return to_float2(*reinterpret_cast<const typename Pair<T>::type*>(&p));
}
// N values of a thread's row, from column `from` on, into and from its tile in
// shared memory (as a TMA box with the row's swizzle has it).  CLIP: kept_pair for
// each pair; tile_keep: for a backward pass to read.
template <class T, int PITCH, bool CLIP = false, int N>
__device__ __forceinline__ void tile_store(uint32_t tile, int lane, int from, const float (&v)[N]) {
#pragma unroll
  for (int u = 0; u < N / 8; ++u) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = v[8 * u + 2 * i], b = v[8 * u + 2 * i + 1];
      p[i] = CLIP ? kept_pair<T>(a, b) : round_pair<T>(a, b);
    }
    st_shared_v4(tile + swz_off<PITCH>(lane, from / 8 + u), p[0], p[1], p[2], p[3]);
  }
}
template <class T, int PITCH, int N>
__device__ __forceinline__ void tile_keep(uint32_t tile, int lane, int from, const float (&v)[N]) {
  if (some_round_to_infinity<T>(v)) tile_store<T, PITCH, true>(tile, lane, from, v);
  else tile_store<T, PITCH>(tile, lane, from, v);
}
template <class T, int PITCH, int N>
__device__ __forceinline__ void tile_load(uint32_t tile, int lane, int from, float (&v)[N]) {
#pragma unroll
  for (int u = 0; u < N / 8; ++u) {
    uint32_t p[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
                 : "r"(tile + swz_off<PITCH>(lane, from / 8 + u))
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = widen<T>(p[i]);
      v[8 * u + 2 * i] = f.x;
      v[8 * u + 2 * i + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  tmem_ld_wait_x16(taddr, r);
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ float most_of(float most, const float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) most = max_abs(most, v[i], v[i + 1]);
  return most;
}

template <class T, int EPI, int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kProductThreads, 1)
    product_kernel(const __grid_constant__ ProductArgs p) {
  using Cfg = ProductCfg<EPI, TN>;
  constexpr int ST = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;  // the same offset in both CTAs
  uint8_t* gbase = smem_raw + (sbase - raw);
  const uint32_t s_stage = sbase + Cfg::OFF_STAGE, s_bar = sbase + Cfg::OFF_BAR;
  auto bar_full = [&](int s) { return s_bar + 8u * s; };          // leader: both CTAs' loads have landed
  auto bar_empty = [&](int s) { return s_bar + 8u * (ST + s); };  // both: the products have read the stage
  auto bar_acc = [&](int b) { return s_bar + 8u * (2 * ST + b); };       // both: accumulator b is complete
  auto bar_free = [&](int b) { return s_bar + 8u * (2 * ST + 2 + b); };  // leader: both epilogues have read it
  const uint32_t bar_done = s_bar + 8u * (2 * ST + 4);
  auto bar_in = [&](int w) { return s_bar + 8u * (2 * ST + 5 + w); };  // a warp's tiles of `in` have landed
  const uint32_t s_tmem = sbase + Cfg::OFF_MISC;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + Cfg::OFF_MISC + 4);
  volatile int no_abort = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int total = p.items;
  const int step = static_cast<int>(cluster_count());
  int* const status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc(b), 1);
      mbar_init(bar_free(b), 2 * kEpiWarps);
    }
    mbar_init(bar_done, 1);
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(bar_in(w), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(s_tmem, 2 * TN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // the barriers of both CTAs are there before either arrives on the other's
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gbase + Cfg::OFF_MISC);
  pdl_enter();

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (elect_one()) {
      int issued = 0, s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = cluster_id(); ok && t < total; t += step) {
        const ItemAt item = product_item(p, t);
        const TileAt at = item.tile;
        const int k0 = item.k0, k1 = item.k1;
        const int row = at.m * kPairRows + static_cast<int>(rank) * 128;
        // A pair's half of B: columns, or for the gate its own matrix.
        const int col = EPI == kEpiGated ? at.n * (TN / 2) : at.n * p.tile_cols + static_cast<int>(rank) * (p.tile_cols / 2);
        const int own_a = p.out_a ? at.output : 0;
        const int own_b = EPI == kEpiGated ? static_cast<int>(rank) : p.out_a ? 0 : at.output;
        for (int kb = k0; kb < k1; ++kb, ++issued) {
          if (!mbar_wait_to(bar_empty(s), phase, abort_flag, kDevTimeoutEmpty, status)) {
            ok = false;
            break;
          }
          // The leader expects the bytes of both CTAs.  (An arrival of each CTA
          // on the leader's barrier, with its own bytes, needs a release at
          // cluster scope for every stage, and the products ran at half their
          // rate: 8192 x 4096 x 4096 bf16 380 us.)
          const uint32_t full = mapa_shared(bar_full(s), 0);
          if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * (Cfg::A_BYTES + p.b_bytes));
          const bool second = kb >= p.nk0;
          const int k = (second ? kb - p.nk0 : kb) * kBlockK;
          const CUtensorMap* ma = &p.a[second ? 1 : own_a];
          const CUtensorMap* mb = &p.b[second ? 1 : own_b];
          const uint32_t sa = s_stage + s * Cfg::STAGE, sb = sa + Cfg::A_BYTES;
          if (p.a_mn) {
#pragma unroll
            for (int c = 0; c < 2; ++c) tma_load_2d_pair(sa + c * kBlockK * 128, ma, full, row + 64 * c, k);
          } else {
            tma_load_2d_pair(sa, ma, full, k, row);
          }
          if (p.b_mn) {
#pragma unroll
            for (int c = 0; c < TN / 128; ++c) tma_load_2d_pair(sb + c * kBlockK * 128, mb, full, col + 64 * c, k);
          } else {
            tma_load_2d_pair(sb, mb, full, k, col);
          }
          if (++s == ST) s = 0, phase ^= 1;
        }
      }
      // After a wait that ran out: nothing of the loads may still be under way
      // when the CTAs end (the leader's barriers count both CTAs' bytes).
      if (!ok && rank == 0)
        for (int b = 0; b < ST && b < issued; ++b) {
          const int uses = (issued - b + ST - 1) / ST;
          mbar_wait_to(bar_full(b), (uses - 1) & 1, &no_abort, kDevTimeoutFull, status);
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ products (leader)
    // One elected thread does all of it: a warp that meets at each stage (a vote
    // on its wait, a __syncwarp behind its instructions) costs the products
    // their run-ahead.
    if (rank == 0 && elect_one()) {
      // K-step of 16: 32 bytes along a K-contiguous row, 16 rows of 128 bytes otherwise.
      const uint64_t a_step = p.a_mn ? 16 * 128 / 16 : 2, b_step = p.b_mn ? 16 * 128 / 16 : 2;
      const uint64_t a_base = make_sdesc(s_stage, p.a_mn ? kBlockK * 128 : 16, 1024, 2);
      const uint64_t b_base = make_sdesc(s_stage + Cfg::A_BYTES, p.b_mn ? kBlockK * 128 : 16, 1024, 2);
      const uint32_t idesc = p.idesc;
      bool ok = true;
      int s = 0, mine = 0;
      uint32_t phase = 0;
      for (int t = cluster_id(); ok && t < total; t += step, ++mine) {
        const ItemAt item = product_item(p, t);
        const int k0 = item.k0, k1 = item.k1;
        const int buf = mine & 1;
        const uint32_t d = tmem + buf * TN;
        ok = mbar_wait_to(bar_free(buf), ((mine >> 1) & 1) ^ 1, abort_flag, kDevTimeoutMma, status);
        if (!ok) break;
        tc_fence_after();
        uint32_t more = 0;  // the first product of a tile overwrites the accumulator
        for (int kb = k0; kb < k1; ++kb) {
          ok = mbar_wait_to(bar_full(s), phase, abort_flag, kDevTimeoutMma, status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = a_base + s * (Cfg::STAGE >> 4), db = b_base + s * (Cfg::STAGE >> 4);
#pragma unroll
          for (int kk = 0; kk < kBlockK / 16; ++kk) {
            umma_f16_pair(d, da + kk * a_step, db + kk * b_step, idesc, more);
            more = 1;
          }
          umma_commit_pair(bar_empty(s));
          if (++s == ST) s = 0, phase ^= 1;
        }
        if (ok) umma_commit_pair(bar_acc(buf));
      }
      umma_commit_pair(bar_done);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int w = warp - 2, quarter = warp & 3, part = w >> 2;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    constexpr int CHUNK = Cfg::CHUNK, PITCH = Cfg::PITCH;
    const uint32_t s_buf = sbase + Cfg::OFF_EPI + w * Cfg::BUFS * Cfg::TILE;
    // A warp's chunks: together where a group of columns has a scale, otherwise
    // every fourth, so that a tile may have any number of them.
    const bool together = EPI == kEpiGated || EPI == kEpiGatedBwd || p.keep_kind == kKeep8;
    const int apart = together ? Cfg::PART : CHUNK, next = together ? CHUNK : 4 * CHUNK;
    const bool by_tma = EPI == kEpiGatedBwd && p.keep_kind == kKeep16;  // g and u come as tiles
    bool ok = true;
    int turn = 0;  // tiles stored so far
    // The next of the two buffers, once the store that used it last has read it;
    // and its store.
    auto begin_tile = [&]() -> uint32_t {
      const uint32_t tile = s_buf + (turn++ & 1) * Cfg::TILE;
      if (lane == 0) bulk_wait_group_read<1>();
      __syncwarp();
      return tile;
    };
    auto end_tile = [&](const CUtensorMap* map, uint32_t tile, int col, int row) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(map, tile, col, row);
        bulk_commit_group();
      }
    };
    int mine = 0;
    uint32_t in_phase = 0;
    for (int t = cluster_id(); ok && t < total; t += step, ++mine) {
      const ItemAt item = product_item(p, t);
      const TileAt at = item.tile;
      const int buf = mine & 1;
      const int row0 = at.m * kPairRows + static_cast<int>(rank) * 128 + quarter * 32;
      const int row = row0 + lane;
      const int first = EPI == kEpiGated ? at.n * (TN / 2) : at.n * p.tile_cols;
      const int col0 = first + part * apart, last = min(p.cols, first + (EPI == kEpiGated ? TN / 2 : p.tile_cols));
      // Chunks with something to store.
      int chunks = 0;
      if (row0 < p.rows && col0 < last) chunks = min(Cfg::CHUNKS, (last - col0 + next - 1) / next);
      // g and u of a chunk into the two buffers, once every store has read them.
      auto fetch_tiles = [&](int col) {
        if (lane == 0) {
          bulk_wait_group_read<0>();
          mbar_arrive_expect_tx(bar_in(w), 2 * Cfg::TILE);
          tma_load_2d(s_buf, &p.in[0], bar_in(w), col, row0);
          tma_load_2d(s_buf + Cfg::TILE, &p.in[1], bar_in(w), col, row0);
        }
        __syncwarp();
      };
      // What the thread itself reads, 32 columns ahead.
      uint32_t in0[16] = {}, in1[16] = {};
      auto fetch_row = [&](int col) {
        if (row >= p.rows || col >= p.cols) return;
        if constexpr (EPI == kEpiGatedBwd) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint4* src = reinterpret_cast<const uint4*>(p.q[k] + row * p.q_pitch + col);
            const uint4 x = src[0], y = src[1];
            uint32_t(&in)[16] = k ? in1 : in0;
            in[0] = x.x, in[1] = x.y, in[2] = x.z, in[3] = x.w, in[4] = y.x, in[5] = y.y, in[6] = y.z, in[7] = y.w;
          }
        } else {
          row_load32<T>(p.residual, static_cast<int64_t>(row) * p.cols + col, p.cols - col, in0);
        }
      };
      const bool by_row = (EPI == kEpiLinear && p.residual && item.share < 0) || (EPI == kEpiGatedBwd && !by_tma);
      float sg = 0.0f, su = 0.0f;  // the row's scales of a backward in 8 bits
      if (by_tma && chunks > 0) fetch_tiles(col0);
      if (by_row && chunks > 0) {
        fetch_row(col0);
        if (EPI == kEpiGatedBwd && row < p.rows) {
          const int64_t o = static_cast<int64_t>(row) * p.scale_pitch + col0 / kKeepGroup;
          sg = p.scale[0][o];
          su = p.scale[1][o];
        }
      }
      ok = __all_sync(0xffffffffu, mbar_wait_to(bar_acc(buf), (mine >> 1) & 1, abort_flag, kDevTimeoutEpi, status));
      if (!ok) {
        if (by_tma && chunks > 0) mbar_wait_to(bar_in(w), in_phase, &no_abort, kDevTimeoutEpi, status);
        break;
      }
      tc_fence_after();
      const uint32_t t_acc = t_lane + buf * TN, t_part = t_acc + part * apart;
      if constexpr (EPI == kEpiPlain || EPI == kEpiLinear) {
        if (item.share >= 0) {
          // Both buffers together: 32 rows x 32 columns of fp32, a run of the
          // workspace (share_unit; with what lies outside the output, as zeros).
          static_assert(2 * Cfg::TILE == 4096 && CHUNK == 32, "a share's run");
          float* dst = p.partials + (static_cast<int64_t>(item.share) * 32 + rank * 16 + w) * (Cfg::CHUNKS * 1024);
#pragma unroll 1
          for (int c = 0; c < Cfg::CHUNKS; ++c) {
            float v[32];
            tmem_load32(t_part + next * c, v);
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 8; ++u)
              st_shared_v4(s_buf + lane * 128 + ((u ^ (lane & 7)) << 4), __float_as_uint(v[4 * u]),
                           __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3]));
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              bulk_store(dst + c * 1024, s_buf, 4096);
              bulk_commit_group();
            }
          }
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          chunks = 0;  // the rest of the epilogue is tail_sum_kernel's
        }
      }
      if constexpr (EPI == kEpiPlain) {
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          float v[32];
          tmem_load32(t_part + next * c, v);
          const uint32_t tile = begin_tile();
          tile_store<T, PITCH>(tile, lane, 0, v);
          end_tile(&p.out[at.output], tile, col0 + next * c, row0);
        }
      } else if constexpr (EPI == kEpiLinear) {
        float inv = 0.0f;
        if (p.keep_kind == kKeep8 && chunks > 0) {
          // The largest magnitude of the row's 128 columns: a half of a wide
          // tile, or all of a narrow one.
          const int g0 = first + part * apart / kKeepGroup * kKeepGroup;
          float most = 0.0f;
#pragma unroll 1
          for (int c = 0; c < kKeepGroup && g0 + c < p.cols; c += 32) {
            float v[32];
            tmem_load32(t_acc + (g0 - first) + c, v);
            if (p.bias) add_bias<T>(p, g0 + c, v);
            most = most_of(most, v);
          }
          const float s = checkpoint_scale(most, &inv);
          if (row < p.rows && g0 == col0) p.scale[0][static_cast<int64_t>(row) * p.scale_pitch + g0 / kKeepGroup] = s;
        }
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          const int col = col0 + next * c;
          float v[32];
          uint32_t r[16];
          tmem_load32(t_part + next * c, v);
          if (p.residual) {
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = in0[i];
            if (c + 1 < chunks) fetch_row(col + next);
          }
          if (p.bias) add_bias<T>(p, col, v);
          if (p.keep_kind == kKeep16) {
            const uint32_t tile = begin_tile();
            tile_keep<T, PITCH>(tile, lane, 0, v);
            end_tile(&p.keep[0], tile, col, row0);
          } else if (p.keep_kind == kKeep8 && row < p.rows) {
            store_fp8x32(p.q[0] + row * p.q_pitch + col, v, inv);
          }
          with_act(p.act, [&](auto a) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = act_value<decltype(a)::value>(v[i]);
          });
          if (p.residual) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 f = widen<T>(r[i]);
              v[2 * i] += f.x;
              v[2 * i + 1] += f.y;
            }
          }
          const uint32_t tile = begin_tile();
          tile_store<T, PITCH>(tile, lane, 0, v);
          end_tile(&p.out[0], tile, col, row0);
        }
      } else if constexpr (EPI == kEpiGated) {
        // The gate's columns come first, its partner's after them.
        float inv_g = 0.0f, inv_u = 0.0f;
        if (p.keep_kind == kKeep8 && chunks > 0) {
          float most_g = 0.0f, most_u = 0.0f;
#pragma unroll 1
          for (int c = 0; c < Cfg::OUT_COLS; c += 32) {
            float v[32];
            tmem_load32(t_acc + c, v);
            most_g = most_of(most_g, v);
            tmem_load32(t_acc + TN / 2 + c, v);
            most_u = most_of(most_u, v);
          }
          const float s_g = checkpoint_scale(most_g, &inv_g), s_u = checkpoint_scale(most_u, &inv_u);
          if (row < p.rows && part == 0) {
            const int64_t o = static_cast<int64_t>(row) * p.scale_pitch + first / kKeepGroup;
            p.scale[0][o] = s_g;
            p.scale[1][o] = s_u;
          }
        }
        if (chunks > 0) {  // one: a warp's part is a chunk
          float g[CHUNK], u[CHUNK];
#pragma unroll
          for (int from = 0; from < CHUNK; from += 16) {
            float v[16];
            tmem_load16(t_part + from, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) g[from + i] = v[i];
            tmem_load16(t_part + TN / 2 + from, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) u[from + i] = v[i];
          }
          if (p.keep_kind == kKeep16) {
            uint32_t tile = begin_tile();
            tile_keep<T, PITCH>(tile, lane, 0, g);
            end_tile(&p.keep[0], tile, col0, row0);
            tile = begin_tile();
            tile_keep<T, PITCH>(tile, lane, 0, u);
            end_tile(&p.keep[1], tile, col0, row0);
          }
          if constexpr (CHUNK == 32) {
            if (p.keep_kind == kKeep8 && row < p.rows) {
              store_fp8x32(p.q[0] + row * p.q_pitch + col0, g, inv_g);
              store_fp8x32(p.q[1] + row * p.q_pitch + col0, u, inv_u);
            }
          }
          with_act(p.act, [&](auto a) {
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) g[i] = act_value<decltype(a)::value>(g[i]) * u[i];
          });
          const uint32_t tile = begin_tile();
          tile_store<T, PITCH>(tile, lane, 0, g);
          end_tile(&p.out[0], tile, col0, row0);
        }
      } else {  // kEpiGatedBwd
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          const int col = col0 + CHUNK * c;
          const uint32_t tile_g = s_buf, tile_u = s_buf + Cfg::TILE;
          if (by_tma) {
            ok = __all_sync(0xffffffffu, mbar_wait_to(bar_in(w), in_phase, abort_flag, kDevTimeoutEpi, status));
            if (!ok) {
              mbar_wait_to(bar_in(w), in_phase, &no_abort, kDevTimeoutEpi, status);
              break;
            }
            in_phase ^= 1;
          } else {
            if (fmaxf(sg, su) >= kLargestScale) {
#pragma unroll
              for (int i = 0; i < 8; ++i) in0[i] = below_256(in0[i]), in1[i] = below_256(in1[i]);
            }
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
          }
          // dg and du take g's and u's places; h waits in registers for a free
          // buffer.  16 columns at a time, for the registers' sake.
          uint32_t h[CHUNK / 2];
#pragma unroll
          for (int from = 0; from < CHUNK; from += 16) {
            float g[16], u[16], d[16];
            tmem_load16(t_part + CHUNK * c + from, d);
            if (by_tma) {
              tile_load<T, PITCH>(tile_g, lane, from, g);
              tile_load<T, PITCH>(tile_u, lane, from, u);
            } else {
              widen_fp8x16(in0 + from / 4, sg, g);
              widen_fp8x16(in1 + from / 4, su, u);
              if (from + 16 == CHUNK && c + 1 < chunks) fetch_row(col + CHUNK);
            }
            with_act(p.act, [&](auto a) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float slope;
                const float v = act_both<decltype(a)::value>(g[i], slope);
                g[i] = d[i] * (u[i] * slope);  // dg
                d[i] *= v;                     // du
                u[i] *= v;                     // h
              }
            });
            tile_store<T, PITCH>(tile_g, lane, from, g);
            tile_store<T, PITCH>(tile_u, lane, from, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[from / 2 + i] = round_pair<T>(u[2 * i], u[2 * i + 1]);
            if (some_round_to_infinity<T>(u)) {
#pragma unroll
              for (int i = 0; i < 8; ++i) h[from / 2 + i] = kept_pair<T>(u[2 * i], u[2 * i + 1]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.out[0], tile_g, col, row0);
            bulk_commit_group();
            tma_store_2d(&p.out[1], tile_u, col, row0);
            bulk_commit_group();
            bulk_wait_group_read<1>();
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < CHUNK / 8; ++u)
            st_shared_v4(tile_g + swz_off<PITCH>(lane, u), h[4 * u], h[4 * u + 1], h[4 * u + 2], h[4 * u + 3]);
          end_tile(&p.keep[0], tile_g, col, row0);
          if (by_tma && c + 1 < chunks) fetch_tiles(col + CHUNK);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(bar_free(buf), 0));
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  // Every product that writes this CTA's accumulators is complete (waited for
  // here, where the rest of the CTA is through: the wait's bound is no bound on
  // the kernel's time).
  if (threadIdx.x == 32) mbar_wait_to(bar_done, 0, &no_abort, kDevTimeoutMma, status);
  __syncwarp();
  cluster_sync();  // neither CTA leaves while the other may still signal its barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * TN);
  }
}

}  // namespace mlpk
