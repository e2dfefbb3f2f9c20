// The matrix products of the feed-forward operators on tensor cores, with what
// stands behind each product in its epilogue:
//
//   kEpiPlain     D = A B                                     (dx, dW)
//   kEpiPartial   the same in fp32, of a share of the reduction (dW, split)
//   kEpiLinear    z = A B + bias; out = act(z) + residual; z kept for the backward
//   kEpiGated     g = A Bg, u = A Bu; h = act(g) u; g and u kept for the backward
//   kEpiGatedBwd  dh = A B; dg = dh u act'(g), du = dh act(g), h = act(g) u again
//
// A tile of D is 256 rows x TN columns of a pair of CTAs (pair.cuh), reduced in
// blocks of 64 through a ring of TMA loads; operands are fp16 or bf16 in either
// order (K contiguous, or the row / column index), chosen at run time by the
// descriptors alone.  Roles of a CTA: warp 0 loads, warp 1 of the leader issues
// the tcgen05 instructions, warps 2..9 are the epilogue (thread = row; two warps
// share the 32 rows of a TMEM lane quarter and halve the columns).  Two
// accumulators of TN columns, so the epilogue of a tile runs beside the products
// of the next.  The kernel is persistent: tiles are taken in groups of `group`
// row tiles over all column tiles, so that the pairs at work share rows and
// columns in L2.
//
// Everything between the operands and the stored values is fp32: accumulators,
// bias, activation, residual.  What is kept for the backward is rounded once, to
// the operands' type (as a 16-bit activation is anywhere else in training) or to
// 8 bits with a scale for each row and 128 columns (act.cuh).
#pragma once
#include "act.cuh"
#include "layout.cuh"
#include "pair.cuh"
#include "product_epi.cuh"

namespace mlpk {

enum Keep : int { kKeepNone = 0, kKeep16 = 1, kKeep8 = 2 };

constexpr int kPairRows = 256;      // rows of a pair's tile
constexpr int kBlockK = 64;         // reduction of a stage: one 128-byte row of 16-bit values
constexpr int kKeepGroup = 128;     // columns that share a scale
constexpr int kProductThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kTileBytes = 2048;    // 32 rows x 32 columns of 16-bit values, a warp's unit of TMA traffic

struct alignas(64) ProductArgs {
  CUtensorMap a[2], b[2];  // [1]: the second reduction range (nk0 < nk), or the gate's partner / second output's B
  CUtensorMap in[2];       // linear: residual; gated backward: g, u (16 bits)
  CUtensorMap out[2];      // plain: D (two of them with `outputs` 2); linear: out; gated: h; backward: dg, du
  CUtensorMap keep[2];     // linear: z; gated: g, u; backward: h
  int rows, cols;          // of each output
  int nk0, nk;             // blocks of the first reduction range, and of both
  int tiles_m, tiles_n, outputs, splits, group;
  int a_mn, b_mn;          // the operand's contiguous index is the row / column, not the reduction
  int out_a;               // with two outputs: A differs, not B
  uint32_t idesc;
  int act, keep_kind, residual, bias32;
  const void* bias;
  uint8_t* q[2];           // 8-bit values, rows of q_pitch bytes
  float* scale[2];         // [rows][scale_pitch]
  int64_t q_pitch;
  int scale_pitch;
  float* partials;         // [splits][outputs][rows][cols]
  int* status;
};

template <int EPI, int TN>
struct ProductCfg {
  static constexpr int A_BYTES = 128 * kBlockK * 2;
  static constexpr int B_BYTES = TN / 2 * kBlockK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  // A warp's buffers of 2 KB: two for outputs in turn; residual / out and z, two
  // of each; a ring of four for h, g, u; two pairs g / dg, u / du and one for h.
  static constexpr int BUFS = EPI == kEpiPlain ? 2 : EPI == kEpiPartial ? 0 : EPI == kEpiGatedBwd ? 5 : 4;
  static constexpr int OFF_EPI = 0;
  static constexpr int EPI_BYTES = kEpiWarps * BUFS * kTileBytes;
  static constexpr int STAGES_FIT = (227 * 1024 - 2048 - EPI_BYTES) / STAGE;
  static constexpr int STAGES = STAGES_FIT < 8 ? STAGES_FIT : 8;
  static constexpr int OFF_STAGE = EPI_BYTES;
  static constexpr int OFF_BAR = OFF_STAGE + STAGES * STAGE;
  static constexpr int NUM_BARS = 2 * STAGES + 5 + 2 * kEpiWarps;
  static constexpr int OFF_MISC = OFF_BAR + 8 * NUM_BARS;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
  static constexpr int OUT_COLS = EPI == kEpiGated ? TN / 2 : TN;  // columns of an output that a tile has
  static constexpr int HALF = OUT_COLS / 2;
  static constexpr int CHUNKS = HALF / 32;
  static_assert(EPI_BYTES % 1024 == 0 && STAGE % 1024 == 0 && SMEM <= 227 * 1024, "shared memory");
  static_assert(STAGES >= 3 && (TN == 128 || TN == 256), "tile");
};

struct TileAt {
  int m, n, output, split;
};
__host__ __device__ inline TileAt product_tile(int t, int tiles_m, int tiles_n, int outputs, int group) {
  const int wide = tiles_n * outputs, each = tiles_m * wide;
  TileAt at;
  at.split = t / each;
  t -= at.split * each;
  const int first = t / (group * wide) * group;
  const int high = tiles_m - first < group ? tiles_m - first : group;
  t -= first * wide;
  at.m = first + t % high;
  const int n = t / high;
  at.output = n / tiles_n;
  at.n = n - at.output * tiles_n;
  return at;
}

// 32 values as pairs of the type.
template <class T>
__device__ __forceinline__ void pack32(const float (&v)[32], uint32_t (&p)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const typename Pair<T>::type x = Pair<T>::round(v[2 * i], v[2 * i + 1]);
    p[i] = *reinterpret_cast<const uint32_t*>(&x);
  }
}
template <class T>
__device__ __forceinline__ void unpack32(const uint32_t (&p)[16], float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 f = to_float2(*reinterpret_cast<const typename Pair<T>::type*>(&p[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// A thread's row of a 32 x 32 tile in shared memory (64-byte rows, as a TMA box
// with the 64-byte swizzle has them).
__device__ __forceinline__ void tile_row_store(uint32_t tile, int lane, const uint32_t (&p)[16]) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
    st_shared_v4(tile + swz_off<64>(lane, u), p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]);
}
__device__ __forceinline__ void tile_row_load(uint32_t tile, int lane, uint32_t (&p)[16]) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(p[4 * u]), "=r"(p[4 * u + 1]), "=r"(p[4 * u + 2]), "=r"(p[4 * u + 3])
                 : "r"(tile + swz_off<64>(lane, u))
                 : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld_wait_x32(taddr, r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 values of a row to 8 bits (q is 32-byte aligned) and back.
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
__device__ __forceinline__ void load_fp8x32(const uint8_t* q, float scale, float (&v)[32]) {
  const Raw<uint16_t, 8> a = load_raw<uint16_t, 8>(reinterpret_cast<const uint16_t*>(q));
  const Raw<uint16_t, 8> b = load_raw<uint16_t, 8>(reinterpret_cast<const uint16_t*>(q) + 8);
  float2 f[8];
  unpack_fp8<16>(a, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[2 * i] = f[i].x * scale, v[2 * i + 1] = f[i].y * scale;
  unpack_fp8<16>(b, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[16 + 2 * i] = f[i].x * scale, v[17 + 2 * i] = f[i].y * scale;
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
  auto bar_in = [&](int w, int b) { return s_bar + 8u * (2 * ST + 5 + 2 * w + b); };  // a warp's tiles of `in`
  const uint32_t s_tmem = sbase + Cfg::OFF_MISC;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + Cfg::OFF_MISC + 4);
  volatile int no_abort = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int total = p.tiles_m * p.tiles_n * p.outputs * p.splits;
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
    for (int w = 0; w < 2 * kEpiWarps; ++w) mbar_init(bar_in(0, w), 1);
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
        const TileAt at = product_tile(t, p.tiles_m, p.tiles_n, p.outputs, p.group);
        const int k0 = static_cast<int>(static_cast<int64_t>(at.split) * p.nk / p.splits);
        const int k1 = static_cast<int>(static_cast<int64_t>(at.split + 1) * p.nk / p.splits);
        const int row = at.m * kPairRows + static_cast<int>(rank) * 128;
        // A pair's half of B: columns, or for the gate its own matrix.
        const int col = EPI == kEpiGated ? at.n * (TN / 2) : at.n * TN + static_cast<int>(rank) * (TN / 2);
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
          if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * Cfg::STAGE);
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
        const TileAt at = product_tile(t, p.tiles_m, p.tiles_n, p.outputs, p.group);
        const int k0 = static_cast<int>(static_cast<int64_t>(at.split) * p.nk / p.splits);
        const int k1 = static_cast<int>(static_cast<int64_t>(at.split + 1) * p.nk / p.splits);
        const int buf = mine & 1;
        const uint32_t d = tmem + buf * TN;
        ok = mbar_wait_cluster(bar_free(buf), ((mine >> 1) & 1) ^ 1, abort_flag, kDevTimeoutMma, status);
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
    const int w = warp - 2, quarter = warp & 3, half = w >> 2;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_buf = sbase + Cfg::OFF_EPI + w * Cfg::BUFS * kTileBytes;
    const bool with_in = (EPI == kEpiLinear && p.residual) || (EPI == kEpiGatedBwd && p.keep_kind == kKeep16);
    bool ok = true;
    int it = 0;       // chunks so far: the turn of the buffers
    int fetched = 0;  // chunks whose `in` has been asked for
    int ring = 0;  // tiles stored so far (buffers in turn)
    // A tile into the next buffer of the ring, and its store.
    auto put = [&](const CUtensorMap* map, const float(&v)[32], int col, int row) {
      constexpr int N = Cfg::BUFS > 0 ? Cfg::BUFS : 1;
      const uint32_t tile = s_buf + (ring++ % N) * kTileBytes;
      if (lane == 0) bulk_wait_group_read<N - 1>();
      __syncwarp();
      uint32_t packed[16];
      pack32<T>(v, packed);
      tile_row_store(tile, lane, packed);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(map, tile, col, row);
        bulk_commit_group();
      }
    };
    // The tile(s) of `in` for the it-th chunk, into its turn's buffers, once
    // every store so far has read its buffer.
    auto fetch = [&](int turn, int col, int row) {
      fetched = turn + 1;
      if (lane == 0) {
        bulk_wait_group_read<0>();
        const uint32_t tile = s_buf + (turn & 1) * (EPI == kEpiGatedBwd ? 2 : 1) * kTileBytes;
        mbar_arrive_expect_tx(bar_in(w, turn & 1), EPI == kEpiGatedBwd ? 2 * kTileBytes : kTileBytes);
        tma_load_2d(tile, &p.in[0], bar_in(w, turn & 1), col, row);
        if (EPI == kEpiGatedBwd) tma_load_2d(tile + kTileBytes, &p.in[1], bar_in(w, turn & 1), col, row);
      }
    };
    int mine = 0;
    for (int t = cluster_id(); ok && t < total; t += step, ++mine) {
      const TileAt at = product_tile(t, p.tiles_m, p.tiles_n, p.outputs, p.group);
      const int buf = mine & 1;
      const int row0 = at.m * kPairRows + static_cast<int>(rank) * 128 + quarter * 32;
      const int row = row0 + lane;
      const int first = at.n * Cfg::OUT_COLS, col0 = first + half * Cfg::HALF;
      // Chunks with something to store.
      int chunks = 0;
      if (row0 < p.rows && col0 < p.cols) chunks = min(Cfg::CHUNKS, (p.cols - col0 + 31) / 32);
      if (with_in && chunks > 0) fetch(it, col0, row0);
      ok = __all_sync(0xffffffffu, mbar_wait_to(bar_acc(buf), (mine >> 1) & 1, abort_flag, kDevTimeoutEpi, status));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_acc = t_lane + buf * TN;
      if constexpr (EPI == kEpiPlain) {
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          float v[32];
          tmem_load32(t_acc + half * Cfg::HALF + 32 * c, v);
          put(&p.out[at.output], v, col0 + 32 * c, row0);
        }
      } else if constexpr (EPI == kEpiPartial) {
        float* dst = p.partials + ((static_cast<int64_t>(at.split) * p.outputs + at.output) * p.rows + row) * p.cols;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          float v[32];
          tmem_load32(t_acc + half * Cfg::HALF + 32 * c, v);
          if (row < p.rows) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int col = col0 + 32 * c + 8 * k;
              float2 f[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = make_float2(v[8 * k + 2 * e], v[8 * k + 2 * e + 1]);
              if (col < p.cols) store_32b(dst + col, f);
            }
          }
        }
      } else if constexpr (EPI == kEpiLinear) {
        float inv = 0.0f;
        if (p.keep_kind == kKeep8 && chunks > 0) {
          // The largest magnitude of the row's 128 columns: a half of a wide
          // tile, or all of a narrow one.
          const int g0 = TN == 256 ? col0 : first;
          float most = 0.0f;
#pragma unroll 1
          for (int c = 0; c < 4 && g0 + 32 * c < p.cols; ++c) {
            float v[32];
            tmem_load32(t_acc + (g0 - first) + 32 * c, v);
            if (p.bias) add_bias<T>(p, g0 + 32 * c, v);
            most = most_of(most, v);
          }
          const float s = checkpoint_scale(most, &inv);
          if (row < p.rows && g0 == col0) p.scale[0][static_cast<int64_t>(row) * p.scale_pitch + g0 / kKeepGroup] = s;
        }
#pragma unroll 1
        for (int c = 0; c < chunks; ++c, ++it) {
          const int col = col0 + 32 * c;
          if (with_in && c + 1 < chunks) fetch(it + 1, col + 32, row0);
          if (!with_in) {
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
          }
          const uint32_t tile = s_buf + (it & 1) * kTileBytes, ztile = tile + 2 * kTileBytes;
          float v[32];
          uint32_t packed[16];
          tmem_load32(t_acc + half * Cfg::HALF + 32 * c, v);
          if (p.bias) add_bias<T>(p, col, v);
          if (p.keep_kind == kKeep16) {
            pack32<T>(v, packed);
            tile_row_store(ztile, lane, packed);
          } else if (p.keep_kind == kKeep8 && row < p.rows) {
            store_fp8x32(p.q[0] + row * p.q_pitch + col, v, inv);
          }
          with_act(p.act, [&](auto a) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = act_value<decltype(a)::value>(v[i]);
          });
          if (with_in) {
            ok = __all_sync(0xffffffffu,
                            mbar_wait_to(bar_in(w, it & 1), (it >> 1) & 1, abort_flag, kDevTimeoutEpi, status));
            if (!ok) break;
            float r[32];
            tile_row_load(tile, lane, packed);
            unpack32<T>(packed, r);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += r[i];
          }
          pack32<T>(v, packed);
          tile_row_store(tile, lane, packed);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.out[0], tile, col, row0);
            if (p.keep_kind == kKeep16) tma_store_2d(&p.keep[0], ztile, col, row0);
            bulk_commit_group();
          }
        }
      } else if constexpr (EPI == kEpiGated) {
        // The gate's columns come first, its partner's after them.
        float inv_g = 0.0f, inv_u = 0.0f;
        if (p.keep_kind == kKeep8 && chunks > 0) {
          float most_g = 0.0f, most_u = 0.0f;
#pragma unroll 1
          for (int c = 0; c < Cfg::OUT_COLS / 32; ++c) {
            float v[32];
            tmem_load32(t_acc + 32 * c, v);
            most_g = most_of(most_g, v);
            tmem_load32(t_acc + TN / 2 + 32 * c, v);
            most_u = most_of(most_u, v);
          }
          const float sg = checkpoint_scale(most_g, &inv_g), su = checkpoint_scale(most_u, &inv_u);
          if (row < p.rows && half == 0) {
            const int64_t o = static_cast<int64_t>(row) * p.scale_pitch + first / kKeepGroup;
            p.scale[0][o] = sg;
            p.scale[1][o] = su;
          }
        }
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          const int col = col0 + 32 * c;
          float g[32], u[32];
          tmem_load32(t_acc + half * Cfg::HALF + 32 * c, g);
          tmem_load32(t_acc + TN / 2 + half * Cfg::HALF + 32 * c, u);
          if (p.keep_kind == kKeep16) {
            put(&p.keep[0], g, col, row0);
            put(&p.keep[1], u, col, row0);
          } else if (p.keep_kind == kKeep8 && row < p.rows) {
            store_fp8x32(p.q[0] + row * p.q_pitch + col, g, inv_g);
            store_fp8x32(p.q[1] + row * p.q_pitch + col, u, inv_u);
          }
          with_act(p.act, [&](auto a) {
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = act_value<decltype(a)::value>(g[i]) * u[i];
          });
          put(&p.out[0], g, col, row0);
        }
      } else {  // kEpiGatedBwd
        float sg = 0.0f, su = 0.0f;
        if (p.keep_kind == kKeep8 && chunks > 0 && row < p.rows && TN == 256) {
          const int64_t o = static_cast<int64_t>(row) * p.scale_pitch + col0 / kKeepGroup;
          sg = p.scale[0][o];
          su = p.scale[1][o];
        }
#pragma unroll 1
        for (int c = 0; c < chunks; ++c, ++it) {
          const int col = col0 + 32 * c;
          const uint32_t tile = s_buf + (it & 1) * 2 * kTileBytes, htile = s_buf + 4 * kTileBytes;
          float g[32], u[32], d[32];
          uint32_t packed[16];
          if (with_in) {
            if (c + 1 < chunks) fetch(it + 1, col + 32, row0);
            else if (lane == 0) bulk_wait_group_read<0>();
            ok = __all_sync(0xffffffffu,
                            mbar_wait_to(bar_in(w, it & 1), (it >> 1) & 1, abort_flag, kDevTimeoutEpi, status));
            if (!ok) break;
            tile_row_load(tile, lane, packed);
            unpack32<T>(packed, g);
            tile_row_load(tile + kTileBytes, lane, packed);
            unpack32<T>(packed, u);
          } else {
            if (row < p.rows) {
              load_fp8x32(p.q[0] + row * p.q_pitch + col, sg, g);
              load_fp8x32(p.q[1] + row * p.q_pitch + col, su, u);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) g[i] = u[i] = 0.0f;
            }
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
          }
          tmem_load32(t_acc + half * Cfg::HALF + 32 * c, d);
          with_act(p.act, [&](auto a) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float slope;
              const float v = act_both<decltype(a)::value>(g[i], slope);
              g[i] = d[i] * (u[i] * slope);  // dg
              d[i] *= v;                     // du
              u[i] *= v;                     // h
            }
          });
          pack32<T>(g, packed);
          tile_row_store(tile, lane, packed);
          pack32<T>(d, packed);
          tile_row_store(tile + kTileBytes, lane, packed);
          pack32<T>(u, packed);
          tile_row_store(htile, lane, packed);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.out[0], tile, col, row0);
            tma_store_2d(&p.out[1], tile + kTileBytes, col, row0);
            tma_store_2d(&p.keep[0], htile, col, row0);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(bar_free(buf), 0));
    }
    if (lane == 0) {
      // After a wait that ran out: no load may still be under way.
      for (; !ok && it < fetched; ++it)
        mbar_wait_to(bar_in(w, it & 1), (it >> 1) & 1, &no_abort, kDevTimeoutEpi, status);
      bulk_wait_group<0>();
    }
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
