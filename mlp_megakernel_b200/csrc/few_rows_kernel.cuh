// The feed-forward products for few rows (a decoding step, a small batch): what
// bounds them is reading the weights once, so the weights take the instruction's
// M = 128 side and the rows its N side:
//
//   D^T tile [128 weight columns][NT rows] = W^T x^T,   NT = 16 .. 256.
//
// A 256-row tile of product_kernel.cuh would leave most SMs without a tile and
// most of each tile empty: 1 x 4096 x 4096 bf16 ran 30 us there.  Here a tile is
// reduced by a cluster of S CTAs, each over its share of the reduction, so that
// all SMs read weights at once; the shares meet in shared memory: every CTA
// leaves its fp32 tile in its own, and after a cluster barrier each adds a part of
// the tile over all of them (in the order of the ranks: the same bits every
// time) and runs the epilogue on it.  No workspace, one launch.
//
// For the gate a tile is 64 columns of its matrix above the same 64 of its
// partner's, so that act(g) u has both.
//
// Roles: warp 0 loads (a ring of 64-deep stages: 16 KB of weights, NT x 128 B of
// rows), warp 1 issues, warps 2..9 empty the accumulator (two to a quarter of its
// lanes); all warps run the epilogue.
#pragma once
#include "few_rows_plan.cuh"
#include "product_kernel.cuh"

namespace mlpk {

constexpr int kFewThreads = 320;
struct alignas(64) FewArgs {
  CUtensorMap x[2], w[2];  // [1]: the second reduction range, or the gate's partner (w)
  int rows, cols;
  int nk0, nk;
  int w_mn;
  int nt, stages;          // rows of a tile, depth of the ring
  uint32_t idesc;
  int act, keep_kind, bias32;
  const void* bias;
  const void* in[2];       // residual; or g, u (16 bits)
  void* out[2];
  void* keep[2];
  uint8_t* q[2];
  float* scale[2];
  int64_t q_pitch;
  int scale_pitch;
  int* status;
};

// 4 values of a peer's shared memory.
__device__ __forceinline__ float4 peer_load4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}
template <class T>
__device__ __forceinline__ void load4(const T* p, float (&f)[4]) {
  unpack<T, 4>(load_raw<T, 4>(p), f);
}
template <class T>
__device__ __forceinline__ void store4(T* p, const float (&f)[4]) {
  store_vec<T, 4>(p, f);
}
template <class T>
__device__ __forceinline__ void store_kept4(T* p, const float (&f)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(kept_pair<T>(f[0], f[1]), kept_pair<T>(f[2], f[3]));
}
__device__ __forceinline__ void load_fp8x4(const uint8_t* q, float scale, float (&f)[4]) {
  float2 v[2];
  uint32_t w = *reinterpret_cast<const uint32_t*>(q);
  if (scale >= kLargestScale) w = below_256(w);
  unpack_fp8<4>(*reinterpret_cast<const Raw<uint16_t, 2>*>(&w), v);
  f[0] = v[0].x * scale, f[1] = v[0].y * scale, f[2] = v[1].x * scale, f[3] = v[1].y * scale;
}

template <class T, int EPI>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const __grid_constant__ FewArgs p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;  // the same offset in all CTAs
  uint8_t* gbase = smem_raw + (sbase - raw);
  const int nt = p.nt, ST = p.stages;
  const int stage_bytes = kFewWBytes + nt * kBlockK * 2;
  const int ring = max(ST * stage_bytes, nt * 128 * 4);
  const uint32_t s_bar = sbase + ring;
  auto bar_full = [&](int s) { return s_bar + 8u * s; };
  auto bar_empty = [&](int s) { return s_bar + 8u * (kFewMaxStages + s); };
  const uint32_t bar_acc = s_bar + 8u * (2 * kFewMaxStages);
  const uint32_t s_tmem = bar_acc + 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + (s_tmem - sbase) + 4);
  volatile int no_abort = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_ctarank(), ranks = cluster_size();
  const int tile = blockIdx.x / ranks, row0 = blockIdx.y * nt;
  constexpr bool GATED = EPI == kEpiGated;
  constexpr int TILE_COLS = GATED ? 64 : 128;
  const int col0 = tile * TILE_COLS;
  const int k0 = static_cast<int>(static_cast<int64_t>(rank) * p.nk / ranks);
  const int k1 = static_cast<int>(static_cast<int64_t>(rank + 1) * p.nk / ranks);
  const uint32_t columns = nt <= 32 ? 32 : nt <= 64 ? 64 : nt <= 128 ? 128 : 256;  // of TMEM
  int* const status = p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    mbar_init(bar_acc, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, columns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gbase + (s_tmem - sbase));
  pdl_enter();

  if (warp == 0) {
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int kb = k0; kb < k1; ++kb, ++issued) {
        if (!mbar_wait_to(bar_empty(s), phase, abort_flag, kDevTimeoutEmpty, status)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(bar_full(s), stage_bytes);
        const bool second = kb >= p.nk0;
        const int k = (second ? kb - p.nk0 : kb) * kBlockK;
        const uint32_t sw = sbase + s * stage_bytes, sx = sw + kFewWBytes;
        const CUtensorMap* mw = &p.w[second];
        if (GATED) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            tma_load_2d(sw + c * 64 * 128, &p.w[c], bar_full(s), p.w_mn ? col0 : k, p.w_mn ? k : col0);
        } else if (p.w_mn) {
#pragma unroll
          for (int c = 0; c < 2; ++c) tma_load_2d(sw + c * 64 * 128, mw, bar_full(s), col0 + 64 * c, k);
        } else {
          tma_load_2d(sw, mw, bar_full(s), k, col0);
        }
        tma_load_2d(sx, &p.x[second], bar_full(s), k, row0);
        if (++s == ST) s = 0, phase ^= 1;
      }
      if (!ok)  // nothing of the loads may still be under way when the CTA ends
        for (int b = 0; b < ST && b < issued; ++b)
          mbar_wait_to(bar_full(b), ((issued - b + ST - 1) / ST - 1) & 1, &no_abort, kDevTimeoutFull, status);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t w_step = p.w_mn ? 16 * 128 / 16 : 2;
      const uint64_t w_base = make_sdesc(sbase, p.w_mn ? kBlockK * 128 : 16, 1024, 2);
      const uint64_t x_base = make_sdesc(sbase + kFewWBytes, 16, 1024, 2);
      uint32_t more = 0, phase = 0;
      int s = 0;
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait_to(bar_full(s), phase, abort_flag, kDevTimeoutMma, status)) break;
        tc_fence_after();
        const uint64_t at = static_cast<uint64_t>(s * stage_bytes) >> 4;
#pragma unroll
        for (int kk = 0; kk < kBlockK / 16; ++kk) {
          umma_f16(tmem, w_base + at + kk * w_step, x_base + at + kk * 2, p.idesc, more);
          more = 1;
        }
        umma_commit(bar_empty(s));
        if (++s == ST) s = 0, phase ^= 1;
      }
      umma_commit(bar_acc);
      // The products have read the ring before the tile below reuses it; waited
      // for even after a wait that ran out.
      mbar_wait_to(bar_acc, 0, &no_abort, kDevTimeoutMma, status);
    }
    __syncwarp();
  } else {
    // The accumulator to shared memory, [row][128 columns] (warp's TMEM lanes = columns).
    if (__all_sync(0xffffffffu, mbar_wait_to(bar_acc, 0, abort_flag, kDevTimeoutEpi, status))) {
      tc_fence_after();
      const int quarter = warp & 3;
      const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
      float* dst = reinterpret_cast<float*>(gbase) + quarter * 32 + lane;
      const int live = min(nt, p.rows - row0);
#pragma unroll 1
      for (int c = (warp - 2) / 4 * 16; c < live; c += 32) {
        uint32_t r[16];
        tmem_ld_wait_x16(t_lane + c, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) dst[(c + i) * 128] = __uint_as_float(r[i]);
      }
      tc_fence_before();
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, columns);
  }
  cluster_sync();

  // A warp takes a row of the tile: 128 columns, 4 a thread (the gate: 64, two
  // rows a warp).  Four rows at once, so that their reads of the other CTAs'
  // shared memory are under way together (one at a time: 128 x 256 x 256 took 12.6
  // us instead of 7).
  constexpr int PER_ROW = TILE_COLS / 4, ROWS = 4;
  const int live = min(nt, p.rows - row0);
  const int sub = lane % PER_ROW, own = lane / PER_ROW, step = ranks * (kFewThreads / 32) * (32 / PER_ROW);
  const int col = col0 + 4 * sub;
  for (int base = (rank * (kFewThreads / 32) + warp) * (32 / PER_ROW); base < live; base += ROWS * step) {
    float all[ROWS][4] = {}, partner[ROWS][4] = {};
#pragma unroll 2
    for (int k = 0; k < ranks; ++k) {
      const uint32_t peer = mapa_shared(sbase + 16 * sub, k);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = base + own + i * step;
        if (r >= live) break;
        const float4 f = peer_load4(peer + r * 512);
        all[i][0] += f.x, all[i][1] += f.y, all[i][2] += f.z, all[i][3] += f.w;
        if (GATED) {
          const float4 g = peer_load4(peer + r * 512 + 256);
          partner[i][0] += g.x, partner[i][1] += g.y, partner[i][2] += g.z, partner[i][3] += g.w;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (base + i * step >= live) break;
      const int r = base + own + i * step;
      const bool here = r < live && col < p.cols;
      float(&v)[4] = all[i];
      float(&u)[4] = partner[i];
      const int64_t row = row0 + r, at = row * p.cols + col;
      if constexpr (EPI == kEpiPlain) {
        if (here) store4(static_cast<T*>(p.out[0]) + at, v);
      } else if constexpr (EPI == kEpiLinear) {
        if (here && p.bias) {
          float b[4];
          if (p.bias32) load4(static_cast<const float*>(p.bias) + col, b);
          else load4(static_cast<const T*>(p.bias) + col, b);
  #pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += b[e];
        }
        if (p.keep_kind == kKeep16 && here) store_kept4(static_cast<T*>(p.keep[0]) + at, v);
        if (p.keep_kind == kKeep8) {  // a whole warp has the row's 128 columns (zeros beyond the last)
          float inv, most = max_abs(max_abs(0.0f, v[0], v[1]), v[2], v[3]);
          if (!here) most = 0.0f;
  #pragma unroll
          for (int o = 16; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
          const float s = checkpoint_scale(most, &inv);
          if (here) {
            const uint32_t lo = to_fp8x2(make_float2(v[0] * inv, v[1] * inv));
            const uint32_t hi = to_fp8x2(make_float2(v[2] * inv, v[3] * inv));
            *reinterpret_cast<uint32_t*>(p.q[0] + row * p.q_pitch + col) = lo | hi << 16;
            if (sub == 0) p.scale[0][row * p.scale_pitch + col0 / kKeepGroup] = s;
          }
        }
        with_act(p.act, [&](auto a) {
  #pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = act_value<decltype(a)::value>(v[e]);
        });
        if (here) {
          if (p.in[0]) {
            float f[4];
            load4(static_cast<const T*>(p.in[0]) + at, f);
  #pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += f[e];
          }
          store4(static_cast<T*>(p.out[0]) + at, v);
        }
      } else if constexpr (EPI == kEpiGated) {
        if (here) {
          if (p.keep_kind == kKeep16) {
            store_kept4(static_cast<T*>(p.keep[0]) + at, v);
            store_kept4(static_cast<T*>(p.keep[1]) + at, u);
          }
          with_act(p.act, [&](auto a) {
  #pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = act_value<decltype(a)::value>(v[e]) * u[e];
          });
          store4(static_cast<T*>(p.out[0]) + at, v);
        }
      } else {  // kEpiGatedBwd
        if (here) {
          float g[4], h[4];
          if (p.keep_kind == kKeep16) {
            load4(static_cast<const T*>(p.in[0]) + at, g);
            load4(static_cast<const T*>(p.in[1]) + at, u);
          } else {
            const int64_t s = row * p.scale_pitch + col / kKeepGroup;
            load_fp8x4(p.q[0] + row * p.q_pitch + col, p.scale[0][s], g);
            load_fp8x4(p.q[1] + row * p.q_pitch + col, p.scale[1][s], u);
          }
          with_act(p.act, [&](auto a) {
  #pragma unroll
            for (int e = 0; e < 4; ++e) {
              float slope;
              const float value = act_both<decltype(a)::value>(g[e], slope);
              g[e] = v[e] * (u[e] * slope);
              h[e] = u[e] * value;
              v[e] *= value;
            }
          });
          store4(static_cast<T*>(p.out[0]) + at, g);
          store4(static_cast<T*>(p.out[1]) + at, v);
          store_kept4(static_cast<T*>(p.keep[0]) + at, h);
        }
      }
    }
  }
  cluster_sync();  // no CTA leaves while another may read its tile
}

}  // namespace mlpk
