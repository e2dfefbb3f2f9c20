// Root-mean-square norm with the residual's addition, its 8-bit output and
// its backward pass.
//
// Per row, all in fp32 from the loads on:
//   h = x + r;   s = rsqrt(mean_j h_j^2 + eps);   y_j = h_j s w_j
// y is computed from the unrounded h; h is rounded once, as it is stored.  The
// 8-bit output stores e4m3(y / scale) with scale = max|y| / 448 over the row
// or over each 128 columns.  Backward, from the stored h and s (G = dL/dy):
//   n_j = h_j s;   c = mean_j G_j w_j n_j
//   dx_j = dr_j = s (G_j w_j - n_j c) + dL/dh_j;   dw_j = sum_rows G_j n_j
// (c uses the norm of the rounded h: it differs from the forward's by the
// rounding of h alone.)
//
// Layout: TPR threads share a row and hold it in registers (NV vectors each,
// vector i of lane l is the row's vector i * TPR + l), so every value is read
// once.  Up to 32 threads a row's sum is a warp shuffle and several rows share
// a block; above, a block has one row and sums through shared memory.
#pragma once
#include "pdl.cuh"
#include "vec.cuh"

namespace mlpk {

constexpr int kNormThreads = 256;  // threads of a block of several rows
constexpr int kNormGroup = 128;    // columns that share a scale
constexpr int kNormMaxWidth = 32768;

// Sum of v over the row's threads.  TPR > 32: `red` is one float per warp;
// two calls in a row take different halves of it (`half`), so one barrier
// separates a write from the reads of the call before the last.
__device__ __forceinline__ float norm_row_sum(float v, int tpr, float* red, int half) {
  if (tpr <= 32) {
    for (int o = tpr / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  red += half * 32;
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.0f;
  for (int k = 0; k < tpr / 32; ++k) t += red[k];  // the same order in every thread
  return t;
}

__device__ __forceinline__ uint32_t norm_row_max(uint32_t v, int tpr, float* red, int half) {
  for (int o = (tpr < 32 ? tpr : 32) / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr <= 32) return v;
  uint32_t* r = reinterpret_cast<uint32_t*>(red) + half * 32;
  if (threadIdx.x % 32 == 0) r[threadIdx.x / 32] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int k = 0; k < tpr / 32; ++k) t = max(t, r[k]);
  return t;
}

struct NormArgs {
  int64_t rows;
  int width;
  int tpr;  // threads of a row: a power of two up to 32, else a multiple of 32
  float eps;
  const void* x;
  const void* r;  // null: no residual
  const void* w;  // null: ones
  void* y;        // T, or e4m3 with FP8
  void* h;        // null: not stored
  float* rstd;    // null: not stored
  float* scale;   // FP8: [rows][groups]
  int group;      // FP8: columns that share a scale: 128, or 0 for the row
};

template <class T, class W, int VEC, int NV, bool FP8>
__global__ void __launch_bounds__(1024) rms_norm_fwd_kernel(const NormArgs a) {
  extern __shared__ float smem[];  // 64 floats, then with FP8 and VEC 1 a maximum per group
  pdl_enter();
  const int lane = threadIdx.x % a.tpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / a.tpr) + threadIdx.x / a.tpr;
  const bool live = row < a.rows;  // whole rows: the other threads take part in the shuffles and barriers
  const int64_t base = row * a.width;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* r = a.r ? static_cast<const T*>(a.r) + base : nullptr;
  const W* w = static_cast<const W*>(a.w);
  const int nvec = a.width / VEC;

  float h[NV][VEC];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * a.tpr + lane;
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[i][e] = 0.0f;
    if (live && v < nvec) {
      unpack(load_raw<T, VEC>(x + v * VEC), h[i]);
      if (r) {
        float f[VEC];
        unpack(load_raw<T, VEC>(r + v * VEC), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i][e] += f[e];
      }
      if (a.h) store_vec<T, VEC>(static_cast<T*>(a.h) + base + v * VEC, h[i]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += h[i][e] * h[i][e];
  }
  const float s = rsqrtf(norm_row_sum(sum, a.tpr, smem, 0) / static_cast<float>(a.width) + a.eps);
  if (a.rstd && live && lane == 0) a.rstd[row] = s;

  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * a.tpr + lane;
    if (live && v < nvec) {
      float f[VEC];
      if (w) {
        unpack(load_raw<W, VEC>(w + v * VEC), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i][e] = h[i][e] * s * f[e];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i][e] *= s;
      }
      if constexpr (FP8) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) amax = max(amax, abs_bits(h[i][e]));
      } else {
        store_vec<T, VEC>(static_cast<T*>(a.y) + base + v * VEC, h[i]);
      }
    }
  }
  if constexpr (FP8) {
    uint8_t* q = static_cast<uint8_t*>(a.y) + base;
    if (a.group == 0) {
      float inv;
      const float scale = fp8_scale(norm_row_max(amax, a.tpr, smem, 1), &inv);
      if (live && lane == 0) a.scale[row] = scale;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = i * a.tpr + lane;
        if (live && v < nvec) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) h[i][e] *= inv;
          store_fp8<VEC>(q + v * VEC, h[i]);
        }
      }
      return;
    }
    const int groups = (a.width + kNormGroup - 1) / kNormGroup;
    if constexpr (VEC > 1) {
      // The 128 / VEC lanes of a group are neighbours: a power of two, and a
      // divisor of tpr unless the row is narrower than a group.
      const int gl = min(kNormGroup / VEC, a.tpr);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = i * a.tpr + lane;
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = max(m, abs_bits(h[i][e]));
        for (int o = gl / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        float inv;
        const float scale = fp8_scale(m, &inv);
        if (live && v < nvec) {
          if (v % gl == 0) a.scale[row * groups + v / gl] = scale;
#pragma unroll
          for (int e = 0; e < VEC; ++e) h[i][e] *= inv;
          store_fp8<VEC>(q + v * VEC, h[i]);
        }
      }
    } else {
      // One element per lane: 32 neighbours lie in one group (32 divides both
      // 128 and every offset i * tpr, or the whole row is one group), and the
      // warps of a group meet in shared memory.  A maximum does not depend on
      // the order.
      uint32_t* gmax = reinterpret_cast<uint32_t*>(smem + 64) + (threadIdx.x / a.tpr) * groups;
      for (int k = lane; k < groups; k += a.tpr) gmax[k] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = i * a.tpr + lane;
        if (live && v < nvec) atomicMax(gmax + v / kNormGroup, abs_bits(h[i][0]));
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = i * a.tpr + lane;
        if (live && v < nvec) {
          float inv;
          const float scale = fp8_scale(gmax[v / kNormGroup], &inv);
          if (v % kNormGroup == 0) a.scale[row * groups + v / kNormGroup] = scale;
          h[i][0] *= inv;
          store_fp8<1>(q + v, h[i]);
        }
      }
    }
  }
}

struct NormBwdArgs {
  int64_t rows;
  int width;
  int tpr;
  const void* h;
  const float* rstd;
  const void* w;   // null: ones
  const void* gy;
  const void* gh;  // null: none
  void* dx;
  float* part;     // null: no weight gradient; else [gridDim.x][width]
};

// A block takes rows blockIdx.x * rows-per-block + k * gridDim.x * ..., its
// threads keep their columns' share of dw in registers, and the block's sum
// over its row groups (through shared memory, in order) is one row of `part`.
template <class T, class W, int VEC, int NV>
__global__ void __launch_bounds__(1024) rms_norm_bwd_kernel(const NormBwdArgs a) {
  extern __shared__ float smem[];  // 64 floats, then [row groups][width] if there are several
  pdl_enter();
  const int lane = threadIdx.x % a.tpr;
  const int sub = threadIdx.x / a.tpr, subs = blockDim.x / a.tpr;
  const int nvec = a.width / VEC;
  const W* w = static_cast<const W*>(a.w);
  float dw[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = 0.0f;

  int half = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * subs; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * subs, half ^= 1) {
    const int64_t row = row0 + sub;
    const bool live = row < a.rows;
    const int64_t base = row * a.width;
    const float s = live ? a.rstd[row] : 0.0f;
    float n[NV][VEC], g[NV][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = i * a.tpr + lane;
#pragma unroll
      for (int e = 0; e < VEC; ++e) n[i][e] = g[i][e] = 0.0f;
      if (live && v < nvec) {
        unpack(load_raw<T, VEC>(static_cast<const T*>(a.h) + base + v * VEC), n[i]);
        unpack(load_raw<T, VEC>(static_cast<const T*>(a.gy) + base + v * VEC), g[i]);
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 1.0f;
        if (w) unpack(load_raw<W, VEC>(w + v * VEC), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          n[i][e] *= s;
          dw[i][e] += g[i][e] * n[i][e];
          g[i][e] *= f[e];
          sum += g[i][e] * n[i][e];
        }
      }
    }
    const float c = norm_row_sum(sum, a.tpr, smem, half) / static_cast<float>(a.width);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = i * a.tpr + lane;
      if (live && v < nvec) {
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 0.0f;
        if (a.gh) unpack(load_raw<T, VEC>(static_cast<const T*>(a.gh) + base + v * VEC), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] += s * (g[i][e] - n[i][e] * c);
        store_vec<T, VEC>(static_cast<T*>(a.dx) + base + v * VEC, f);
      }
    }
  }
  if (!a.part) return;
  float* out = a.part + static_cast<int64_t>(blockIdx.x) * a.width;
  if (subs == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = i * a.tpr + lane;
      if (v < nvec) store_vec<float, VEC>(out + v * VEC, dw[i]);
    }
    return;
  }
  float* acc = smem + 64;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * a.tpr + lane;
    if (v < nvec)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[sub * a.width + v * VEC + e] = dw[i][e];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < a.width; j += blockDim.x) {
    float t = 0.0f;
    for (int k = 0; k < subs; ++k) t += acc[k * a.width + j];
    out[j] = t;
  }
}

// dw[j] = sum over the blocks' rows of `part`, in a fixed order: 32 columns x
// 32 row groups a block, the groups' sums added in order.
template <class W>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* __restrict__ part, int nparts, int width,
                                                           W* __restrict__ dw) {
  __shared__ float red[32][33];
  pdl_enter();
  const int c = threadIdx.x % 32, k = threadIdx.x / 32;
  const int j = blockIdx.x * 32 + c;
  float t = 0.0f;
  if (j < width)
    for (int p = k; p < nparts; p += 32) t += part[static_cast<int64_t>(p) * width + j];
  red[k][c] = t;
  __syncthreads();
  if (k == 0 && j < width) {
    t = 0.0f;
#pragma unroll
    for (int q = 0; q < 32; ++q) t += red[q][c];
    dw[j] = from_float<W>(t);
  }
}

}  // namespace mlpk
