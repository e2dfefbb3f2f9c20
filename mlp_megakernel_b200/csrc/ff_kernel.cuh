// What stands beside the products (product_kernel.cuh): checkpoints in 8 bits,
// and the activation's backward with the bias gradient.
// All of them are streams over memory, bound by it.
#pragma once
#include "act.cuh"
#include "pdl.cuh"

namespace mlpk {

constexpr int kStreamThreads = 256;
constexpr int kGroupCols = 128;  // columns that share a scale

// ---------------------------------------------------------------- checkpoints
// A group of 128 columns of a row is taken by 16 threads, 8 values each, in
// vectors; or, where the rows are of no whole number of vectors, by a warp, in
// single values (neighbouring threads take neighbouring values).
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    unpack<T, 8>(load_raw<T, 8>(p), f);
  } else {
    const Raw<float, 4> a = load_raw<float, 4>(p), b = load_raw<float, 4>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a.v[e], f[4 + e] = b.v[e];
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    store_vec<T, 8>(p, f);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

template <class T, bool VECTORS>
__global__ void __launch_bounds__(kStreamThreads)
    checkpoint_kernel(int64_t rows, int width, int groups, const T* __restrict__ x, uint8_t* __restrict__ q,
                      float* __restrict__ scale) {
  pdl_enter();
  constexpr int TEAM = VECTORS ? 16 : 32;
  const int64_t teams = static_cast<int64_t>(gridDim.x) * (kStreamThreads / TEAM);
  const int64_t work = rows * groups, id = threadIdx.x % TEAM;
  // All threads of a warp take the same number of turns (they exchange values).
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kStreamThreads / TEAM); base < work; base += teams) {
    const int64_t i = base + threadIdx.x / TEAM;
    const bool live = i < work;
    const int64_t row = live ? i / groups : 0;
    const int g = static_cast<int>(live ? i - row * groups : 0);
    const int64_t at = row * width + g * kGroupCols;
    const int cols = min(kGroupCols, width - g * kGroupCols);
    float inv, most = 0.0f;
    if constexpr (VECTORS) {
      float f[8];
      const bool here = live && id * 8 < cols;
      if (here) load8(x + at + id * 8, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = here ? f[e] : 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) most = max_abs(most, f[e], f[e + 1]);
#pragma unroll
      for (int o = 8; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float s = checkpoint_scale(most, &inv);
      if (here) {
        uint32_t w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
          w[k] = to_fp8x2(make_float2(f[4 * k] * inv, f[4 * k + 1] * inv)) |
                 static_cast<uint32_t>(to_fp8x2(make_float2(f[4 * k + 2] * inv, f[4 * k + 3] * inv))) << 16;
        *reinterpret_cast<uint2*>(q + at + id * 8) = make_uint2(w[0], w[1]);
        if (id == 0) scale[i] = s;
      }
    } else {
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = live && id + 32 * e < cols ? to_float(x[at + id + 32 * e]) : 0.0f;
      most = max_abs(max_abs(0.0f, f[0], f[1]), f[2], f[3]);
#pragma unroll
      for (int o = 16; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float s = checkpoint_scale(most, &inv);
      if (live) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (id + 32 * e < cols)
            q[at + id + 32 * e] = static_cast<uint8_t>(to_fp8x2(make_float2(f[e] * inv, 0.0f)));
        if (id == 0) scale[i] = s;
      }
    }
  }
}

// The largest finite value of a type: rounding up to e4m3 may pass it.
template <class T>
__device__ __forceinline__ float finite_max() {
  return sizeof(T) == 4 ? 3.402823466e+38f : std::is_same_v<T, __half> ? 65504.0f : 3.3895313892515355e+38f;
}
__device__ __forceinline__ float clip(float v, float most) {  // a NaN stays
  return v > most ? most : v < -most ? -most : v;
}

template <class T, bool VECTORS>
__global__ void __launch_bounds__(kStreamThreads)
    restore_kernel(int64_t rows, int width, int groups, const uint8_t* __restrict__ q,
                   const float* __restrict__ scale, T* __restrict__ x) {
  pdl_enter();
  constexpr int EACH = VECTORS ? 8 : 1;
  const int per_row = width / EACH;
  const int64_t total = rows * per_row, step = static_cast<int64_t>(gridDim.x) * kStreamThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kStreamThreads + threadIdx.x; i < total; i += step) {
    const int64_t row = i / per_row;
    const int col = static_cast<int>(i - row * per_row) * EACH;
    const float s = scale[row * groups + col / kGroupCols];
    if constexpr (VECTORS) {
      float2 f[4];
      float v[8];
      unpack_fp8<8>(load_raw<uint16_t, 4>(reinterpret_cast<const uint16_t*>(q + i * 8)), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = clip(f[e].x * s, finite_max<T>());
        v[2 * e + 1] = clip(f[e].y * s, finite_max<T>());
      }
      store8(x + i * 8, v);
    } else {
      Raw<uint16_t, 1> r;
      r.v[0] = q[i];
      float2 f[1];
      unpack_fp8<2>(r, f);
      x[i] = from_float<T>(clip(f[0].x * s, finite_max<T>()));
    }
  }
}

// ---------------------------------------------------------------- the activation's backward
// dz = grad_out act'(z), rounded to the operands' type for the products, and the
// sum of dz over the rows for the bias (from the values before that rounding).  A
// block has 32 vectors of 8 columns by 8 rows of threads and takes every
// gridDim.y-th run of 8 rows; its column sums go to partial[blockIdx.y], which
// bias_grad_kernel adds in order.
struct DzArgs {
  int64_t rows;
  int width, act, keep_kind, scale_pitch;
  int64_t q_pitch;
  const void* grad;
  const void* z;         // 16 bits, or 8
  const float* scale;
  void* dz;              // NULL: not wanted
  float* partial;        // NULL: not wanted
};
constexpr int kDzVectors = 32, kDzRows = kStreamThreads / kDzVectors;

template <class T>
__global__ void __launch_bounds__(kStreamThreads) linear_dz_kernel(const DzArgs a) {
  pdl_enter();
  const int v = threadIdx.x % kDzVectors, r = threadIdx.x / kDzVectors;
  const int col = (blockIdx.x * kDzVectors + v) * 8;
  const bool live = col < a.width;
  float sum[8] = {};
  if (live)
    for (int64_t row = static_cast<int64_t>(blockIdx.y) * kDzRows + r; row < a.rows;
         row += static_cast<int64_t>(gridDim.y) * kDzRows) {
      const int64_t at = row * a.width + col;
      float d[8];
      load8(static_cast<const T*>(a.grad) + at, d);
      if (a.act != kActNone) {
        float z[8];
        if (a.keep_kind == 2) {
          const float s = a.scale[row * a.scale_pitch + col / kGroupCols];
          float2 f[4];
          unpack_fp8<8>(load_raw<uint16_t, 4>(reinterpret_cast<const uint16_t*>(
                            static_cast<const uint8_t*>(a.z) + row * a.q_pitch + col)),
                        f);
#pragma unroll
          for (int e = 0; e < 4; ++e) z[2 * e] = f[e].x * s, z[2 * e + 1] = f[e].y * s;
        } else {
          load8(static_cast<const T*>(a.z) + at, z);
        }
        with_act(a.act, [&](auto act) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float slope;
            act_both<decltype(act)::value>(z[e], slope);
            d[e] *= slope;
          }
        });
      }
      if (a.dz) store8(static_cast<T*>(a.dz) + at, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += d[e];
    }
  if (!a.partial) return;
  __shared__ float s_sum[kDzRows][kDzVectors * 8 + 4];
#pragma unroll
  for (int e = 0; e < 8; ++e) s_sum[r][v * 8 + e] = sum[e];
  __syncthreads();
  const int c = threadIdx.x;  // as many columns as threads
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < kDzRows; ++k) s += s_sum[k][c];
  const int at = blockIdx.x * kDzVectors * 8 + c;
  if (at < a.width) a.partial[static_cast<int64_t>(blockIdx.y) * a.width + at] = s;
}

template <class W>
__global__ void __launch_bounds__(kStreamThreads)
    bias_grad_kernel(int width, int parts, const float* __restrict__ partial, W* __restrict__ db) {
  pdl_enter();
  const int lane = threadIdx.x % 32, part = threadIdx.x / 32;  // 32 columns by 8 shares of the parts
  const int col = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (col < width)
    for (int k = part; k < parts; k += kStreamThreads / 32) s += partial[static_cast<int64_t>(k) * width + col];
  __shared__ float s_sum[kStreamThreads / 32][33];
  s_sum[part][lane] = s;
  __syncthreads();
  if (part == 0 && col < width) {
    float all = 0.0f;
#pragma unroll
    for (int k = 0; k < kStreamThreads / 32; ++k) all += s_sum[k][lane];
    db[col] = from_float<W>(all);
  }
}

}  // namespace mlpk
