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
// A group of 128 columns of a row is taken by 8 threads, 16 values each, in
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

// Where a team's or thread's work lies, step by step: the divisions are done once
// (one for each item of 8 values cost more than the rest of it).
struct Steps {
  int64_t major, major_step;
  int minor, minor_step, minors;
  __host__ __device__ Steps(int64_t first, int64_t step, int minors_) : minors(minors_) {
    major = first / minors;
    minor = static_cast<int>(first - major * minors);
    major_step = step / minors;
    minor_step = static_cast<int>(step - major_step * minors);
  }
  __host__ __device__ __forceinline__ void next() {
    // Unsigned: both are below 2^31, their sum need not be.
    const uint32_t next = static_cast<uint32_t>(minor) + static_cast<uint32_t>(minor_step);
    const bool over = next >= static_cast<uint32_t>(minors);
    minor = static_cast<int>(over ? next - static_cast<uint32_t>(minors) : next);
    major += major_step + over;
  }
};

// Groups of a team under way together: one at a time left memory waiting
// (16384 x 8192 bf16, both ways: 167 us).
template <bool VECTORS>
constexpr int kGroupsAtOnce = VECTORS ? 2 : 4;

template <class T, bool VECTORS>
__global__ void __launch_bounds__(kStreamThreads)
    checkpoint_kernel(int64_t rows, int width, int groups, const T* __restrict__ x, uint8_t* __restrict__ q,
                      float* __restrict__ scale) {
  pdl_enter();
  constexpr int TEAM = VECTORS ? 8 : 32, N = VECTORS ? 16 : 4, AT_ONCE = kGroupsAtOnce<VECTORS>;
  const bool wide = width % 16 == 0;  // 16-byte vectors of 8-bit values
  const int64_t teams = static_cast<int64_t>(gridDim.x) * (kStreamThreads / TEAM);
  const int id = threadIdx.x % TEAM;
  const int64_t block_first = static_cast<int64_t>(blockIdx.x) * (kStreamThreads / TEAM);
  Steps at(block_first + threadIdx.x / TEAM, teams, groups);
  // All threads of a warp take the same number of turns (they exchange values).
  for (int64_t base = block_first; base < rows * groups; base += AT_ONCE * teams) {
    float f[AT_ONCE][N];
    int64_t first[AT_ONCE], group[AT_ONCE];
    int cols[AT_ONCE];  // of the group; 0: there is none
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      cols[k] = at.major < rows ? min(kGroupCols, width - at.minor * kGroupCols) : 0;
      first[k] = at.major * width + at.minor * kGroupCols;
      group[k] = at.major * groups + at.minor;
      at.next();
#pragma unroll
      for (int e = 0; e < N; ++e) f[k][e] = 0.0f;
      if constexpr (VECTORS) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (id * 16 + 8 * v < cols[k])
            load8(x + first[k] + id * 16 + 8 * v, *reinterpret_cast<float(*)[8]>(&f[k][8 * v]));
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (id + 32 * e < cols[k]) f[k][e] = to_float(x[first[k] + id + 32 * e]);
      }
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      float inv, most = 0.0f;
#pragma unroll
      for (int e = 0; e < N; e += 2) most = max_abs(most, f[k][e], f[k][e + 1]);
#pragma unroll
      for (int o = TEAM / 2; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float s = checkpoint_scale(most, &inv);
      uint32_t w[N / 4];
#pragma unroll
      for (int v = 0; v < N / 4; ++v)
        w[v] = to_fp8x2(make_float2(f[k][4 * v] * inv, f[k][4 * v + 1] * inv)) |
               static_cast<uint32_t>(to_fp8x2(make_float2(f[k][4 * v + 2] * inv, f[k][4 * v + 3] * inv))) << 16;
      if constexpr (VECTORS) {
        uint8_t* to = q + first[k] + id * 16;
        if (wide && id * 16 < cols[k]) {
          *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int v = 0; v < 2; ++v)
            if (id * 16 + 8 * v < cols[k]) *reinterpret_cast<uint2*>(to + 8 * v) = make_uint2(w[2 * v], w[2 * v + 1]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (id + 32 * e < cols[k]) q[first[k] + id + 32 * e] = static_cast<uint8_t>(w[0] >> 8 * e);
      }
      if (id == 0 && cols[k] > 0) scale[group[k]] = s;
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

// 16 values of the flat tensor at a time, whatever the width: they have one
// scale (always where 16 divides the width, ONE: what follows costs 16384 x 8192
// bf16 84 -> 100 us), or two (the rest of a group and the beginning of the next),
// or, where a row's last group is shorter than that, each looks up its own.
template <class T, bool ONE>
__global__ void __launch_bounds__(kStreamThreads)
    restore_kernel(int64_t total, int width, int groups, const uint8_t* __restrict__ q,
                   const float* __restrict__ scale, T* __restrict__ x) {
  pdl_enter();
  constexpr int AT_ONCE = 2, N = 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kStreamThreads * N;
  int64_t i = (static_cast<int64_t>(blockIdx.x) * kStreamThreads + threadIdx.x) * N;
  Steps at(i, step, width);
  for (; i < total; i += AT_ONCE * step) {
    Raw<uint16_t, N / 2> raw[AT_ONCE];
    float s[AT_ONCE], next[AT_ONCE];
    int64_t row[AT_ONCE];
    int col[AT_ONCE], here[AT_ONCE], there[AT_ONCE];  // values of this group, and of the next, from the first on
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      row[k] = at.major;
      col[k] = at.minor;
      at.next();
      const int64_t p = i + k * step;
      here[k] = min(kGroupCols - col[k] % kGroupCols, width - col[k]);
      there[k] = N;
      next[k] = 0.0f;
      if (p + N <= total) {
        raw[k] = load_raw<uint16_t, N / 2>(reinterpret_cast<const uint16_t*>(q + p));
        const int64_t group = row[k] * groups + col[k] / kGroupCols;  // the next one follows it, on the next row too
        s[k] = scale[group];
        if (!ONE && here[k] < N) {
          const int begin = col[k] + here[k] == width ? 0 : col[k] + here[k];
          there[k] = min(kGroupCols, width - begin);
          next[k] = scale[group + 1];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int64_t p = i + k * step;
      int64_t r = row[k];
      int c = col[k];
      if (p + N <= total) {
        float2 f[N / 2];
        float v[N];
        unpack_fp8<N>(raw[k], f);
        const bool two = ONE || here[k] + there[k] >= N;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float each = ONE || e < here[k] ? s[k] : next[k];
          if (!two) {
            each = scale[r * groups + c / kGroupCols];
            if (++c == width) c = 0, ++r;
          }
          v[e] = clip((e % 2 ? f[e / 2].y : f[e / 2].x) * each, finite_max<T>());
        }
        if constexpr (sizeof(T) == 2) {
          uint32_t w[N / 2];
#pragma unroll
          for (int e = 0; e < N / 2; ++e) {
            const typename Pair<T>::type y = Pair<T>::round(v[2 * e], v[2 * e + 1]);
            w[e] = *reinterpret_cast<const uint32_t*>(&y);
          }
          if (reinterpret_cast<uintptr_t>(x) % 32 == 0) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(x + p), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
          } else {
            reinterpret_cast<uint4*>(x + p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(x + p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
          }
        } else {
          store8(x + p, *reinterpret_cast<const float(*)[8]>(&v[0]));
          store8(x + p + 8, *reinterpret_cast<const float(*)[8]>(&v[8]));
        }
      } else {
        for (int64_t e = p; e < total; ++e) {
          Raw<uint16_t, 1> one_value;
          one_value.v[0] = q[e];
          float2 f[1];
          unpack_fp8<2>(one_value, f);
          x[e] = from_float<T>(clip(f[0].x * scale[r * groups + c / kGroupCols], finite_max<T>()));
          if (++c == width) c = 0, ++r;
        }
      }
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
  int width, scale_pitch;
  int64_t q_pitch;
  const void* grad;
  const void* z;         // 16 bits, or 8
  const float* scale;
  void* dz;              // NULL: not wanted
  float* partial;        // NULL: not wanted
};
constexpr int kDzVectors = 32, kDzRows = kStreamThreads / kDzVectors;
constexpr int kDzBlocks = 4;  // of an SM

template <class T, int ACT, bool FP8>
__global__ void __launch_bounds__(kStreamThreads, kDzBlocks) linear_dz_kernel(const DzArgs a) {
  pdl_enter();
  constexpr int AT_ONCE = 2;  // rows under way
  const int v = threadIdx.x % kDzVectors, r = threadIdx.x / kDzVectors;
  const int col = (blockIdx.x * kDzVectors + v) * 8;
  const int64_t step = static_cast<int64_t>(gridDim.y) * kDzRows;
  float sum[8] = {};
  if (col < a.width)
    for (int64_t first = static_cast<int64_t>(blockIdx.y) * kDzRows + r; first < a.rows; first += AT_ONCE * step) {
      uint4 graw[AT_ONCE], zraw[AT_ONCE];
      float s[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int64_t row = first + k * step;
        graw[k] = zraw[k] = make_uint4(0, 0, 0, 0);
        s[k] = 0.0f;
        if (row < a.rows) {
          graw[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.grad) + row * a.width + col);
          if constexpr (ACT != kActNone && FP8) {
            s[k] = a.scale[row * a.scale_pitch + col / kGroupCols];
            const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.z) + row * a.q_pitch + col);
            zraw[k].x = x.x;
            zraw[k].y = x.y;
          } else if constexpr (ACT != kActNone) {
            zraw[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.z) + row * a.width + col);
          }
        }
      }
      if constexpr (ACT != kActNone && FP8) {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
          if (s[k] >= kLargestScale) zraw[k].x = below_256(zraw[k].x), zraw[k].y = below_256(zraw[k].y);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int64_t row = first + k * step;
        float d[8];
        unpack<T, 8>(*reinterpret_cast<const Raw<T, 8>*>(&graw[k]), d);
        if constexpr (ACT != kActNone) {
          float z[8];
          if constexpr (FP8) {
            const uint2 x = make_uint2(zraw[k].x, zraw[k].y);
            float2 f[4];
            unpack_fp8<8>(*reinterpret_cast<const Raw<uint16_t, 4>*>(&x), f);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[2 * e] = f[e].x * s[k], z[2 * e + 1] = f[e].y * s[k];
          } else {
            unpack<T, 8>(*reinterpret_cast<const Raw<T, 8>*>(&zraw[k]), z);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float slope;
            act_both<ACT>(z[e], slope);
            d[e] *= slope;
          }
        }
        if (row < a.rows) {
          if (a.dz) store8(static_cast<T*>(a.dz) + row * a.width + col, d);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += d[e];
        }
      }
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
