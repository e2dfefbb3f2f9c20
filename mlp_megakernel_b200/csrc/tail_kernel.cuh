// The sum of the shares of a product's last tiles (product_kernel.cuh): z = the
// sum over s of share s, in the order of s; out = act(z + bias) + residual,
// rounded once.  Bound by reading the shares; a thread takes 8 columns of a row,
// four shares under way at a time.
#pragma once
#include "act.cuh"
#include "pdl.cuh"
#include "product_plan.cuh"
#include "vec.cuh"

namespace mlpk {

constexpr int kTailThreads = 256;

struct TailArgs {
  const float* partials;
  void* out[2];
  int rows, cols;
  int tiles_m, tiles_n, outputs, group;
  int full, splits;
  int act, bias32;
  const void* bias;      // NULL: none
  const void* residual;  // NULL: none
};

template <class T, int TN>
__global__ void __launch_bounds__(kTailThreads) tail_sum_kernel(const TailArgs a) {
  pdl_enter();
  constexpr int VECTORS = TN / 8;
  const int i = blockIdx.x * kTailThreads + threadIdx.x, row = i / VECTORS, col = i % VECTORS * 8;
  const TileAt at = product_tile(a.full + blockIdx.y, a.tiles_m, a.tiles_n, a.outputs, a.group);
  const int64_t out_row = static_cast<int64_t>(at.m) * 256 + row;
  const int out_col = at.n * TN + col;
  if (out_row >= a.rows || out_col >= a.cols) return;
  const float4* p = reinterpret_cast<const float4*>(a.partials) + static_cast<int64_t>(blockIdx.y) * (64 * TN);
  const int first = share_unit(row, col, TN), second = share_unit(row, col + 4, TN);
  const int64_t apart = static_cast<int64_t>(gridDim.y) * (64 * TN);
  float f[8] = {};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float4 x = p[s * apart + first], y = p[s * apart + second];
    f[0] += x.x, f[1] += x.y, f[2] += x.z, f[3] += x.w;
    f[4] += y.x, f[5] += y.y, f[6] += y.z, f[7] += y.w;
  }
  const int64_t o = out_row * a.cols + out_col;
  if (a.bias && a.bias32) {
    const float4* b = reinterpret_cast<const float4*>(static_cast<const float*>(a.bias) + out_col);
    const float4 x = b[0], y = b[1];
    f[0] += x.x, f[1] += x.y, f[2] += x.z, f[3] += x.w;
    f[4] += y.x, f[5] += y.y, f[6] += y.z, f[7] += y.w;
  } else if (a.bias) {
    float b[8];
    unpack<T, 8>(load_raw<T, 8>(static_cast<const T*>(a.bias) + out_col), b);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += b[e];
  }
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = act_value<decltype(act)::value>(f[e]);
  });
  if (a.residual) {
    float r[8];
    unpack<T, 8>(load_raw<T, 8>(static_cast<const T*>(a.residual) + o), r);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += r[e];
  }
  store_vec<T, 8>(static_cast<T*>(a.out[at.output]) + o, f);
}

}  // namespace mlpk
